"""64-bit statements of the operators that prepare what a view reads: dropout (Philox4x32-10), 4-bit SH rows, the product of
SH coefficients with the viewing direction's basis and its gradients.  numpy only."""
import numpy as np

U = 2.0 ** -24                       # half a step of fp32, relative
C0 = 0.28209479177387814
CAP = 0.999
DROPPED = -64.0
BANDS = ((0, 3), (3, 8), (8, 15))


def philox(blocks, seed, offset):
    """uint32 [m][4]: the words of the given block numbers."""
    m32 = np.uint64(0xffffffff)
    s32 = np.uint64(32)
    b = np.asarray(blocks, np.uint64)
    c = [b & m32, b >> s32, np.full_like(b, offset & 0xffffffff), np.full_like(b, (offset >> 32) & 0xffffffff)]
    k0, k1 = seed & 0xffffffff, (seed >> 32) & 0xffffffff
    for _ in range(10):
        p, q = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(q >> s32) ^ c[1] ^ np.uint64(k0), q & m32, (p >> s32) ^ c[3] ^ np.uint64(k1), p & m32]
        k0, k1 = (k0 + 0x9E3779B9) & 0xffffffff, (k1 + 0xBB67AE85) & 0xffffffff
    return np.stack(c, 1).astype(np.uint32)


def dropped(first, count, group, rate, seed, offset):
    """bool [count]: whether value first + k of the array is dropped.  rate: the fp32 number the call gets."""
    g = (np.arange(first, first + count, dtype=object) if first + count >= 2 ** 63 else np.arange(first, first + count, dtype=np.uint64)) // group
    g = g.astype(np.uint64)
    uniq, inv = np.unique(g >> np.uint64(2), return_inverse=True)
    w = philox(uniq, seed, offset)[inv, (g & np.uint64(3)).astype(np.int64)]
    return w.astype(np.float64) < np.floor(float(np.float32(rate)) * 2.0 ** 32)


def dropout(x, first, group, rate, seed, offset):
    d = dropped(first, x.size, group, rate, seed, offset)
    with np.errstate(all="ignore"):
        return np.where(d, 0.0, x.astype(np.float64) / (1.0 - float(np.float32(rate))))


def dropout_opacities(x, first, rate, seed, offset):
    """(logits, slope, error bound of an fp32 evaluation of the logits); the slope is zero where dropped or limited."""
    r = float(np.float32(rate))
    x = x.astype(np.float64)
    if r == 0.0:
        return x, np.ones_like(x), np.zeros_like(x)
    d = dropped(first, x.size, 1, rate, seed, offset)
    with np.errstate(all="ignore"):
        # e = (1 - z) / z of the compensated opacity z = s / (1 - r)
        e = (1.0 - r) * np.exp(-x) - r
        capped = e <= (1.0 - CAP) / CAP
        a = -np.log1p(-r)
        lw = np.log1p(-np.exp(-(np.log((1.0 - r) / r) - x)))
        y = np.where(capped, np.log(CAP / (1.0 - CAP)), x + a - lw)
        slope = np.where(capped, 0.0, (e + r) / e)
        slope = np.where(np.isposinf(e), 1.0, slope)
        # ln w: w = 1 - e^-d with d off by 2 U relative, which w / (e^d - 1) d <= 1 hands on, and 1 - e^-d by another 2 U relative,
        # together 4 U relative in w; a base-2 logarithm off by 2^-22 = 4 U absolute above w = 1/2 and relative below, times ln 2
        # (itself half a U off); then the rounding of a, of x + a and of the final multiply-add
        bound = np.where(capped, U * np.abs(y), U * (4.0 + np.maximum(4.0 * np.log(2.0), 4.0 * np.abs(lw)) + 0.5 * np.abs(lw) + a + np.abs(x + a) + np.abs(y)))
    y = np.where(d, DROPPED, y)
    return y, np.where(d, 0.0, slope), np.where(d, 0.0, bound)


def encode_rows(sh):
    """(codes int [n][15][3], scales fp64 [n][3]) of fp32 values [n][15][3]."""
    v = np.asarray(sh, np.float32).astype(np.float64)
    n = v.shape[0]
    q = np.zeros((n, 15, 3), np.int64)
    scales = np.zeros((n, 3))
    for b, (lo, hi) in enumerate(BANDS):
        x = v[:, lo:hi]
        m = np.where(np.isfinite(x), np.abs(x), 0.0).reshape(n, -1).max(axis=1)
        f, e = np.frexp(m / 7.0)
        s = np.ldexp(np.ceil(np.ldexp(f, 8)), e - 8)         # rounded up to eight significant bits
        s = np.where(7 * s > np.finfo(np.float32).max, s - np.ldexp(1.0, e - 8), s)
        s = np.where(m >= 2.0 ** -100, s, 0.0)
        safe = np.where(s > 0, s, 1.0)[:, None, None]
        with np.errstate(all="ignore"):
            t = np.clip(np.nan_to_num(x / safe, nan=0.0, posinf=7.0, neginf=-7.0), -7, 7)
        q[:, lo:hi] = np.where(s[:, None, None] > 0, np.rint(t), 0).astype(np.int64)
        scales[:, b] = s
    return q, scales


def row_values(q, scales):
    out = q.astype(np.float64)
    for b, (lo, hi) in enumerate(BANDS):
        out[:, lo:hi] *= scales[:, b][:, None, None]
    return out


def pack_rows(q, scales):
    """uint8 [n][32]."""
    n = q.shape[0]
    w = np.zeros((n, 8), np.uint32)
    for c in range(3):
        for j in range(15):
            w[:, 2 * c + j // 8] |= ((q[:, j, c] + 8).astype(np.uint32) << np.uint32(4 * (j % 8)))
    sb = scales.astype(np.float32).view(np.uint32) >> np.uint32(16)
    w[:, 6] = sb[:, 0] | (sb[:, 1] << np.uint32(16))
    w[:, 7] = sb[:, 2]
    return w.view(np.uint8).reshape(n, 32)


def unpack_rows(rows):
    w = np.ascontiguousarray(rows).view(np.uint32).reshape(-1, 8)
    q = np.zeros((w.shape[0], 15, 3), np.int64)
    for c in range(3):
        for j in range(15):
            q[:, j, c] = ((w[:, 2 * c + j // 8] >> np.uint32(4 * (j % 8))) & np.uint32(15)).astype(np.int64) - 8
    sb = np.stack([w[:, 6] << np.uint32(16), w[:, 6] & np.uint32(0xffff0000), w[:, 7] << np.uint32(16)], 1)
    return q, np.ascontiguousarray(sb).view(np.float32).astype(np.float64)


def _parts(d):
    x, y, z = d[..., 0], d[..., 1], d[..., 2]
    return x, y, z


def basis(d):
    """[..., 15] at unit directions [..., 3]."""
    x, y, z = _parts(d)
    a, b, c = np.sqrt(3 / (4 * np.pi)), np.sqrt(15 / (4 * np.pi)), np.sqrt(5 / (16 * np.pi))
    e, f, g, h = np.sqrt(35 / (32 * np.pi)), np.sqrt(105 / (4 * np.pi)), np.sqrt(21 / (32 * np.pi)), np.sqrt(7 / (16 * np.pi))
    return np.stack([-a * y, a * z, -a * x,
                     b * x * y, -b * y * z, c * (3 * z * z - 1), -b * x * z, b / 2 * (x * x - y * y),
                     -e * y * (3 * x * x - y * y), f * x * y * z, -g * y * (5 * z * z - 1), h * z * (5 * z * z - 3), -g * x * (5 * z * z - 1),
                     f / 2 * z * (x * x - y * y), -e * x * (x * x - 3 * y * y)], -1)


def basis_grad(d):
    """[..., 15, 3]: derivatives of the polynomials of `basis`."""
    x, y, z = _parts(d)
    o = np.zeros_like(x)
    a, b, c = np.sqrt(3 / (4 * np.pi)), np.sqrt(15 / (4 * np.pi)), np.sqrt(5 / (16 * np.pi))
    e, f, g, h = np.sqrt(35 / (32 * np.pi)), np.sqrt(105 / (4 * np.pi)), np.sqrt(21 / (32 * np.pi)), np.sqrt(7 / (16 * np.pi))
    rows = [(o, o - a, o), (o, o, o + a), (o - a, o, o),
            (b * y, b * x, o), (o, -b * z, -b * y), (o, o, 6 * c * z), (-b * z, o, -b * x), (b * x, -b * y, o),
            (-6 * e * x * y, -3 * e * (x * x - y * y), o), (f * y * z, f * x * z, f * x * y), (o, -g * (5 * z * z - 1), -10 * g * y * z),
            (o, o, h * (15 * z * z - 3)), (-g * (5 * z * z - 1), o, -10 * g * x * z), (f * x * z, -f * y * z, f / 2 * (x * x - y * y)),
            (-3 * e * (x * x - y * y), 6 * e * x * y, o)]
    return np.stack([np.stack(r, -1) for r in rows], -2)


def directions(means, viewmat):
    """(unit directions [n][3], distances [n])."""
    m = np.asarray(viewmat, np.float64).reshape(4, 4)
    d = np.asarray(means, np.float64) + (m[:3, :3].T @ m[:3, 3])[None]
    big = np.abs(d).max(axis=1, keepdims=True)
    big = np.where(big > 0, big, 1.0)
    r = np.linalg.norm(d / big, axis=1) * big[:, 0]
    return np.where(r[:, None] > 0, d / np.where(r > 0, r, 1.0)[:, None], 0.0), r


# Errors of an fp32 evaluation in units of U.  A component of the difference mean - centre is off by 2 (two additions), the
# squared length by 8, the reciprocal root (2 ulps are 4 U) by 4 + 8/2, a unit component by 12 in all.  With the largest magnitudes
# of the monomials that makes, per band: the basis function (summed by itself, or with its monomials' coefficients gathered first:
# b = c z^2 - c/3 at z^2 = 1/3 loses no more than 2 c/3 times the roundings that follow, within the 27); its largest value and the
# error and the largest value of a component of its gradient.
BASIS_ERR = (7.0, 27.0, 100.0)
GRAD_ERR = (10.0, 40.0, 240.0)
GRAD_MAX = (0.49, 2.2, 7.0)


def _per_coefficient(t):
    return np.repeat(np.array(t), [3, 5, 7])


def sh_eval(means, dc, sh, viewmats, degree=3):
    """(values [V][n][3], error bound of an fp32 evaluation)."""
    used = (degree + 1) ** 2 - 1
    W = np.asarray(sh, np.float64)[:, :used]
    dc = np.zeros((len(means), 3)) if dc is None else np.asarray(dc, np.float64)
    out, tol = [], []
    for vm in np.asarray(viewmats).reshape(-1, 16):
        d, r = directions(means, vm)
        b = np.where(r[:, None] > 0, basis(d), 0.0)[:, :used]
        out.append(C0 * dc + np.einsum("nj,njc->nc", b, W))
        # eighteen roundings of the sum of at most sixteen products, plus the basis functions' own errors
        tol.append(U * (np.einsum("nj,njc->nc", _per_coefficient(BASIS_ERR)[None, :used] + 18 * np.abs(b), np.abs(W)) + 18 * C0 * np.abs(dc)))
    return np.stack(out), np.stack(tol)


def sh_eval_bwd(means, sh, viewmats, v, degree=3):
    """((v_means, v_dc, v_sh), (their error bounds))."""
    used = (degree + 1) ** 2 - 1
    W = np.asarray(sh, np.float64)[:, :used]
    n = len(means)
    vms = np.asarray(viewmats).reshape(-1, 16)
    gm, gd, gs = np.zeros((n, 3)), np.zeros((n, 3)), np.zeros((n, 15, 3))
    tm, td, ts = np.zeros((n, 3)), np.zeros((n, 3)), np.zeros((n, 15, 3))
    sums = len(vms) + 3
    for i, vm in enumerate(vms):
        g = np.asarray(v[i], np.float64)
        d, r = directions(means, vm)
        ok = (r > 0)[:, None]
        inv = np.where(r > 0, 1.0 / np.where(r > 0, r, 1.0), 0.0)[:, None]
        b = np.where(ok, basis(d), 0.0)[:, :used]
        gd += C0 * g
        td += sums * U * C0 * np.abs(g)
        gs[:, :used] += b[:, :, None] * g[:, None]
        ts[:, :used] += U * ((_per_coefficient(BASIS_ERR)[None, :used] * ok + sums * np.abs(b))[:, :, None] * np.abs(g)[:, None])
        w = np.einsum("njc,nc->nj", W, g)
        wa = np.einsum("njc,nc->nj", np.abs(W), np.abs(g))
        vn = np.einsum("nj,njk->nk", w, basis_grad(d)[:, :used])
        gm += np.where(ok, vn - d * (d * vn).sum(1, keepdims=True), 0.0) * inv
        # the gradient's components, w (five roundings) and the projection onto the sphere (a unit vector off by 12 used four
        # times, eight roundings, the reciprocal distance), in units of the largest gradient; then the sum over the views
        tm += U * inv * (wa * (_per_coefficient(GRAD_ERR) + (75 + sums) * _per_coefficient(GRAD_MAX))[None, :used]).sum(1, keepdims=True)
    return (gm, gd, gs), (tm, td, ts)
