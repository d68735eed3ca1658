"""Performance cases of the operators that prepare what the views of a training iteration (or a viewer's frame) read
in place of the stored splat parameters: dropout with a mask that is regenerated from a counter, the 4-bit spherical
harmonic (SH) rows, and the product of such a row with the basis of a viewing direction.

`own` chooses between the plain form (elementary torch operations) and the calls of libssb_b200.
"""
import ctypes
import math

import numpy as np
import torch

own = False

DEV = "cuda"
C0 = 0.28209479177387814
CAP = 0.999                    # largest opacity after compensation
DROPPED = -64.0                # logit of a dropped splat
BANDS = ((0, 3), (3, 8), (8, 15))


# ---------------------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------------------

def listed():
    return [
        # SH coefficients dropped whole (three colour values share a decision) before an iteration of the 1M-splat scene
        dict(name="dropout_coefficients_1m", kind="dropout", n=1_000_000, width=45, group=3, rate=0.1, first=0),
        # value by value over the SH array of the 3M-splat scene; the backward pass is the same call on the gradients
        dict(name="dropout_values_3m", kind="dropout", n=3_000_000, width=45, group=1, rate=0.25, first=0),
        # one rank's odd-sized shard of a 10M-splat scene, whole splats dropped (45 values share a decision)
        dict(name="dropout_shard_rows", kind="dropout", n=50_001, width=45, group=45, rate=0.1, first=1_250_003),
        # opacities, forward and backward, of the small scene: launch latency counts
        dict(name="opacity_50k", kind="opacity", n=50_000, rate=0.1, first=0),
        # opacities, forward and backward, of the largest scene
        dict(name="opacity_10m", kind="opacity", n=10_000_000, rate=0.2, first=0),
        # SH rows to 4 bits and back: the small scene, and the wide scene after loading
        dict(name="rows_50k", kind="rows", n=50_000),
        dict(name="rows_5m", kind="rows", n=5_000_000),
        # a viewer's frame: one direction per splat; a small object (latency), and the largest scene
        dict(name="eval_6k_1_view", kind="eval", n=6_007, views=1, degree=3, extent=1.0),
        dict(name="eval_10m_1_view", kind="eval", n=10_000_000, views=1, degree=3, extent=20.0),
        # the batch of the 1M-splat scene: every row against sixteen directions
        dict(name="eval_1m_16_views", kind="eval", n=1_000_000, views=16, degree=3, extent=4.0),
        # gradients through the 4-bit rows: one view of the dense scene, the batch of the 1M-splat scene
        dict(name="eval_bwd_3m_1_view", kind="eval_bwd", n=3_000_000, views=1, degree=3, extent=4.0),
        dict(name="eval_bwd_1m_16_views", kind="eval_bwd", n=1_000_000, views=16, degree=3, extent=4.0),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["dropout", "opacity", "rows", "eval", "eval_bwd"])
    rate = rng.choice([0.0, 0.01, 0.1, 0.2, 0.25, 0.5, 0.9, round(rng.uniform(0.02, 0.7), 3)])
    if kind == "dropout":
        width = rng.choice([1, 3, 4, 45])
        return dict(kind=kind, n=_log_int(rng, 1, 3_000_000), width=width, group=rng.choice([1, 2, 3, 4, 9, 45]), rate=rate,
                    first=rng.choice([0, 0, _log_int(rng, 1, 7_000_000)]))
    if kind == "opacity":
        return dict(kind=kind, n=_log_int(rng, 1, 10_000_000), rate=rate, first=rng.choice([0, _log_int(rng, 1, 5_000_000)]))
    if kind == "rows":
        return dict(kind=kind, n=_log_int(rng, 1, 5_000_000))
    degree = rng.choice([3, 3, 3, 2, 1, 0])
    extent = rng.choice([1.0, 4.0, 15.0, 20.0])
    views = rng.choice([1, 1, 2, 3, 7, 16, 33])
    if kind == "eval":
        n = _log_int(rng, 1, 10_000_000 if views == 1 else 16_000_000 // views)
    else:
        n = _log_int(rng, 1, 3_000_000 if views == 1 else 16_000_000 // max(views, 8))
    return dict(kind=kind, n=n, views=views, degree=degree, extent=extent)


def work(case):
    n, kind = case["n"], case["kind"]
    if kind == "dropout":
        return dict(bytes=8 * n * case["width"], flops=n * case["width"])
    if kind == "opacity":
        # forward reads and writes a logit; backward reads a logit and a gradient and writes a gradient
        return dict(bytes=16 * n, flops=16 * n)
    if kind == "rows":
        return dict(bytes=(180 + 180) * n, flops=4 * 45 * n)
    used = (case["degree"] + 1) ** 2 - 1
    pairs = n * case["views"]
    row = 32 if used else 0
    if kind == "eval":
        return dict(bytes=(row + 24) * n + 12 * pairs, flops=(2 * 3 * used + 60) * pairs)
    return dict(bytes=(row + 12 + 204) * n + 12 * pairs, flops=(4 * 3 * used + 150) * pairs)


# ---------------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------------

def _encode(sh):
    """Plain 4-bit rows of sh [n][15][3]: (codes int64 [n][15][3] in -7..7, scales fp32 [n][3])."""
    n = sh.shape[0]
    q = torch.empty(n, 15, 3, dtype=torch.int64, device=sh.device)
    scales = torch.empty(n, 3, dtype=torch.float32, device=sh.device)
    for b, (lo, hi) in enumerate(BANDS):
        v = sh[:, lo:hi]
        mag = v.abs()
        m = torch.where(mag <= torch.finfo(torch.float32).max, mag, torch.zeros_like(mag)).amax(dim=(1, 2))
        # smallest bf16 s with 7 s >= m: take a bf16 near m / 7 and move to the neighbour that qualifies (7 s is exact in fp32)
        near = (m.double() / 7.0).float()
        bits = near.view(torch.int32) & ~0xffff
        s = bits.view(torch.float32)
        s = torch.where(7.0 * s.double() < m.double(), (bits + 0x10000).view(torch.float32), s)
        s = torch.where(m < 2.0 ** -100, torch.zeros_like(s), s)
        safe = torch.where(s > 0, s, torch.ones_like(s))[:, None, None].double()
        t = torch.nan_to_num(v.double() / safe, nan=0.0, posinf=7.0, neginf=-7.0)
        code = torch.round(t).clamp(-7, 7).to(torch.int64)
        q[:, lo:hi] = torch.where(s[:, None, None] > 0, code, torch.zeros_like(code))
        scales[:, b] = s
    return q, scales


def _pack(q, scales):
    """uint8 [n][32]: words 2c and 2c + 1 hold channel c's codes + 8, four bits each; words 6 and 7 the three bf16 scales."""
    n = q.shape[0]
    words = torch.zeros(n, 8, dtype=torch.int64, device=q.device)
    for c in range(3):
        for j in range(15):
            words[:, 2 * c + j // 8] |= (q[:, j, c] + 8) << (4 * (j % 8))
    sb = (scales.contiguous().view(torch.int32).to(torch.int64) >> 16) & 0xffff
    words[:, 6] = sb[:, 0] | (sb[:, 1] << 16)
    words[:, 7] = sb[:, 2]
    words = torch.where(words >= 2 ** 31, words - 2 ** 32, words).to(torch.int32)
    return words.contiguous().view(torch.uint8).reshape(n, 32)


def _unpack(rows):
    """(codes fp32 [n][15][3], scales fp32 [n][3]) of the bytes."""
    words = rows.reshape(-1).view(torch.int32).reshape(-1, 8)
    q = torch.empty(words.shape[0], 15, 3, dtype=torch.float32, device=rows.device)
    for c in range(3):
        for j in range(15):
            q[:, j, c] = (((words[:, 2 * c + j // 8] >> (4 * (j % 8))) & 15) - 8).float()
    scales = torch.stack([words[:, 6] << 16, words[:, 6] & ~0xffff, words[:, 7] << 16], dim=1).contiguous().view(torch.float32)
    return q, scales


def _cameras(views, extent, g):
    """World-to-camera matrices of cameras on a ring of radius 2 extent, looking at the middle."""
    ang = 2 * math.pi * (torch.arange(views, dtype=torch.float64) + torch.rand(1, generator=g, dtype=torch.float64)) / views
    h = (torch.rand(views, generator=g, dtype=torch.float64) * 2 - 1) * 0.25 * extent
    eye = torch.stack([2 * extent * torch.cos(ang), h, 2 * extent * torch.sin(ang)], 1)
    fwd = -eye / eye.norm(dim=1, keepdim=True)
    down = torch.tensor([0.0, 1.0, 0.0], dtype=torch.float64).expand_as(fwd)
    right = torch.linalg.cross(down, fwd)
    right = right / right.norm(dim=1, keepdim=True)
    R = torch.stack([right, torch.linalg.cross(fwd, right), fwd], 1)
    vm = torch.zeros(views, 4, 4, dtype=torch.float64)
    vm[:, :3, :3] = R
    vm[:, :3, 3] = -(R @ eye[:, :, None])[:, :, 0]
    vm[:, 3, 3] = 1
    return vm.float().reshape(views, 16)


def prepare(case, seed):
    n, kind = case["n"], case["kind"]
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    gc = torch.Generator()
    gc.manual_seed(seed)
    normal = lambda *s: torch.randn(*s, generator=g, device=DEV)
    st = dict(case=case)
    if kind in ("dropout", "opacity"):
        st["seed"] = int(torch.randint(0, 2 ** 62, (1,), generator=gc))
        st["offset"] = int(torch.randint(0, 30_000, (1,), generator=gc))        # the iteration number
        st["rate"] = float(np.float32(case["rate"]))
    if kind == "dropout":
        st["x"] = 0.05 * normal(n * case["width"])
        if own:
            st["y"] = torch.empty_like(st["x"])
    elif kind == "opacity":
        # trained logits: mostly N(0, 1), some splats nearly opaque or nearly gone
        x = normal(n)
        st["x"] = torch.where(torch.rand(n, generator=g, device=DEV) < 0.1, 4.0 * x, x)
        st["v"] = 1e-4 * normal(n)
        if own:
            st["y"], st["gx"] = torch.empty_like(st["x"]), torch.empty_like(st["x"])
    else:
        sh = 0.05 * normal(n, 15, 3)
        sh[torch.rand(n, generator=g, device=DEV) < 0.02] = 0.0                  # splats whose bands have not been trained yet
        if kind == "rows":
            st["sh"] = sh
            if own:
                st["rows"] = torch.empty(n, 32, dtype=torch.uint8, device=DEV)
                st["out"] = torch.empty_like(sh)
        else:
            st["rows"] = _pack(*_encode(sh))
            st["dc"] = 0.3 * normal(n, 3)
            st["means"] = case["extent"] * (2 * torch.rand(n, 3, generator=g, device=DEV) - 1)
            st["viewmats"] = _cameras(case["views"], case["extent"], gc).to(DEV)
            if kind == "eval_bwd":
                st["v"] = 1e-3 * normal(case["views"], n, 3)
                if own:
                    st["v_means"], st["v_dc"], st["v_sh"] = (torch.empty(n, 3, device=DEV), torch.empty(n, 3, device=DEV),
                                                             torch.empty(n, 15, 3, device=DEV))
            elif own:
                st["out"] = torch.empty(case["views"], n, 3, device=DEV)
        del sh
    return st


# ---------------------------------------------------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------------------------------------------------

def _mul32(a, m):
    """(high, low) 32 bits of a * m for a an int64 tensor of 32-bit values."""
    lo = (a & 0xffff) * m
    hi = (a >> 16) * m + (lo >> 16)
    return hi >> 16, ((hi & 0xffff) << 16) | (lo & 0xffff)


def _dropped(first_group, n_groups, rate, seed, offset):
    """Truth values [n_groups]: which groups Philox4x32-10 drops."""
    b0, b1 = first_group // 4, (first_group + n_groups - 1) // 4 + 1
    block = torch.arange(b0, b1, dtype=torch.int64, device=DEV)
    c = [block & 0xffffffff, block >> 32, torch.full_like(block, offset & 0xffffffff), torch.full_like(block, offset >> 32)]
    k0, k1 = seed & 0xffffffff, seed >> 32
    for _ in range(10):
        h0, l0 = _mul32(c[0], 0xD2511F53)
        h1, l1 = _mul32(c[2], 0xCD9E8D57)
        c = [h1 ^ c[1] ^ k0, l1, h0 ^ c[3] ^ k1, l0]
        k0, k1 = (k0 + 0x9E3779B9) & 0xffffffff, (k1 + 0xBB67AE85) & 0xffffffff
    threshold = int(math.floor(rate * 2.0 ** 32))
    out = torch.stack([w < threshold for w in c], dim=1).reshape(-1)
    skip = first_group - 4 * b0
    return out[skip:skip + n_groups]


def _plain_dropout(st):
    case = st["case"]
    group, first, count = case["group"], case["first"] * case["width"], st["x"].numel()
    g0, g1 = first // group, (first + count - 1) // group
    drop = _dropped(g0, g1 - g0 + 1, st["rate"], st["seed"], st["offset"])
    drop = drop.repeat_interleave(group)[first - g0 * group:first - g0 * group + count] if group > 1 else drop
    scale = float(np.float32(1.0 / (1.0 - st["rate"])))
    return torch.where(drop, torch.zeros_like(st["x"]), st["x"] * scale)


def _plain_opacity(st):
    x, r = st["x"], st["rate"]
    if r == 0.0:
        return [x.clone(), st["v"].clone()]
    drop = _dropped(st["case"]["first"], x.numel(), r, st["seed"], st["offset"])
    # 64 bits: e^-x - r / (1 - r) cancels near the cap
    e = (1.0 - r) * torch.exp(-x.double()) - r                # (1 - z) / z of the compensated opacity z
    capped = e <= (1.0 - CAP) / CAP
    y = torch.where(capped, torch.full_like(e, math.log(CAP / (1.0 - CAP))), -torch.log(torch.where(capped, torch.ones_like(e), e)))
    slope = torch.where(capped, torch.zeros_like(e), (e + r) / torch.where(capped, torch.ones_like(e), e))
    y = torch.where(drop, torch.full_like(y, DROPPED), y).float()
    gx = torch.where(drop, torch.zeros_like(slope), slope * st["v"]).float()
    return [y, gx]


def _basis(d):
    """Real SH basis, bands 1..3, of unit directions [n][3]: a list of fifteen [n]."""
    x, y, z = d[:, 0], d[:, 1], d[:, 2]
    z2 = z * z
    c1, s1 = x * x - y * y, 2 * x * y
    c2, s2 = x * c1 - y * s1, x * s1 + y * c1
    t = 0.4570457994644658 - 2.285228997322329 * z2
    return [-0.4886025119029199 * y, 0.4886025119029199 * z, -0.4886025119029199 * x,
            0.5462742152960396 * s1, -1.0925484305920792 * z * y, 0.9461746957575601 * z2 - 0.31539156525252005, -1.0925484305920792 * z * x,
            0.5462742152960396 * c1,
            -0.5900435899266435 * s2, 1.445305721320277 * z * s1, t * y, z * (1.8658816629505769 * z2 - 1.1195289977703462), t * x,
            1.445305721320277 * z * c1, -0.5900435899266435 * c2]


def _basis_vjp(d, w):
    """Gradient of sum_j w_j b_j with respect to the direction: [n][3]."""
    x, y, z = d[:, 0], d[:, 1], d[:, 2]
    z2 = z * z
    c1, s1 = x * x - y * y, 2 * x * y
    t = 0.4570457994644658 - 2.285228997322329 * z2
    k1, k2, k2h, k3, k3h = 0.4886025119029199, 1.0925484305920792, 0.5462742152960396, 0.5900435899266435, 1.445305721320277
    gx = -k1 * w[2] + 2 * k2h * y * w[3] - k2 * z * w[6] + 2 * k2h * x * w[7] \
        - 3 * k3 * s1 * w[8] + 2 * k3h * y * z * w[9] + t * w[12] + 2 * k3h * z * x * w[13] - 3 * k3 * c1 * w[14]
    gy = -k1 * w[0] + 2 * k2h * x * w[3] - k2 * z * w[4] - 2 * k2h * y * w[7] \
        - 3 * k3 * c1 * w[8] + 2 * k3h * x * z * w[9] + t * w[10] - 2 * k3h * z * y * w[13] + 3 * k3 * s1 * w[14]
    gz = k1 * w[1] - k2 * y * w[4] + 2 * 0.9461746957575601 * z * w[5] - k2 * x * w[6] + k3h * s1 * w[9] \
        - 2 * 2.285228997322329 * z * y * w[10] + (3 * 1.8658816629505769 * z2 - 1.1195289977703462) * w[11] \
        - 2 * 2.285228997322329 * z * x * w[12] + k3h * c1 * w[13]
    return torch.stack([gx, gy, gz], 1)


def _directions(st, v):
    """Unit direction and inverse distance from camera v to every splat (64 bits: the difference of two positions), in fp32."""
    m = st["viewmats"][v].reshape(4, 4).double()
    d = st["means"].double() + (m[:3, :3].T @ m[:3, 3])[None]
    inv = 1.0 / d.norm(dim=1, keepdim=True)
    return (d * inv).float(), inv.float()


def _plain_values(st):
    q, scales = _unpack(st["rows"])
    for b, (lo, hi) in enumerate(BANDS):
        q[:, lo:hi] *= scales[:, b][:, None, None]
    return q


def _plain_eval(st):
    case = st["case"]
    used = (case["degree"] + 1) ** 2 - 1
    sh = _plain_values(st)
    out = torch.empty(case["views"], case["n"], 3, device=DEV)
    for v in range(case["views"]):
        d, _ = _directions(st, v)
        b = _basis(d)
        o = C0 * st["dc"]
        for j in range(used):
            o += b[j][:, None] * sh[:, j]
        out[v] = o
    return out


def _plain_eval_bwd(st):
    case = st["case"]
    used = (case["degree"] + 1) ** 2 - 1
    sh = _plain_values(st)
    v_means, v_dc, v_sh = torch.zeros(case["n"], 3, device=DEV), torch.zeros(case["n"], 3, device=DEV), torch.zeros(case["n"], 15, 3, device=DEV)
    zero = torch.zeros(case["n"], device=DEV)
    for v in range(case["views"]):
        gv = st["v"][v]
        d, inv = _directions(st, v)
        b = _basis(d)
        v_dc += C0 * gv
        w = [zero] * 15
        for j in range(used):
            v_sh[:, j] += b[j][:, None] * gv
            w[j] = (sh[:, j] * gv).sum(1)
        gd = _basis_vjp(d, w)
        v_means += (gd - d * (d * gd).sum(1, keepdim=True)) * inv
    return [v_means, v_dc, v_sh]


def _plain_rows(st):
    q, scales = _encode(st["sh"])
    out = q.float()
    for b, (lo, hi) in enumerate(BANDS):
        out[:, lo:hi] *= scales[:, b][:, None, None]
    return out


# ---------------------------------------------------------------------------------------------------------------------
# the framework's calls
# ---------------------------------------------------------------------------------------------------------------------

def _describe(st):
    """The argument blocks a program builds once for its buffers."""
    from spirula_studio_b200 import lib as L
    case, kind = st["case"], st["case"]["kind"]
    d = dict(L=L, lib=L.load())
    if kind in ("dropout", "opacity"):
        d["dropout"] = L.dropout_struct(st["rate"], st["seed"], st["offset"])
    elif kind in ("eval", "eval_bwd"):
        d["splats"] = L.splats_struct(dict(means=st["means"], features_dc=st["dc"]))
        d["shq"] = L.shq_struct(st["rows"], None, 4, 0)
        d["cams"] = L.cameras_struct(st["viewmats"], st["viewmats"], 1, 1, sh_degree=case["degree"])
        if kind == "eval_bwd":
            d["grads"] = L.splats_struct(dict(means=st["v_means"], features_dc=st["v_dc"], features_sh=st["v_sh"]))
    return d


def _own_run(st):
    if "call" not in st:
        st["call"] = _describe(st)
    d = st["call"]
    L, lib = d["L"], d["lib"]
    case, kind = st["case"], st["case"]["kind"]
    n = case["n"]
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    ref = ctypes.byref
    if kind == "dropout":
        L.check(lib.ssb_dropout(L.ptr(st["x"]), case["first"] * case["width"], n * case["width"], case["group"], ref(d["dropout"]),
                                L.ptr(st["y"]), stream))
        return st["y"]
    if kind == "opacity":
        L.check(lib.ssb_dropout_opacities(L.ptr(st["x"]), case["first"], n, ref(d["dropout"]), L.ptr(st["y"]), stream))
        L.check(lib.ssb_dropout_opacities_bwd(L.ptr(st["x"]), L.ptr(st["v"]), case["first"], n, ref(d["dropout"]), L.ptr(st["gx"]), stream))
        return [st["y"], st["gx"]]
    if kind == "rows":
        L.check(lib.ssb_quant_encode(L.ptr(st["sh"]), n * 45, 4, L.ptr(st["rows"]), None, stream))
        L.check(lib.ssb_quant_decode(L.ptr(st["rows"]), None, n * 45, 4, L.ptr(st["out"]), stream))
        return st["out"]
    if kind == "eval":
        L.check(lib.ssb_sh_eval_fwd(ref(d["splats"]), ref(d["shq"]), n, ref(d["cams"]), L.ptr(st["out"]), stream))
        return st["out"]
    L.check(lib.ssb_sh_eval_bwd(ref(d["splats"]), ref(d["shq"]), n, ref(d["cams"]), L.ptr(st["v"]), ref(d["grads"]), 0, stream))
    return [st["v_means"], st["v_dc"], st["v_sh"]]


def run(state):
    if own:
        return _own_run(state)
    return {"dropout": _plain_dropout, "opacity": _plain_opacity, "rows": _plain_rows, "eval": _plain_eval,
            "eval_bwd": _plain_eval_bwd}[state["case"]["kind"]](state)


# ---------------------------------------------------------------------------------------------------------------------
# 64-bit values, from the definitions
# ---------------------------------------------------------------------------------------------------------------------

def _exact_words(blocks, seed, offset):
    """Philox4x32-10 of int64 block numbers by unsigned 64-bit products: the 64-bit pattern of a product of two 32-bit numbers
    fits int64 arithmetic modulo 2^64."""
    mask = 0xffffffff
    s = [blocks & mask, (blocks >> 32) & mask, torch.full_like(blocks, offset & mask), torch.full_like(blocks, (offset >> 32) & mask)]
    keys = [((seed & mask) + i * 0x9E3779B9) & mask for i in range(10)], [((seed >> 32) + i * 0xBB67AE85) & mask for i in range(10)]
    for ka, kb in zip(*keys):
        p = s[0] * 0xD2511F53
        q = s[2] * 0xCD9E8D57
        s = [((q >> 32) & mask) ^ s[1] ^ ka, q & mask, ((p >> 32) & mask) ^ s[3] ^ kb, p & mask]
    return s


def _exact_keep(groups, rate, seed, offset):
    """Keep factor (0 or 1) of each group number."""
    first, last = int(groups[0]) >> 2, int(groups[-1]) >> 2
    words = _exact_words(torch.arange(first, last + 1, device=DEV, dtype=torch.int64), seed, offset)
    table = torch.stack(words, 1).reshape(-1)
    return table[groups - 4 * first] >= math.floor(rate * 4294967296.0)


def _exact_basis(x, y, z):
    """The Cartesian forms, normalised over the sphere, with the Condon-Shortley sign."""
    pi = math.pi
    a = math.sqrt(3 / (4 * pi))
    b = math.sqrt(15 / (4 * pi))
    c = math.sqrt(5 / (16 * pi))
    e, f, g, h = math.sqrt(35 / (32 * pi)), math.sqrt(105 / (4 * pi)), math.sqrt(21 / (32 * pi)), math.sqrt(7 / (16 * pi))
    return torch.stack([-a * y, a * z, -a * x,
                        b * x * y, -b * y * z, c * (3 * z * z - 1), -b * x * z, 0.5 * b * (x * x - y * y),
                        -e * y * (3 * x * x - y * y), f * x * y * z, -g * y * (5 * z * z - 1), h * z * (5 * z * z - 3), -g * x * (5 * z * z - 1),
                        0.5 * f * z * (x * x - y * y), -e * x * (x * x - 3 * y * y)], 1)


def _exact_rows(sh):
    """Values the 4-bit rows stand for, in 64 bits."""
    v = sh.double()
    out = torch.zeros_like(v)
    for lo, hi in BANDS:
        m = v[:, lo:hi].abs().amax(dim=(1, 2))
        # bf16 has 8 significant bits: m / 7 = f 2^e with f in [0.5, 1), rounded up to a multiple of 2^(e - 8)
        f, e = torch.frexp(m / 7.0)
        s = torch.ldexp(torch.ceil(torch.ldexp(f, torch.full_like(e, 8))), e - 8)
        ok = m > 0
        t = torch.where(ok, s, torch.ones_like(s))[:, None, None]
        out[:, lo:hi] = torch.where(ok[:, None, None], torch.round(v[:, lo:hi] / t) * t, torch.zeros_like(v[:, lo:hi]))
    return out


def exact(case, seed):
    st = prepare(case, seed)
    kind, n = case["kind"], case["n"]
    if kind == "dropout":
        first = case["first"] * case["width"]
        out = torch.empty(st["x"].numel(), dtype=torch.float64, device=DEV)
        step = 1 << 24
        for i in range(0, out.numel(), step):
            j = min(out.numel(), i + step)
            idx = torch.arange(first + i, first + j, device=DEV, dtype=torch.int64) // case["group"]
            keep = _exact_keep(idx, st["rate"], st["seed"], st["offset"])
            out[i:j] = torch.where(keep, st["x"][i:j].double() / (1.0 - st["rate"]), torch.zeros(j - i, dtype=torch.float64, device=DEV))
        return out
    if kind == "opacity":
        x, r = st["x"].double(), st["rate"]
        if r == 0.0:
            return [x, st["v"].double()]
        keep = _exact_keep(torch.arange(case["first"], case["first"] + n, device=DEV, dtype=torch.int64), r, st["seed"], st["offset"])
        s = 1.0 / (1.0 + torch.exp(-x))
        z = s / (1.0 - r)
        free = z < CAP
        zz = torch.clamp(z, max=CAP)
        y = torch.where(keep, torch.log(zz) - torch.log1p(-zz), torch.full_like(x, DROPPED))
        slope = s * (1.0 - s) / (1.0 - r) / (zz * (1.0 - zz))
        return [y, torch.where(keep & free, slope * st["v"].double(), torch.zeros_like(x))]
    if kind == "rows":
        return _exact_rows(st["sh"])
    used = (case["degree"] + 1) ** 2 - 1
    vm = st["viewmats"].double().reshape(-1, 4, 4)
    centre = -(vm[:, :3, :3].transpose(1, 2) @ vm[:, :3, 3:])[:, :, 0]
    words = st["rows"].reshape(-1).view(torch.int32).reshape(n, 8)
    back = kind == "eval_bwd"
    outs = [torch.zeros(n, 3, dtype=torch.float64, device=DEV), torch.zeros(n, 3, dtype=torch.float64, device=DEV),
            torch.zeros(n, 15, 3, dtype=torch.float64, device=DEV)] if back else torch.zeros(case["views"], n, 3, dtype=torch.float64, device=DEV)
    shift = torch.arange(8, device=DEV, dtype=torch.int32) * 4
    step = 1 << 18
    for i in range(0, n, step):
        sl = slice(i, min(n, i + step))
        w = words[sl]
        codes = ((w[:, :6, None] >> shift) & 15).reshape(-1, 3, 16)[:, :, :15].transpose(1, 2).double() - 8.0
        sc = torch.stack([w[:, 6] << 16, w[:, 6] & -65536, w[:, 7] << 16], 1).contiguous().view(torch.float32).double()
        sh = codes * torch.repeat_interleave(sc, torch.tensor([3, 5, 7], device=DEV), dim=1)[:, :, None]
        mean, dc = st["means"][sl].double(), st["dc"][sl].double()
        if back:
            mean.requires_grad_(True); dc.requires_grad_(True); sh = sh.requires_grad_(True)
        for v in range(case["views"]):
            with torch.enable_grad():
                d = mean - centre[v]
                d = d / torch.sqrt((d * d).sum(1, keepdim=True))
                o = C0 * dc + (_exact_basis(d[:, 0], d[:, 1], d[:, 2])[:, :used, None] * sh[:, :used]).sum(1)
                if back:
                    o.backward(st["v"][v][sl].double())
                else:
                    outs[v][sl] = o
        if back:
            for o, leaf in zip(outs, (mean, dc, sh)):
                if leaf.grad is not None:
                    o[sl] = leaf.grad
    return outs
