"""Dropout, 4-bit SH rows and the SH product without a GPU: the statements the GPU tests compare against, and the refusals of
the entry points (checked before any device call)."""
import ctypes as C

import numpy as np
import pytest

import view_ops_oracle as O
from spirula_studio_b200 import lib as L

ONE = C.c_void_p(64)


def test_philox_known_answers():
    # the published known-answer vectors of Philox4x32-10 whose counter's upper words are the offset
    def words(ctr, key):
        return [int(w) for w in O.philox([ctr[0] | ctr[1] << 32], key[0] | key[1] << 32, ctr[2] | ctr[3] << 32)[0]]
    assert words((0, 0, 0, 0), (0, 0)) == [0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8]
    f = 0xffffffff
    assert words((f, f, f, f), (f, f)) == [0x408f276d, 0x41c83b0e, 0xa20bc7c6, 0x6d5451fd]
    assert words((0x243f6a88, 0x85a308d3, 0x13198a2e, 0x03707344), (0xa4093822, 0x299f31d0)) == [0xd16cfe09, 0x94fdcceb, 0x5001e420, 0x24126ea1]


def test_opacity_slope_is_the_derivative():
    x = np.linspace(-9, 9, 4001).astype(np.float32)
    for rate in (0.01, 0.1, 0.5, 0.9):
        h = 1e-5
        def f(t):
            r = float(np.float32(rate))
            z = np.minimum(1 / (1 + np.exp(-t)) / (1 - r), O.CAP)
            return np.log(z / (1 - z))
        y, slope, _ = O.dropout_opacities(x, 0, rate, 3, 5)
        kept = ~O.dropped(0, x.size, 1, rate, 3, 5)
        xd = x.astype(np.float64)
        z = 1 / (1 + np.exp(-xd)) / (1 - float(np.float32(rate)))
        smooth = kept & (np.abs(z - O.CAP) > 1e-3)
        diff = (f(xd + h) - f(xd - h)) / (2 * h)
        assert np.allclose(y[kept], f(xd)[kept], rtol=1e-9, atol=1e-9)
        # central differences: h^2 / 6 times the third derivative, which stays below 1e9 (1 / (1 - z)^3 at the cap) next to the kink
        far = smooth & (z < 0.9)
        assert np.allclose(slope[far], diff[far], rtol=1e-6, atol=1e-8)
        assert np.all(slope[kept & (z > O.CAP)] == 0)


def test_basis_gradients_are_derivatives_and_backward_is_the_adjoint():
    rng = np.random.default_rng(5)
    d = rng.normal(size=(50, 3))
    d /= np.linalg.norm(d, axis=1, keepdims=True)
    h = 1e-6
    num = np.stack([(O.basis(d + h * e) - O.basis(d - h * e)) / (2 * h) for e in np.eye(3)], -1)
    assert np.allclose(num, O.basis_grad(d), atol=1e-8)
    # orthonormal over the sphere (Gauss-Legendre x uniform angles integrate degree 6 exactly)
    t, wt = np.polynomial.legendre.leggauss(8)
    ph = 2 * np.pi * np.arange(16) / 16
    s = np.sqrt(1 - t ** 2)
    pts = np.stack([np.outer(s, np.cos(ph)), np.outer(s, np.sin(ph)), np.outer(t, np.ones(16))], -1).reshape(-1, 3)
    w = np.repeat(wt, 16) * 2 * np.pi / 16
    B = O.basis(pts)
    assert np.allclose(np.einsum("p,pi,pj->ij", w, B, B), np.eye(15), atol=1e-12)
    # gradients against differences of the forward statement
    means, sh, dc = rng.normal(size=(7, 3)), rng.normal(size=(7, 15, 3)), rng.normal(size=(7, 3))
    vm = np.stack([np.eye(4), np.eye(4)])
    vm[1, :3, 3] = (0.3, -2.0, 5.0)
    v = rng.normal(size=(2, 7, 3))
    (gm, gd, gs), _ = O.sh_eval_bwd(means, sh, vm, v)
    val = lambda m, c, s_: (O.sh_eval(m, c, s_, vm)[0] * v).sum()
    for k in range(3):
        e = np.zeros((7, 3)); e[3, k] = 1e-6
        assert abs((val(means + e, dc, sh) - val(means - e, dc, sh)) / 2e-6 - gm[3, k]) < 1e-6
        assert abs((val(means, dc + e, sh) - val(means, dc - e, sh)) / 2e-6 - gd[3, k]) < 1e-6
    e = np.zeros_like(sh); e[2, 9, 1] = 1e-6
    assert abs((val(means, dc, sh + e) - val(means, dc, sh - e)) / 2e-6 - gs[2, 9, 1]) < 1e-6


def test_row_oracle_round_trips():
    rng = np.random.default_rng(1)
    sh = (0.05 * rng.normal(size=(200, 15, 3))).astype(np.float32)
    q, s = O.encode_rows(sh)
    q2, s2 = O.unpack_rows(O.pack_rows(q, s))
    assert np.array_equal(q, q2) and np.array_equal(s, s2)
    assert np.abs(q).max() <= 7
    err = np.abs(O.row_values(q, s) - sh)
    for b, (lo, hi) in enumerate(O.BANDS):
        assert np.all(err[:, lo:hi] <= s[:, b][:, None, None] / 2)
        m = np.abs(sh[:, lo:hi]).reshape(200, -1).max(1)
        assert np.all(7 * s[:, b] >= m) and np.all(7 * s[:, b] * (1 - 2.0 ** -7) < m)
    assert not O.row_values(*O.unpack_rows(np.zeros((3, 32), np.uint8))).any()


@pytest.mark.parametrize("rate", [-0.1, 1.0, 2.0, float("nan"), float("inf")])
def test_dropout_refuses_rates_outside_the_range(rate):
    lib = L.load()
    d = L.dropout_struct(rate)
    assert lib.ssb_dropout(ONE, 0, 4, 1, C.byref(d), ONE, None) == L.SSB_ERR_INVALID_ARGUMENT
    assert b"rate" in lib.ssb_last_error_string()
    assert lib.ssb_dropout_opacities(ONE, 0, 4, C.byref(d), ONE, None) == L.SSB_ERR_INVALID_ARGUMENT
    assert lib.ssb_dropout_opacities_bwd(ONE, ONE, 0, 4, C.byref(d), ONE, None) == L.SSB_ERR_INVALID_ARGUMENT


def test_dropout_refusals():
    lib = L.load()
    ok = L.dropout_struct(0.1, 3, 4)
    bad = L.SSB_ERR_INVALID_ARGUMENT
    assert lib.ssb_dropout(ONE, 0, 4, 1, None, ONE, None) == bad
    assert lib.ssb_dropout(None, 0, 4, 1, C.byref(ok), ONE, None) == bad
    assert lib.ssb_dropout(ONE, 0, 4, 1, C.byref(ok), None, None) == bad
    assert lib.ssb_dropout(ONE, 0, 4, 0, C.byref(ok), ONE, None) == bad
    assert lib.ssb_dropout(ONE, 0, 4, -3, C.byref(ok), ONE, None) == bad
    assert lib.ssb_dropout(ONE, -1, 4, 1, C.byref(ok), ONE, None) == bad
    assert lib.ssb_dropout(ONE, 0, -1, 1, C.byref(ok), ONE, None) == bad
    assert lib.ssb_dropout(ONE, 2 ** 62, 2 ** 62, 1, C.byref(ok), ONE, None) == bad
    assert lib.ssb_dropout(C.c_void_p(66), 0, 4, 1, C.byref(ok), ONE, None) == bad            # not on a float boundary
    assert lib.ssb_dropout_opacities(None, 0, 4, C.byref(ok), ONE, None) == bad
    assert lib.ssb_dropout_opacities(ONE, -1, 4, C.byref(ok), ONE, None) == bad
    assert lib.ssb_dropout_opacities_bwd(ONE, None, 0, 4, C.byref(ok), ONE, None) == bad
    assert lib.ssb_dropout_opacities_bwd(ONE, ONE, 0, 4, None, ONE, None) == bad
    r = L.dropout_struct(0.1); r.reserved = 1
    assert lib.ssb_dropout(ONE, 0, 4, 1, C.byref(r), ONE, None) == bad
    r = L.dropout_struct(0.1); r.d_offset = 4
    assert lib.ssb_dropout(ONE, 0, 4, 1, C.byref(r), ONE, None) == bad
    # nothing to do is not an error
    assert lib.ssb_dropout(None, 0, 0, 1, C.byref(ok), None, None) == L.SSB_OK
    assert lib.ssb_dropout_opacities(None, 7, 0, C.byref(ok), None, None) == L.SSB_OK
    assert lib.ssb_dropout_opacities_bwd(None, None, 7, 0, C.byref(ok), None, None) == L.SSB_OK


def test_sh_row_refusals():
    lib = L.load()
    bad = L.SSB_ERR_INVALID_ARGUMENT
    assert lib.ssb_quant_encode(ONE, 44, 4, ONE, None, None) == bad                   # not whole splats
    assert lib.ssb_quant_encode(ONE, -45, 4, ONE, None, None) == bad
    assert lib.ssb_quant_encode(None, 45, 4, ONE, None, None) == bad
    assert lib.ssb_quant_encode(ONE, 45, 4, C.c_void_p(80), None, None) == bad        # rows off the 32-byte boundary
    assert lib.ssb_quant_decode(C.c_void_p(16), None, 45, 4, ONE, None) == bad
    assert lib.ssb_quant_decode(ONE, None, 46, 4, ONE, None) == bad
    assert lib.ssb_quant_encode(ONE, 45, 3, ONE, ONE, None) == bad
    assert lib.ssb_quant_encode(None, 0, 4, None, None, None) == L.SSB_OK
    cfg = L.SsbAdamConfig(0, 0, 0, 0, 0, 1e-3, 0, 1, 1, 0)
    assert lib.ssb_adam_step_sh_quantized(ONE, ONE, ONE, ONE, ONE, 4, 0, 256, 256, C.byref(cfg), None) == bad     # rows are not updated in place


def test_sh_eval_refusals():
    lib = L.load()
    bad = L.SSB_ERR_INVALID_ARGUMENT
    sp, cams, gr = L.SsbSplats(), L.SsbCameras(), L.SsbSplats()
    sp.means, cams.d_viewmats, cams.count = 64, 64, 1
    rows = L.SsbShQuant(64, None, 4, 0, 0)
    fwd = lambda s=sp, q=rows, n=4, c=cams, o=ONE: lib.ssb_sh_eval_fwd(C.byref(s) if s else None, C.byref(q) if q else None, n, C.byref(c) if c else None, o, None)
    bwd = lambda s=sp, q=rows, n=4, c=cams, v=ONE, g=gr: lib.ssb_sh_eval_bwd(C.byref(s), C.byref(q) if q else None, n, C.byref(c), v, C.byref(g) if g else None, 0, None)
    assert fwd(s=None) == bad and fwd(c=None) == bad and fwd(o=None) == bad and fwd(n=-1) == bad
    assert fwd(q=None) == bad                                                          # neither fp32 values nor codes
    assert fwd(q=L.SsbShQuant(80, None, 4, 0, 0)) == bad                               # rows off the 32-byte boundary
    assert fwd(q=L.SsbShQuant(64, None, 16, 0, 256)) == bad                            # 16-bit codes without bounds
    assert bwd(v=None) == bad and bwd(g=None) == bad and bwd(n=-1) == bad
    for field, value in (("sh_degree_plus1", 5), ("sh_degree_plus1", -1), ("count", -1)):
        c = L.SsbCameras(); c.d_viewmats, c.count = 64, 1
        setattr(c, field, value)
        assert fwd(c=c) == bad and bwd(c=c) == bad, field
    c = L.SsbCameras(); c.count = 1
    assert fwd(c=c) == bad
    s = L.SsbSplats()
    assert fwd(s=s) == bad and bwd(s=s) == bad                                         # no means
    assert fwd(n=0) == L.SSB_OK and bwd(n=0) == L.SSB_OK
    c = L.SsbCameras()
    assert fwd(c=c) == L.SSB_OK                                                        # no views


def test_fused_backward_without_sh_values_to_update_is_refused():
    """Views may read rows while the fp32 values are absent, but then the 16-bit-moment step has nothing to update."""
    lib = L.load()
    sp, cams, m, cfg = L.SsbSplats(), L.SsbCameras(), L.SsbSplats(), L.SsbAdamConfig(0, 0, 0, 0, 0, 1e-3, 0, 1, 1, 0)
    m.features_sh = 64
    q16, rows = L.SsbMomentsQ16(), L.SsbShQuant(64, None, 4, 0, 0)
    ws = C.c_void_p(256)
    assert lib.ssb_project_bwd_optimize_q16(C.byref(sp), C.byref(rows), 1000, C.byref(cams), ONE, ONE, C.byref(q16), C.byref(m), C.byref(m), None,
                                            C.byref(cfg), None, ws, 1 << 30, None) == L.SSB_ERR_INVALID_ARGUMENT
    assert b"SH values" in lib.ssb_last_error_string()
