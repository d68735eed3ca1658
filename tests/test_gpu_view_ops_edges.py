"""The SH product and the dropout of opacities where the ordinary sizes and layouts of their tests do not reach."""
import ctypes as C

import numpy as np
import pytest

torch = pytest.importorskip("torch")

import view_ops_oracle as O  # noqa: E402
from spirula_studio_b200 import lib as L  # noqa: E402
from test_gpu_view_ops import DEV, dev, eval_case, run_bwd, run_fwd, shifted, sources, untouched, within  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def lib():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return L.load()


@pytest.mark.parametrize("fmt", [None, 4, 32])
@pytest.mark.parametrize("n,views", [(700, 1), (700, 2), (700, 35), (40_000, 3)])
def test_degree_zero_does_not_depend_on_the_positions(lib, fmt, n, views):
    """The sum over no coefficient: the value is the DC term and the position has no gradient, whatever the position is."""
    c = eval_case(n, views, seed=5)
    c["means"][0] = np.nan
    c["means"][130, 1], c["means"][259, 2], c["means"][n - 1] = np.inf, -np.inf, (np.nan, np.inf, 1e30)
    src = (None, None) if fmt is None else sources(lib, c["sh"], fmt)
    want = np.broadcast_to(O.C0 * c["dc"].astype(np.float64), (views, n, 3))
    within(run_fwd(lib, c, src, degree=0), want, 2 * O.U * np.abs(want))            # C0 and the product
    g = run_bwd(lib, c, src, degree=0)
    assert not g["means"].any() and not g["features_sh"].any()
    v = c["v"].astype(np.float64)
    within(g["features_dc"], O.C0 * v.sum(0), (views + 2) * O.U * O.C0 * np.abs(v).sum(0))


@pytest.mark.parametrize("rate", [1e-6, 0.1, 0.5, 0.9, 0.9999])
@pytest.mark.parametrize("count,first,sx,sv,so", [
    # 16-byte accesses: every array's offset follows the numbering
    (40001, 0, 0, 0, 0), (40001, 12345, 1, 1, 1), (4099, 6, 2, 2, 2), (2049, 7, 3, 3, 3), (7, 1, 1, 1, 1),
    # one array does not
    (4099, 6, 2, 3, 2), (4099, 6, 2, 2, 0), (4099, 6, 1, 2, 2)])
def test_opacities_on_every_alignment(lib, rate, count, first, sx, sv, so):
    rng = np.random.default_rng(count + first)
    x = rng.normal(size=count).astype(np.float32) * np.where(rng.random(count) < 0.3, 6.0, 1.0).astype(np.float32)
    r = float(np.float32(rate))
    if count > 100:          # next to the limit, where 1 - z cancels, at both ends, and around the change of form at d = 1.375
        edge = np.log(O.CAP * (1 - r) / (1 - O.CAP * (1 - r)))
        x[10:60] = (edge + np.linspace(-1e-3, 1e-3, 50)).astype(np.float32)
        x[60:68] = [80, -80, 1e30, -1e30, np.inf, -np.inf, 0.0, -88.0]
        x[68:168] = (np.log((1 - r) / r) - np.linspace(1.3, 1.45, 100)).astype(np.float32)
    v = rng.normal(size=count).astype(np.float32)
    d = L.dropout_struct(rate, 0x123456789abcdef, 99)
    (bx, vx), (bv, vv), (by, vy), (bg, vg) = (shifted(count, s) for s in (sx, sv, so, so))
    vx.copy_(torch.from_numpy(x)); vv.copy_(torch.from_numpy(v))
    L.check(lib.ssb_dropout_opacities(L.ptr(vx), first, count, C.byref(d), L.ptr(vy), None))
    L.check(lib.ssb_dropout_opacities_bwd(L.ptr(vx), L.ptr(vv), first, count, C.byref(d), L.ptr(vg), None))
    torch.cuda.synchronize()
    y, slope, bound = O.dropout_opacities(x, first, rate, 0x123456789abcdef, 99)
    drop = O.dropped(first, count, 1, rate, 0x123456789abcdef, 99)
    got = vy.cpu().numpy().astype(np.float64)
    inf = ~np.isfinite(y)
    assert np.array_equal(got[inf], y[inf]) and np.all(got[drop] == O.DROPPED)
    within(torch.from_numpy(got[~inf]), y[~inf], bound[~inf])
    within(vg, slope * v, 8 * O.U * np.abs(slope * v))          # w off by 4 U, a quotient of two ulps
    assert not vg.cpu().numpy()[slope == 0].any()
    for b, t in ((bx, vx), (bv, vv), (by, vy), (bg, vg)):
        assert untouched(b, t)
