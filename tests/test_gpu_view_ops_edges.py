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
