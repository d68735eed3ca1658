"""Refusals of the SH product's arguments that a device would answer with a fault."""
import ctypes as C

import pytest

from spirula_studio_b200 import lib as L


@pytest.mark.parametrize("packed,bounds,bits", [(65, 64, 16), (64, 68, 16), (64, 68, 8), (65, 66, 16)])
def test_codes_and_bounds_off_their_boundaries_are_refused(packed, bounds, bits):
    """The kernels read 16-bit codes and (min, max) pairs as such: an address between two of them is a misaligned access."""
    lib = L.load()
    sp, cams, gr = L.SsbSplats(), L.SsbCameras(), L.SsbSplats()
    sp.means = sp.quats = sp.scales = sp.opacities = sp.features_dc = 64
    cams.d_viewmats, cams.d_intrins, cams.count, cams.width, cams.height = 64, 64, 1, 16, 16
    q = L.SsbShQuant(packed, bounds, bits, 0, 256)
    one = C.c_void_p(64)
    for status in (lib.ssb_sh_eval_fwd(C.byref(sp), C.byref(q), 4, C.byref(cams), one, None),
                   lib.ssb_sh_eval_bwd(C.byref(sp), C.byref(q), 4, C.byref(cams), one, C.byref(gr), 0, None),
                   lib.ssb_project_fwd(C.byref(sp), C.byref(q), 4, C.byref(cams), one, one, None, one, None)):
        assert status == L.SSB_ERR_INVALID_ARGUMENT
        assert b"boundary" in lib.ssb_last_error_string()
