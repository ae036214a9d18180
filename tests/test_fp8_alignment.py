"""Addresses that are no multiple of their element's size are refused by the 8-bit
operators (no GPU needed): a kernel's access there would be misaligned."""
import ctypes as C

import pytest

import libcmol_b200 as pkg
from libcmol_b200 import BF16, F16, F32

P = 1 << 20          # an address that no refused call may touch


def _norm(x=P, xt=F32, res=None, out=None, rt=F32, w=P, s=P):
    return pkg.lib().cmolcu_fp8_rmsnorm(0, x, xt, 256, res, 256, out, 256, rt, w, 1e-5, 4, 256, P, 256, s, 1, 4, None)


@pytest.mark.parametrize("kw", [
    dict(x=P + 2), dict(x=P + 1, xt=BF16), dict(res=P + 2, out=P), dict(res=P, out=P + 2),
    dict(res=P + 1, out=P, rt=F16), dict(w=P + 2), dict(s=P + 1), dict(s=P + 2),
])
def test_rmsnorm(kw):
    assert _norm(**kw) == -1
    assert pkg.last_error() == "cmolcu_fp8_rmsnorm: an address is no multiple of its element's size"


@pytest.mark.parametrize("g, u, t, s", [(P + 2, P, F32, P), (P, P + 1, BF16, P), (P, P, F16, P + 2)])
def test_swiglu(g, u, t, s):
    assert pkg.lib().cmolcu_fp8_swiglu(0, g, 512, u, 512, t, 4, 256, P, 256, s, 1, 4, None) == -1
    assert pkg.last_error() == "cmolcu_fp8_swiglu: an address is no multiple of its element's size"


def test_weights():
    L = pkg.lib()
    for rc, who in [
        (lambda h: L.cmolcu_fp8_weight_upload_dev(0, P, 128, P + 2, 128, 128, None, h), "upload_dev"),
        (lambda h: L.cmolcu_fp8_weight_quantize_dev(0, P + 2, F32, 128, 128, 128, None, h), "quantize_dev"),
        (lambda h: L.cmolcu_fp8_weight_quantize_dev(0, P + 1, BF16, 128, 128, 128, None, h), "quantize_dev"),
    ]:
        h = C.c_void_p(7)
        assert rc(C.byref(h)) == -1 and h.value is None
        assert pkg.last_error() == f"cmolcu_fp8_weight_{who}: an address is no multiple of its element's size"


def test_the_product_checks_before_it_looks_at_a_gpu():
    """A weight stands in by its bytes alone: the refusal comes before any device call."""
    fake = (C.c_char * 256)()
    L = pkg.lib()
    for s, y, t in [(P + 2, P, F32), (P, P + 2, F32), (P, P + 1, BF16)]:
        C.memset(fake, 0, 256)
        C.cast(C.addressof(fake) + 16, C.POINTER(C.c_int))[0] = 128      # rows
        C.cast(C.addressof(fake) + 20, C.POINTER(C.c_int))[0] = 128      # k
        assert L.cmolcu_fp8_matmul(C.addressof(fake), P, 128, s, 1, 4, 4, y, t, 128, None) == -1
        assert pkg.last_error() == "cmolcu_fp8_matmul: an address is no multiple of its element's size"
