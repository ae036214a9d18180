"""The 8-bit floating point operators' argument checks (no GPU needed): every
refusal comes before any device work, with a message that names the call."""
import ctypes as C

import pytest

import libcmol_b200 as pkg
from libcmol_b200 import BF16, F16, F32

P = 1 << 20          # an address that no refused call may touch
LL = C.c_longlong


def _norm(device=0, x=P, xt=F32, x_ld=256, res=None, res_ld=0, out=None, out_ld=0, rt=F32, w=P, eps=1e-5, n=4, k=256,
          q=P, q_ld=256, s=P, s_ld=1, s_inc=4):
    return pkg.lib().cmolcu_fp8_rmsnorm(device, x, xt, x_ld, res, res_ld, out, out_ld, rt, w, eps, n, k, q, q_ld, s,
                                        s_ld, s_inc, None)


def _swiglu(g=P, g_ld=512, u=P, u_ld=512, t=BF16, n=4, k=256, q=P, q_ld=256, s=P, s_ld=1, s_inc=4):
    return pkg.lib().cmolcu_fp8_swiglu(0, g, g_ld, u, u_ld, t, n, k, q, q_ld, s, s_ld, s_inc, None)


@pytest.mark.parametrize("kw, says", [
    (dict(k=250), "multiple of 16"), (dict(k=0), "multiple of 16"), (dict(n=-1), "n=-1"),
    (dict(xt=2), "dtype 2"), (dict(res=P, out=P, out_ld=256, rt=8), "dtype 8"),
    (dict(x=None), "NULL"), (dict(q=None), "NULL"), (dict(s=None), "NULL"),
    (dict(res=P, res_ld=256), "NULL"), (dict(out=P, out_ld=256), "NULL"),
    (dict(res=P, res_ld=256, out=P, out_ld=255), "overlap"),
    (dict(q=P + 8), "16-byte"), (dict(q_ld=264), "16-byte"), (dict(q_ld=240), "16-byte"),
    (dict(s_ld=1, s_inc=3), "overlap"), (dict(s_ld=0), "overlap"), (dict(s_ld=1, s_inc=1), "overlap"),
])
def test_rmsnorm_refusals(kw, says):
    assert _norm(**kw) == -1
    msg = pkg.last_error()
    assert msg.startswith("cmolcu_fp8_rmsnorm") and says in msg, msg


@pytest.mark.parametrize("kw, says", [
    (dict(k=8), "multiple of 16"), (dict(n=-3), "n=-3"), (dict(t=14), "dtype 14"), (dict(g=None), "NULL"),
    (dict(u=None), "NULL"), (dict(q=P + 4), "16-byte"), (dict(q_ld=128), "16-byte"), (dict(s_inc=0), "overlap"),
])
def test_swiglu_refusals(kw, says):
    assert _swiglu(**kw) == -1
    msg = pkg.last_error()
    assert msg.startswith("cmolcu_fp8_swiglu") and says in msg, msg


def test_no_rows_do_nothing():
    assert _norm(n=0, x=None, q=None, s=None) == 0
    assert _swiglu(n=0, g=None, u=None, q=None, s=None) == 0


def test_weight_refusals():
    L = pkg.lib()
    h = C.c_void_p(7)

    def refused(rc, says):
        assert rc == -1 and h.value is None and says in pkg.last_error(), pkg.last_error()
        h.value = 7

    refused(L.cmolcu_fp8_weight_upload(0, None, P, 128, 128, C.byref(h)), "NULL")
    refused(L.cmolcu_fp8_weight_upload(0, P, None, 128, 128, C.byref(h)), "NULL")
    refused(L.cmolcu_fp8_weight_upload(0, P, P, 0, 128, C.byref(h)), "rows=0")
    refused(L.cmolcu_fp8_weight_upload(0, P, P, 128, 120, C.byref(h)), "multiple of 16")
    refused(L.cmolcu_fp8_weight_upload_dev(0, P, 112, P, 128, 128, None, C.byref(h)), "ld=112")
    refused(L.cmolcu_fp8_weight_upload_dev(0, P, 136, P, 128, 128, None, C.byref(h)), "16-byte")
    refused(L.cmolcu_fp8_weight_upload_dev(0, P + 8, 128, P, 128, 128, None, C.byref(h)), "16-byte")
    refused(L.cmolcu_fp8_weight_quantize_dev(0, P, 8, 128, 128, 128, None, C.byref(h)), "dtype 8")
    refused(L.cmolcu_fp8_weight_quantize_dev(0, P, F16, 128, 1 << 24, 128, None, C.byref(h)), "too many")
    assert L.cmolcu_fp8_weight_upload(0, P, P, 128, 128, None) == -1
    L.cmolcu_fp8_weight_free(None)
    assert L.cmolcu_fp8_weight_bytes(None) == 0


def test_product_without_a_weight_is_refused():
    assert pkg.lib().cmolcu_fp8_matmul(None, P, 128, P, 1, 4, 4, P, F32, 128, None) == -1
    assert pkg.last_error() == "cmolcu_fp8_matmul: NULL argument"
    assert pkg.lib().cmolcu_fp8_weight_read_dev(None, P, 128, P, None) == -1


def test_tensor_checks_name_the_argument():
    import torch
    from libcmol_b200 import CmolError, fp8
    x = torch.zeros(2, 256)
    for call, says in [
        (lambda: fp8.rmsnorm(x.double(), None), "x: dtype"),
        (lambda: fp8.rmsnorm(x, None), "wanted a GPU"),
        (lambda: fp8.rmsnorm(x[0], None), "two dimensions"),
        (lambda: fp8.swiglu(x.to(torch.int8), x), "gate: dtype"),
        (lambda: fp8.Fp8Weight(x, x), "float8_e4m3fn"),
        (lambda: fp8.Fp8Weight(x.to(torch.float8_e4m3fn), torch.zeros(2, 2)), "scales are float32 (1, 2)"),
        (lambda: fp8.Fp8Weight.quantize(x), "wanted a GPU"),
    ]:
        with pytest.raises(CmolError, match=None) as e:
            call()
        assert says in str(e.value), str(e.value)
