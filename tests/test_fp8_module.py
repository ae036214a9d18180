"""libcmol_b200.fp8 above the library (no GPU needed): what it passes on, with a
stand-in for the library where a call would need a GPU."""
import ctypes as C

import pytest
import torch

import libcmol_b200 as pkg
from libcmol_b200 import fp8


class _Word:
    """A library whose fault word holds `code`."""

    def __init__(self, code):
        self.code, self.asked = code, []

    def cmolcu_fault_status(self, device, out, clear):
        self.asked.append((device, clear))
        C.cast(out, C.POINTER(C.c_uint))[0] = self.code
        if clear:
            self.code = 0
        return 0


def test_a_wait_that_ran_out_is_seen(monkeypatch):
    word = _Word(2)
    monkeypatch.setattr(fp8, "lib", lambda: word)
    assert fp8.fault() == 2 and fp8.fault(3) == 2
    assert fp8.fault(3, clear=True) == 2 and fp8.fault(3) == 0
    assert word.asked == [(0, 0), (3, 0), (3, 1), (3, 0)]


def test_no_word_is_an_error():
    with pytest.raises(pkg.CmolError, match="fp8.fault: cmolcu_fault_status: no fault word for device 99"):
        fp8.fault(99)


def test_activations_that_require_a_gradient_are_refused():
    """While gradients are recorded; the results would be cut from the graph without a word."""
    g, x = torch.zeros(2, 256, requires_grad=True), torch.zeros(2, 256)
    s = torch.zeros(2, 2, requires_grad=True)
    W = fp8.Fp8Weight.__new__(fp8.Fp8Weight)
    W.h, W.rows, W.k, W.index = None, 2, 256, 0
    q = x.to(torch.float8_e4m3fn)
    gains = torch.nn.Parameter(torch.ones(256))
    for call, name in [
        (lambda: fp8.rmsnorm(g, gains), "fp8.rmsnorm: x"),
        (lambda: fp8.rmsnorm(x, gains, residual=g), "fp8.rmsnorm: residual"),
        (lambda: fp8.rmsnorm(x, gains, residual=x, residual_out=g), "fp8.rmsnorm: residual_out"),
        (lambda: fp8.rmsnorm(x, gains, scales=s), "fp8.rmsnorm: scales"),
        (lambda: fp8.quantize(g), "fp8.rmsnorm: x"),
        (lambda: fp8.swiglu(g, x), "fp8.swiglu: gate"),
        (lambda: fp8.swiglu(x, g), "fp8.swiglu: up"),
        (lambda: W.matmul(q, s), "Fp8Weight.matmul: scales"),
        (lambda: W.matmul(q, x[:, :2], y=g), "Fp8Weight.matmul: y"),
    ]:
        with pytest.raises(pkg.CmolError) as e:
            call()
        assert str(e.value).startswith(name + " requires a gradient"), str(e.value)
        with torch.no_grad(), pytest.raises(pkg.CmolError, match="on cpu|shape|scales are"):
            call()
    with pytest.raises(pkg.CmolError, match="wanted a GPU"):         # gains may be a parameter
        fp8.rmsnorm(x, gains)
    with pytest.raises(pkg.CmolError, match="wanted a GPU"):         # and so may a weight that is quantised
        fp8.Fp8Weight.quantize(torch.nn.Parameter(torch.zeros(2, 256)))


def test_forms_of_the_product_are_refused_by_name():
    L = pkg.lib()
    P = 1 << 20
    for form, n, says in [(0, 4, "no form 0"), (7, 4, "no form 7"), (512, 4, "no form 512"),
                          (8, 17, "n=17 is too many for form 8"), (64, 4, "NULL argument"), (256, 4, "NULL argument")]:
        assert L.cmolcu_fp8_matmul_as(form, None, P, 128, P, 1, 4, n, P, 0, 128, None) == -1
        assert pkg.last_error() == f"cmolcu_fp8_matmul_as: {says}"
    assert L.cmolcu_fp8_matmul_form(None, 4) == 0


def test_copies_of_a_weight_are_the_weight(monkeypatch):
    """A weight does not change, and its memory is given back once however it was copied."""
    import copy
    import pickle
    freed = []

    class Lib:
        def cmolcu_fp8_weight_free(self, h):
            freed.append(h)

    monkeypatch.setattr(fp8, "lib", Lib)
    W = fp8.Fp8Weight.__new__(fp8.Fp8Weight)
    W._set(C.c_void_p(64), 2, 256, 0)
    layer = {"w": W}
    for other in (copy.copy(W), copy.deepcopy(W), copy.deepcopy(layer)["w"]):
        assert other is W
    with pytest.raises(pkg.CmolError, match="Fp8Weight: .* read"):
        pickle.dumps(W)
    other.free()
    W.free()
    assert len(freed) == 1
