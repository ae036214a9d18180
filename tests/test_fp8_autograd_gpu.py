"""What the 8-bit operators write counts as modified: a backward pass that saved it
refuses to go on with other values."""
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _device(gpu):
    pass


@pytest.mark.parametrize("what", ["residual in place", "residual_out", "scales", "swiglu scales", "y"])
def test_a_saved_tensor_that_is_written_fails_the_backward_pass(what):
    from libcmol_b200 import fp8
    x, gains = torch.randn(4, 256, device="cuda"), torch.ones(256, device="cuda")
    W = fp8.Fp8Weight.quantize(torch.randn(64, 256, device="cuda"))
    q, s = fp8.quantize(x)
    saved = {"residual in place": x, "residual_out": x, "y": torch.randn(4, 64, device="cuda")}.get(what, s)
    p = torch.ones(1, device="cuda", requires_grad=True)
    z = (saved * p).sum()                       # keeps `saved` for p's gradient
    with torch.no_grad():
        if what == "residual in place":
            fp8.rmsnorm(x.clone(), gains, residual=x)
        elif what == "residual_out":
            fp8.rmsnorm(x.clone(), gains, residual=x.clone(), residual_out=x)
        elif what == "scales":
            fp8.quantize(x, q=q, scales=s)
        elif what == "swiglu scales":
            fp8.swiglu(x, x, q=q, scales=s)
        else:
            W.matmul(q, s, y=saved)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        z.backward()


def test_in_inference_mode():
    from libcmol_b200 import fp8
    with torch.inference_mode():
        x, h = torch.randn(4, 256, device="cuda"), torch.randn(4, 256, device="cuda")
        h0 = h + x
        W = fp8.Fp8Weight.quantize(torch.randn(64, 256, device="cuda"))
        q, s = fp8.rmsnorm(x, torch.ones(256, device="cuda"), residual=h)
        y = W.matmul(q, s)
        assert torch.equal(h, h0) and torch.isfinite(y).all()
        fp8.swiglu(x, x, q=q, scales=s)
