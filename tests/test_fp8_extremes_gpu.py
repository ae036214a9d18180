"""Values at the ends of f32's range, as cmolcu.h documents them."""
import pytest

torch = pytest.importorskip("torch")

F32, E4M3 = torch.float32, torch.float8_e4m3fn

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _device(gpu):
    pass


@pytest.mark.parametrize("form", [8, 16, 32, 64, 128, 256])
def test_scales_whose_product_is_subnormal(form):
    """The product of two scales is off by at most 2^-150 (half of f32's smallest) where it is
    subnormal, and a block's sum is below 448^2 * 128 < 2^25: 2^-125 a block beside the ordinary
    bound ((128 + 3 + 8 + blocks) * 2^-23 of the sum of magnitudes)."""
    from libcmol_b200 import check, fp8, lib
    n, rows, k = (12 if form == 8 else 200), 400, 1040
    g = torch.Generator(device="cuda").manual_seed(form)

    def rand(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    q, wq = ((200 * rand(*s)).clamp(-448, 448).to(E4M3) for s in ((n, k), (rows, k)))
    kb = -(-k // 128)
    s = torch.exp2(-torch.randint(60, 100, (n, kb), generator=g, device="cuda").float()) * (1 + rand(n, kb).abs())
    ws = torch.exp2(-torch.randint(26, 60, (-(-rows // 128), kb), generator=g, device="cuda").float()) * 1.37
    W = fp8.Fp8Weight(wq, ws)
    y = torch.empty(n, rows, device="cuda")
    check(lib().cmolcu_fp8_matmul_as(form, W.h, q.data_ptr(), k, s.data_ptr(), s.stride(0), s.stride(1), n, y.data_ptr(),
                                     0, rows, torch.cuda.current_stream().cuda_stream), "product")
    x = q.double() * s.double().repeat_interleave(128, 1)[:, :k]
    w = wq.double() * ws.double().repeat_interleave(128, 0)[:rows].repeat_interleave(128, 1)[:, :k]
    bound = (128 + 3 + 8 + kb) * 2.0 ** -23 * (x.abs() @ w.abs().t()) + kb * 2.0 ** -125
    assert ((y.double() - x @ w.t()).abs() <= bound).all()


def test_rows_whose_sum_of_squares_passes_f32():
    """They give zeros, and their neighbours what they always give."""
    from libcmol_b200 import fp8
    g = torch.Generator(device="cuda").manual_seed(1)
    w = torch.ones(960, device="cuda")
    x = torch.randn(50, 960, generator=g, device="cuda")
    q0, s0 = fp8.rmsnorm(x, w, 1e-5)
    big = x.clone()
    big[7] *= 1e25
    q, s = fp8.rmsnorm(big, w, 1e-5)
    assert (q[7].float() == 0).all() and (s[7] == 2.0 ** -126).all()
    keep = [i for i in range(50) if i != 7]
    assert torch.equal(q[keep].view(torch.uint8), q0[keep].view(torch.uint8)) and torch.equal(s[keep], s0[keep])
