"""The quantisers' arithmetic, bit for bit: scale = max(amax * r, 2^-126) with r the f32 next to
1 / 448, and q = v / scale rounded to nearest even after IEEE's rounding of the quotient
to f32.  The wanted values come from the CPU, and from f32 torch operations on the GPU.

A quotient whose distance from a midpoint of f32 is below 2^-45 of its size may
fall on the other side (one in 2^20 values); to show in q it has to lie beside a
midpoint of e4m3 as well, so none is expected among the 10^7 values here."""
import pytest

torch = pytest.importorskip("torch")

F32, F16, BF16, E4M3 = torch.float32, torch.float16, torch.bfloat16, torch.float8_e4m3fn
LOWEST = 2.0 ** -126
R = torch.tensor(1.0) / 448.0

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _device(gpu):
    pass


def _same(q, want):
    """The same bytes, any NaN for a NaN."""
    q, want = q.cpu().contiguous(), want.contiguous()
    a, b = q.view(torch.uint8), want.view(torch.uint8)
    ok = (a == b) | (torch.isnan(q.float()) & torch.isnan(want.float()))
    assert ok.all(), f"{(~ok).sum().item()} of {ok.numel()} values differ"


def _quotients(b, s):
    return (b / s).clamp(-448, 448).to(E4M3)     # a NaN passes the clamp


def _want_rows(x):
    """q and scales of rows, by the CPU."""
    x = x.float().cpu()
    n, k = x.shape
    kb = -(-k // 128)
    b = torch.nn.functional.pad(x, (0, kb * 128 - k)).view(n, kb, 128)
    s = (b.abs().amax(-1) * R).clamp_min(LOWEST)
    return _quotients(b, s.unsqueeze(-1)).view(n, -1)[:, :k], s


def _check_rows(x):
    from libcmol_b200 import fp8
    q, s = fp8.quantize(x)
    wq, ws = _want_rows(x)
    s = s.cpu()
    assert ((s == ws) | (s.isnan() & ws.isnan())).all(), f"{(s != ws).sum().item()} of {s.numel()} scales differ"
    _same(q, wq)


@pytest.mark.parametrize("t", [F32, F16, BF16])
@pytest.mark.parametrize("n, k", [(1021, 2064), (3, 208), (257, 11008)])
def test_scales_and_quotients_of_rows(n, k, t):
    g = torch.Generator(device="cuda").manual_seed(n)
    x = torch.randn(n, k, generator=g, device="cuda")
    x[:, ::61] *= 30
    _check_rows(x.to(t))


def test_scales_from_the_smallest_to_the_largest():
    """Blocks of every binary exponent, subnormal ones among them."""
    g = torch.Generator().manual_seed(1)
    e = torch.arange(-149, 128).double().repeat_interleave(8)
    m = 1 + torch.rand(e.numel(), 128, generator=g, dtype=torch.float64)
    sign = torch.randint(0, 2, m.shape, generator=g) * 2 - 1
    small = torch.randint(0, 14, m.shape, generator=g)
    x = (m * torch.exp2(e[:, None] - small) * sign).float()
    assert torch.isfinite(x).all()
    _check_rows(x.cuda())


def test_values_between_two_of_e4m3():
    """v / scale next to and at the midpoints of e4m3: a tie goes to the even one."""
    g = torch.Generator().manual_seed(2)
    top = 448 * torch.exp2(torch.randint(-20, 20, (512, 1), generator=g).float()) * (
        1 + torch.randint(0, 1 << 10, (512, 1), generator=g).float() / (1 << 10))
    s = top * R
    grid = torch.arange(0, 127, dtype=torch.uint8).view(E4M3).float()
    mid = (grid[1:] + grid[:-1]) / 2
    v = s * mid[torch.randint(0, 126, (512, 126), generator=g)]
    x = torch.cat([top, v, torch.zeros(512, 1)], 1)
    for y in (x, x.nextafter(torch.tensor(0.0)), x.nextafter(torch.tensor(float("inf")))):
        y[:, 0] = top[:, 0]
        y[::2, 1::3] *= -1
        _check_rows(y.cuda())


def test_infinite_and_nan_blocks_and_signed_zeros():
    """Beside an infinity finite values are zero, with their sign; a NaN makes its block NaN."""
    x = torch.randn(6, 384, generator=torch.Generator().manual_seed(3))
    x[0, 130], x[1, 3], x[2, 200] = float("inf"), -float("inf"), float("nan")
    x[3, :] = -0.0
    x[4, ::2] = -0.0
    x[5, 128:] = -1e-45
    for t in (F32, BF16):
        _check_rows(x.to(t).cuda())


@pytest.mark.parametrize("t", [F32, F16, BF16])
def test_weights(t):
    from libcmol_b200 import fp8
    rows, k = 1025, 2064
    g = torch.Generator(device="cuda").manual_seed(4)
    w = (0.02 * torch.randn(rows, k, generator=g, device="cuda")).to(t)
    if t == F32:
        w[:128] *= 1e-34                   # scales below the smallest whose products are exact
        w[128:256, 128:256] = 0
        w[700, 300] = float("inf")
    q, s = fp8.Fp8Weight.quantize(w).read()
    rb, kb = -(-rows // 128), -(-k // 128)
    p = torch.zeros(rb * 128, kb * 128)
    p[:rows, :k] = w.float().cpu()
    p = p.view(rb, 128, kb, 128)
    want = (p.abs().amax((1, 3)) * R).clamp_min(LOWEST)
    assert (s.cpu() == want).all()
    _same(q, _quotients(p, want[:, None, :, None]).reshape(rb * 128, kb * 128)[:rows, :k])


@pytest.mark.parametrize("t", [F32, F16, BF16])
def test_the_bits_of_torch_operations_on_the_gpu(t):
    from libcmol_b200 import fp8
    g = torch.Generator(device="cuda").manual_seed(6)
    x = torch.randn(1000, 2560, generator=g, device="cuda").to(t)
    q, s = fp8.quantize(x)
    b = x.float().view(1000, 20, 128)
    ws = (b.abs().amax(-1) / 448.0).clamp_min(LOWEST)
    assert torch.equal(s, ws)
    _same(q, (b / ws.unsqueeze(-1)).clamp(-448, 448).to(E4M3).view(1000, 2560).cpu())
