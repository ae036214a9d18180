"""SwiGLU's value before its rounding to 8 bits, read from the scales: with one
gate that is not zero in a block, the block's scale is |v| / 448 in f32.

Bound, u = 2^-24.  Up to |gate| = 87: the power of two is within 2 units of its
last place (4 u), 1 + exp(-gate) takes two roundings (2 u), the reciprocal is within
one unit (2 u), the two products u each, the scale's product with 1/448 (off by 0.75 u)
1.75 u: 11.75 u, and 87 times the error of f32's ln(2) in the exponent, 2.75e-9: 4.01 u.
Below -87, v = gate * exp(gate/2) * up * exp(gate/2): two exponentials (2 units, 4 u each), three
products and the scale's: 12.75 u.  Terms of second order are below 0.1 u: 16 u for both."""
import pytest

torch = pytest.importorskip("torch")

F32, F16, BF16, E4M3 = torch.float32, torch.float16, torch.bfloat16, torch.float8_e4m3fn
U = 2.0 ** -24
LOWEST = 2.0 ** -126

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _device(gpu):
    pass


def _value(g, u):
    """gate * sigmoid(gate) * up in 64 bits, without overflow."""
    g, u = g.double(), u.double()
    return torch.where(g < 0, g * torch.exp(g) / (1 + torch.exp(g)), g / (1 + torch.exp(-g.clamp_min(0)))) * u


def _one_a_block(g, u, where):
    """Rows of two blocks with gate g[i] at column where[i] of the first and zeros elsewhere."""
    n = g.numel()
    gate, up = torch.zeros(n, 256, device="cuda", dtype=g.dtype), torch.ones(n, 256, device="cuda", dtype=g.dtype)
    i = torch.arange(n, device="cuda")
    gate[i, where], up[i, where] = g, u
    return gate, up


@pytest.mark.parametrize("lo, hi", [(-16, 16), (-30, -16), (-60, -30), (-80, -60), (-88.7, -80), (-104, -88), (-170, -104), (86, 88),
                                    (16, 1000)])
@pytest.mark.parametrize("t", [F32, BF16])
def test_accuracy(lo, hi, t):
    from libcmol_b200 import fp8
    n = 20000
    r = torch.Generator(device="cuda").manual_seed(abs(int(lo)))
    g = (lo + (hi - lo) * torch.rand(n, generator=r, device="cuda", dtype=torch.float64)).to(t)
    # up large enough that v stays well inside f32's normal numbers
    u = ((1 + torch.rand(n, generator=r, device="cuda")) * (2.0 ** 120 if lo < -88.5 else 2.0 ** 30 if lo < -60 else 1.0)).to(t)
    where = torch.randint(0, 128, (n,), generator=r, device="cuda")
    q, s = fp8.swiglu(*_one_a_block(g, u, where))
    want = _value(g, u)
    keep = want.abs() >= 448 * LOWEST
    assert keep.any()
    err = (s[:, 0].double() * 448 - want.abs()).abs()[keep]
    assert (err <= 16 * U * want.abs()[keep]).all(), (err / want.abs()[keep]).max().item() / U
    top = q[torch.arange(n, device="cuda"), where].double()[keep]
    assert (top == 448 * want[keep].sign()).all()
    assert (s[:, 1] == LOWEST).all()


@pytest.mark.parametrize("t", [F32, BF16])
def test_a_value_does_not_depend_on_its_neighbours(t):
    """Gates far out beside an ordinary one, whose value sets the scale, leave its bits as they are."""
    from libcmol_b200 import fp8
    n = 4096
    r = torch.Generator(device="cuda").manual_seed(7)
    g = (3 * torch.randn(n, generator=r, device="cuda")).to(t)
    u = (1 + torch.rand(n, generator=r, device="cuda")).to(t)
    where = 32 + torch.randint(0, 64, (n,), generator=r, device="cuda")
    gate, up = _one_a_block(g, u, where)
    q0, s0 = fp8.swiglu(gate, up)
    for far in (-86.9, -87.1, -88.5, -89.0, -200.0, -3e38):
        for col in (0, 31, 96, 127, 130):
            other = gate.clone()
            other[:, col] = far
            q1, s1 = fp8.swiglu(other, up)
            assert torch.equal(s0[:, 0], s1[:, 0])
            keep = q0.view(torch.uint8)[:, :128] == q1.view(torch.uint8)[:, :128]
            if col < 128:
                keep[:, col] = True
            assert keep.all()


def test_nan_and_infinite_gates_stay_in_their_block():
    from libcmol_b200 import fp8
    r = torch.Generator(device="cuda").manual_seed(8)
    gate, up = 3 * torch.randn(64, 1024, generator=r, device="cuda"), torch.randn(64, 1024, generator=r, device="cuda")
    q0, s0 = fp8.swiglu(gate, up)
    for bad in (float("nan"), float("inf"), -float("inf")):
        far = gate.clone()
        far[:, 300] = bad
        q1, s1 = fp8.swiglu(far, up)
        keep = [b for b in range(8) if b != 2]
        assert torch.equal(s0[:, keep], s1[:, keep])
        a, b = (q.view(torch.uint8).view(64, 8, 128)[:, keep] for q in (q0, q1))
        assert torch.equal(a, b)
        assert torch.isinf(s1[:, 2]).all() if bad == float("inf") else torch.isnan(s1[:, 2]).all()


def test_infinite_gates():
    """gate = inf gives inf * up, as the formula does; -inf gives NaN."""
    from libcmol_b200 import fp8
    gate, up = torch.zeros(4, 128, device="cuda"), torch.ones(4, 128, device="cuda")
    gate[0, 5], gate[1, 5], gate[2, 5], gate[3, 5] = float("inf"), -float("inf"), 3e38, -3e38
    q, s = fp8.swiglu(gate, up)
    assert torch.isinf(s[0, 0]) and torch.isnan(q[0, 5].float()) and torch.isnan(s[1, 0])
    assert s[2, 0].item() == (torch.tensor(3e38) * (torch.tensor(1.0) / 448)).item() and s[3, 0] == LOWEST and (q[3].float() == 0).all()


@pytest.mark.parametrize("t", [F32, F16, BF16])
def test_the_bits_of_f32_arithmetic(t):
    """Ordinary gates: q and scales are those of f32 operations in the formula's order, but for the exponential's last bit."""
    from libcmol_b200 import fp8
    r = torch.Generator(device="cuda").manual_seed(11)
    gate = (3 * torch.randn(300, 2560, generator=r, device="cuda")).to(t)
    up = torch.randn(300, 2560, generator=r, device="cuda").to(t)
    q, s = fp8.swiglu(gate, up)
    g = gate.float()
    b = (g / (1 + torch.exp(-g)) * up.float()).view(300, 20, 128)
    ws = (b.abs().amax(-1) / 448).clamp_min(LOWEST)
    assert ((s - ws).abs() <= 8 * U * ws).all()
    wq = (b / ws.unsqueeze(-1)).to(E4M3).view(300, 2560)
    # two values 16 u apart lie on two sides of one of e4m3's midpoints (2^-3 to 2^-4 of the value apart) once in 2^16
    assert (q.view(torch.uint8) != wq.view(torch.uint8)).float().mean() < 1e-4
