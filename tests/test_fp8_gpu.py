"""The 8-bit floating point operators (cmolcu_fp8_*, libcmol_b200.fp8) against
plain implementations in 64 bits.

Bounds.  u = 2^-24 is half a step of f32.
 - A sum of squares adds at most L = 8 * max(8, ceil(k / 2048)) terms one after
   another in a lane and then 10 partial sums, all positive: relative error at
   most (L + 12) u, half of that in 1/sqrt(mean + eps) and 4 u more for the
   quotients and the root; h, g * (h * ir) and the scale's quotient add 4 u.  So
   v / s is within DELTA = ((L + 12) / 2 + 10) u of the exact one, and q lies
   between the roundings of v / s (1 - DELTA) and v / s (1 + DELTA).  A scale is
   within DELTA of its own.
 - SwiGLU: exp(-g) is within 4 u (its own error) + 2 u |g| (its argument's, for
   an exponential formed in base 2) and enters 1 + exp(-g) with weight at most
   one; the quotient, two products and the scale's add 8 u.  With |g| <= 16 here
   DELTA = 50 u.
 - A stored residual is off by half a step of its type, and u for the f32 sum.
 - The product: a block's 128 products are exact in f32 and their sum is off by
   at most 128 * 2^-23 of the sum of magnitudes (each addition may truncate);
   scaling and adding the blocks cost (3 + blocks) * 2^-23 more, the output half
   a step of its type.
"""
import itertools

import numpy as np
import pytest

torch = pytest.importorskip("torch")

F32, F16, BF16, E4M3 = torch.float32, torch.float16, torch.bfloat16, torch.float8_e4m3fn
U = 2.0 ** -24
MIN_SCALE = 2.0 ** -126

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _device(gpu):
    torch.backends.cuda.matmul.allow_tf32 = False


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape, dtype=F32):
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def _round(v):
    """e4m3 rounding of f64 values, as f64."""
    return v.clamp(-448, 448).float().to(E4M3).double()


def _blocked(v):
    n, k = v.shape
    kb = -(-k // 128)
    return torch.nn.functional.pad(v, (0, kb * 128 - k)).view(n, kb, 128)


def _check_eight_bits(v, q, s, delta):
    """q, s are the 8-bit form of the f64 values v up to a relative delta."""
    n, k = v.shape
    b = _blocked(v)
    want = (b.abs().amax(-1) / 448).clamp_min(MIN_SCALE)
    assert s.shape == want.shape and s.dtype == F32 and q.dtype == E4M3
    assert ((s.double() - want).abs() <= delta * want + 2 ** -149).all()
    r = (b / want.unsqueeze(-1)).view(n, -1)[:, :k]
    a, c = _round(r * (1 - delta)), _round(r * (1 + delta))
    got = q.double()
    assert ((got >= torch.minimum(a, c)) & (got <= torch.maximum(a, c))).all()


def _norm_delta(k):
    return ((8 * max(8, -(-k // 2048)) + 12) / 2 + 10) * U


def _norm_ref(x, r, g, eps):
    h = x.double() + (r.double() if r is not None else 0)
    v = h if g is None else g.double() * h / torch.sqrt((h * h).mean(-1, keepdim=True) + eps)
    return h, v


STEP = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}


# every width of the kernel's choice of lanes, ragged last blocks, a row that is read twice
@pytest.mark.parametrize("n, k", [(1, 16), (1, 960), (3, 576), (5, 128), (2, 144), (257, 2048), (33, 8192), (700, 11008),
                                  (2, 12288), (2, 16400), (1, 40016), (1500, 256), (4099, 64), (9000, 960), (3, 3824)])
@pytest.mark.parametrize("xt, rt", [(F32, F32), (BF16, BF16), (F16, None), (BF16, F32)])
def test_rmsnorm(n, k, xt, rt):
    from libcmol_b200 import fp8
    g = _gen(n + k)
    x = _randn(g, n, k, dtype=xt)
    r = None if rt is None else (3 * _randn(g, n, k)).to(rt)
    w = 1 + 0.1 * _randn(g, k)
    out = None if r is None else torch.empty_like(r)
    q, s = fp8.rmsnorm(x, w, 1e-5, residual=r, residual_out=out)
    h, v = _norm_ref(x, r, w, 1e-5)
    _check_eight_bits(v, q, s, _norm_delta(k))
    if r is not None:
        assert ((out.double() - h).abs() <= (STEP[rt] + U) * h.abs() + 2 ** -25).all()


@pytest.mark.parametrize("n, k", [(1, 16), (7, 960), (300, 2064), (9, 17008), (130, 400), (77, 64), (3, 992)])
@pytest.mark.parametrize("xt", [F32, F16, BF16])
def test_quantize(n, k, xt):
    from libcmol_b200 import fp8
    x = _randn(_gen(k), n, k, dtype=xt)
    x[:, ::37] *= 50
    q, s = fp8.quantize(x)
    _check_eight_bits(x.double(), q, s, 4 * U)


def test_rmsnorm_residual_in_place_and_repeated():
    from libcmol_b200 import fp8
    g = _gen(5)
    x, r, w = _randn(g, 9, 960, dtype=BF16), _randn(g, 9, 960), 1 + 0.1 * _randn(g, 960)
    out = torch.empty_like(r)
    q0, s0 = fp8.rmsnorm(x, w, 1e-5, residual=r, residual_out=out)
    q1, s1 = fp8.rmsnorm(x, w, 1e-5, residual=r)
    assert torch.equal(r, out) and torch.equal(q0.view(torch.uint8), q1.view(torch.uint8)) and torch.equal(s0, s1)


def test_rmsnorm_strides_and_what_lies_between():
    """Rows of wider buffers at any alignment; bytes between the rows stay."""
    from libcmol_b200 import fp8
    g = _gen(6)
    n, k = 13, 336
    for off, pad in [(0, 0), (8, 8), (1, 7), (3, 0), (0, 5)]:
        x = _randn(g, n, k + off + pad, dtype=BF16)[:, off:off + k]
        r = _randn(g, n, k + off + pad + 1)[:, off:off + k]
        wfull = 1 + 0.1 * _randn(g, k + off)
        w = wfull[off:]
        rbuf = torch.full((n, k + off + pad), 7.0, device="cuda")
        qbuf = torch.full((n, k + 32), 0x55, dtype=torch.uint8, device="cuda")
        sbuf = torch.full((n, 8), -1.0, device="cuda")
        rout, q, s = rbuf[:, off:off + k], qbuf[:, 16:16 + k].view(E4M3), sbuf[:, 1:7:2]
        fp8.rmsnorm(x, w, 1e-6, residual=r, residual_out=rout, q=q, scales=s)
        h, v = _norm_ref(x, r, w, 1e-6)
        _check_eight_bits(v, q, s, _norm_delta(k))
        assert ((rout.double() - h).abs() <= 2 * U * h.abs()).all()
        assert (qbuf[:, :16] == 0x55).all() and (qbuf[:, 16 + k:] == 0x55).all()
        assert (sbuf[:, ::2] == -1).all() and sbuf[:, 7].eq(-1).all()
        assert (rbuf[:, :off] == 7).all() and (rbuf[:, off + k:] == 7).all()


def test_quantisers_at_the_edges_of_the_range():
    """Zeros, subnormals, the largest values, NaN and infinities: each block by itself."""
    from libcmol_b200 import fp8
    x = torch.zeros(8, 384, device="cuda")
    x[1, 0] = 1e-44                      # the scale's floor
    x[2, 5] = 3.4e38
    x[2, 6] = -1e30
    x[3, 130] = float("nan")
    x[4, 130] = float("inf")
    x[5, 130] = -float("inf")
    x[3:6, 0] = x[3:6, 300] = 2.0
    x[6] = 1e-40
    x[7] = -448.0
    q, s = fp8.quantize(x)
    qd = q.double()
    ok = [0, 1, 2, 6, 7]
    _check_eight_bits(x[ok].double(), q[ok], s[ok], 4 * U)
    assert torch.isnan(s[3, 1]) and torch.isinf(s[4, 1]) and torch.isinf(s[5, 1])
    assert torch.isnan(qd[3, 130]) and torch.isnan(qd[4, 130]) and torch.isnan(qd[5, 130])
    for row in (3, 4, 5):                # the other blocks of the row are as ever
        assert s[row, 0] == s[row, 2] == torch.tensor(2.0 / 448) and qd[row, 0] == qd[row, 300] == 448
    w = torch.ones(384, device="cuda")
    q, s = fp8.rmsnorm(x[3:6], w, 1e-5)
    assert (s.isnan() | s.isinf() | q.double().isnan().view(3, 3, 128).any(-1) | (s == MIN_SCALE)).all()
    q, s = fp8.rmsnorm(x[:1], w, 1e-5)   # a row of zeros
    assert (q.double() == 0).all() and (s == MIN_SCALE).all()


def test_broadcast_row():
    """One row read for all (stride 0)."""
    from libcmol_b200 import fp8
    g = _gen(8)
    x, r, w = _randn(g, 1, 576), _randn(g, 6, 576), torch.ones(576, device="cuda")
    q, s = fp8.rmsnorm(x.expand(6, 576), w, 1e-5, residual=r, residual_out=torch.empty_like(r))
    _check_eight_bits(_norm_ref(x.expand(6, 576), r, w, 1e-5)[1], q, s, _norm_delta(576))


@pytest.mark.parametrize("n, k", [(1, 16), (1, 2560), (6, 144), (301, 8192), (64, 11008), (3, 2064), (1000, 48), (130, 400), (5, 208)])
@pytest.mark.parametrize("t", [F32, F16, BF16])
def test_swiglu(n, k, t):
    from libcmol_b200 import fp8
    g = _gen(n * k)
    both = (3 * _randn(g, n, 2 * k)).clamp(-16, 16).to(t)
    q, s = fp8.swiglu(both[:, :k], both[:, k:])
    gd = both[:, :k].double()
    _check_eight_bits(gd / (1 + torch.exp(-gd)) * both[:, k:].double(), q, s, 50 * U)


def test_swiglu_saturated_gates_and_strides():
    """Gates far out on both sides; unaligned halves; bytes between the rows stay."""
    from libcmol_b200 import fp8
    g = _gen(3)
    n, k = 5, 208
    buf = _randn(g, n, 2 * k + 3)
    gate, up = buf[:, 1:1 + k], buf[:, k + 2:2 * k + 2]
    gate[0, :4] = torch.tensor([-1e4, 1e4, -90.0, 90.0], device="cuda")
    gate[1] = -200.0                      # every product vanishes
    qbuf = torch.full((n, k + 16), 0x11, dtype=torch.uint8, device="cuda")
    q, s = fp8.swiglu(gate, up, q=qbuf[:, :k].view(E4M3))
    gd = gate.double()
    v = gd / (1 + torch.exp(-gd)) * up.double()
    rows = [0, 2, 3, 4]
    _check_eight_bits(v[rows], q[rows], s[rows], 250 * U)    # |g| <= 1e4, but exp(-g) counts only up to g = -90 here
    assert (q[1].double() == 0).all() and (s[1] == MIN_SCALE).all()
    assert (qbuf[:, k:] == 0x11).all()


# ---------------------------------------------------------------------------
# Weights and the product
# ---------------------------------------------------------------------------
def _weight(g, rows, k, dtype=F32):
    return (0.02 * _randn(g, rows, k) * torch.exp(_randn(g, rows, 1))).to(dtype)


@pytest.mark.parametrize("rows, k", [(1, 16), (128, 128), (200, 960), (129, 1040), (576, 64)])
@pytest.mark.parametrize("t", [F32, F16, BF16])
def test_weight_quantize_and_read(rows, k, t):
    from libcmol_b200 import fp8
    w = _weight(_gen(rows + k), rows, k, t)
    W = fp8.Fp8Weight.quantize(w)
    q, s = W.read()
    rb, kb = -(-rows // 128), -(-k // 128)
    p = torch.zeros(rb * 128, kb * 128, dtype=torch.float64, device="cuda")
    p[:rows, :k] = w.double()
    p = p.view(rb, 128, kb, 128)
    want = (p.abs().amax((1, 3)) / 448).clamp_min(MIN_SCALE)
    assert ((s.double() - want).abs() <= U * 2 * want).all()
    r = (p / want[:, None, :, None]).reshape(rb * 128, kb * 128)[:rows, :k]
    a, c = _round(r * (1 - 4 * U)), _round(r * (1 + 4 * U))
    assert ((q.double() >= torch.minimum(a, c)) & (q.double() <= torch.maximum(a, c))).all()
    assert W.nbytes == rows * k + 4 * rb * kb
    # the same weight from its own values: from the device, a wider buffer, the host
    wide = torch.full((rows, k + 16), 0x7F, dtype=torch.uint8, device="cuda")
    wide[:, :k] = q.view(torch.uint8)
    for V in (fp8.Fp8Weight(q, s), fp8.Fp8Weight(wide.view(E4M3)[:, :k], s), fp8.Fp8Weight(q.cpu(), s.cpu())):
        q2, s2 = V.read()
        assert torch.equal(q2.view(torch.uint8), q.view(torch.uint8)) and torch.equal(s2, s)
        V.free()


def _acts(g, n, k):
    """Any e4m3 values with any scales (not only those that a quantiser leaves)."""
    q = (200 * _randn(g, n, k)).clamp(-448, 448).to(E4M3)
    s = torch.exp(_randn(g, -(-k // 128), n)).t()
    return q, s


def _mm_ref(q, s, wq, ws):
    """(exact product, sum of magnitudes)."""
    n, k = q.shape
    rows = wq.shape[0]
    x = q.double() * s.double().repeat_interleave(128, 1)[:, :k]
    w = wq.double() * ws.double().repeat_interleave(128, 0)[:rows].repeat_interleave(128, 1)[:, :k]
    return x @ w.t(), x.abs() @ w.abs().t()


def _mm_check(y, q, s, wq, ws):
    want, mag = _mm_ref(q, s, wq, ws)
    kb = -(-q.shape[1] // 128)
    bound = (128 + 3 + kb) * 2.0 ** -23 * mag + (STEP[y.dtype] if y.dtype != F32 else 0) * want.abs()
    if y.dtype == F16:
        bound += 2.0 ** -25
    err = (y.double() - want).abs()
    assert torch.isfinite(y).all() and (err <= bound).all(), (err / bound).max().item()


MM = [(1, 16, 16), (1, 128, 128), (1, 960, 2560), (2, 300, 960), (1, 2048, 11008), (3, 129, 144), (4, 4096, 576),
      (5, 257, 1040), (8, 2048, 2048), (13, 1000, 1296), (16, 64, 4096), (17, 384, 2064), (31, 2049, 640), (37, 2048, 1100 * 16),
      (64, 515, 2048), (65, 515, 2048), (100, 640, 960), (128, 1536, 576), (129, 256, 256), (200, 2304, 2048),
      (256, 5000, 1024), (257, 384, 512), (300, 130, 4112), (511, 2560, 960), (777, 641, 1536), (1025, 1281, 400), (2000, 4100, 96), (384, 960, 2560), (130, 2048, 11008),
      (3000, 2500, 2048)]


@pytest.mark.parametrize("n, rows, k", MM, ids=["x".join(map(str, c)) for c in MM])
@pytest.mark.parametrize("t", [F32, F16, BF16])
def test_matmul(n, rows, k, t):
    from libcmol_b200 import fp8
    g = _gen(n + rows + k)
    q, s = _acts(g, n, k)
    W = fp8.Fp8Weight.quantize(_weight(g, rows, k))
    wq, ws = W.read()
    if t == F16:
        s = s * 1e-3                      # keeps |y| inside f16
    y = W.matmul(q, s, dtype=t)
    _mm_check(y, q, s, wq, ws)
    again = W.matmul(q, s, dtype=t)
    assert torch.equal(y, again)


@pytest.mark.parametrize("n", [1, 2, 4, 7, 40, 150, 400])
def test_matmul_strides_and_what_lies_between(n):
    """Rows of wider buffers whose other bytes are NaN; both orders of the
    scales; what lies between the rows of y stays."""
    from libcmol_b200 import fp8
    g = _gen(n)
    rows, k = 333, 400
    q0, s0 = _acts(g, n, k)
    qbuf = torch.full((n + 2, k + 48), 0x7F, dtype=torch.uint8, device="cuda")
    q = qbuf[1:n + 1, 16:16 + k].view(E4M3)
    q.view(torch.uint8).copy_(q0.view(torch.uint8))
    W = fp8.Fp8Weight.quantize(_weight(g, rows, k))
    wq, ws = W.read()
    sbuf = torch.full((n, 9), float("nan"), device="cuda")
    for s in (s0, s0.contiguous(), sbuf[:, 1:9:2]):
        s.copy_(s0)
        for off, pad, t in [(0, 3, F32), (1, 0, BF16), (8, 3, F16), (16, 7, F32)]:
            f = 1e-3 if t == F16 else 1.0
            ybuf = torch.full((n, off + rows + pad), 5.0, dtype=t, device="cuda")
            y = ybuf[:, off:off + rows]
            W.matmul(q, (s * f) if t == F16 else s, y=y)
            _mm_check(y, q0, s0 * f, wq, ws)
            assert (ybuf[:, :off] == 5).all() and (ybuf[:, off + rows:] == 5).all()


@pytest.mark.parametrize("n", [1, 3, 20, 200, 600])
def test_matmul_nan_and_infinite_rows_stay_by_themselves(n):
    from libcmol_b200 import fp8
    g = _gen(n)
    rows, k = 300, 640
    q, s = _acts(g, n, k)
    w = _weight(g, rows, k)
    W = fp8.Fp8Weight.quantize(w)
    wq, ws = W.read()
    bad = n // 2
    for what in ("q", "scale nan", "scale inf", "zero scale"):
        q1, s1 = q.clone(), s.clone()
        if what == "q":
            q1.view(torch.uint8)[bad, 200] = 0x7F
        else:
            s1[bad, 2] = {"scale nan": float("nan"), "scale inf": float("inf"), "zero scale": 0.0}[what]
        y = W.matmul(q1, s1)
        if what == "zero scale":
            _mm_check(y, q1, s1, wq, ws)
            continue
        assert not torch.isfinite(y[bad]).any()
        keep = [i for i in range(n) if i != bad]
        if keep:
            _mm_check(y[keep], q[keep], s[keep], wq, ws)
    w[150, 300] = float("nan")            # a NaN weight reaches the 128 rows of its block alone
    V = fp8.Fp8Weight.quantize(w)
    y = V.matmul(q, s)
    assert torch.isnan(y[:, 128:256]).all()
    _mm_check(y[:, :128], q, s, wq[:128], ws[:1])
    _mm_check(y[:, 256:], q, s, wq[256:], ws[2:])


@pytest.mark.parametrize("n", [1, 6, 50, 300])
def test_matmul_of_zeros_and_of_one_hot(n):
    """Exact cases: every value lands where it belongs."""
    from libcmol_b200 import fp8
    rows, k = 515, 1168
    g = _gen(2)
    wq = (100 * _randn(g, rows, k)).clamp(-448, 448).to(E4M3)
    ws = torch.ones(5, 10, device="cuda")
    W = fp8.Fp8Weight(wq, ws)
    q = torch.zeros(n, k, device="cuda")
    cols = torch.randint(0, k, (n,), generator=g, device="cuda")
    q[torch.arange(n, device="cuda"), cols] = 1
    s = torch.full((n, 10), 2.0, device="cuda")
    assert torch.equal(W.matmul(q.to(E4M3), s), 2 * wq.float()[:, cols].t())
    assert (W.matmul(torch.zeros(n, k, device="cuda").to(E4M3), s) == 0).all()


def test_product_refusals():
    from libcmol_b200 import CmolError, fp8
    W = fp8.Fp8Weight.quantize(torch.ones(64, 256, device="cuda"))
    q, s = fp8.quantize(torch.ones(4, 256, device="cuda"))
    cases = [
        (lambda: W.matmul(q[:, :240], s), "q: shape"),
        (lambda: W.matmul(q.float(), s), "q: dtype"),
        (lambda: W.matmul(q, s[:, :1]), "scales are float32 (4, 2)"),
        (lambda: W.matmul(q, s.half()), "scales are float32"),
        (lambda: W.matmul(q.cpu(), s), "q: on cpu"),
        (lambda: W.matmul(q, s, dtype=torch.float64), "y: dtype"),
        (lambda: W.matmul(q, s, y=torch.empty(4, 63, device="cuda")), "y: shape"),
        (lambda: W.matmul(q, s, y=torch.empty(64, 4, device="cuda").t()), "consecutive"),
        (lambda: W.matmul(q, s, y=torch.empty(1, 64, device="cuda").expand(4, 64)), "rows of y overlap"),
        (lambda: W.matmul(torch.zeros(4, 264, dtype=torch.uint8, device="cuda")[:, :256].view(E4M3), s), "16-byte"),
        (lambda: W.matmul(torch.zeros(4, 288, dtype=torch.uint8, device="cuda")[:, 8:264].view(E4M3), s), "16-byte"),
    ]
    for call, says in cases:
        with pytest.raises(CmolError) as e:
            call()
        assert says in str(e.value), str(e.value)
    assert W.matmul(q[:0], s[:0]).shape == (0, 64)
    W.free()
    with pytest.raises(CmolError, match="NULL"):
        W.matmul(q, s)


# ---------------------------------------------------------------------------
# A run of them together
# ---------------------------------------------------------------------------
def _layer(g, d, ff):
    from libcmol_b200 import fp8
    w = {"gu": _weight(g, 2 * ff, d), "down": _weight(g, d, ff), "norm": 1 + 0.1 * _randn(g, d)}
    return w, fp8.Fp8Weight.quantize(w["gu"]), fp8.Fp8Weight.quantize(w["down"])


def _ffn(x, h, norm, gu, down, ff, dtype):
    from libcmol_b200 import fp8
    q, s = fp8.rmsnorm(x, norm, 1e-5, residual=h)
    a = gu.matmul(q, s, dtype=dtype)
    q, s = fp8.swiglu(a[:, :ff], a[:, ff:])
    return down.matmul(q, s, dtype=dtype)


@pytest.mark.parametrize("n, d, ff", [(1, 576, 1536), (1, 960, 2560), (7, 576, 1536), (64, 960, 2560), (333, 2048, 2560)])
@pytest.mark.parametrize("t", [F32, BF16])
def test_feed_forward_layer(n, d, ff, t):
    """norm -> gate|up -> SwiGLU -> down, each step against the 64-bit step on
    the same 8-bit inputs (what the step before left)."""
    from libcmol_b200 import fp8
    g = _gen(n)
    w, gu, down = _layer(g, d, ff)
    x, h = _randn(g, n, d, dtype=t), _randn(g, n, d)
    h0 = h.clone()
    y = _ffn(x, h, w["norm"], gu, down, ff, t)
    _, v = _norm_ref(x, h0, w["norm"], 1e-5)
    q, s = fp8.rmsnorm(x, w["norm"], 1e-5, residual=h0)
    assert torch.equal(h, h0)
    _check_eight_bits(v, q, s, _norm_delta(d))
    a = gu.matmul(q, s, dtype=t)
    _mm_check(a, q, s, *gu.read())
    q, s = fp8.swiglu(a[:, :ff], a[:, ff:])
    ad = a.double()
    _check_eight_bits(ad[:, :ff] / (1 + torch.exp(-ad[:, :ff])) * ad[:, ff:], q, s, 150 * U)
    _mm_check(y, q, s, *down.read())


def test_captured_and_replayed():
    """The layer in a CUDA graph, replayed on new inputs, and two graphs of one weight on two streams."""
    g = _gen(1)
    w, gu, down = _layer(g, 960, 2560)
    graphs = []
    for n in (1, 48):
        x, h = _randn(g, n, 960, dtype=BF16), _randn(g, n, 960)
        y0 = _ffn(x, h.clone(), w["norm"], gu, down, 2560, BF16)       # first use outside the capture
        graph, hs = torch.cuda.CUDAGraph(), h.clone()
        st = torch.cuda.Stream()
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            with torch.cuda.graph(graph, stream=st):
                y = _ffn(x, hs, w["norm"], gu, down, 2560, BF16)
        hs.copy_(h)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, y0)
        graphs.append((graph, x, hs, y, st))
    want = []
    for graph, x, hs, y, st in graphs:
        x.copy_(_randn(g, *x.shape, dtype=BF16))
        hs.copy_(_randn(g, *hs.shape))
        want.append(_ffn(x, hs.clone(), w["norm"], gu, down, 2560, BF16))
    start = [hs.clone() for _, _, hs, _, _ in graphs]
    torch.cuda.synchronize()
    for _ in range(20):
        for (graph, x, hs, y, st), h0 in zip(graphs, start):
            with torch.cuda.stream(st):
                hs.copy_(h0)
                graph.replay()
    torch.cuda.synchronize()
    for (graph, x, hs, y, st), ref in zip(graphs, want):
        assert torch.equal(y, ref)


def test_two_streams_share_a_weight():
    g = _gen(4)
    _, gu, _ = _layer(g, 960, 2560)
    from libcmol_b200 import fp8
    ins = [_acts(g, n, 960) for n in (1, 33, 300, 1200)]
    want = [gu.matmul(q, s) for q, s in ins]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in ins]
    ys = [torch.empty_like(y) for y in want]
    torch.cuda.synchronize()
    for _ in range(10):
        for (q, s), y, st in zip(ins, ys, streams):
            with torch.cuda.stream(st):
                gu.matmul(q, s, y=y)
    torch.cuda.synchronize()
    for y, ref in zip(ys, want):
        assert torch.equal(y, ref)


def test_current_device_is_left_alone_and_no_fault():
    import ctypes as C
    from libcmol_b200 import lib
    assert torch.cuda.current_device() == 0
    code = C.c_uint(0)
    assert lib().cmolcu_fault_status(0, C.byref(code), 0) == 0 and code.value == 0


# ---------------------------------------------------------------------------
# Calls that the documentation allows and an ordinary program seldom makes
# ---------------------------------------------------------------------------
def test_the_residual_may_be_the_input():
    """h = x + x, written back over x: short and long rows."""
    from libcmol_b200 import fp8
    for n, k in [(300, 960), (3, 20000)]:
        g = _gen(k)
        x, w = _randn(g, n, k), 1 + 0.1 * _randn(g, k)
        x0 = x.clone()
        q, s = fp8.rmsnorm(x, w, 1e-5, residual=x)
        h, v = _norm_ref(x0, x0, w, 1e-5)
        assert torch.equal(x.double(), h)
        _check_eight_bits(v, q, s, _norm_delta(k))


def test_rows_with_nan_among_many():
    """A NaN stays in its row where a CTA goes through several rows."""
    from libcmol_b200 import fp8
    g = _gen(9)
    n, k = 5000, 960
    x, w = _randn(g, n, k, dtype=BF16), 1 + 0.1 * _randn(g, k)
    bad = [0, 17, 2500, n - 1]
    x[bad, 3] = float("nan")
    q, s = fp8.rmsnorm(x, w, 1e-5)
    good = torch.ones(n, dtype=torch.bool, device="cuda")
    good[bad] = False
    assert torch.isnan(s[bad]).all()
    _check_eight_bits(_norm_ref(x[good], None, w, 1e-5)[1], q[good], s[good], _norm_delta(k))


def test_a_wrong_device_is_refused_and_leaves_no_error():
    from libcmol_b200 import last_error, lib
    x = torch.zeros(16, device="cuda")
    p = x.data_ptr()
    assert lib().cmolcu_fp8_rmsnorm(97, p, 0, 16, None, 0, None, 0, 0, None, 0.0, 1, 16, p, 16, p, 1, 1, None) == -1
    assert "cmolcu_fp8_rmsnorm" in last_error()
    assert (x + 1 == 1).all() and torch.cuda.current_device() == 0


def test_first_use_inside_a_capture():
    """Nothing has to run before a capture but the making of the weight."""
    import os
    import subprocess
    import sys
    code = """
import torch
from libcmol_b200 import fp8
W = [fp8.Fp8Weight.quantize(torch.randn(r, 1024, device="cuda")) for r in (256, 24000)]
x = [torch.randn(n, 1024, device="cuda") for n in (1, 12, 40, 600)]
w = torch.ones(1024, device="cuda")
def go():
    out = []
    for a in x:
        q, s = fp8.rmsnorm(a, w, 1e-5)
        q2, s2 = fp8.swiglu(a, a)
        out += [W[0].matmul(q, s), W[1].matmul(q, s, dtype=torch.bfloat16), W[0].matmul(q2, s2, dtype=torch.float16)]
    return out
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    got = go()
g.replay()
torch.cuda.synchronize()
want = go()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(got, want))
print("same")
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "same" in r.stdout, r.stdout + r.stderr


def test_threads_share_a_weight():
    import threading
    from libcmol_b200 import fp8
    g = _gen(12)
    W = fp8.Fp8Weight.quantize(_weight(g, 640, 512))
    ins = [_acts(g, n, 512) for n in (1, 14, 50, 700)]
    want = [W.matmul(q, s) for q, s in ins]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(30):
                y = W.matmul(*ins[i])
                torch.cuda.current_stream().synchronize()
                if not torch.equal(y, want[i]):
                    wrong.append(i)

    ts = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    [t.start() for t in ts]
    [t.join() for t in ts]
    assert not wrong


def test_offsets_past_32_bits():
    """Activations, outputs and a weight of more than 2^32 bytes: what lies at the
    end."""
    from libcmol_b200 import fp8
    g = _gen(13)
    n, k = 2_200_003, 1024                       # x: 4.5 GB, q: 2.25 GB
    x = torch.zeros(n, k, dtype=BF16, device="cuda")
    x[-300:] = _randn(g, 300, k, dtype=BF16)
    w = 1 + 0.1 * _randn(g, k)
    q, s = fp8.rmsnorm(x, w, 1e-5)
    q1, s1 = q[-300:].clone(), s[-300:].clone()
    _check_eight_bits(_norm_ref(x[-300:], None, w, 1e-5)[1], q1, s1, _norm_delta(k))
    assert (q[:1000].double() == 0).all()
    del x
    W = fp8.Fp8Weight.quantize(_weight(g, 600, k))
    y = W.matmul(q, s, dtype=F32)                # 5.3 GB
    assert (y[:1000] == 0).all()
    _mm_check(y[-300:], q1, s1, *W.read())
    del q, s, y
    torch.cuda.empty_cache()
    rows, k = 1_100_033, 4096                    # 4.5 GB
    wq = torch.zeros(rows, k, dtype=torch.uint8, device="cuda")
    tail = (100 * _randn(g, 161, k)).clamp(-448, 448).to(E4M3)
    wq[-161:] = tail.view(torch.uint8)           # the last two row blocks: 128 + 33
    ws = torch.ones(-(-rows // 128), k // 128, device="cuda")
    W = fp8.Fp8Weight(wq.view(E4M3), ws)
    del wq
    for n in (2, 40, 300):
        q, s = _acts(g, n, k)
        y = W.matmul(q, s)
        _mm_check(y[:, -161:], q, s, tail, torch.ones(2, k // 128, device="cuda"))
        assert (y[:, :1000] == 0).all()
        del y
    W.free()


@pytest.mark.parametrize("n", [1, 5, 12, 40, 130, 700])
@pytest.mark.parametrize("t", [F32, BF16])
def test_rows_behind_the_last_stay(n, t):
    """A batch smaller than its buffers: nothing behind row n is written."""
    from libcmol_b200 import fp8
    g = _gen(n)
    rows, k, extra = 384, 768, 130
    q = torch.full((n + extra, k), 0x2A, dtype=torch.uint8, device="cuda")
    s = torch.full((6, n + extra), 3.0, device="cuda").t()
    r = torch.full((n + extra, k), 7.0, dtype=t, device="cuda")
    r[:n] = _randn(g, n, k, dtype=t)
    x, w = _randn(g, n, k, dtype=t), torch.ones(k, device="cuda")
    W = fp8.Fp8Weight.quantize(_weight(g, rows, k))
    for call in (lambda a, b: fp8.rmsnorm(x, w, 1e-5, residual=r[:n], q=a, scales=b), lambda a, b: fp8.swiglu(x, x, q=a, scales=b),
                 lambda a, b: fp8.quantize(x, q=a, scales=b)):
        call(q[:n].view(E4M3), s[:n])
        assert (q[n:] == 0x2A).all() and (s[n:] == 3).all() and (r[n:] == 7).all()
    y = torch.full((n + extra, rows), 5.0, dtype=t, device="cuda")
    W.matmul(q[:n].view(E4M3), s[:n], y=y[:n])
    assert (y[n:] == 5).all()
    _mm_check(y[:n], q[:n].view(E4M3), s[:n], *W.read())


def test_no_rows():
    from libcmol_b200 import fp8
    x = torch.ones(3, 256, device="cuda")[:0]
    W = fp8.Fp8Weight.quantize(torch.ones(64, 256, device="cuda"))
    for q, s in (fp8.quantize(x), fp8.swiglu(x, x), fp8.rmsnorm(x, torch.ones(256, device="cuda"), residual=x)):
        assert q.shape == (0, 256) and s.shape == (0, 2) and W.matmul(q, s).shape == (0, 64)
