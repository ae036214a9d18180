"""Every form of the 8-bit product (cmolcu_fp8_matmul_as) over the range it may be
given, whichever the library's own choice would be.

Bounds as for the product itself: a block's 128 products are exact in f32 and their sum
is off by at most 128 * 2^-23 of the sum of magnitudes (each addition may truncate); scaling
and adding the blocks cost (3 + blocks) * 2^-23 more, where a cluster's partial sums add 8
to the blocks' number; the output half a step of its type."""
import ctypes as C

import pytest

torch = pytest.importorskip("torch")

F32, F16, BF16, E4M3 = torch.float32, torch.float16, torch.bfloat16, torch.float8_e4m3fn
STEP = {F32: 0.0, F16: 2.0 ** -11, BF16: 2.0 ** -8}
FORMS = [8, 16, 32, 64, 128, 256]

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _device(gpu):
    from libcmol_b200 import fp8
    yield
    torch.cuda.synchronize()
    assert fp8.fault() == 0


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _acts(g, n, k):
    q = (200 * torch.randn(n, k, generator=g, device="cuda")).clamp(-448, 448).to(E4M3)
    return q, torch.exp(torch.randn(-(-k // 128), n, generator=g, device="cuda")).t()


def _weight(g, rows, k):
    """A weight of any e4m3 values and any scales: (handle, values in 64 bits)."""
    from libcmol_b200 import fp8
    wq = (150 * torch.randn(rows, k, generator=g, device="cuda")).clamp(-448, 448).to(E4M3)
    ws = 1e-4 * torch.exp(torch.randn(-(-rows // 128), -(-k // 128), generator=g, device="cuda"))
    w = wq.double() * ws.double().repeat_interleave(128, 0)[:rows].repeat_interleave(128, 1)[:, :k]
    return fp8.Fp8Weight(wq, ws), w


def _run(form, W, q, s, y):
    from libcmol_b200 import BF16 as TB, F16 as T6, F32 as T3, check, lib
    tag = {F32: T3, F16: T6, BF16: TB}[y.dtype]
    check(lib().cmolcu_fp8_matmul_as(form, W.h, q.data_ptr(), q.stride(0), s.data_ptr(), s.stride(0), s.stride(1),
                                     q.shape[0], y.data_ptr(), tag, y.stride(0),
                                     torch.cuda.current_stream().cuda_stream), "form %d" % form)
    return y


def _check(y, q, s, w):
    n, k = q.shape
    x = q.double() * s.double().repeat_interleave(128, 1)[:, :k]
    want, mag = x @ w.t(), x.abs() @ w.abs().t()
    bound = (128 + 3 + 8 - -k // 128) * 2.0 ** -23 * mag + STEP[y.dtype] * want.abs()
    if y.dtype == F16:
        bound += 2.0 ** -25
    err = (y.double() - want).abs()
    assert torch.isfinite(y).all() and (err <= bound).all(), (err / bound).max().item()


# (n, rows, k).  Odd and even numbers of 128-blocks along k, of row blocks, ragged last ones; rank 1's
# half past the weight; one tile and several a pair of CTAs, several rows of tiles; single blocks.
WIDE = [(1, 16, 16), (5, 130, 128), (17, 257, 144), (100, 128, 384), (255, 384, 400), (256, 512, 1024), (257, 640, 1296),
        (300, 300, 2064), (513, 900, 96), (700, 7001, 400), (1300, 5000, 272), (2050, 3001, 640), (600, 20000, 144)]
# the cluster forms: k whole, in two to eight parts, parts of unequal length; activation tiles ragged
TALL = [(1, 16, 16), (3, 200, 1296), (9, 128, 4112), (16, 1000, 960), (17, 2050, 2064), (31, 130, 2576), (40, 17000, 272),
        (15, 24000, 144), (33, 8000, 528), (64, 515, 1168), (65, 300, 11008), (100, 9000, 400), (200, 129, 640), (130, 2560, 1536)]
FEW = [(1, 16, 16), (2, 129, 144), (3, 1000, 2576), (8, 333, 400), (9, 16, 4112), (11, 5000, 272), (16, 30000, 144), (16, 130, 17616)]
CASES = [(f, *c) for f in FORMS for c in (FEW if f == 8 else TALL if f <= 64 else WIDE)]


@pytest.mark.parametrize("form, n, rows, k", CASES, ids=["%d-%dx%dx%d" % c for c in CASES])
def test_each_form(form, n, rows, k):
    """All types, rows of y on 16-byte boundaries and off them; the same bits again."""
    g = _gen(form + n + rows + k)
    q, s = _acts(g, n, k)
    W, w = _weight(g, rows, k)
    for t in (F32, F16, BF16):
        f = 1e-4 if t == F16 else 1.0           # keeps |y| inside f16
        for pad in (-rows % 16, -rows % 16 + 16, -rows % 16 + 3):
            buf = torch.full((n + 2, rows + pad), 7.0, dtype=t, device="cuda")
            y = _run(form, W, q, s * f, buf[:n, :rows])
            _check(y, q, s * f, w)
            assert (buf[n:] == 7).all() and (buf[:n, rows:] == 7).all()
        again = _run(form, W, q, s * f, torch.empty(n, rows, dtype=t, device="cuda"))
        assert torch.equal(again, y)


@pytest.mark.parametrize("form", FORMS)
def test_strides_of_each_form(form):
    """Rows of a wider buffer whose other bytes are NaN, scales in both orders, y at an odd address."""
    n, rows, k = (16 if form == 8 else 300), 700, 656
    g = _gen(form)
    q0, s0 = _acts(g, n, k)
    W, w = _weight(g, rows, k)
    buf = torch.full((n + 2, k + 48), 0x7F, dtype=torch.uint8, device="cuda")
    q = buf[1:n + 1, 16:16 + k].view(E4M3)
    q.view(torch.uint8).copy_(q0.view(torch.uint8))
    spread = torch.full((n, 13), float("nan"), device="cuda")
    for s in (s0.contiguous(), spread[:, 1:12:2]):
        s.copy_(s0)
        for t in (F32, BF16):
            ybuf = torch.full((n, rows + 9), 5.0, dtype=t, device="cuda")
            y = _run(form, W, q, s, ybuf[:, 1:1 + rows])
            _check(y, q0, s0, w)
            assert (ybuf[:, 0] == 5).all() and (ybuf[:, 1 + rows:] == 5).all()


@pytest.mark.parametrize("form", FORMS)
def test_nan_rows_of_each_form_stay_by_themselves(form):
    n, rows, k = (16 if form == 8 else 400), 515, 640
    g = _gen(form)
    q, s = _acts(g, n, k)
    W, w = _weight(g, rows, k)
    bad = [0, n // 2, n - 1]
    s[bad[1], 4], s[bad[2], 0] = float("nan"), float("inf")
    q.view(torch.uint8)[0, 639] = 0x7F
    y = _run(form, W, q, s, torch.empty(n, rows, device="cuda"))
    good = [i for i in range(n) if i not in bad]
    assert not torch.isfinite(y[bad]).any()
    _check(y[good], q[good], s[good], w)


@pytest.mark.parametrize("form", FORMS[1:])
def test_forms_in_turn_in_a_graph(form):
    """A form behind every other one, without a pause, captured and replayed."""
    n, rows, k = 12, 1100, 1168
    g = _gen(form)
    q, s = _acts(g, n, k)
    W, _ = _weight(g, rows, k)
    order = [f for other in FORMS for f in (form, other)]
    want = {f: _run(f, W, q, s, torch.empty(n, rows, device="cuda")) for f in FORMS}
    ys = [torch.zeros(n, rows, device="cuda") for _ in order]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for f, y in zip(order, ys):
            _run(f, W, q, s, y)
    for _ in range(20):
        graph.replay()
    torch.cuda.synchronize()
    for f, y in zip(order, ys):
        assert torch.equal(y, want[f])


def test_the_choice_is_one_of_the_forms():
    """Over the sizes a program has, every form is chosen somewhere, and the plain call is that form."""
    from libcmol_b200 import lib
    g = _gen(0)
    chosen = set()
    for rows, k in [(576, 576), (2048, 2048), (960, 2560), (22016, 2048), (2048, 11008), (49152, 960)]:
        W, _ = _weight(g, rows, k)
        assert lib().cmolcu_fp8_matmul_form(W.h, 0) == 0
        for n in (1, 8, 9, 16, 24, 33, 64, 100, 256, 600, 1500):
            f = lib().cmolcu_fp8_matmul_form(W.h, n)
            assert f in FORMS and (f != 8 or n <= 16)
            if f not in chosen:
                q, s = _acts(g, n, k)
                assert torch.equal(W.matmul(q, s), _run(f, W, q, s, torch.empty(n, rows, device="cuda")))
            chosen.add(f)
    assert chosen >= {8, 32, 128, 256}, chosen


def test_the_choice_follows_the_measurements():
    """Sizes at which one form is measured far ahead of the others, on the GPU that the estimates were fitted on."""
    from libcmol_b200 import fp8, lib
    if torch.cuda.get_device_properties(0).multi_processor_count != 148:
        pytest.skip("the estimates are for 148 SMs")
    for n, rows, k, form in [(1, 960, 2560, 8), (4, 2048, 2048, 8), (16, 1536, 576, 8), (8, 32768, 512, 16),
                             (16, 8192, 2048, 16), (64, 5760, 960, 16), (192, 960, 2560, 32), (96, 2048, 8192, 32),
                             (64, 22016, 2048, 64), (256, 22016, 2048, 128), (777, 2049, 8192, 128),
                             (1024, 22016, 2048, 256), (8192, 22016, 2048, 256), (2048, 2048, 11008, 256)]:
        W = fp8.Fp8Weight.quantize(torch.ones(rows, k, device="cuda"))
        assert lib().cmolcu_fp8_matmul_form(W.h, n) == form, (n, rows, k)
        W.free()
