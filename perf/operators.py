"""The 8-bit floating point operators of a dense layer, as measured.

A decoder layer's dense work in 8 bits is a chain of three operators: the RMS
norm that adds the residual stream and leaves e4m3 values with a scale for
each 128 of them, the matrix product of such activations with weights that
hold a scale for each 128 x 128 block, and the SwiGLU between the feed-forward
layer's two products, which leaves the same 8-bit form.  Widths are those of
the decode engine's own models (hidden 576, 960 and 2048, feed-forward 1536,
2560, 8192 and 11008); token counts run from one decoded token over a batch of
sessions to long prompts.

`run` computes an operator's plain form from elementary torch operations, or,
with `own` set, calls the package's kernels.
"""
import math

import torch

own = False

BLOCK = 128
E4M3_MAX = 448.0
SCALE_MIN = 2.0 ** -126
EPS = 1e-5
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}


def listed():
    return [
        # one decoded token of the smallest single-session model: latency
        {"name": "norm 1x960", "op": "norm", "n": 1, "k": 960, "x": "f32", "res": "f32", "norm": True, "pad": 0},
        # one step of a full batch of sessions, f32 residual stream as the engine keeps it
        {"name": "norm 256x2048", "op": "norm", "n": 256, "k": 2048, "x": "f32", "res": "f32", "norm": True, "pad": 0},
        # a long prompt in one call, ragged count, rows of a wider buffer
        {"name": "norm 8191x2048", "op": "norm", "n": 8191, "k": 2048, "x": "bf16", "res": "bf16", "norm": True, "pad": 8},
        # activations that another kernel has formed: only the 8-bit form is made
        {"name": "quantise 4099x11008", "op": "norm", "n": 4099, "k": 11008, "x": "f16", "res": "", "norm": False, "pad": 0},
        # the feed-forward activation of one token, and of a long prompt
        {"name": "swiglu 1x2560", "op": "swiglu", "n": 1, "k": 2560, "x": "f32"},
        {"name": "swiglu 8192x11008", "op": "swiglu", "n": 8192, "k": 11008, "x": "bf16"},
        # one token: a small matrix (latency) and the largest of a layer (the weights' stream)
        {"name": "matmul 1x960x2560", "op": "matmul", "n": 1, "rows": 960, "k": 2560, "y": "f32"},
        {"name": "matmul 1x22016x2048", "op": "matmul", "n": 1, "rows": 22016, "k": 2048, "y": "f32"},
        # a small batch of sessions over a matrix with a long sum and few rows
        {"name": "matmul 37x2048x11008", "op": "matmul", "n": 37, "rows": 2048, "k": 11008, "y": "bf16"},
        # a full batch of sessions, gate and up of the feed-forward layer
        {"name": "matmul 256x22016x2048", "op": "matmul", "n": 256, "rows": 22016, "k": 2048, "y": "f16"},
        # a prompt chunk of odd length, odd rows, f32 out
        {"name": "matmul 777x2049x8192", "op": "matmul", "n": 777, "rows": 2049, "k": 8192, "y": "f32"},
        # a long prompt: bound by the tensor cores
        {"name": "matmul 8192x22016x2048", "op": "matmul", "n": 8192, "rows": 22016, "k": 2048, "y": "bf16"},
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, even over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm", "swiglu", "matmul", "matmul"])
    if op == "matmul":
        k = 16 * _log(rng, 4, 768)
        rows = _log(rng, 64, 32768)
        rows = min(rows, (22016 * 2048) // k)
        n = _log(rng, 1, 8192)
        n = max(1, min(n, (8192 * 22016 * 2048 // 2) // (rows * k), (8192 * 22016 // 2) // rows))
        return {"op": op, "n": n, "rows": rows, "k": k, "y": rng.choice(["f32", "f16", "bf16"])}
    k = 16 * _log(rng, 4, 768)
    n = max(1, min(_log(rng, 1, 16384), 4096 * 11008 // k))
    x = rng.choice(["f32", "f16", "bf16"])
    if op == "swiglu":
        return {"op": op, "n": n, "k": k, "x": x}
    norm = rng.random() < 0.8
    res = rng.choice([x, "f32", ""]) if norm else ""
    return {"op": op, "n": n, "k": k, "x": x, "res": res, "norm": norm, "pad": rng.choice([0, 0, 8])}


def _blocks(k):
    return (k + BLOCK - 1) // BLOCK


def _normal(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda")


def _rows(gen, n, k, dtype, pad):
    """Rows of activations: a normal value per entry, channels of different size, a few of them far larger."""
    size = torch.exp(0.5 * _normal(gen, k))
    size[torch.randint(0, k, (max(1, k // 256),), generator=gen, device="cuda")] *= 20.0
    full = torch.zeros(n, k + pad, dtype=dtype, device="cuda")
    full[:, :k] = _normal(gen, n, k).mul_(size)
    return full[:, :k]


def _eight_bits(v):
    """Rows of f32 values as e4m3 values and a scale for each 128 of a row."""
    n, k = v.shape
    b = torch.nn.functional.pad(v, (0, _blocks(k) * BLOCK - k)).view(n, _blocks(k), BLOCK)
    s = (b.abs().amax(-1) / E4M3_MAX).clamp_min(SCALE_MIN)
    q = (b / s.unsqueeze(-1)).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
    return q.view(n, -1)[:, :k].contiguous(), s


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op, n, k = case["op"], case["n"], case["k"]
    st = {"op": op, "n": n, "k": k}
    if op == "norm":
        st["x"] = _rows(gen, n, k, TYPES[case["x"]], case["pad"])
        st["g"] = 1.0 + 0.1 * _normal(gen, k) if case["norm"] else None
        st["r"] = st["r_out"] = None
        if case["res"]:
            st["r"] = _rows(gen, n, k, TYPES[case["res"]], 0) * 4
            st["r_out"] = torch.empty_like(st["r"])
    elif op == "swiglu":
        # gate and up as the product of their stacked weights leaves them: halves of one row
        both = _normal(gen, n, 2 * k).mul_(2.0).to(TYPES[case["x"]])
        st["gate"], st["up"] = both[:, :k], both[:, k:]
    else:
        rows = case["rows"]
        st["q"], st["s"] = _eight_bits(_rows(gen, n, k, torch.float32, 0))
        # weights of spread 0.02, in blocks of 128 x 128 with a scale each
        rb, kb = _blocks(rows), _blocks(k)
        w = torch.zeros(rb * BLOCK, kb * BLOCK, device="cuda")
        w[:rows, :k] = 0.02 * _normal(gen, rows, k)
        w = w.view(rb, BLOCK, kb, BLOCK)
        ws = (w.abs().amax((1, 3)) / E4M3_MAX).clamp_min(SCALE_MIN)
        wq = (w / ws[:, None, :, None]).to(torch.float8_e4m3fn).view(rb * BLOCK, kb * BLOCK)[:rows, :k].contiguous()
        st["wq"], st["ws"], st["out"] = wq, ws, TYPES[case["y"]]
        if own:     # a program lays its weights out once, when it loads them
            from libcmol_b200 import fp8
            st["w"] = fp8.Fp8Weight(wq, ws)
    if own:         # the buffers that a decode loop keeps
        if op == "matmul":
            st["y"] = torch.empty(n, case["rows"], dtype=st["out"], device="cuda")
        else:
            st["qo"] = torch.empty(n, k, dtype=torch.float8_e4m3fn, device="cuda")
            st["so"] = torch.empty(_blocks(k), n, device="cuda").t()
    return st


def run(st):
    if own:
        return _run_own(st)
    if st["op"] == "norm":
        h = st["x"].float()
        if st["r"] is not None:
            h = h + st["r"].float()
        v = h
        if st["g"] is not None:
            v = st["g"] * (h * torch.rsqrt((h * h).mean(-1, keepdim=True) + EPS))
        q, s = _eight_bits(v)
        return {"q": q, "scales": s, "residual": h.to(st["r"].dtype) if st["r"] is not None else None}
    if st["op"] == "swiglu":
        g = st["gate"].float()
        q, s = _eight_bits(g / (1.0 + torch.exp(-g)) * st["up"].float())
        return {"q": q, "scales": s}
    k, rows = st["k"], st["wq"].shape[0]
    x = st["q"].float() * st["s"].repeat_interleave(BLOCK, 1)[:, :k]
    w = st["wq"].float() * st["ws"].repeat_interleave(BLOCK, 0)[:rows].repeat_interleave(BLOCK, 1)[:, :k]
    return {"y": torch.matmul(x, w.t()).to(st["out"])}


def _run_own(st):
    from libcmol_b200 import fp8
    if st["op"] == "norm":
        q, s = fp8.rmsnorm(st["x"], st["g"], EPS, residual=st["r"], residual_out=st["r_out"], q=st["qo"], scales=st["so"])
        return {"q": q, "scales": s, "residual": st["r_out"]}
    if st["op"] == "swiglu":
        q, s = fp8.swiglu(st["gate"], st["up"], q=st["qo"], scales=st["so"])
        return {"q": q, "scales": s}
    return {"y": st["w"].matmul(st["q"], st["s"], y=st["y"])}


def work(case):
    n, k = case["n"], case["k"]
    eight = n * k + 4 * n * _blocks(k)      # e4m3 values and their scales
    if case["op"] == "norm":
        res = 2 * n * k * SIZE[case["res"]] if case["res"] else 0
        return {"bytes": n * k * SIZE[case["x"]] + res + eight + (4 * k if case["norm"] else 0), "flops": 8 * n * k}
    if case["op"] == "swiglu":
        return {"bytes": 2 * n * k * SIZE[case["x"]] + eight, "flops": 8 * n * k}
    rows = case["rows"]
    weights = rows * k + 4 * _blocks(rows) * _blocks(k)
    return {"bytes": weights + eight + n * rows * SIZE[case["y"]], "flops": 2 * n * rows * k}


def exact(case, seed):
    """The operators in 64 bits.  The e4m3 values are given before their rounding: v / s."""
    st = prepare(case, seed)
    n, k = st["n"], st["k"]
    if st["op"] == "matmul":
        y = torch.zeros(n, st["wq"].shape[0], dtype=torch.float64, device="cuda")
        row_block = torch.arange(st["wq"].shape[0], device="cuda") // BLOCK
        for b in range(_blocks(k)):
            cols = slice(b * BLOCK, min(k, (b + 1) * BLOCK))
            part = st["q"][:, cols].double() @ st["wq"][:, cols].double().t()
            y += part * st["s"][:, b].double()[:, None] * st["ws"][row_block, b].double()[None, :]
        return {"y": y}
    if st["op"] == "norm":
        h = st["x"].double() + (st["r"].double() if st["r"] is not None else 0.0)
        v = h
        if st["g"] is not None:
            v = h / torch.sqrt(torch.linalg.vector_norm(h, dim=-1, keepdim=True) ** 2 / k + EPS) * st["g"].double()
    else:
        g = st["gate"].double()
        v = g * torch.sigmoid(g) * st["up"].double()
    q, s = torch.empty_like(v), torch.empty(n, _blocks(k), dtype=torch.float64, device="cuda")
    for b in range(_blocks(k)):
        part = v[:, b * BLOCK:(b + 1) * BLOCK]
        s[:, b] = (part.abs().max(dim=-1).values / E4M3_MAX).clamp_min(SCALE_MIN)
        q[:, b * BLOCK:(b + 1) * BLOCK] = part / s[:, b, None]
    if st["op"] == "swiglu":
        return {"q": q, "scales": s}
    return {"q": q, "scales": s, "residual": h if st["r"] is not None else None}
