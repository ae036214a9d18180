"""8-bit floating point operators on torch tensors (cmolcu_fp8_* of cmolcu.h).

An activation in 8 bits is a pair: ``q`` [n, k] float8_e4m3fn and ``scales``
[n, ceil(k/128)] float32, its values q * scale with one scale for each 128 of
a row.  A weight (`Fp8Weight`) has one scale for each 128 x 128.  A feed-forward
layer, for instance::

    q, s = fp8.rmsnorm(x, gains, eps, residual=h)           # h += x
    gu = gate_up.matmul(q, s, dtype=torch.bfloat16)        # [n, 2 ff]
    q, s = fp8.swiglu(gu[:, :ff], gu[:, ff:])
    x = down.matmul(q, s, dtype=torch.bfloat16)

Every call launches on torch's current stream of the tensors' device and can
be captured in a CUDA graph (making a weight cannot).  Results go to the
tensors given, or to new ones.  k is a multiple of 16; the rows of a `q` start
on 16-byte boundaries.  Waits inside the products are bounded: `fault` tells whether
one ran out.

The operators are for inference: they have no backward pass, and activations that
require a gradient are refused while gradients are recorded.  Gains and weights may be
parameters and count as constants.
"""

from __future__ import annotations

import ctypes as C

import torch

from . import BF16, F16, F32, CmolError, _vp, check, lib

BLOCK = 128
_TAG = {torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16}
_E4M3 = torch.float8_e4m3fn
_Q = (_E4M3,)


def _blocks(k: int) -> int:
    return (k + BLOCK - 1) // BLOCK


def _refuse(t, what: str, dtypes, shape, index: int):
    """Says what is wrong with a tensor that is not as it should be."""
    if t.dtype not in dtypes:
        raise CmolError(f"{what}: dtype {t.dtype}")
    if tuple(t.shape) != shape:
        raise CmolError(f"{what}: shape {tuple(t.shape)}, wanted {shape}")
    if t.get_device() != index:
        raise CmolError(f"{what}: on {t.device}, wanted cuda:{index}, as the other tensors")
    raise CmolError(f"{what}: the values of a row must be consecutive")


def _rows(t, what: str, dtypes, shape, index: int) -> int:
    """Checks a matrix of consecutive values on GPU `index`; its row stride."""
    if t.shape == shape and t.dtype in dtypes and t.get_device() == index:
        ld, inc = t.stride()
        if inc == 1 or shape[1] == 1:
            return ld
    _refuse(t, what, dtypes, shape, index)


def _first(t, what: str, dtypes):
    """As _rows for the tensor that says where and how large: (index, shape, row stride)."""
    if t.dtype not in dtypes:
        raise CmolError(f"{what}: dtype {t.dtype}")
    if t.dim() != 2:
        raise CmolError(f"{what}: shape {tuple(t.shape)}, wanted two dimensions")
    index = t.get_device()
    if index < 0:
        raise CmolError(f"{what}: on {t.device}, wanted a GPU")
    shape = tuple(t.shape)
    return index, shape, _rows(t, what, dtypes, shape, index)


def _no_grad(what: str, **tensors):
    """Refuses activations that autograd follows: their results would be cut off without a word."""
    for name, t in tensors.items():
        if t is not None and t.requires_grad and torch.is_grad_enabled():
            raise CmolError(f"{what}: {name} requires a gradient and there is none here: call it under torch.no_grad()")


def _scales(t, what: str, shape, index: int):
    if t.shape != shape or t.dtype is not torch.float32 or t.get_device() != index:
        raise CmolError(f"{what}: scales are float32 {shape} on cuda:{index}, got {t.dtype} {tuple(t.shape)} on "
                        f"{t.device}")
    return t.stride()


def _out(q, scales, what: str, shape, index: int):
    """The 8-bit output: checked, or new.  New scales keep a block's rows together."""
    n, k = shape
    kb = (k + 127) >> 7
    if q is None:
        q = torch.empty(shape, dtype=_E4M3, device=index)
    if scales is None:
        scales = torch.empty((kb, n), dtype=torch.float32, device=index).t()
    s_ld, s_inc = _scales(scales, what, (n, kb), index)
    return q, _rows(q, what, _Q, shape, index), scales, s_ld, s_inc


def _stream(index: int) -> int:
    return torch.cuda.current_stream(index).cuda_stream


# The same without building a stream object (2 us a call), where torch offers it.
_stream = getattr(torch._C, "_cuda_getCurrentRawStream", _stream)
# Counts tensors as modified, so that a backward pass which saved one does not take it for
# what it was (the public form checks its argument first, 0.2 us a call).
_modified = getattr(torch._C, "_increment_version", torch.autograd.graph.increment_version)


def rmsnorm(x, norm_w, eps: float = 1e-5, residual=None, residual_out=None, q=None, scales=None):
    """RMS norm of x (+ residual) with an 8-bit output: (q, scales).

    h = x + residual; residual_out = h in the residual's type (the residual
    itself when not given); q, scales of norm_w * h / sqrt(mean(h^2) + eps), or
    of h itself when norm_w is None.  x and residual are [n, k] float32,
    float16 or bfloat16, norm_w is [k] float32."""
    if x.requires_grad or (residual is not None and residual.requires_grad) or (
            residual_out is not None and residual_out.requires_grad) or (scales is not None and scales.requires_grad):
        _no_grad("fp8.rmsnorm", x=x, residual=residual, residual_out=residual_out, scales=scales)
    index, shape, x_ld = _first(x, "fp8.rmsnorm: x", _TAG)
    n, k = shape
    q, q_ld, scales, s_ld, s_inc = _out(q, scales, "fp8.rmsnorm: q", shape, index)
    r_ld = ro_ld = r_tag = 0
    r_ptr = ro_ptr = w_ptr = None
    if residual is not None:
        r_ld = ro_ld = _rows(residual, "fp8.rmsnorm: residual", _TAG, shape, index)
        r_tag = _TAG[residual.dtype]
        r_ptr = ro_ptr = residual.data_ptr()
        if residual_out is not None and residual_out is not residual:
            ro_ld = _rows(residual_out, "fp8.rmsnorm: residual_out", (residual.dtype,), shape, index)
            ro_ptr = residual_out.data_ptr()
    elif residual_out is not None:
        raise CmolError("fp8.rmsnorm: residual_out without residual")
    if norm_w is not None:
        if norm_w.dtype is not torch.float32 or norm_w.shape != (k,) or norm_w.get_device() != index or (
                k > 1 and norm_w.stride(0) != 1):
            raise CmolError(f"fp8.rmsnorm: norm_w is {k} consecutive float32 values on cuda:{index}")
        w_ptr = norm_w.data_ptr()
    if lib().cmolcu_fp8_rmsnorm(index, x.data_ptr(), _TAG[x.dtype], x_ld, r_ptr, r_ld, ro_ptr, ro_ld, r_tag, w_ptr,
                                eps, n, k, q.data_ptr(), q_ld, scales.data_ptr(), s_ld, s_inc, _stream(index)):
        check(-1, "fp8.rmsnorm")
    _modified([scales] if residual is None else [scales, residual if residual_out is None else residual_out])
    return q, scales


def fault(device: int = 0, clear: bool = False) -> int:
    """The fault word of this module's products on a GPU: 0, or the code of a
    bounded wait inside a kernel that ran out (cmolcu_fault_status); the products
    since the last look are then invalid.  It counts what has finished: synchronize
    first.  `clear` resets it."""
    code = C.c_uint(0)
    check(lib().cmolcu_fault_status(device, C.byref(code), int(clear)), "fp8.fault")
    return code.value


def quantize(x, q=None, scales=None):
    """The 8-bit form of activations as they are: (q, scales)."""
    return rmsnorm(x, None, 0.0, q=q, scales=scales)


def swiglu(gate, up, q=None, scales=None):
    """q, scales of gate / (1 + exp(-gate)) * up; gate and up [n, k] of one
    type, which may be halves of one tensor."""
    if gate.requires_grad or up.requires_grad or (scales is not None and scales.requires_grad):
        _no_grad("fp8.swiglu", gate=gate, up=up, scales=scales)
    index, shape, g_ld = _first(gate, "fp8.swiglu: gate", _TAG)
    u_ld = _rows(up, "fp8.swiglu: up", (gate.dtype,), shape, index)
    q, q_ld, scales, s_ld, s_inc = _out(q, scales, "fp8.swiglu: q", shape, index)
    n, k = shape
    if lib().cmolcu_fp8_swiglu(index, gate.data_ptr(), g_ld, up.data_ptr(), u_ld, _TAG[gate.dtype], n, k,
                               q.data_ptr(), q_ld, scales.data_ptr(), s_ld, s_inc, _stream(index)):
        check(-1, "fp8.swiglu")
    _modified([scales])
    return q, scales


class Fp8Weight:
    """A [rows x k] e4m3 weight with a scale for each 128 x 128, on one GPU.

    Fp8Weight(q, scales): q [rows, k] float8_e4m3fn and scales
    [ceil(rows/128), ceil(k/128)] float32, both on a GPU, or both on the host
    (then `device` says where the weight goes).
    Fp8Weight.quantize(w): from a float32, float16 or bfloat16 matrix on a
    GPU.

    The memory goes with the last reference (or with `free`), which may be while a
    stream is captured.  A CUDA graph with a captured product does not keep the
    weight: hold on to it as long as the graph is replayed."""

    def __init__(self, q, scales, device: int = 0):
        what = "Fp8Weight"
        h = _vp()
        self.h = None
        if q.dtype != _E4M3 or q.dim() != 2:
            raise CmolError(f"{what}: q is a float8_e4m3fn matrix, got {q.dtype} of {q.dim()} dimensions")
        rows, k = q.shape
        want = (_blocks(rows), _blocks(k))
        if scales.dtype != torch.float32 or tuple(scales.shape) != want or scales.device != q.device:
            raise CmolError(f"{what}: scales are float32 {want} beside q, got {scales.dtype} {tuple(scales.shape)} "
                            f"on {scales.device}")
        scales = scales.contiguous()
        if q.device.type == "cuda":
            device, _, ld = _first(q, what + ": q", _Q)
            check(lib().cmolcu_fp8_weight_upload_dev(device, q.data_ptr(), k if rows == 1 else ld,
                                                     scales.data_ptr(), rows, k, _stream(device), C.byref(h)), what)
        else:
            q = q.contiguous()
            check(lib().cmolcu_fp8_weight_upload(device, q.data_ptr(), scales.data_ptr(), rows, k, C.byref(h)), what)
        self._set(h, rows, k, device)

    def _set(self, h, rows, k, device):
        self.h, self.rows, self.k, self.index = h, rows, k, device
        self.device = torch.device("cuda", device)

    @classmethod
    def quantize(cls, w):
        """A weight from a float32, float16 or bfloat16 [rows, k] matrix on a GPU."""
        what = "Fp8Weight.quantize"
        index, (rows, k), ld = _first(w, what, _TAG)
        h = _vp()
        check(lib().cmolcu_fp8_weight_quantize_dev(index, w.data_ptr(), _TAG[w.dtype], k if rows == 1 else ld, rows, k,
                                                   _stream(index), C.byref(h)), what)
        self = cls.__new__(cls)
        self._set(h, rows, k, index)
        return self

    # One owner of the memory: a weight does not change, so a copy is the weight itself.
    def __copy__(self):
        return self

    def __deepcopy__(self, memo):
        return self

    def __reduce__(self):
        raise CmolError("Fp8Weight: lies in a GPU's memory and cannot be pickled; read() gives its values")

    @property
    def nbytes(self) -> int:
        return lib().cmolcu_fp8_weight_bytes(self.h)

    def read(self):
        """The weight as it is held: (q [rows, k], scales) on its GPU."""
        q = torch.empty((self.rows, self.k), dtype=_E4M3, device=self.device)
        s = torch.empty((_blocks(self.rows), _blocks(self.k)), dtype=torch.float32, device=self.device)
        check(lib().cmolcu_fp8_weight_read_dev(self.h, q.data_ptr(), self.k, s.data_ptr(), _stream(self.index)),
              "Fp8Weight.read")
        return q, s

    def matmul(self, q, scales, y=None, dtype=torch.float32):
        """y [n, rows] = (q * scales) . W^T in float32, float16 or bfloat16
        (`y`'s type, else `dtype`)."""
        if scales.requires_grad or (y is not None and y.requires_grad):
            _no_grad("Fp8Weight.matmul", scales=scales, y=y)
        index = self.index
        n = q.shape[0]
        q_ld = _rows(q, "Fp8Weight.matmul: q", _Q, (n, self.k), index)
        s_ld, s_inc = _scales(scales, "Fp8Weight.matmul", (n, (self.k + 127) >> 7), index)
        if y is None:
            y = torch.empty((n, self.rows), dtype=dtype, device=index)
        y_ld = _rows(y, "Fp8Weight.matmul: y", _TAG, (n, self.rows), index)
        if lib().cmolcu_fp8_matmul(self.h, q.data_ptr(), q_ld, scales.data_ptr(), s_ld, s_inc, n, y.data_ptr(),
                                   _TAG[y.dtype], y_ld, _stream(index)):
            check(-1, "Fp8Weight.matmul")
        _modified([y])
        return y

    def free(self):
        if self.h:
            lib().cmolcu_fp8_weight_free(self.h)
            self.h = None

    def __del__(self):
        try:
            self.free()
        except Exception:
            pass
