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
on 16-byte boundaries.
"""

from __future__ import annotations

import ctypes as C

import torch

from . import BF16, F16, F32, CmolError, _vp, check, lib

BLOCK = 128
_TAG = {torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16}
_E4M3 = torch.float8_e4m3fn


def _blocks(k: int) -> int:
    return (k + BLOCK - 1) // BLOCK


def _rows(t, what: str, dtypes, shape, device):
    """Checks a matrix of consecutive values on `device`; its row stride."""
    if t.dtype not in dtypes:
        raise CmolError(f"{what}: dtype {t.dtype}")
    if t.dim() != 2 or (shape is not None and tuple(t.shape) != shape):
        raise CmolError(f"{what}: shape {tuple(t.shape)}, wanted {shape or 'two dimensions'}")
    if t.device != device or device.type != "cuda":
        raise CmolError(f"{what}: on {t.device}, wanted a GPU and one device for all tensors")
    ld, inc = t.stride()
    if inc != 1 and t.shape[1] > 1:
        raise CmolError(f"{what}: the values of a row must be consecutive")
    return ld


def _scales(t, what: str, n: int, kb: int, device):
    if t.dtype != torch.float32 or tuple(t.shape) != (n, kb) or t.device != device:
        raise CmolError(f"{what}: scales are float32 {(n, kb)} on {device}, got {t.dtype} {tuple(t.shape)} on {t.device}")
    return t.stride()


def _out(q, scales, what: str, n: int, k: int, device):
    """The 8-bit output: checked, or new.  New scales keep a block's rows together."""
    if q is None:
        q = torch.empty((n, k), dtype=_E4M3, device=device)
    if scales is None:
        scales = torch.empty((_blocks(k), n), dtype=torch.float32, device=device).t()
    return q, _rows(q, what + ": q", (_E4M3,), (n, k), device), scales, _scales(scales, what, n, _blocks(k), device)


def _stream(device) -> int:
    return torch.cuda.current_stream(device).cuda_stream


def rmsnorm(x, norm_w, eps: float = 1e-5, residual=None, residual_out=None, q=None, scales=None):
    """RMS norm of x (+ residual) with an 8-bit output: (q, scales).

    h = x + residual; residual_out = h in the residual's type (the residual
    itself when not given); q, scales of norm_w * h / sqrt(mean(h^2) + eps), or
    of h itself when norm_w is None.  x and residual are [n, k] float32,
    float16 or bfloat16, norm_w is [k] float32."""
    what = "fp8.rmsnorm"
    dev = x.device
    x_ld = _rows(x, what + ": x", _TAG, None, dev)
    n, k = x.shape
    q, q_ld, scales, (s_ld, s_inc) = _out(q, scales, what, n, k, dev)
    r_ld = ro_ld = r_tag = 0
    r_ptr = ro_ptr = w_ptr = None
    if residual is not None:
        r_ld = _rows(residual, what + ": residual", _TAG, (n, k), dev)
        if residual_out is None:
            residual_out = residual
        ro_ld = _rows(residual_out, what + ": residual_out", (residual.dtype,), (n, k), dev)
        r_tag, r_ptr, ro_ptr = _TAG[residual.dtype], residual.data_ptr(), residual_out.data_ptr()
    elif residual_out is not None:
        raise CmolError(f"{what}: residual_out without residual")
    if norm_w is not None:
        if norm_w.dtype != torch.float32 or tuple(norm_w.shape) != (k,) or norm_w.device != dev or (
                k > 1 and norm_w.stride(0) != 1):
            raise CmolError(f"{what}: norm_w is {k} consecutive float32 values on {dev}")
        w_ptr = norm_w.data_ptr()
    if lib().cmolcu_fp8_rmsnorm(dev.index, x.data_ptr(), _TAG[x.dtype], x_ld, r_ptr, r_ld, ro_ptr, ro_ld, r_tag, w_ptr,
                                eps, n, k, q.data_ptr(), q_ld, scales.data_ptr(), s_ld, s_inc, _stream(dev)):
        check(-1, what)
    return q, scales


def quantize(x, q=None, scales=None):
    """The 8-bit form of activations as they are: (q, scales)."""
    return rmsnorm(x, None, 0.0, q=q, scales=scales)


def swiglu(gate, up, q=None, scales=None):
    """q, scales of gate / (1 + exp(-gate)) * up; gate and up [n, k] of one
    type, which may be halves of one tensor."""
    what = "fp8.swiglu"
    dev = gate.device
    g_ld = _rows(gate, what + ": gate", _TAG, None, dev)
    n, k = gate.shape
    u_ld = _rows(up, what + ": up", (gate.dtype,), (n, k), dev)
    q, q_ld, scales, (s_ld, s_inc) = _out(q, scales, what, n, k, dev)
    if lib().cmolcu_fp8_swiglu(dev.index, gate.data_ptr(), g_ld, up.data_ptr(), u_ld, _TAG[gate.dtype], n, k,
                               q.data_ptr(), q_ld, scales.data_ptr(), s_ld, s_inc, _stream(dev)):
        check(-1, what)
    return q, scales


class Fp8Weight:
    """A [rows x k] e4m3 weight with a scale for each 128 x 128, on one GPU.

    Fp8Weight(q, scales): q [rows, k] float8_e4m3fn and scales
    [ceil(rows/128), ceil(k/128)] float32, both on a GPU, or both on the host
    (then `device` says where the weight goes).
    Fp8Weight.quantize(w): from a float32, float16 or bfloat16 matrix on a
    GPU."""

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
            device = q.device.index
            ld = _rows(q, what + ": q", (_E4M3,), None, q.device)
            check(lib().cmolcu_fp8_weight_upload_dev(device, q.data_ptr(), k if rows == 1 else ld,
                                                     scales.data_ptr(), rows, k, _stream(q.device), C.byref(h)), what)
        else:
            q = q.contiguous()
            check(lib().cmolcu_fp8_weight_upload(device, q.data_ptr(), scales.data_ptr(), rows, k, C.byref(h)), what)
        self._set(h, rows, k, device)

    def _set(self, h, rows, k, device):
        self.h, self.rows, self.k = h, rows, k
        self.device = torch.device("cuda", device)

    @classmethod
    def quantize(cls, w):
        """A weight from a float32, float16 or bfloat16 [rows, k] matrix on a GPU."""
        what = "Fp8Weight.quantize"
        ld = _rows(w, what, _TAG, None, w.device)
        h = _vp()
        rows, k = w.shape
        check(lib().cmolcu_fp8_weight_quantize_dev(w.device.index, w.data_ptr(), _TAG[w.dtype],
                                                   k if rows == 1 else ld, rows, k, _stream(w.device),
                                                   C.byref(h)), what)
        self = cls.__new__(cls)
        self._set(h, rows, k, w.device.index)
        return self

    @property
    def nbytes(self) -> int:
        return lib().cmolcu_fp8_weight_bytes(self.h)

    def read(self):
        """The weight as it is held: (q [rows, k], scales) on its GPU."""
        q = torch.empty((self.rows, self.k), dtype=_E4M3, device=self.device)
        s = torch.empty((_blocks(self.rows), _blocks(self.k)), dtype=torch.float32, device=self.device)
        check(lib().cmolcu_fp8_weight_read_dev(self.h, q.data_ptr(), self.k, s.data_ptr(), _stream(self.device)),
              "Fp8Weight.read")
        return q, s

    def matmul(self, q, scales, y=None, dtype=torch.float32):
        """y [n, rows] = (q * scales) . W^T in float32, float16 or bfloat16
        (`y`'s type, else `dtype`)."""
        what = "Fp8Weight.matmul"
        dev = self.device
        q_ld = _rows(q, what + ": q", (_E4M3,), (q.shape[0], self.k), dev)
        n = q.shape[0]
        s_ld, s_inc = _scales(scales, what, n, _blocks(self.k), dev)
        if y is None:
            y = torch.empty((n, self.rows), dtype=dtype, device=dev)
        y_ld = _rows(y, what + ": y", _TAG, (n, self.rows), dev)
        if lib().cmolcu_fp8_matmul(self.h, q.data_ptr(), q_ld, scales.data_ptr(), s_ld, s_inc, n, y.data_ptr(),
                                   _TAG[y.dtype], y_ld, _stream(dev)):
            check(-1, what)
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
