"""Activation checkpoints in 8 bits, and the backward pass that reads them.

The module API's autograd keeps the encoder's input ``[B, d]``, the
pre-activations ``[B, F]`` and the decoder's input ``[B, F]`` for the backward
(as the reference's does); at F = 49152 the last two are all of its memory.
Here each is held at one byte per element:

* ``checkpoint8(x)`` -> ``Act8``: int8 codes with one power-of-two step per 32
  columns of a row. ``Act8.weight_grad(g)`` is the weight gradient straight
  from the codes, ``Act8.dequantize()`` the values.
* ``jumprelu8(pre, log_threshold, ste_bandwidth)``: the JumpReLU whose
  backward keeps a byte that says off, on, or where inside the STE band.

``B200JumpReLUSAE.checkpoint_bits = 8`` makes the module use them. The
reference has no counterpart (its autograd keeps the tensors).
"""
from __future__ import annotations

import ctypes
import functools
from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from . import _lib as L

GROUP = 32   # columns that share a step


_CODES = {torch.float32: L.DTYPE_F32, torch.bfloat16: L.DTYPE_BF16}
# current_stream() builds a Stream object, a third of a small call's time on the host.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)
_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device


def _cuda_float(name: str, t: torch.Tensor) -> None:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a tensor, got {type(t).__name__}")
    if not t.is_cuda:
        raise RuntimeError(f"{name} must be a CUDA tensor: sae_b200 computes on CUDA devices only")
    if t.dtype not in _CODES:
        raise TypeError(f"{name} must be float32 or bfloat16, got {t.dtype}")


def _launch(index: int, name: str, *args) -> None:
    """The library call with device ``index`` current, on its current stream (the last argument)."""
    if _current_device() == index:     # a CUDA tensor is at hand: CUDA is initialised
        L.call(name, *args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            L.call(name, *args, _raw_stream(index))


def _f32(v) -> float:
    """A number as the kernels hold it."""
    return ctypes.c_float(float(v)).value


def _rows(t: torch.Tensor) -> torch.Tensor:
    """t as rows of its last dimension, contiguous inside a row (the rows may be apart)."""
    if t.dim() != 2:
        t = t.detach().reshape(-1, t.shape[-1])
    if t.is_contiguous():
        return t
    rows, cols = t.shape
    if (cols > 1 and t.stride(1) != 1) or (rows > 1 and t.stride(0) < cols):
        t = t.detach().contiguous()
    return t


def _pitch(t: torch.Tensor) -> int:
    return t.stride(0) if t.shape[0] > 1 else max(t.shape[1], 1)


class Act8:
    """A ``[..., D]`` tensor held as int8 ``codes [T, pitch]`` and one step byte
    per 32 columns, ``steps [T, pitch / 32]`` (T: the leading dimensions
    together, pitch: D rounded up to 32). Made by ``checkpoint8``."""

    def __init__(self, codes: torch.Tensor, step_rows: torch.Tensor, shape, dtype: torch.dtype):
        self.codes, self.step_rows = codes, step_rows   # the latter in rows of 16 k bytes
        self.shape, self.dtype = torch.Size(shape), dtype
        self.device = codes.device

    @property
    def steps(self) -> torch.Tensor:
        return self.step_rows[:, :self.codes.shape[1] // GROUP]

    @property
    def n_cols(self) -> int:
        return self.shape[-1]

    @property
    def n_tokens(self) -> int:
        return self.codes.shape[0]

    @property
    def nbytes(self) -> int:
        return self.codes.numel() + self.step_rows.numel()

    def dequantize(self, dtype: Optional[torch.dtype] = None,
                   out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """The values, as ``dtype`` (default: the saved tensor's) or into ``out``
        (same shape, rows contiguous inside). Exact in bfloat16 and float32."""
        if out is None:
            dtype = dtype or self.dtype
            if dtype not in _CODES:
                raise TypeError(f"dtype must be float32 or bfloat16, got {dtype}")
            out = torch.empty(self.shape, device=self.device, dtype=dtype)
        elif dtype is not None and dtype != out.dtype:
            raise TypeError(f"out is {out.dtype}, not {dtype}")
        else:
            _cuda_float("out", out)
        if out.shape != self.shape or out.device != self.device:
            raise ValueError(f"out must have shape {tuple(self.shape)} on {self.device}")
        if out.numel() == 0:
            return out
        o = out.detach()
        o = o if o.dim() == 2 else o.view(-1, self.n_cols)
        if (o.shape[1] > 1 and o.stride(1) != 1) or (o.shape[0] > 1 and o.stride(0) < o.shape[1]):
            raise ValueError("out must be contiguous inside its rows, the rows not overlapping")
        _launch(o.get_device(), "sae_b200_act8_load", self.codes.data_ptr(),
                self.step_rows.data_ptr(), self.n_tokens, self.n_cols, o.data_ptr(),
                _CODES[o.dtype], _pitch(o))
        torch.autograd.graph.increment_version(out)   # for whoever saved the old values
        return out

    def weight_grad(self, g: torch.Tensor, *, transposed: bool = False,
                    out: Optional[torch.Tensor] = None, accumulate: bool = False) -> torch.Tensor:
        """``sum_t g[t, n] v[t, c]`` over the tokens, v the checkpoint's values:
        float32 ``[N, D]``, or ``[D, N]`` when ``transposed``. ``g``: ``[..., N]``
        float32 or bfloat16 with the checkpoint's leading dimensions. ``out`` is
        written, or added to when ``accumulate``. No gradient is recorded."""
        _cuda_float("g", g)
        if g.dim() != len(self.shape) or g.shape[:-1] != self.shape[:-1]:
            raise ValueError(f"g must have the checkpoint's leading dimensions "
                             f"{tuple(self.shape[:-1])}, got {tuple(g.shape)}")
        if g.device != self.device:
            raise ValueError(f"g is on {g.device}, the checkpoint on {self.device}")
        N = g.shape[-1]
        shape = (self.n_cols, N) if transposed else (N, self.n_cols)
        if out is None:
            if accumulate:
                raise ValueError("accumulate needs out")
            out = torch.empty(shape, device=self.device, dtype=torch.float32)
        elif (out.shape != shape or out.dtype != torch.float32 or out.device != self.device
              or (out.numel() and ((shape[1] > 1 and out.stride(1) != 1)
                                   or (shape[0] > 1 and out.stride(0) < shape[1])))):
            raise ValueError(f"out must be float32 {shape} on {self.device}, contiguous inside rows")
        if out.numel() == 0:
            return out
        if self.n_tokens == 0:
            return out if accumulate else out.zero_()
        g = _rows(g)
        need = ctypes.c_size_t(0)
        index, gcode, gpitch = g.get_device(), _CODES[g.dtype], _pitch(g)
        with torch.cuda.device(index):    # the plan depends on the device
            L.call("sae_b200_weight_grad8_workspace_bytes", self.n_tokens, self.n_cols,
                   g.data_ptr(), gcode, N, gpitch, ctypes.byref(need))
        ws = torch.empty(need.value, device=self.device, dtype=torch.uint8)
        _launch(index, "sae_b200_weight_grad8", self.codes.data_ptr(), self.step_rows.data_ptr(),
                self.n_tokens, self.n_cols, g.data_ptr(), gcode, N, gpitch, int(bool(transposed)),
                1.0 if accumulate else 0.0, out.data_ptr(), _pitch(out), ws.data_ptr(), need.value)
        torch.autograd.graph.increment_version(out)
        return out


def checkpoint8(x: torch.Tensor) -> Act8:
    """Hold ``x [..., D]`` (float32 or bfloat16) at 8 bits per element; see ``Act8``.
    An element is off by at most half its group's step; the step is at most
    max|x| / 63.75 of its 32 columns, or 2^-126. A group with an infinity or a NaN reads
    back as NaN."""
    _cuda_float("x", x)
    if x.dim() < 2 or x.shape[-1] == 0:
        raise ValueError("x must be [..., D] with at least two dimensions and D >= 1")
    rows = _rows(x)
    T, D = rows.shape
    pitch = (D + GROUP - 1) // GROUP * GROUP
    codes = torch.empty(T, pitch, device=x.device, dtype=torch.int8)
    steps = torch.empty(T, (pitch // GROUP + 15) // 16 * 16, device=x.device, dtype=torch.uint8)
    if T:
        _launch(x.get_device(), "sae_b200_act8_save", rows.data_ptr(), _CODES[rows.dtype], T, D,
                _pitch(rows), codes.data_ptr(), steps.data_ptr())
    return Act8(codes, steps, x.shape, x.dtype)


@functools.lru_cache(maxsize=1024)
def _jumprelu8_scratch(index: int, T: int, F: int) -> int:
    need = ctypes.c_size_t(0)
    with torch.cuda.device(index):
        L.call("sae_b200_jumprelu8_workspace_bytes", T, F, ctypes.byref(need))
    return need.value


class _JumpReLU8(torch.autograd.Function):
    """(feat, gate) of the JumpReLU, keeping a byte per element. ``sae``: the
    module whose ste_bandwidth must still be the forward's in the backward."""

    @staticmethod
    def forward(ctx, pre, log_threshold, eps, sae):
        ctx.set_materialize_grads(False)
        shape, dev, code = pre.shape, pre.device, _CODES[pre.dtype]
        F = shape[-1]
        rows = pre if pre.dim() == 2 and pre.is_contiguous() else pre.reshape(-1, F).contiguous()
        T = rows.shape[0]
        feat = torch.empty(shape, device=dev, dtype=torch.float32)
        gate = torch.empty(shape, device=dev, dtype=torch.float32)
        codes = torch.empty((T, (F + 15) // 16 * 16), device=dev, dtype=torch.int8)
        if T:
            _launch(pre.get_device(), "sae_b200_jumprelu8_forward", rows.data_ptr(), code,
                    log_threshold.data_ptr(), T, F, eps, feat.data_ptr(), gate.data_ptr(),
                    codes.data_ptr())
        ctx.save_for_backward(codes, log_threshold)
        ctx.held = eps, sae, shape, pre.dtype, T, F
        return feat, gate

    @staticmethod
    def _grads(ctx, grad_feat, grad_gate):
        codes, log_threshold = ctx.saved_tensors
        eps, sae, shape, dtype, T, F = ctx.held
        if sae is not None and _f32(sae.ste_bandwidth) != eps:
            raise RuntimeError(
                "ste_bandwidth changed between forward and backward: an 8-bit JumpReLU checkpoint "
                f"holds positions in the forward's band ({eps}, now {sae.ste_bandwidth})")
        dev = codes.device
        grad_pre = torch.empty(shape, device=dev, dtype=dtype) if ctx.needs_input_grad[0] else None
        grad_thr = torch.empty(F, device=dev, dtype=torch.float32)
        if T == 0:
            return grad_pre, grad_thr.zero_(), None, None
        gf = None if grad_feat is None else grad_feat.float().contiguous()
        # read by stride where it is used: the sparsity loss hands in one expanded number
        gg = None if grad_gate is None else grad_gate.float().reshape(T, F)
        st, sf = (0, 0) if gg is None else gg.stride()
        index = codes.get_device()
        need = _jumprelu8_scratch(index, T, F)
        ws = torch.empty(need, device=dev, dtype=torch.uint8)
        _launch(index, "sae_b200_jumprelu8_backward", codes.data_ptr(), log_threshold.data_ptr(),
                T, F, eps, L.ptr(gf), L.ptr(gg), st, sf, L.ptr(grad_pre), _CODES[dtype],
                grad_thr.data_ptr(), ws.data_ptr(), need)
        return grad_pre, grad_thr, None, None

    @staticmethod
    def backward(ctx, grad_feat, grad_gate):
        # The wrapper that refuses a second differentiation is needed, and paid for,
        # only where a graph of the gradients is asked for.
        if torch.is_grad_enabled():
            return once_differentiable(_JumpReLU8._grads)(ctx, grad_feat, grad_gate)
        return _JumpReLU8._grads(ctx, grad_feat, grad_gate)


def _jumprelu8(pre, log_threshold, eps, sae):
    _cuda_float("pre", pre)
    _cuda_float("log_threshold", log_threshold)
    if pre.dim() < 2 or pre.shape[-1] == 0:
        raise ValueError("pre must be [..., F] with at least two dimensions and F >= 1")
    if (log_threshold.dtype != torch.float32 or log_threshold.shape != pre.shape[-1:]
            or not log_threshold.is_contiguous() or log_threshold.device != pre.device):
        raise ValueError(f"log_threshold must be a contiguous float32 [{pre.shape[-1]}] on "
                         f"{pre.device}")
    eps = _f32(eps)
    if not 0.0 < eps < float("inf"):
        raise ValueError(f"ste_bandwidth must be positive and finite, got {eps}")
    return _JumpReLU8.apply(pre, log_threshold, eps, sae)


def jumprelu8(pre: torch.Tensor, log_threshold: torch.Tensor, ste_bandwidth: float):
    """``(feat, gate)`` = (pre where pre > exp(log_threshold) else 0, the gate as
    0 / 1), float32, with the straight-through threshold gradient; the backward
    reads one byte per element instead of ``pre``. In the band
    |pre - theta| < ste_bandwidth the byte is good to ste_bandwidth / 252; gate
    and band are exact."""
    return _jumprelu8(pre, log_threshold, ste_bandwidth, None)
