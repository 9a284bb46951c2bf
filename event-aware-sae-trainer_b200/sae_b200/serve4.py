"""Serving an SAE from 4-bit weights.

``quantize4(sae)`` -> ``B200SAE4``: encoder and decoder at 4 bits per weight
with a scale per 32, 64 or 128 columns of a row. At 1536 x 49152 that is 80 MB
instead of the 302 MB of bf16 copies ``reconstruct`` reads, which is what bounds a few
tokens next to a decoding language model. Same calls as the module's
inference side (``encode_pre``, ``encode``, ``decode``, ``reconstruct``); the
reference has no counterpart.
"""
from __future__ import annotations

import ctypes
from typing import Optional, Tuple

import torch

from . import _lib as L
from .act8 import _CODES, _cuda_float, _launch, _pitch, _rows

GROUPS = (32, 64, 128)
MAX_D_IN = 12288
_MAX_WEIGHT = 2.0 ** 60    # partial sums stay in float32's range
# Tokens per library call of reconstruct: its [tokens, F] float32 scratch stays
# at 200 MB for F = 49152.
_RECONSTRUCT_TOKENS = 1024
_CALL_TOKENS = 65535


def _check_shape(F: int, d: int, group: int) -> None:
    if group not in GROUPS:
        raise ValueError(f"group must be one of {GROUPS}, got {group}")
    if F <= 0 or d <= 0 or d % 2 or d > MAX_D_IN:
        raise ValueError(f"4-bit weights need F >= 1 and an even d_in of at most {MAX_D_IN}, "
                         f"got [{F}, {d}]")


def quantize4_rows(W: torch.Tensor, group: int = 64) -> Tuple[torch.Tensor, torch.Tensor]:
    """``W [F, d]`` float32 as 4-bit codes ``uint8 [F, d / 2]`` (byte i: the
    code of column 2 i in the low half, of column 2 i + 1 in the high one, each
    as q + 8) and ``bfloat16
    [F, ceil(d / group)]`` scales: max|w| / 7 rounded up to 5 significant bits."""
    _cuda_float("W", W)
    if W.dim() != 2 or W.dtype != torch.float32:
        raise TypeError("W must be a float32 [F, d] tensor")
    F, d = W.shape
    _check_shape(F, d, group)
    W = W.detach().contiguous()
    if not bool((W.abs() <= _MAX_WEIGHT).all()):
        raise ValueError("W must be finite, with |w| <= 2^60")
    codes = torch.empty(F, d // 2, device=W.device, dtype=torch.uint8)
    scales = torch.empty(F, -(-d // group), device=W.device, dtype=torch.bfloat16)
    _launch(W.get_device(), "sae_b200_sae4_quantize", L.ptr(W), F, d, group, L.ptr(codes),
            L.ptr(scales))
    return codes, scales


def _check_codes(name: str, codes: torch.Tensor, scales: torch.Tensor, F: int, d: int,
                 group: int) -> None:
    if codes.dtype != torch.uint8 or codes.shape != (F, d // 2):
        raise ValueError(f"{name} codes must be uint8 [{F}, {d // 2}]")
    if scales.dtype != torch.bfloat16 or scales.shape != (F, -(-d // group)):
        raise ValueError(f"{name} scales must be bfloat16 [{F}, {-(-d // group)}]")
    s = scales.float()
    ok = (s == 0) | ((s >= 2.0 ** -100) & (s <= _MAX_WEIGHT))
    if not bool((ok & ((scales.contiguous().view(torch.int16) & 7) == 0)).all()):
        raise ValueError(f"{name} scales must be 0 or within [2^-100, 2^60], with at most 5 "
                         "significant bits (the weights are then exact in bfloat16)")


class B200SAE4:
    """An SAE held for inference in 4 bits; made by ``quantize4`` or
    ``from_codes``. It keeps no state between calls and allocates its scratch
    per call, so it may be used from several streams and captured into graphs."""

    def __init__(self):
        raise TypeError("use quantize4(sae) or B200SAE4.from_codes(...)")

    @classmethod
    def from_codes(cls, enc_codes, enc_scales, b_enc, dec_codes, dec_scales, b_dec,
                   log_threshold, *, group: int = 64) -> "B200SAE4":
        """From row-major codes and scales of the encoder and of the
        feature-major decoder (``quantize4_rows``'s format), ``b_enc [F]``,
        ``b_dec [d]`` and ``log_threshold [F]``."""
        ts = (enc_codes, enc_scales, b_enc, dec_codes, dec_scales, b_dec, log_threshold)
        dev = enc_codes.device
        if any(not t.is_cuda or t.device != dev for t in ts):
            raise RuntimeError("B200SAE4 needs all its tensors on one CUDA device")
        if b_enc.dim() != 1 or b_dec.dim() != 1:
            raise ValueError("b_enc must be [F] and b_dec [d]")
        F, d = b_enc.shape[0], b_dec.shape[0]
        _check_shape(F, d, group)
        if log_threshold.shape != (F,):
            raise ValueError(f"log_threshold must be [{F}]")
        if bool(log_threshold.isnan().any()):
            raise ValueError("log_threshold holds a NaN")
        _check_codes("encoder", enc_codes, enc_scales, F, d, group)
        _check_codes("decoder", dec_codes, dec_scales, F, d, group)
        self = cls.__new__(cls)
        self.d_in, self.n_features, self.group, self.device = d, F, group, dev
        need = ctypes.c_size_t(0)
        L.call("sae_b200_sae4_packed_bytes", F, d, group, ctypes.byref(need))
        self._enc = torch.empty(need.value, device=dev, dtype=torch.uint8)
        ec, es = enc_codes.contiguous(), enc_scales.contiguous()
        _launch(ec.get_device(), "sae_b200_sae4_pack", L.ptr(ec), L.ptr(es), F, d, group,
                L.ptr(self._enc))
        pitch = (d // 2 + 15) // 16 * 16
        self._dec = torch.full((F, pitch), 0x88, device=dev, dtype=torch.uint8)
        self._dec[:, :d // 2] = dec_codes
        self._dec_scale = dec_scales.detach().contiguous().clone()
        self._b_enc = b_enc.detach().float().contiguous().clone()
        self._b_dec = b_dec.detach().float().contiguous().clone()
        self._theta = log_threshold.detach().float().exp().contiguous()
        self._index = ec.get_device()
        self._struct = L.Sae4(d, F, group, 0, L.ptr(self._enc), L.ptr(self._dec),
                              L.ptr(self._dec_scale), L.ptr(self._b_enc), L.ptr(self._b_dec),
                              L.ptr(self._theta))
        self._model = ctypes.byref(self._struct)
        self._scratch_bytes = {}   # by token count
        torch.cuda.current_stream(dev).synchronize()   # any stream may use it from here on
        return self

    @property
    def nbytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in (
            self._enc, self._dec, self._dec_scale, self._b_enc, self._b_dec, self._theta))

    def _input(self, name: str, x: torch.Tensor, width: int) -> torch.Tensor:
        _cuda_float(name, x)
        if x.dim() != 2 or x.shape[1] != width:
            raise ValueError(f"{name} must be [tokens, {width}], got {tuple(x.shape)}")
        if x.device != self.device:
            raise ValueError(f"{name} is on {x.device}, the weights on {self.device}")
        return _rows(x)

    def _scratch(self, n_tokens: int, which: int) -> torch.Tensor:
        """Scratch of encode (0), decode (1) or reconstruct (2), for this call alone."""
        need = self._scratch_bytes.get(n_tokens)
        if need is None:
            out = (ctypes.c_size_t(0), ctypes.c_size_t(0), ctypes.c_size_t(0))
            L.call("sae_b200_sae4_workspace_bytes", n_tokens, self.d_in, self.n_features,
                   *(ctypes.byref(n) for n in out))
            if len(self._scratch_bytes) >= 1024:
                self._scratch_bytes.clear()
            need = self._scratch_bytes[n_tokens] = tuple(n.value for n in out)
        return torch.empty(need[which], device=self.device, dtype=torch.uint8)

    def _encode(self, x: torch.Tensor, gated: bool) -> torch.Tensor:
        x = self._input("x", x, self.d_in)
        T, F = x.shape[0], self.n_features
        out = torch.empty(T, F, device=self.device, dtype=torch.float32)
        pitch = _pitch(x)
        for t in range(0, T, _CALL_TOKENS):
            n = min(T - t, _CALL_TOKENS)
            ws = self._scratch(n, 0)
            _launch(self._index, "sae_b200_sae4_encode", self._model,
                    x.data_ptr() + t * pitch * x.element_size(), _CODES[x.dtype], n, pitch,
                    int(gated), out.data_ptr() + 4 * t * F, F, ws.data_ptr(), ws.numel())
        return out

    def encode_pre(self, x: torch.Tensor) -> torch.Tensor:
        """``W bf16(x - b_dec) + b_enc``, float32 ``[tokens, F]``. No gradient is
        recorded, here and below. The features of a token that holds an infinity
        or a NaN mean nothing; other tokens are not touched by it."""
        return self._encode(x, False)

    def encode(self, x: torch.Tensor) -> torch.Tensor:
        """The features: pre-activations above their threshold, 0 elsewhere."""
        return self._encode(x, True)

    def decode(self, acts: torch.Tensor) -> torch.Tensor:
        """``acts D + b_dec``, float32 ``[tokens, d]``, reading the decoder rows
        of nonzero activations only (features edited for steering included)."""
        acts = self._input("acts", acts.detach(), self.n_features)
        if acts.dtype != torch.float32:
            acts = acts.float()
        T, d = acts.shape[0], self.d_in
        out = torch.empty(T, d, device=self.device, dtype=torch.float32)
        pitch = _pitch(acts)
        for t in range(0, T, _CALL_TOKENS):
            n = min(T - t, _CALL_TOKENS)
            ws = self._scratch(n, 1)
            _launch(self._index, "sae_b200_sae4_decode", self._model,
                    acts.data_ptr() + 4 * t * pitch, n, pitch, out.data_ptr() + 4 * t * d,
                    ws.data_ptr(), ws.numel())
        return out

    def reconstruct(self, x: torch.Tensor, fired: Optional[torch.Tensor] = None):
        """``(x_hat float32 [tokens, d], active features per token int32)``;
        ``fired`` (uint8 [F]) is OR-accumulated. The 4-bit counterpart of
        ``B200JumpReLUSAE.reconstruct``."""
        x = self._input("x", x, self.d_in)
        if fired is not None and (fired.dtype != torch.uint8 or not fired.is_contiguous()
                                  or fired.shape != (self.n_features,)
                                  or fired.device != self.device):
            raise ValueError(f"fired must be a contiguous uint8 [{self.n_features}] on "
                             f"{self.device}")
        T, d = x.shape[0], self.d_in
        x_hat = torch.empty(T, d, device=self.device, dtype=torch.float32)
        counts = torch.empty(T, device=self.device, dtype=torch.int32)
        if T == 0:
            return x_hat, counts
        ws = self._scratch(min(T, _RECONSTRUCT_TOKENS), 2)
        pitch = _pitch(x)
        for t in range(0, T, _RECONSTRUCT_TOKENS):
            _launch(self._index, "sae_b200_sae4_reconstruct", self._model,
                    x.data_ptr() + t * pitch * x.element_size(), _CODES[x.dtype],
                    min(T - t, _RECONSTRUCT_TOKENS), pitch, x_hat.data_ptr() + 4 * t * d,
                    counts.data_ptr() + 4 * t, L.ptr(fired), ws.data_ptr(), ws.numel())
        return x_hat, counts


def quantize4(sae, group: int = 64) -> B200SAE4:
    """A 4-bit inference copy of a ``B200JumpReLUSAE`` (later training of ``sae``
    does not reach it)."""
    with torch.no_grad():
        enc = quantize4_rows(sae.W_enc.weight, group)
        dec = quantize4_rows(sae._dec_fm(), group)
        return B200SAE4.from_codes(*enc, sae.W_enc.bias, *dec, sae.b_dec, sae.log_threshold,
                                   group=group)
