"""A head held in 8 bits (include/qws.h qws_fp8_*): the approximate logits that `HeadSelect` refines, and the scoring of
given tokens without the logits in memory, on torch tensors."""
from __future__ import annotations

import ctypes as C
from typing import Optional

import torch

from . import _lib
from ._lib import check
from .logprobs import given, on_stream, rows_of
from .sampling import ValidationError


class Fp8Head:
    """The weights w [N, K] (bf16 or fp32, on the GPU) packed once into 8 bits; w is not kept.  Calls allocate their
    workspace, so they may run on any streams (the first ones ordered behind the packing, which ran on the current one).

        head = Fp8Head(w)
        logits = head(x)                      # x bf16 [T, K] -> fp32 [T, N] (dtype=torch.bfloat16: bf16)
        logprobs, entropy = head.score(x, tokens)"""

    def __init__(self, w: torch.Tensor):
        self.lib = _lib.load()
        if w.device.type != "cuda" or w.dtype not in (torch.float32, torch.bfloat16) or w.dim() != 2 or not w.numel():
            raise ValidationError("w must be a CUDA fp32 / bf16 [N, K] tensor", "w")
        self.N, self.K = w.shape
        self.device = w.device
        self._ws_bytes = {}
        stride = rows_of(w, "w")[1]
        n = self.lib.qws_fp8_pack_bytes(self.N, self.K)
        if n == 0:
            raise ValidationError("w is larger than 2^24 x 2^20", "w")
        where, stream = on_stream(self.device.index)
        with where:
            self.packed = torch.empty(n, dtype=torch.uint8, device=self.device)
            check(self.lib.qws_fp8_pack(w.data_ptr(), _lib.DTYPE_F32 if w.dtype == torch.float32 else _lib.DTYPE_BF16, self.N, self.K, stride,
                                        self.packed.data_ptr(), stream), "qws_fp8_pack")
        self._w = self.packed.data_ptr()

    def _states(self, x):
        if x.dtype != torch.bfloat16 or x.device != self.device or x.dim() != 2 or x.shape[1] != self.K:
            raise ValidationError(f"x must be a bf16 [T, {self.K}] tensor on {self.device}", "x")
        return rows_of(x, "x")

    def _workspace(self, T, score):
        n = self._ws_bytes.get((T, score))
        if n is None:
            n = self._ws_bytes[T, score] = (self.lib.qws_fp8_score_ws_bytes if score else self.lib.qws_fp8_head_ws_bytes)(T, self.N, self.K)
        return torch.empty(n, dtype=torch.uint8, device=self.device), n

    def __call__(self, x: torch.Tensor, dtype=torch.float32, out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """The logits [T, N] of hidden states x [T, K] in fp32 or bf16; out: a tensor of that type to write them into."""
        T, stride = self._states(x)
        where, stream = on_stream(self.device.index)
        with where:
            if out is None:
                if dtype != torch.float32 and dtype != torch.bfloat16:
                    raise ValidationError("dtype must be fp32 or bf16", "dtype")
                out = torch.empty(T, self.N, dtype=dtype, device=self.device)
                out_stride = self.N
            else:
                dtype = out.dtype
                if dtype not in (torch.float32, torch.bfloat16) or out.device != self.device or out.shape != (T, self.N):
                    raise ValidationError(f"out must be a fp32 / bf16 [{T}, {self.N}] tensor on {self.device}", "out")
                out_stride = rows_of(out, "out")[1]
                if T > 1 and out_stride < self.N:
                    raise ValidationError("out: its rows overlap", "out")
            if T:
                ws, n = self._workspace(T, False)
                err = self.lib.qws_fp8_head(self._w, self.N, self.K, x.data_ptr(), stride, T, out.data_ptr(),
                                            _lib.DTYPE_F32 if dtype == torch.float32 else _lib.DTYPE_BF16, out_stride, ws.data_ptr(), n, stream)
                if err:
                    check(err, "qws_fp8_head")
        return out

    def score(self, x: torch.Tensor, tokens: torch.Tensor, temperature: Optional[torch.Tensor] = None):
        """(log probabilities, entropies), fp32 [T]: of tokens int32 [T] under softmax(logits of x / temperature); a token
        outside [0, N) is skipped (log probability 0).  temperature: fp32 [T] (0, negative or NaN: as 1) or None."""
        T, stride = self._states(x)
        given(tokens, (T,), torch.int32, self.device, "tokens")
        if temperature is not None:
            given(temperature, (T,), torch.float32, self.device, "temperature")
        where, stream = on_stream(self.device.index)
        with where:
            lp = torch.empty(T, dtype=torch.float32, device=self.device)
            h = torch.empty(T, dtype=torch.float32, device=self.device)
            if T:
                ws, n = self._workspace(T, True)
                err = self.lib.qws_fp8_score(self._w, self.N, self.K, x.data_ptr(), stride, T, tokens.data_ptr(),
                                             temperature.data_ptr() if temperature is not None else None, lp.data_ptr(), h.data_ptr(), ws.data_ptr(), n, stream)
                if err:
                    check(err, "qws_fp8_score")
        return lp, h
