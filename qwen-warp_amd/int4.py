"""A head held in 4 bits (include/qws.h qws_int4_*): logits of a few hidden states from weights with a scale and a zero point
for each group of them, on torch tensors."""
from __future__ import annotations

from typing import Optional

import torch

from . import _lib
from ._lib import check
from .logprobs import no_tangent, on_stream, rows_of
from .sampling import ValidationError

GROUPS = (32, 64, 128)


class Int4Head:
    """The weights w [N, K] (bf16 or fp32, on the GPU) packed once into 4 bits, `group` of a row's values (32, 64 or 128) to a
    scale and a zero point; w is not kept.  `from_codes` takes a quantised checkpoint's codes instead.  Calls allocate their
    workspace, so they may run on any streams (the first ones ordered behind the packing, which ran on the current one).

        head = Int4Head(w)                                    # or Int4Head.from_codes(codes, scales, zeros, group=64)
        logits = head(x)                                      # x bf16 [T, K] -> fp32 [T, N] (dtype=torch.bfloat16: bf16)"""

    def __init__(self, w: torch.Tensor, group: int = 128):
        if w.device.type != "cuda" or w.dtype not in (torch.float32, torch.bfloat16) or w.dim() != 2 or not w.numel():
            raise ValidationError("w must be a CUDA fp32 / bf16 [N, K] tensor", "w")
        stride = rows_of(w, "w")[1]
        self._pack(w.device, *w.shape, group, lambda lib, packed, stream: lib.qws_int4_pack(
            w.data_ptr(), _lib.DTYPE_F32 if w.dtype == torch.float32 else _lib.DTYPE_BF16, self.N, self.K, stride, self.group, packed, stream))

    @classmethod
    def from_codes(cls, codes: torch.Tensor, scales: torch.Tensor, zeros: Optional[torch.Tensor] = None, group: int = 128) -> "Int4Head":
        """Weights (codes - zeros) * scales: codes uint8 [N, K] (the low four bits count), scales bf16 or fp16 [N, groups] with
        groups = ceil(K / group), zeros uint8 [N, groups] (the low four bits) or None (8 everywhere)."""
        if codes.device.type != "cuda" or codes.dtype != torch.uint8 or codes.dim() != 2 or not codes.numel():
            raise ValidationError("codes must be a CUDA uint8 [N, K] tensor", "codes")
        if group not in GROUPS:
            raise ValidationError(f"group must be one of {GROUPS}", "group", group)
        shape = (codes.shape[0], -(-codes.shape[1] // group))
        if scales.dtype not in (torch.bfloat16, torch.float16) or scales.device != codes.device or scales.shape != shape:
            raise ValidationError(f"scales must be a bf16 / fp16 tensor of shape {shape} on {codes.device}", "scales")
        if zeros is not None and (zeros.dtype != torch.uint8 or zeros.device != codes.device or zeros.shape != shape):
            raise ValidationError(f"zeros must be a uint8 tensor of shape {shape} on {codes.device}", "zeros")
        steps = [rows_of(t, name)[1] if t is not None else 0 for t, name in ((codes, "codes"), (scales, "scales"), (zeros, "zeros"))]
        head = cls.__new__(cls)
        head._pack(codes.device, *codes.shape, group, lambda lib, packed, stream: lib.qws_int4_pack_codes(
            codes.data_ptr(), steps[0], scales.data_ptr(), int(scales.dtype == torch.float16), steps[1], zeros.data_ptr() if zeros is not None else None, steps[2],
            head.N, head.K, head.group, packed, stream))
        return head

    def _pack(self, device, N, K, group, pack):
        self.lib = _lib.load()
        if group not in GROUPS:
            raise ValidationError(f"group must be one of {GROUPS}", "group", group)
        self.N, self.K, self.group, self.device = N, K, int(group), device
        self._ws_bytes = {}
        n = self.lib.qws_int4_pack_bytes(N, K, self.group)
        if n == 0:
            raise ValidationError("the weights are larger than 2^24 x 2^20", "w")
        where, stream = on_stream(device.index)
        with where:
            self.packed = torch.empty(n, dtype=torch.uint8, device=device)
            check(pack(self.lib, self.packed.data_ptr(), stream), "qws_int4_pack")
        self._w = self.packed.data_ptr()

    def __call__(self, x: torch.Tensor, dtype=torch.float32, out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """The logits [T, N] of hidden states x [T, K] in fp32 or bf16; out: a tensor of that type to write them into.  They are
        constants: an x that requires a gradient is taken under torch.no_grad() alone."""
        if x.requires_grad and torch.is_grad_enabled():
            raise ValidationError("x requires a gradient, which the head does not give: detach it, or call under torch.no_grad()", "x")
        no_tangent(x, "x")
        if x.dtype != torch.bfloat16 or x.device != self.device or x.dim() != 2 or x.shape[1] != self.K:
            raise ValidationError(f"x must be a bf16 [T, {self.K}] tensor on {self.device}", "x")
        T, stride = rows_of(x, "x")
        where, on = on_stream(self.device.index)
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
                n = self._ws_bytes.get(T)
                if n is None:
                    n = self._ws_bytes[T] = self.lib.qws_int4_head_ws_bytes(T, self.N, self.K, self.group)
                ws = torch.empty(n, dtype=torch.uint8, device=self.device)
                err = self.lib.qws_int4_head(self._w, self.N, self.K, self.group, x.data_ptr(), stride, T, out.data_ptr(),
                                             _lib.DTYPE_F32 if dtype == torch.float32 else _lib.DTYPE_BF16, out_stride, ws.data_ptr(), n, on)
                if err:
                    check(err, "qws_int4_head")
        return out
