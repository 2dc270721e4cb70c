"""Log probabilities of given tokens, their ranks, the rows' entropies and their best alternatives (include/qws.h
qws_logprobs) on torch tensors."""
from __future__ import annotations

import ctypes as C
from typing import NamedTuple, Optional

import torch

from . import _lib
from ._lib import check
from .sampling import ValidationError

LOGPROBS_MAX = 64  # given tokens and alternatives of a row at most


class LogProbsResult(NamedTuple):
    logprobs: Optional[torch.Tensor]      # fp32, the shape of `tokens` (None without tokens)
    ranks: Optional[torch.Tensor]         # int32, the shape of `tokens`: 0 = the best token, -1 = skipped
    entropy: torch.Tensor                 # fp32 [...]
    top_ids: torch.Tensor                 # int32 [..., top], best first, -1 past the last token above -inf
    top_logprobs: torch.Tensor            # fp32 [..., top]


def rows_of(x: torch.Tensor, name: str):
    """(rows, stride) of a tensor [..., n] read as rows of n contiguous elements at one stride."""
    if x.dim() < 2 or (x.shape[-1] > 1 and x.stride(-1) != 1):
        raise ValidationError(f"{name} must be [..., n] with contiguous rows", name)
    rows, stride = 1, 0
    for size, step in zip(reversed(x.shape[:-1]), reversed(x.stride()[:-1])):
        if size == 1:
            continue
        if rows == 1:
            stride = step
        elif rows and step != rows * stride:
            raise ValidationError(f"{name}: the leading dimensions must lie at one stride (reshape it to two dimensions)", name)
        rows *= size
    return rows, stride


def given(t: torch.Tensor, shape, dtype, device, name: str):
    if t.dtype != dtype or t.device != device or tuple(t.shape) != tuple(shape) or not t.is_contiguous():
        raise ValidationError(f"{name} must be a contiguous {dtype} tensor of shape {tuple(shape)} on {device}", name)


class LogProbs:
    """One call per batch of logits, on the current stream; the workspace is allocated with each call, so calls may run on
    any streams.

        out = LogProbs("cuda")(logits, tokens, top=5)      # logits [B, V] or [B, K + 1, V]; tokens [B] or [B, K + 1]
        out.logprobs, out.ranks, out.entropy, out.top_ids, out.top_logprobs

    logits: fp32 or bf16 [..., V] on the GPU, rows contiguous, at any stride.  tokens: int32 [...] (one token a row: those
    that `Sampler` returned; -1 = skipped: log probability 0, rank -1) or [..., M] (several: labels); None: no tokens.
    temperature: fp32 [...] (0: as 1) or None.  ranks=False leaves the ranks out."""

    def __init__(self, device="cuda"):
        self.lib = _lib.load()
        self.device = torch.device(device)

    def __call__(self, logits: torch.Tensor, tokens: Optional[torch.Tensor] = None, top: int = 0, temperature: Optional[torch.Tensor] = None,
                 ranks: bool = True) -> LogProbsResult:
        if logits.device.type != "cuda" or logits.dtype not in (torch.float32, torch.bfloat16):
            raise ValidationError("logits must be a CUDA fp32 / bf16 tensor", "logits")
        R, stride = rows_of(logits, "logits")
        lead, V, dev = logits.shape[:-1], logits.shape[-1], logits.device
        top = int(top)
        if V < 1 or not 0 <= top <= LOGPROBS_MAX:
            raise ValidationError(f"top must be in [0, {LOGPROBS_MAX}]", "top", top)
        M = 0
        if tokens is not None:
            M = 1 if tokens.dim() < logits.dim() else tokens.shape[-1]
            if not 1 <= M <= LOGPROBS_MAX:
                raise ValidationError(f"at most {LOGPROBS_MAX} tokens a row", "tokens", M)
            given(tokens, lead if tokens.dim() < logits.dim() else (*lead, M), torch.int32, dev, "tokens")
        if temperature is not None:
            given(temperature, lead, torch.float32, dev, "temperature")
        with torch.cuda.device(dev):
            lp = torch.empty(tokens.shape, dtype=torch.float32, device=dev) if M else None
            rk = torch.empty(tokens.shape, dtype=torch.int32, device=dev) if M and ranks else None
            h = torch.empty(lead, dtype=torch.float32, device=dev)
            ids = torch.empty((*lead, top), dtype=torch.int32, device=dev)
            tlp = torch.empty((*lead, top), dtype=torch.float32, device=dev)
            if R:
                dt = _lib.DTYPE_F32 if logits.dtype == torch.float32 else _lib.DTYPE_BF16
                ptr = lambda t: t.data_ptr() if t is not None and t.numel() else None  # noqa: E731
                b = _lib.LogprobsBatch(logits.data_ptr(), dt, R, V, stride, ptr(tokens), M, top, ptr(temperature), ptr(lp), ptr(rk), ptr(h), ptr(ids), ptr(tlp))
                ws = torch.empty(self.lib.qws_logprobs_ws_bytes(dt, R, V, M, top), dtype=torch.uint8, device=dev)
                check(self.lib.qws_logprobs(C.byref(b), ws.data_ptr(), ws.numel(), C.c_void_p(torch.cuda.current_stream(dev).cuda_stream)), "qws_logprobs")
        return LogProbsResult(lp, rk, h, ids, tlp)
