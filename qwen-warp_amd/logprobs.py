"""Log probabilities of given tokens, their ranks, the rows' entropies and their best alternatives (include/qws.h
qws_logprobs) on torch tensors."""
from __future__ import annotations

import contextlib
import ctypes as C
import math
from typing import NamedTuple, Optional

import torch
from torch.autograd import forward_ad

from . import _lib
from ._lib import check
from .sampling import ValidationError

LOGPROBS_MAX = 64  # given tokens and alternatives of a row at most
INT_MAX = 2 ** 31 - 1


class LogProbsResult(NamedTuple):
    logprobs: Optional[torch.Tensor]      # fp32, the shape of `tokens` (None without tokens)
    ranks: Optional[torch.Tensor]         # int32, the shape of `tokens`: 0 = the best token, -1 = skipped
    entropy: torch.Tensor                 # fp32 [...]
    top_ids: torch.Tensor                 # int32 [..., top], best first, -1 past the last token above -inf
    top_logprobs: torch.Tensor            # fp32 [..., top]


def rows_of(x: torch.Tensor, name: str):
    """(rows, stride) of a tensor [..., n] read as rows of n contiguous elements at one stride.  Both counts fit an int."""
    shape, strides = x.shape, x.stride()
    if len(shape) < 2 or (shape[-1] > 1 and strides[-1] != 1):
        raise ValidationError(f"{name} must be [..., n] with contiguous rows", name)
    if max(shape) > INT_MAX or (len(shape) > 2 and math.prod(shape[:-1]) > INT_MAX):
        raise ValidationError(f"{name}: at most 2^31 - 1 rows of as many elements", name)
    if len(shape) == 2:
        return shape[0], strides[0] if shape[0] > 1 else 0
    rows, stride = 1, 0
    for size, step in zip(reversed(shape[:-1]), reversed(strides[:-1])):
        if size == 1:
            continue
        if rows == 1:
            stride = step
        elif rows and step != rows * stride:
            raise ValidationError(f"{name}: the leading dimensions must lie at one stride (reshape it to two dimensions)", name)
        rows *= size
    return rows, stride


def given(t: torch.Tensor, shape, dtype, device, name: str):
    if t.dtype != dtype or t.device != device or t.shape != shape or not t.is_contiguous():
        raise ValidationError(f"{name} must be a contiguous {dtype} tensor of shape {tuple(shape)} on {device}", name)


def no_tangent(t, name):
    """Forward-mode derivatives are not given: without a refusal a result would come back as one that does not depend on `t`."""
    if forward_ad._current_level >= 0 and forward_ad.unpack_dual(t).tangent is not None:
        raise ValidationError(f"{name} carries a tangent: no forward-mode derivatives", name)


def on_stream(index: int):
    """(a context that makes GPU `index` the current one, its current stream's handle).  These calls are small next to the
    kernels they start only if the host is quick: the context is left out where nothing changes, and the handle comes without
    a stream object (2 us)."""
    same = torch._C._cuda_getDevice() == index
    return NOTHING if same else torch.cuda.device(index), torch._C._cuda_getCurrentRawStream(index)


NOTHING = contextlib.nullcontext()


class LogProbs:
    """One call per batch of logits, on the current stream; the workspace is allocated with each call, so calls may run on
    any streams.

        out = LogProbs("cuda")(logits, tokens, top=5)      # logits [B, V] or [B, K + 1, V]; tokens [B] or [B, K + 1]
        out.logprobs, out.ranks, out.entropy, out.top_ids, out.top_logprobs

    logits: fp32 or bf16 [..., V] on the GPU, rows contiguous, at any stride.  tokens: int32 [...] (one token a row: those
    that `Sampler` returned; -1 = skipped: log probability 0, rank -1) or [..., M] (several: labels); None: no tokens.
    temperature: fp32 [...] (0, negative or NaN: as 1) or None.  ranks=False leaves the ranks out.  device: the logits';
    without an index, any GPU's."""

    def __init__(self, device="cuda"):
        self.lib = _lib.load()
        self.device = torch.device(device)
        self._ws_bytes = {}

    def __call__(self, logits: torch.Tensor, tokens: Optional[torch.Tensor] = None, top: int = 0, temperature: Optional[torch.Tensor] = None,
                 ranks: bool = True) -> LogProbsResult:
        dtype, dev = logits.dtype, logits.device
        if not logits.is_cuda or (dtype != torch.float32 and dtype != torch.bfloat16):
            raise ValidationError("logits must be a CUDA fp32 / bf16 tensor", "logits")
        if dev != self.device and (self.device.type != "cuda" or self.device.index is not None):
            raise ValidationError(f"logits must be on {self.device}", "logits")
        R, stride = rows_of(logits, "logits")
        lead, V, top = logits.shape[:-1], logits.shape[-1], int(top)
        if V < 1 or not 0 <= top <= LOGPROBS_MAX:
            raise ValidationError(f"top must be in [0, {LOGPROBS_MAX}]", "top", top)
        M, lp, rk = 0, None, None
        if tokens is not None:
            shape = lead
            M = 1
            if tokens.dim() > len(lead):
                M = tokens.shape[-1]
                shape = (*lead, M)
                if not 1 <= M <= LOGPROBS_MAX:
                    raise ValidationError(f"at most {LOGPROBS_MAX} tokens a row", "tokens", M)
            given(tokens, shape, torch.int32, dev, "tokens")
        if temperature is not None:
            given(temperature, lead, torch.float32, dev, "temperature")
        where, stream = on_stream(dev.index)
        with where:
            h = torch.empty(lead, dtype=torch.float32, device=dev)
            ids = torch.empty((*lead, top), dtype=torch.int32, device=dev)
            tlp = h.new_empty((*lead, top))
            if M:
                lp = h.new_empty(shape)
                if ranks:
                    rk = ids.new_empty(shape)
            if R:
                dt = _lib.DTYPE_F32 if dtype == torch.float32 else _lib.DTYPE_BF16
                key = (dt, R, V, M, top)
                n = self._ws_bytes.get(key)
                if n is None:
                    n = self._ws_bytes[key] = self.lib.qws_logprobs_ws_bytes(*key)
                ws = torch.empty(n, dtype=torch.uint8, device=dev)
                b = _lib.LogprobsBatch(logits.data_ptr(), dt, R, V, stride, tokens.data_ptr() if M else None, M, top,
                                       temperature.data_ptr() if temperature is not None else None, lp.data_ptr() if M else None,
                                       rk.data_ptr() if rk is not None else None, h.data_ptr(), ids.data_ptr() if top else None, tlp.data_ptr() if top else None)
                err = self.lib.qws_logprobs(C.byref(b), ws.data_ptr(), n, stream)
                if err:
                    check(err, "qws_logprobs")
        return LogProbsResult(lp, rk, h, ids, tlp)
