"""Losses over drawn tokens with their gradient at the logits (include/qws.h qws_policy_loss, qws_preference_loss) on torch
tensors: what follows `Sampler` and `LogProbs` where a model learns from its own samples."""
from __future__ import annotations

import ctypes as C
import math
from typing import NamedTuple, Optional, Sequence, Tuple

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from ._lib import check
from .logprobs import INT_MAX, given, no_tangent, on_stream
from .sampling import ValidationError


class PolicyLossResult(NamedTuple):
    loss: torch.Tensor                    # fp32, one value; differentiable where the logits are
    logprobs: torch.Tensor                # fp32 [...]: the tokens' log probabilities (0 for rows left out)
    ratio: torch.Tensor                   # fp32 [...]: e^(logprobs - old_logprobs) (1 for rows left out)
    kl: Optional[torch.Tensor]            # fp32 [...]: e^d - 1 - d, d = ref_logprobs - logprobs (None without ref_logprobs)


class PreferenceLossResult(NamedTuple):
    loss: torch.Tensor                    # fp32, one value; differentiable where the logits are
    logprobs: torch.Tensor                # fp32 [2 P]: the sequences' summed (or mean) log probabilities
    margins: torch.Tensor                 # fp32 [P]: what the sigmoid is taken of
    token_logprobs: torch.Tensor          # fp32 [...] (0 for rows left out)


def blocks_of(x: torch.Tensor, name: str):
    """(rows, rows of a block, row stride, block stride) of a tensor [..., n] read as rows of n contiguous elements in blocks at one
    stride, each of rows at one stride: what a slice [:, :-1] of [B, L, n] is.  One block: 0 rows of a block."""
    shape, strides = x.shape, x.stride()
    if len(shape) < 2 or (shape[-1] > 1 and strides[-1] != 1):
        raise ValidationError(f"{name} must be [..., n] with contiguous rows", name)
    if max(shape) > INT_MAX or (len(shape) > 2 and math.prod(shape[:-1]) > INT_MAX):
        raise ValidationError(f"{name}: at most 2^31 - 1 rows of as many elements", name)
    if len(shape) == 2:
        return shape[0], 0, strides[0] if shape[0] > 1 else 0, 0
    levels = []  # (rows, stride), innermost first
    for size, step in zip(reversed(shape[:-1]), reversed(strides[:-1])):
        if size == 1:
            continue
        if levels and step == levels[-1][0] * levels[-1][1]:
            levels[-1] = (levels[-1][0] * size, levels[-1][1])
        else:
            levels.append((size, step))
    rows = math.prod(shape[:-1])
    if rows == 0 or not levels:
        return rows, 0, 0, 0
    if len(levels) == 1:
        return rows, 0, levels[0][1], 0
    if len(levels) == 2:
        return rows, levels[0][0], levels[0][1], levels[1][1]
    raise ValidationError(f"{name}: the leading dimensions must lie at two strides at most (reshape it)", name)


def structure(logits, tokens: int, temperature: Optional[int] = None):
    """The rows of logits fp32 / bf16 [..., V] as the library takes them; tokens, temperature: addresses."""
    R, block, stride, block_stride = blocks_of(logits, "logits")
    return _lib.LossRows(logits.data_ptr(), _lib.DTYPE_F32 if logits.dtype == torch.float32 else _lib.DTYPE_BF16, R, logits.shape[-1], block, stride, block_stride,
                         tokens, temperature)


def not_captured():
    """A backward pass there ends the process where an eager graph of the same leaves lives (a leaf's node belongs to that graph's
    stream, which is not captured).  Of a loss whose forward pass ran before, replays would read logits and state that were given
    back since."""
    if torch.cuda.is_current_stream_capturing():
        raise ValidationError("inside a captured graph the gradient is value_and_grad's", "logits")


class _Loss(torch.autograd.Function):
    """The loss as a function of the logits; `call(grad, scale)` runs it and returns (loss, rows, state, what they refer to).  With
    `ahead` (not 0) the gradient is written by the forward pass, for an upstream gradient of that value; the first backward pass
    hands it out, after a launch that writes it anew for any other.  Later ones write their own.  The logits of a backward pass are
    those that autograd hands out: under hooks on saved tensors (an offload to the host, a checkpoint that makes them anew) another
    tensor than the forward pass read, whose memory may be gone, and in strides of its own."""

    @staticmethod
    def forward(ctx, logits, owner, call, ahead):
        ctx.grad = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device) if ahead else None
        loss, rows, ctx.state, ctx.keep = call(ctx.grad, ahead)
        ctx.owner, ctx.ahead, ctx.tokens, ctx.of = owner, ahead, rows.tokens, (logits.shape, logits.dtype, logits.device)
        ctx.save_for_backward(logits)
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, upstream):
        not_captured()
        (logits,) = ctx.saved_tensors
        if (logits.shape, logits.dtype, logits.device) != ctx.of:
            raise ValidationError(f"the saved logits came back as {logits.dtype} {tuple(logits.shape)} on {logits.device}", "logits")
        where, stream = on_stream(logits.device.index)
        with where:
            grad, ctx.grad = ctx.grad, None
            written = ctx.ahead
            if grad is None:
                written = 0.0
                grad = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
            try:
                rows = structure(logits, ctx.tokens)
            except ValidationError:  # strides that the forward pass would have refused
                logits = logits.contiguous()
                rows = structure(logits, ctx.tokens)
            err = ctx.owner.lib.qws_loss_grad(C.byref(rows), ctx.state.data_ptr(), upstream.data_ptr(), grad.data_ptr(), rows.V, written, stream)
            if err:
                check(err, "qws_loss_grad")
        return grad, None, None, None


class _Base:
    def __init__(self, device):
        self.lib = _lib.load()
        self.device = torch.device(device)
        self._bytes = {}

    def _rows(self, logits, tokens, temperature=None):
        """The checks of the rows, and their structure."""
        dtype, dev = logits.dtype, logits.device
        no_tangent(logits, "logits")
        if not logits.is_cuda or (dtype != torch.float32 and dtype != torch.bfloat16):
            raise ValidationError("logits must be a CUDA fp32 / bf16 tensor", "logits")
        if dev != self.device and (self.device.type != "cuda" or self.device.index is not None):
            raise ValidationError(f"logits must be on {self.device}", "logits")
        if logits.dim() and logits.shape[-1] < 1:
            raise ValidationError("logits must have a value a row", "logits")
        lead = logits.shape[:-1]
        given(tokens, lead, torch.int32, dev, "tokens")
        return structure(logits, tokens.data_ptr(), self._number(temperature, lead, dev, "temperature") if temperature is not None else None)

    @staticmethod
    def _number(t, shape, dev, name):
        if t is None:
            raise ValidationError(f"{name} is needed", name)
        if t.dtype != torch.float32 or t.device != dev or t.shape != shape or not t.is_contiguous():
            given(t, shape, torch.float32, dev, name)
        if t.requires_grad:
            raise ValidationError(f"{name} is taken as a constant: detach it", name)
        no_tangent(t, name)
        return t.data_ptr()

    def _state(self, query, *key):
        n = self._bytes.get(key)
        if not n:
            n = self._bytes[key] = query(*key)
            if n == 0:
                raise ValidationError("logits: fewer than 2^24 rows of at most 2^24 values", "logits")
        return n

    def _forward(self, logits, call, ahead=0.0):
        """The loss, with autograd where the logits ask for it."""
        if not (logits.requires_grad and torch.is_grad_enabled()):
            return call(None, 1.0)[0]
        not_captured()
        return _Loss.apply(logits, self, call, ahead)


class PolicyLoss(_Base):
    """The clipped policy loss of drawn tokens, with a KL term towards reference log probabilities.

        loss_fn = PolicyLoss("cuda", clip=(0.2, 0.2), kl=0.0)
        out = loss_fn(logits, tokens, old_logprobs, advantages)   # logits [..., V]; the others [...]
        out.loss.backward()
        out, grad = loss_fn.value_and_grad(logits, tokens, old_logprobs, advantages)   # without autograd, in one call

    Per row with r = e^(log p - old_logprobs) and d = ref_logprobs - log p:
    -min(r A, clamp(r, 1 - clip[0], 1 + clip[1]) A) + kl (e^d - 1 - d), times its weight; without weights the mean over the rows with a token.
    logits: fp32 or bf16, rows contiguous, the leading dimensions at up to two strides.  tokens: int32 (`Sampler`'s; one
    outside [0, V), as -1, leaves its row out).  old_logprobs (`LogProbs`'), advantages, ref_logprobs, weights,
    temperature (0, negative or NaN: as 1): fp32, constants.  Calls run on any streams; the workspace is allocated with each call.
    upstream: the upstream gradient that backward passes will most often bring (1 / n for a loss that is divided by n, a loss
    scaler's factor); it may be set between calls.  Any other is right too, but costs another way over the logits."""

    def __init__(self, device="cuda", clip: Sequence[float] = (0.2, 0.2), kl: float = 0.0, upstream: float = 1.0):
        super().__init__(device)
        low, high = (float(c) for c in clip)
        if not (0.0 <= low <= 1.0 and 0.0 <= high < 1e38):
            raise ValidationError("clip must be (in [0, 1], >= 0)", "clip", clip)
        if not abs(float(kl)) < 1e38:
            raise ValidationError("kl must be finite", "kl", kl)
        if not abs(float(upstream)) < 1e38:
            raise ValidationError("upstream must be finite", "upstream", upstream)
        self.clip, self.kl, self.upstream = (low, high), float(kl), float(upstream)

    def __call__(self, logits: torch.Tensor, tokens: torch.Tensor, old_logprobs: torch.Tensor, advantages: torch.Tensor, ref_logprobs: Optional[torch.Tensor] = None,
                 weights: Optional[torch.Tensor] = None, temperature: Optional[torch.Tensor] = None) -> PolicyLossResult:
        call, others = self._prepare(logits, tokens, old_logprobs, advantages, ref_logprobs, weights, temperature)
        # from some size on the gradient comes on the loss's own way over the logits
        ahead = 0.0
        if logits.requires_grad and self.lib.qws_policy_one_pass(_lib.DTYPE_F32 if logits.dtype == torch.float32 else _lib.DTYPE_BF16, others[0].numel(), logits.shape[-1]):
            ahead = self.upstream
        return PolicyLossResult(self._forward(logits, call, ahead), *others)

    def value_and_grad(self, logits: torch.Tensor, tokens: torch.Tensor, old_logprobs: torch.Tensor, advantages: torch.Tensor,
                       ref_logprobs: Optional[torch.Tensor] = None, weights: Optional[torch.Tensor] = None,
                       temperature: Optional[torch.Tensor] = None) -> Tuple[PolicyLossResult, torch.Tensor]:
        """(the result, the loss's gradient at the logits: their type and shape, contiguous)."""
        call, others = self._prepare(logits, tokens, old_logprobs, advantages, ref_logprobs, weights, temperature)
        grad = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
        return PolicyLossResult(call(grad, 1.0)[0], *others), grad

    def _prepare(self, logits, tokens, old, adv, ref, weights, temperature):
        rows = self._rows(logits, tokens, temperature)
        lead, dev, number = logits.shape[:-1], logits.device, self._number
        inputs = (number(old, lead, dev, "old_logprobs"), number(adv, lead, dev, "advantages"), number(ref, lead, dev, "ref_logprobs") if ref is not None else None,
                  number(weights, lead, dev, "weights") if weights is not None else None)
        n = self._state(self.lib.qws_policy_state_bytes, rows.dtype, rows.R, rows.V)
        where, stream = on_stream(dev.index)
        with where:
            lp = torch.empty(lead, dtype=torch.float32, device=dev)
            ratio = torch.empty_like(lp)
            kl = torch.empty_like(lp) if ref is not None else None

        def call(grad, scale):
            with where:
                loss = lp.new_empty(())
                state = torch.empty(n, dtype=torch.uint8, device=dev)
                b = _lib.PolicyBatch(rows, *inputs, *self.clip, self.kl, loss.data_ptr(), lp.data_ptr(), ratio.data_ptr(), kl.data_ptr() if kl is not None else None)
                err = self.lib.qws_policy_loss(C.byref(b), state.data_ptr(), n, grad.data_ptr() if grad is not None else None, rows.V, scale, stream)
                if err:
                    check(err, "qws_policy_loss")
            return loss, rows, state, tokens

        return call, (lp, ratio, kl)


class PreferenceLoss(_Base):
    """The loss of pairs of texts by the log ratio of their probabilities, the first of each pair preferred.

        loss_fn = PreferenceLoss("cuda", beta=0.1)
        out = loss_fn(logits, tokens, starts, ref=ref_logprobs)   # logits [R, V], tokens [R], starts [2 P + 1]
        out.loss.backward()
        out, grad = loss_fn.value_and_grad(logits, tokens, starts)   # without autograd, in one call

    Sequence i is rows starts[i] .. starts[i + 1], 2 p the preferred one of pair p and 2 p + 1 the other; s_i is the sum (average:
    the mean) of its tokens' log probabilities; with u = beta ((s_2p - ref_2p) - (s_2p+1 - ref_2p+1)) - margin a pair's loss is
    -(1 - smoothing) ln sigmoid(u) - smoothing ln sigmoid(-u), times its weight; without weights the mean over the pairs.
    logits: fp32 or bf16 [..., V], rows contiguous, the leading dimensions at up to two strides.  tokens: int32 [...]
    (one outside [0, V), as -1 for a prompt's positions and padding, leaves its row out).  starts: int32 [2 P + 1],
    ascending; None with logits [2 P, L, V]: a sequence each.  ref (the reference's s) [2 P], weights [P]: fp32, constants."""

    def __init__(self, device="cuda", beta: float = 0.1, margin: float = 0.0, smoothing: float = 0.0, average: bool = False):
        super().__init__(device)
        if not (abs(float(beta)) < 1e38 and abs(float(margin)) < 1e38):
            raise ValidationError("beta and margin must be finite", "beta", beta)
        if not 0.0 <= float(smoothing) <= 1.0:
            raise ValidationError("smoothing must be in [0, 1]", "smoothing", smoothing)
        self.beta, self.margin, self.smoothing, self.average = float(beta), float(margin), float(smoothing), bool(average)

    def __call__(self, logits: torch.Tensor, tokens: torch.Tensor, starts: Optional[torch.Tensor] = None, ref: Optional[torch.Tensor] = None,
                 weights: Optional[torch.Tensor] = None) -> PreferenceLossResult:
        call, others = self._prepare(logits, tokens, starts, ref, weights)
        return PreferenceLossResult(self._forward(logits, call), *others)

    def value_and_grad(self, logits: torch.Tensor, tokens: torch.Tensor, starts: Optional[torch.Tensor] = None, ref: Optional[torch.Tensor] = None,
                       weights: Optional[torch.Tensor] = None) -> Tuple[PreferenceLossResult, torch.Tensor]:
        """(the result, the loss's gradient at the logits: their type and shape, contiguous)."""
        call, others = self._prepare(logits, tokens, starts, ref, weights)
        grad = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
        return PreferenceLossResult(call(grad, 1.0)[0], *others), grad

    def _prepare(self, logits, tokens, starts, ref, weights):
        rows = self._rows(logits, tokens)
        lead, dev = logits.shape[:-1], logits.device
        if starts is None:
            if len(lead) != 2 or lead[0] % 2:
                raise ValidationError("without starts logits must be [2 P, L, V]", "starts")
            P = lead[0] // 2
        else:
            if starts.dim() != 1 or starts.numel() % 2 == 0:
                raise ValidationError("starts must be [2 P + 1]", "starts")
            given(starts, starts.shape, torch.int32, dev, "starts")
            P = starts.numel() // 2
        inputs = (self._number(ref, (2 * P,), dev, "ref") if ref is not None else None, self._number(weights, (P,), dev, "weights") if weights is not None else None)
        n = self._state(self.lib.qws_preference_state_bytes, rows.dtype, rows.R, rows.V, P)
        where, stream = on_stream(dev.index)
        with where:
            if starts is None:
                starts = torch.arange(0, 2 * P + 1, dtype=torch.int32, device=dev).mul_(lead[1])
            lp = torch.empty(lead, dtype=torch.float32, device=dev)
            sums, margins = lp.new_empty(2 * P), lp.new_empty(P)

        def call(grad, scale):
            with where:
                loss = lp.new_empty(())
                state = torch.empty(n, dtype=torch.uint8, device=dev)
                b = _lib.PreferenceBatch(rows, starts.data_ptr(), P, self.average, *inputs, self.beta, self.margin, self.smoothing, loss.data_ptr(), sums.data_ptr(),
                                         margins.data_ptr(), lp.data_ptr())
                err = self.lib.qws_preference_loss(C.byref(b), state.data_ptr(), n, grad.data_ptr() if grad is not None else None, rows.V, scale, stream)
                if err:
                    check(err, "qws_preference_loss")
            return loss, rows, state, tokens

        return call, (sums, margins, lp)
