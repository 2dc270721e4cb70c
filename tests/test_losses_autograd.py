"""What the losses' autograd node hands to qws_loss_grad, without a GPU: a stand-in for the library records the calls."""
import contextlib
import ctypes as C
from types import SimpleNamespace

import pytest
import torch
from torch.autograd import forward_ad
from torch.utils.checkpoint import checkpoint

import qwen_warp_amd as q
from qwen_warp_amd import _lib, losses


class Library:
    """qws_loss_grad: keeps the rows' structure and copies the logits that it points at into the gradient."""

    def __init__(self):
        self.calls = []

    def qws_loss_grad(self, rows, state, upstream, grad, stride, written, stream):
        r = C.cast(rows, C.POINTER(_lib.LossRows)).contents
        self.calls.append(SimpleNamespace(logits=r.logits, R=r.R, V=r.V, block=r.block, row_stride=r.row_stride, block_stride=r.block_stride, written=written))
        block = r.block or r.R
        for i in range(r.R):
            C.memmove(grad + 4 * i * stride, r.logits + 4 * (i // block * r.block_stride + i % block * r.row_stride), 4 * r.V)
        return 0


@pytest.fixture
def lib(monkeypatch):
    monkeypatch.setattr(losses, "on_stream", lambda index: (contextlib.nullcontext(), None))
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    return Library()


def loss_of(lib, logits, ahead=0.0):
    """A loss whose node is PolicyLoss's and PreferenceLoss's; the forward pass writes no gradient."""
    tokens = torch.zeros(logits.shape[:-1], dtype=torch.int32)

    def call(grad, scale):
        R, block, stride, block_stride = losses.blocks_of(logits, "logits")
        rows = _lib.LossRows(logits.data_ptr(), _lib.DTYPE_F32, R, logits.shape[-1], block, stride, block_stride, tokens.data_ptr(), None)
        return torch.zeros(()), rows, torch.empty(256, dtype=torch.uint8), tokens

    return losses._Loss.apply(logits, SimpleNamespace(lib=lib), call, ahead)


def test_backward_reads_the_logits_it_is_given(lib):
    """Hooks on saved tensors hand out another tensor than the forward pass saw, in other strides: the kernel gets that one's."""
    kept = []

    def unpack(t):
        kept.append(t.transpose(0, 1).contiguous().transpose(0, 1) if wide else t)
        return kept[-1]

    for wide in (False, True):  # wide: the leading dimensions in another order
        x = torch.randn(2, 3, 5, requires_grad=True)
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t.clone(), unpack):
            loss = loss_of(lib, x * 2.0)
        loss.backward()
        call = lib.calls[-1]
        assert call.logits == kept[-1].data_ptr() and (call.R, call.V) == (6, 5)
        assert (call.block, call.row_stride, call.block_stride) == ((3, 10, 5) if wide else (0, 5, 0))
        assert torch.equal(x.grad, 4.0 * x.detach())  # the gradient is the product's of what the kernel read


def test_backward_of_unpacked_logits_in_any_layout(lib):
    """A layout that the kernel does not take is copied."""
    x = torch.randn(4, 6, requires_grad=True)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t.t().contiguous().t()):
        loss = loss_of(lib, x * 2.0)
    loss.backward()
    assert torch.equal(x.grad, 4.0 * x.detach())


def test_backward_under_a_checkpoint(lib):
    """The logits are made anew for the backward pass; those of the first forward pass may be gone."""
    seen = []

    def head(x):
        logits = x * 2.0
        seen.append(logits.data_ptr())
        return loss_of(lib, logits)

    x = torch.randn(3, 7, requires_grad=True)
    loss = checkpoint(head, x, use_reentrant=False)
    held = [torch.full((3, 7), 9.0) for _ in range(8)]  # what was freed is used again
    loss.backward()
    assert lib.calls[-1].logits == seen[-1] and len(seen) == 2 and held
    assert torch.equal(x.grad, 4.0 * x.detach())


def test_backward_refuses_other_logits(lib):
    """A hook that hands out something else than the saved tensor's values: refused before the kernel reads it."""
    for change in (lambda t: t[:-1], lambda t: t.double(), lambda t: t[:, :-1].contiguous(), lambda t: t.to("meta")):
        x = torch.randn(4, 6, requires_grad=True)
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, change):
            loss = loss_of(lib, x * 2.0)
        with pytest.raises(q.ValidationError):
            loss.backward()
    assert not lib.calls


def test_forward_mode_is_refused():
    """A dual tensor does not require a gradient, and a loss without a tangent would read as one that does not depend on it."""
    x, t, v = torch.zeros(2, 3), torch.zeros(2, dtype=torch.int32), torch.zeros(2)
    fn, pl = q.PolicyLoss("cuda"), q.PreferenceLoss("cuda")
    with forward_ad.dual_level():
        d = forward_ad.make_dual(x, torch.ones(2, 3))
        for call in (lambda: fn(d, t, v, v), lambda: fn.value_and_grad(d, t, v, v), lambda: pl(d, t, torch.tensor([0, 1, 2], dtype=torch.int32))):
            with pytest.raises(q.ValidationError, match="tangent"):
                call()
        c = forward_ad.make_dual(v, torch.ones(2))
        with pytest.raises(q.ValidationError, match="advantages.*tangent"):
            fn._number(c, (2,), v.device, "advantages")
        assert fn._number(v, (2,), v.device, "advantages") == v.data_ptr()
    with pytest.raises(q.ValidationError, match="CUDA"):
        fn(x, t, v, v)


@pytest.mark.parametrize("ahead", [0.0, 1.0])
def test_backward_in_a_captured_graph_is_refused(lib, monkeypatch, ahead):
    """Of a loss whose forward pass ran before: a replay would read logits and state that were given back, or find a gradient
    written that is someone else's by then.  Outside, the same loss still has its gradient."""
    x = torch.randn(3, 7, requires_grad=True)
    loss = loss_of(lib, x * 2.0, ahead)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(q.ValidationError, match="captured"):
        loss.backward(retain_graph=True)
    assert x.grad is None and not lib.calls
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    loss.backward()
    assert torch.equal(x.grad, 4.0 * x.detach()) and lib.calls[-1].written == ahead
