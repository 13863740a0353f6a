"""GPU losses over a large vocabulary (``csrc/kernels/vocab_loss.hip``): cross-entropy behind the output projection, and the
divergence from a teacher's top logits, on given logits or behind the projection.

Role parity: nn.CrossEntropyLoss at /root/reference/src/main.py:62,76,78 (on a classifier's logits).
"""

from __future__ import annotations

import os

import torch

from .hip import SHADOWS, _axpy_dev, _check, _derivative_wanted, _grad_sink, _on, _once_differentiable, _ptr, _round_up, _stream, zero_padded
from .hip_transformer import _f, _i, _ll, _sig, _vp

_head_scratch = _sig("pdt_head_loss_scratch", [_i] * 8)
_head_scratch.restype = _ll
_head = _sig("pdt_head_loss", [_vp] * 9 + [_ll] + [_i] * 5 + [_f, _vp])
_scale_gradients = _sig("pdt_scale_gradients", [_vp, _ll, _i, _vp, _ll, _i, _vp, _vp])
_distill_scratch = _sig("pdt_distill_scratch", [_i] * 2)
_distill_scratch.restype = _ll
_distill = _sig("pdt_distill", [_vp] * 6 + [_ll] + [_i] * 3 + [_ll, _ll, _f, _i, _vp])

# Rows worked off at a time: their exponentials (2 bytes per row and vocabulary entry; the size of the logits in bf16) are the one
# large buffer, without a gradient the groups' statistics (8 bytes per row and 64 entries).  8192 rows
# of 130 001 entries, width 2048: 10.6 ms in one piece (2.1 GB), 11.6 in pieces of 1 GB, 14.1 in pieces of 256 MB.
CHUNK_BYTES = int(os.environ.get("PDT_VOCAB_CHUNK_MB", "8192")) << 20
MAX_ROWS = (1 << 22) - 63  # rows of a call stay below (rounded up to 64, with up to 1024 threads each: fewer than 2^32 in a launch)


def _check_rows(n: int) -> None:
    if n >= MAX_ROWS:
        raise ValueError(f"the vocabulary losses take fewer than {MAX_ROWS} rows at a time, got {n}")


def _matrix(x: torch.Tensor, width: int) -> torch.Tensor:
    x = x.reshape(-1, width)
    if x.dtype != torch.bfloat16:
        x = x.to(torch.bfloat16)
    if not x.is_contiguous() or x.data_ptr() % 16:
        x = x.clone(memory_format=torch.contiguous_format)
    return x


def _weight(weight: torch.Tensor) -> torch.Tensor:
    """bf16 copy of a parameter (the one every linear layer uses and the optimizer refreshes), or the bf16 tensor itself."""
    if weight.dtype == torch.float32 and isinstance(weight, torch.nn.Parameter):
        return SHADOWS.fwd(weight)
    return _matrix(weight.detach(), weight.shape[1])


def _head_forward(x, weight, ids, teacher, tau: float, want_dx: bool, want_dw: bool):
    """(loss, dx, dW), the gradients for an incoming one of 1."""
    vocab, width = weight.shape
    dev = x.device
    with _on(dev):
        x2, w = _matrix(x, width), _weight(weight)
        n, top = ids.shape
        _check_rows(n)
        groups = -(-vocab // 64)
        chunk = min(n, CHUNK_BYTES // (groups * (128 if want_dx or want_dw else 8)))
        if chunk < n:
            chunk = min(n, max(256, chunk - chunk % 256))
        # one chunk and a bf16 weight: the gradient is rounded once, in the product's epilogue; else it is summed in fp32
        direct = want_dw and chunk == n and weight.dtype == torch.bfloat16
        dx = torch.empty((n, width), dtype=torch.bfloat16, device=dev) if want_dx else None
        dw = torch.empty((vocab, width), dtype=torch.bfloat16 if direct else torch.float32, device=dev) if want_dw else None
        loss = torch.empty((), dtype=torch.float32, device=dev)
        size = _head_scratch(n, top, vocab, width, chunk, int(teacher is not None), int(want_dx), int(want_dw))
        if size < 0:
            raise ValueError(f"the vocabulary kernels do not take {n} rows of {width} features against {vocab} entries")
        scratch = torch.empty(size, dtype=torch.uint8, device=dev)
        _check(_head(x2.data_ptr(), w.data_ptr(), ids.data_ptr(), _ptr(teacher), loss.data_ptr(), _ptr(dx), _ptr(dw) if direct else None,
                     None if direct else _ptr(dw), scratch.data_ptr(), size, n, top, vocab, width, chunk, tau, _stream()), "head_loss")
    return loss, dx, dw


def _scale(g, *grads) -> None:
    """Gradients (bf16 or fp32, up to two) times a device scalar, in place."""
    args = []
    for d in (*grads, None)[:2]:
        args += (None, 0, 0) if d is None else (d.data_ptr(), d.numel(), int(d.dtype == torch.float32))
    _check(_scale_gradients(*args, g.data_ptr(), _stream()), "scale_gradients")


def _check_capture(ctx) -> None:
    """A graph of the backward pass alone would scale the forward pass's buffers again at every replay."""
    if not ctx.captured and torch.cuda.is_current_stream_capturing():
        raise RuntimeError("the backward pass of a vocabulary loss is captured without its forward pass; capture both, in one graph or one each")


class _HeadLoss(torch.autograd.Function):
    """Loss of ``x W^T`` against a few targets per row.  The rows are worked off in chunks; the forward pass leaves ``dx``
    and ``dW`` for an incoming gradient of 1, the backward pass multiplies them by the incoming one (a device scalar; where it
    is neither 1 nor another power of two, gradients in bf16 are rounded a second time)."""

    @staticmethod
    def forward(ctx, x, weight, ids, teacher, tau: float):
        loss, *ctx.grads = _head_forward(x, weight, ids, teacher, tau, *ctx.needs_input_grad[:2])
        ctx.weight, ctx.shape, ctx.captured = weight, x.shape, torch.cuda.is_current_stream_capturing()
        return loss

    @staticmethod
    @_once_differentiable
    def backward(ctx, g):
        dx, dw = ctx.grads
        if dx is None and dw is None:
            raise RuntimeError("the loss behind a projection handed its gradients out already (backward ran twice)")
        _check_capture(ctx)
        ctx.grads = [None, None]
        weight = ctx.weight
        with _on(g.device):
            g1 = g if g.dtype == torch.float32 else g.to(torch.float32)
            sink = _grad_sink(weight, tuple(weight.shape)) if dw is not None and dw.dtype == torch.float32 else None
            if sink is not None:
                _check(_axpy_dev(sink.data_ptr(), dw.data_ptr(), g1.data_ptr(), dw.numel(), _stream()), "axpy")
                dw = None
            _scale(g1, dx, dw)
            if dw is not None:
                dw = dw.to(weight.dtype)
        return None if dx is None else dx.view(ctx.shape), dw, None, None, None


def head_loss(x, weight, ids, teacher, tau: float):
    if not _derivative_wanted(x, weight):
        return _head_forward(x, weight, ids, teacher, tau, False, False)[0]
    return _HeadLoss.apply(x, weight, ids, teacher, tau)


def _distill_forward(logits, ids, teacher, tau: float, want: bool):
    """(loss, gradient of the logits for an incoming one of 1, rows padded with zeros to 64 entries as ``ops.linear`` takes them)."""
    vocab = logits.shape[-1]
    dev = logits.device
    with _on(dev):
        z = logits.reshape(-1, vocab)
        if z.dtype not in (torch.bfloat16, torch.float32):
            z = z.to(torch.float32)
        if z.stride(1) != 1 and vocab > 1:
            z = z.contiguous()
        n, top = ids.shape
        _check_rows(n)
        dz = torch.empty((n, _round_up(vocab, 64)), dtype=z.dtype, device=dev) if want else None
        loss = torch.empty((), dtype=torch.float32, device=dev)
        size = _distill_scratch(n, top)
        scratch = torch.empty(size, dtype=torch.uint8, device=dev)
        _check(_distill(z.data_ptr(), _ptr(dz), ids.data_ptr(), teacher.data_ptr(), loss.data_ptr(), scratch.data_ptr(), size, n, vocab, top,
                        z.stride(0), 0 if dz is None else dz.stride(0), tau, int(z.dtype == torch.bfloat16), _stream()), "distill")
    return loss, dz


class _LogitsDistill(torch.autograd.Function):
    """The forward pass leaves the gradient for an incoming one of 1 (the logits are read once), as the cross-entropy does."""

    @staticmethod
    def forward(ctx, logits, ids, teacher, tau: float):
        loss, ctx.dz = _distill_forward(logits, ids, teacher, tau, True)
        ctx.shape, ctx.captured = logits.shape, torch.cuda.is_current_stream_capturing()
        return loss

    @staticmethod
    @_once_differentiable
    def backward(ctx, g):
        dz = ctx.dz
        if dz is None:
            raise RuntimeError("the distillation loss handed its gradient out already (backward ran twice)")
        _check_capture(ctx)
        ctx.dz = None
        with _on(g.device):
            g1 = g if g.dtype == torch.float32 else g.to(torch.float32)
            _scale(g1, dz)
        if dz.shape[1] != ctx.shape[-1]:
            dz = zero_padded(dz)[:, :ctx.shape[-1]]
        return dz.reshape(ctx.shape), None, None, None


def logits_distill(logits, ids, teacher, tau: float):
    if not _derivative_wanted(logits):
        return _distill_forward(logits, ids, teacher, tau, False)[0]
    return _LogitsDistill.apply(logits, ids, teacher, tau)
