"""GPU losses over a large vocabulary (``csrc/kernels/vocab_loss.hip``): cross-entropy behind the output projection, and the
divergence from a teacher's top logits, on given logits or behind the projection.

Role parity: nn.CrossEntropyLoss at /root/reference/src/main.py:62,76,78 (on a classifier's logits).
"""

from __future__ import annotations

import os

import torch

from .hip import SHADOWS, _axpy_dev, _check, _grad_sink, _ptr, _round_up, _scale_by_scalar, _stream
from .hip_transformer import _f, _i, _ll, _sig, _vp

_scores = _sig("pdt_vocab_scores", [_vp] * 4 + [_i] * 3 + [_ll, _f, _vp])
_targets = _sig("pdt_vocab_targets", [_vp] * 9 + [_i] * 4 + [_f, _vp])
_rows = _sig("pdt_vocab_rows", [_vp] * 7 + [_i] * 3 + [_ll, _vp])
_mean = _sig("pdt_vocab_mean", [_vp] * 3 + [_i, _vp])
_part_floats = _sig("pdt_vocab_part_floats", [_i] * 4)
_part_floats.restype = _ll
_dx = _sig("pdt_vocab_dx", [_vp] * 5 + [_i] * 3 + [_ll, _vp])
_dw = _sig("pdt_vocab_dw", [_vp] * 4 + [_i, _vp, _vp] + [_i] * 3 + [_ll, _vp])
_distill = _sig("pdt_logits_distill", [_vp] * 8 + [_i] * 3 + [_ll, _ll, _f, _i, _vp])

MAX_TOP = 1024  # targets of a row that fit the kernels' table
# Rows worked off at a time: their exponentials (2 bytes per row and vocabulary entry) are the one large buffer.
CHUNK_BYTES = int(os.environ.get("PDT_VOCAB_CHUNK_MB", "8192")) << 20


class _Targets:
    """Weights of the rows' targets, and the two factors (tau, tau^2 over the rows that have one)."""

    def __init__(self, ids, teacher, vocab: int, tau: float, x=None, w=None, x_used=None):
        n, top = ids.shape
        dev = ids.device
        self.ids, self.tau = ids, tau
        self.p = torch.empty((n, top), dtype=torch.float32, device=dev) if teacher is not None else None
        self.base = torch.empty(n, dtype=torch.float32, device=dev)
        self.valid = torch.empty(n, dtype=torch.int32, device=dev)
        self.scal = torch.empty(2, dtype=torch.float32, device=dev)
        _check(_targets(ids.data_ptr(), _ptr(teacher), _ptr(self.p), self.base.data_ptr(), self.valid.data_ptr(), self.scal.data_ptr(), _ptr(x),
                        _ptr(w), _ptr(x_used), n, top, 0 if x is None else x.shape[1], vocab, tau, _stream()), "vocab_targets")

    def mean(self, row_loss):
        loss = torch.empty((), dtype=torch.float32, device=row_loss.device)
        _check(_mean(row_loss.data_ptr(), self.scal.data_ptr(), loss.data_ptr(), row_loss.numel(), _stream()), "vocab_mean")
        return loss


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


class _HeadLoss(torch.autograd.Function):
    """Loss of ``x W^T`` against a few targets per row.  The rows are worked off in chunks; the forward pass leaves ``dx``
    and ``dW`` for an incoming gradient of 1, the backward pass multiplies them by the incoming one (a device scalar)."""

    @staticmethod
    def forward(ctx, x, weight, ids, teacher, tau: float):
        vocab, width = weight.shape
        want_dx, want_dw = ctx.needs_input_grad[0], ctx.needs_input_grad[1]
        with torch.cuda.device(x.device):
            x2, w = _matrix(x, width), _weight(weight)
            n, dev, top = x2.shape[0], x.device, ids.shape[1]
            x_used = torch.empty((_round_up(n, 64), width), dtype=torch.bfloat16, device=dev) if want_dw else None
            t = _Targets(ids, teacher, vocab, tau, x2, w, x_used)
            train = want_dx or want_dw
            pitch, groups = _round_up(vocab, 64), -(-vocab // 64)
            rows_c = n if not train else max(1, min(n, CHUNK_BYTES // (2 * pitch)))
            if rows_c < n:
                rows_c = max(256, rows_c - rows_c % 256)
            stats = torch.empty((rows_c, groups, 2), dtype=torch.float32, device=dev)
            e = torch.empty((_round_up(rows_c, 64), pitch), dtype=torch.bfloat16, device=dev) if train else None
            row_loss = torch.empty(n, dtype=torch.float32, device=dev)
            dx = torch.empty((n, width), dtype=torch.bfloat16, device=dev) if want_dx else None
            # one chunk and a bf16 weight: the gradient is rounded once, in the product's epilogue; else it is summed in fp32
            direct = want_dw and rows_c == n and weight.dtype == torch.bfloat16
            dw = torch.empty((vocab, width), dtype=torch.bfloat16 if direct else torch.float32, device=dev) if want_dw else None
            chunks = {rows_c, n % rows_c or rows_c}
            need = max(_part_floats(which, rows, vocab, width) for rows in chunks for which in (1, 2)) if train else 0
            part = torch.empty(need, dtype=torch.float32, device=dev) if need > 0 else None
            for r0 in range(0, n, rows_c):
                rows = min(rows_c, n - r0)
                xc, idc = x2[r0:r0 + rows], ids[r0:r0 + rows]
                _check(_scores(xc.data_ptr(), w.data_ptr(), stats.data_ptr(), _ptr(e), rows, vocab, width, pitch, 1.0 / tau, _stream()),
                       "vocab_scores")
                _check(_rows(stats.data_ptr(), _ptr(e), idc.data_ptr(), None if t.p is None else t.p[r0:].data_ptr(), t.base[r0:].data_ptr(),
                             t.valid[r0:].data_ptr(), row_loss[r0:].data_ptr(), rows, vocab, top, pitch, _stream()), "vocab_rows")
                if want_dx:
                    _check(_dx(e.data_ptr(), w.data_ptr(), dx[r0:].data_ptr(), _ptr(part), t.scal.data_ptr(), rows, vocab, width, pitch,
                               _stream()), "vocab_dx")
                if want_dw:
                    _check(_dw(e.data_ptr(), x_used[r0:].data_ptr(), dw.data_ptr() if direct else None, None if direct else dw.data_ptr(), int(r0 > 0),
                               _ptr(part), t.scal.data_ptr(), rows, vocab, width, pitch, _stream()), "vocab_dw")
            loss = t.mean(row_loss)
        ctx.grads = [dx, dw]
        ctx.weight, ctx.shape = weight, x.shape
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g):
        dx, dw = ctx.grads
        ctx.grads = [None, None]
        if dx is None and dw is None:
            raise RuntimeError("the loss behind a projection handed its gradients out already (backward ran twice)")
        weight = ctx.weight
        with torch.cuda.device(g.device):
            g1 = g.reshape(1).to(torch.float32).contiguous()
            for d in (dx, dw):
                if d is not None and d.dtype == torch.bfloat16:
                    _check(_scale_by_scalar(d.data_ptr(), g1.data_ptr(), d.numel(), _stream()), "scale_by_scalar")
            if dw is not None and dw.dtype == torch.float32:
                sink = _grad_sink(weight, tuple(weight.shape))
                if sink is not None:
                    _check(_axpy_dev(sink.data_ptr(), dw.data_ptr(), g1.data_ptr(), dw.numel(), _stream()), "axpy")
                    dw = None
                else:
                    dw = (dw * g1).to(weight.dtype)
        return None if dx is None else dx.view(ctx.shape), dw, None, None, None


def head_loss(x, weight, ids, teacher, tau: float):
    return _HeadLoss.apply(x, weight, ids, teacher, tau)


class _LogitsDistill(torch.autograd.Function):
    """The forward pass leaves the gradient for an incoming one of 1 (the logits are read once), as the cross-entropy does."""

    @staticmethod
    def forward(ctx, logits, ids, teacher, tau: float):
        vocab = logits.shape[-1]
        with torch.cuda.device(logits.device):
            z = logits.reshape(-1, vocab)
            if z.dtype not in (torch.bfloat16, torch.float32):
                z = z.to(torch.float32)
            if z.stride(1) != 1 and vocab > 1:
                z = z.contiguous()
            n, top = ids.shape
            t = _Targets(ids, teacher, vocab, tau)
            row_loss = torch.empty(n, dtype=torch.float32, device=z.device)
            dz = None
            if ctx.needs_input_grad[0]:
                dz = torch.empty((n, _round_up(vocab, 64)), dtype=z.dtype, device=z.device)
            _check(_distill(z.data_ptr(), _ptr(dz), ids.data_ptr(), t.p.data_ptr(), t.base.data_ptr(), t.valid.data_ptr(), t.scal.data_ptr(),
                            row_loss.data_ptr(), n, vocab, top, z.stride(0), 0 if dz is None else dz.stride(0), 1.0 / tau,
                            int(z.dtype == torch.bfloat16), _stream()), "logits_distill")
            loss = t.mean(row_loss)
        ctx.dz, ctx.shape = dz, logits.shape
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g):
        dz, ctx.dz = ctx.dz, None
        if dz is None:
            raise RuntimeError("the distillation loss handed its gradient out already (backward ran twice)")
        with torch.cuda.device(g.device):
            g1 = g.reshape(1).to(torch.float32).contiguous()
            if dz.dtype == torch.bfloat16:
                _check(_scale_by_scalar(dz.data_ptr(), g1.data_ptr(), dz.numel(), _stream()), "scale_by_scalar")
            else:
                dz.mul_(g1)
        return dz[:, :ctx.shape[-1]].reshape(ctx.shape), None, None, None


def logits_distill(logits, ids, teacher, tau: float):
    return _LogitsDistill.apply(logits, ids, teacher, tau)
