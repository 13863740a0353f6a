"""GPU attention over packed sequences with grouped heads (``csrc/kernels/attention_packed.hip``).

Not exercised by the reference (its model is a CNN, /root/reference/src/main.py:49).
"""

from __future__ import annotations

import ctypes

import torch

from .hip import _check, _derivative_wanted, _on, _once_differentiable, _ptr, _stream
from .hip_transformer import _f, _i, _sig, _vp

_pack_spans = _sig("pdt_pack_spans", [_vp, _i, _i] + [_vp] * 5)
_fwd = _sig("pdt_packed_attention_fwd", [_vp] * 9 + [_i] * 4 + [_f, _i, _vp])
_bwd = _sig("pdt_packed_attention_bwd", [_vp] * 12 + [_i, _vp, _vp, _vp] + [_i] * 4 + [_f, _i, _vp])
_splits = _sig("pdt_packed_attention_splits", [_i] * 3)

HEAD_DIMS = (64, 128)
BLOCK_ROWS = 128  # rows of a workgroup


def pack_plan(offsets, rows: int):
    """One int64 buffer: ``rows`` positions, ``rows`` spans (two int32), three orders of the blocks (four int32 each) and as much scratch."""
    with _on(offsets.device):
        if offsets.dtype == torch.int64:
            offsets = offsets.clamp(-1, rows)  # (what lies beyond is cut off, and must not wrap around in 32 bits)
        offsets = offsets.to(torch.int32).contiguous()
        blocks = -(-rows // BLOCK_ROWS)
        plan = torch.empty(2 * rows + 12 * blocks, dtype=torch.int64, device=offsets.device)
        if rows:
            at = plan.data_ptr()
            order = at + 16 * rows
            _check(_pack_spans(offsets.data_ptr(), offsets.numel() - 1, rows, at + 8 * rows, at, order, order + 48 * blocks, _stream()), "pack_spans")
    return plan


def _heads(x: torch.Tensor) -> torch.Tensor:
    """[T, heads, D] in bf16 with unit stride along D and rows and heads on 16-byte boundaries (a view where it is one already)."""
    if x.dtype != torch.bfloat16:
        x = x.to(torch.bfloat16)
    rows, heads, one = x.stride()
    if one != 1 or rows % 8 or heads % 8 or not 0 < rows < 1 << 24 or heads <= 0 or x.data_ptr() % 16:
        x = x.clone(memory_format=torch.contiguous_format)
    return x


def _strides(*xs):
    vals = [s for x in xs for s in x.stride()[:2]]
    return (ctypes.c_longlong * len(vals))(*vals)


def _forward(q, k, v, plan, causal: bool, scale: float, train: bool):
    """(out, what the backward pass needs beside it: a byte per element of out, what its rounding took, then the fp32 row
    terms ``[h, t]``; without a backward pass the row terms alone)."""
    t, h, d = q.shape
    out = torch.empty((t, h, d), dtype=torch.bfloat16, device=q.device)
    aside = torch.empty(t * h * (1 + d // 4 if train else 1), dtype=torch.float32, device=q.device)
    if out.numel():
        rest = aside.data_ptr() if train else None
        lse = aside.data_ptr() + (t * h * d if train else 0)
        _check(_fwd(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), rest, lse, plan.data_ptr() + 8 * t,
                    plan.data_ptr() + 16 * t, _strides(q, k, v), t, h, k.shape[1], d, scale, int(causal), _stream()), "packed_attention_fwd")
    return out, aside


def _backward(q, k, v, out, aside, g, plan, causal: bool, scale: float, dq, dk, dv) -> None:
    t, h, d = q.shape
    hk = k.shape[1]
    if t == 0:
        return
    if g.dtype != torch.bfloat16:
        g = g.to(torch.bfloat16)
    if not g.is_contiguous() or g.data_ptr() % 16:
        g = g.clone(memory_format=torch.contiguous_format)
    delta = torch.empty((h, t), dtype=torch.float32, device=q.device)
    splits = _splits(t, h, hk)
    part = torch.empty((splits, 2, t, hk, d), dtype=torch.float32, device=q.device) if splits > 1 else None
    _check(_bwd(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), aside.data_ptr(), g.data_ptr(), aside.data_ptr() + t * h * d, delta.data_ptr(),
                dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), _ptr(part), splits, plan.data_ptr() + 8 * t, plan.data_ptr() + 16 * t, _strides(q, k, v, dq, dk, dv), t, h, hk, d, scale,
                int(causal), _stream()), "packed_attention_bwd")


class _AttentionPacked(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, plan, causal: bool, scale: float):
        with _on(q.device):
            q, k, v = _heads(q), _heads(k), _heads(v)
            out, aside = _forward(q, k, v, plan, causal, scale, any(ctx.needs_input_grad[:3]))
        ctx.save_for_backward(q, k, v, out, aside, plan)
        ctx.meta = (causal, scale)
        return out

    @staticmethod
    @_once_differentiable
    def backward(ctx, g):
        q, k, v, out, aside, plan = ctx.saved_tensors
        with _on(q.device):
            dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
            _backward(q, k, v, out, aside, g, plan, *ctx.meta, dq, dk, dv)
        return dq, dk, dv, None, None, None


def _split_qkv(qkv, heads: int, kv_heads: int):
    t, width = qkv.shape
    d = width // (heads + 2 * kv_heads)
    x = qkv.view(t, heads + 2 * kv_heads, d)
    return x[:, :heads], x[:, heads:heads + kv_heads], x[:, heads + kv_heads:]


class _AttentionPackedQKV(torch.autograd.Function):
    """On the projection's output, whose gradient is written as one tensor (no split in forward, no concatenation behind)."""

    @staticmethod
    def forward(ctx, qkv, heads: int, kv_heads: int, plan, causal: bool, scale: float):
        with _on(qkv.device):
            if qkv.dtype != torch.bfloat16:
                qkv = qkv.to(torch.bfloat16)
            if not qkv.is_contiguous() or qkv.data_ptr() % 16:
                qkv = qkv.clone(memory_format=torch.contiguous_format)
            out, aside = _forward(*_split_qkv(qkv, heads, kv_heads), plan, causal, scale, ctx.needs_input_grad[0])
        ctx.save_for_backward(qkv, out, aside, plan)
        ctx.meta = (heads, kv_heads, causal, scale)
        return out.flatten(1)

    @staticmethod
    @_once_differentiable
    def backward(ctx, g):
        qkv, out, aside, plan = ctx.saved_tensors
        heads, kv_heads, causal, scale = ctx.meta
        with _on(qkv.device):
            dqkv = torch.empty_like(qkv)
            _backward(*_split_qkv(qkv, heads, kv_heads), out, aside, g.reshape(out.shape), plan, causal, scale,
                      *_split_qkv(dqkv, heads, kv_heads))
        return dqkv, None, None, None, None, None


def _check_head_dim(d: int) -> None:
    if d not in HEAD_DIMS:
        raise ValueError(f"the packed attention kernels need a head_dim of 64 or 128, got {d}")


def attention_packed(q, k, v, pack, causal: bool, scale: float):
    _check_head_dim(q.shape[2])
    if not _derivative_wanted(q, k, v):
        with _on(q.device):
            return _forward(_heads(q), _heads(k), _heads(v), pack.plan, causal, scale, False)[0]
    return _AttentionPacked.apply(q, k, v, pack.plan, bool(causal), scale)


def attention_packed_qkv(qkv, pack, heads: int, kv_heads: int, causal: bool, scale: float):
    _check_head_dim(qkv.shape[1] // (heads + 2 * kv_heads))
    return _AttentionPackedQKV.apply(qkv, heads, kv_heads, pack.plan, bool(causal), scale)
