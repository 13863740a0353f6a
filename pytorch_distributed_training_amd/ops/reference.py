"""Plain PyTorch implementations of every fused op.

They define the semantics: the HIP kernels are tested against them, and they are what runs
for CPU tensors (the gloo plumbing configuration and unit tests).  They are ordinary
differentiable compositions, so autograd provides their backward passes.
"""

from __future__ import annotations

import math
from typing import Optional, Tuple

import torch
import torch.nn as nn
import torch.nn.functional as F
from torch.autograd import forward_ad


def any_tangent(*xs: torch.Tensor) -> bool:
    """Whether a forward-mode derivative is carried by one of these (outside every dual level, nearly always, none is looked at:
    half a microsecond each)."""
    return getattr(forward_ad, "_current_level", 0) >= 0 and any(forward_ad.unpack_dual(x).tangent is not None for x in xs)


def batch_norm(y: torch.Tensor, bn: nn.BatchNorm2d) -> torch.Tensor:
    """Training-mode batch statistics (and running-stat update) or eval-mode running statistics."""
    if bn.training and bn.track_running_stats and bn.num_batches_tracked is not None:
        bn.num_batches_tracked.add_(1)
    use_batch = bn.training or not bn.track_running_stats
    return F.batch_norm(
        y,
        bn.running_mean if bn.track_running_stats else None,
        bn.running_var if bn.track_running_stats else None,
        bn.weight,
        bn.bias,
        use_batch,
        bn.momentum if bn.momentum is not None else 0.1,
        bn.eps,
    )


def conv2d_stats(x, weight, stride: int = 1, padding: int = 0, want_stats: bool = True, link=None, link_out=None):
    return F.conv2d(x, weight, None, stride, padding), None


def bn_act(y, stats, bn, relu: bool = True):
    z = batch_norm(y, bn)
    return F.relu(z) if relu else z


def bn_relu_conv2d(y_prev, stats_prev, bn, weight, stride: int = 1, padding: int = 0):
    return F.conv2d(F.relu(batch_norm(y_prev, bn)), weight, None, stride, padding), None


def bn_add_relu(y, stats, bn, identity, id_stats=None, id_bn=None, link=None):
    z = batch_norm(y, bn)
    if id_bn is not None:
        identity = batch_norm(identity, id_bn)
    return F.relu(z + identity)


def bn_relu_maxpool(y, stats, bn):
    return F.max_pool2d(F.relu(batch_norm(y, bn)), kernel_size=3, stride=2, padding=1)


def global_avgpool(a: torch.Tensor) -> torch.Tensor:
    return a.mean(dim=(2, 3))


def linear(x, weight, bias=None, activation: Optional[str] = None, residual=None, link=None):
    out = F.linear(x, weight, bias)
    if residual is not None:
        out = out + residual
    if activation == "gelu":
        out = F.gelu(out, approximate="tanh")
    elif activation is not None:
        raise ValueError("activation must be None or 'gelu'")
    return out


def softmax_cross_entropy(logits: torch.Tensor, labels: torch.Tensor) -> torch.Tensor:
    """Mean softmax cross-entropy over the rows with a label (not -100), 0 without any (role of ``nn.CrossEntropyLoss()`` at
    /root/reference/src/main.py:62,76)."""
    y = labels.reshape(-1)
    none = not y.is_cuda and not bool((y != -100).any())  # (not asked of the GPU, which would have to be waited for: NaN there)
    return F.cross_entropy(logits.float().reshape(-1, logits.shape[-1]), y, reduction="sum" if none else "mean")


def without_others(labels, vocab: int):
    """Labels outside the vocabulary as -100."""
    y = labels.reshape(-1).to(torch.int64)
    return torch.where((y >= 0) & (y < vocab), y, torch.full_like(y, -100))


def linear_cross_entropy(x, weight, labels):
    """Mean cross-entropy of ``x W^T`` over the rows whose label lies in the vocabulary; 0 without any."""
    up = torch.promote_types(x.dtype, torch.float32)
    z = F.linear(x.reshape(-1, x.shape[-1]).to(up), weight.to(up))
    y = without_others(labels, weight.shape[0])
    return F.cross_entropy(z, y, ignore_index=-100, reduction="sum") / (y >= 0).sum().clamp(min=1)


def distillation_loss(logits, teacher_logits, teacher_ids, temperature: float):
    """``tau^2 sum_k p_k (log p_k - log q[id_k])``, mean over the rows with a present entry; 0 without any."""
    up = torch.promote_types(logits.dtype, torch.float32)
    vocab, top = logits.shape[-1], teacher_ids.shape[-1]
    ids = teacher_ids.reshape(-1, top).to(torch.int64)
    t = teacher_logits.reshape(-1, top).to(up)
    t = t.masked_fill((ids < 0) | (ids >= vocab), float("-inf"))
    some = (t != float("-inf")).any(1)
    logp = torch.log_softmax((t - t.amax(1, keepdim=True)).masked_fill(~some[:, None], 0.0) / temperature, 1)
    logq = torch.log_softmax(logits.reshape(-1, vocab).to(up) / temperature, 1).gather(1, ids.clamp(0, vocab - 1))
    p = logp.exp()
    each = torch.where((p != 0) & some[:, None], p * (torch.where(p != 0, logp, 0.0) - torch.where(p != 0, logq, 0.0)), 0.0)
    return temperature ** 2 * each.sum() / some.sum().clamp(min=1)


def layer_norm(x, weight, bias, eps: float = 1e-5, link=None):
    return F.layer_norm(x, (x.shape[-1],), weight, bias, eps)


def gelu(x):
    return F.gelu(x, approximate="tanh")


def attention(q, k, v, causal: bool = False, scale: Optional[float] = None):
    """softmax(q k^T * scale [+ causal mask]) v for [B, H, S, D] tensors."""
    d = q.shape[-1]
    scale = scale if scale is not None else 1.0 / math.sqrt(d)
    s = torch.matmul(q.float(), k.float().transpose(-1, -2)) * scale
    if causal:
        sq, sk = s.shape[-2], s.shape[-1]
        mask = torch.ones(sq, sk, dtype=torch.bool, device=s.device).tril(sk - sq)
        s = s.masked_fill(~mask, float("-inf"))
    p = torch.softmax(s, dim=-1)
    return torch.matmul(p, v.float()).to(q.dtype)


def attention_qkv(qkv, heads: int, causal: bool = False):
    """Multi-head self-attention on the packed projection output ``[B, S, 3*H*Dh]`` -> ``[B, S, H*Dh]``."""
    b, s, three_d = qkv.shape
    d = three_d // 3
    dh = d // heads
    x = qkv.view(b, s, 3, heads, dh)
    q, k, v = (x[:, :, i].transpose(1, 2) for i in range(3))
    return attention(q, k, v, causal).transpose(1, 2).reshape(b, s, d)


def attention_packed(q, k, v, spans, causal: bool, scale: float):
    """Attention inside the sequences given by ``spans`` (``[T, 2]``, first row and end of each row's sequence); heads of
    ``k`` / ``v`` are shared by equal groups of heads of ``q``.  Rows outside every sequence give zeros."""
    group = q.shape[1] // k.shape[1]
    out = q.new_zeros(q.shape) + 0.0 * q[:0].sum()  # (differentiable also where there is no sequence at all)
    parts, end = [], 0
    for first, stop in torch.unique(spans, dim=0).tolist():
        if stop > first:
            qs, ks, vs = (x[first:stop].transpose(0, 1) for x in (q, k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)))
            up = torch.promote_types(q.dtype, torch.float32)
            s = (qs.to(up) @ ks.to(up).transpose(1, 2)) * scale
            if causal:
                s = s.masked_fill(torch.ones(s.shape[1:], dtype=torch.bool, device=s.device).triu(1), float("-inf"))
            parts += [out[end:first], (torch.softmax(s, dim=-1) @ vs.to(up)).transpose(0, 1).to(q.dtype)]
            end = stop
    return torch.cat(parts + [out[end:]])


def embedding(ids, weight):
    return F.embedding(ids, weight)


def token_position_embedding(ids, wte, wpe):
    """``wte[ids] + wpe[0..S)`` for ``ids`` of shape ``[B, S]``."""
    s_ = ids.shape[1]
    return F.embedding(ids, wte) + wpe[:s_].unsqueeze(0)


def packed_embedding(ids, positions, wte, wpe):
    return F.embedding(ids, wte) + F.embedding(positions, wpe)


def vit_assemble(tok, cls, pos):
    """``cat([cls, tok], dim=1) + pos``: class token in front of the patch tokens, position table added."""
    b = tok.shape[0]
    return torch.cat([cls.to(tok.dtype).expand(b, -1, -1), tok], dim=1) + pos.to(tok.dtype)


def add_bias_residual(x, bias, residual):
    out = x
    if bias is not None:
        out = out + bias
    if residual is not None:
        out = out + residual
    return out
