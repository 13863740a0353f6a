"""Fused operators.

Every op has exactly one GPU implementation - a hand-written gfx950 HIP kernel wrapped in
an ``autograd.Function`` (``ops.hip``) - and a plain PyTorch definition (``ops.reference``)
that states its semantics, runs for CPU tensors and is the oracle in numerics tests.
Dispatch is by device only: a GPU tensor never takes the PyTorch composition, and a missing
kernel library is an error, not a fallback.
"""

from __future__ import annotations

import math
from typing import Optional

import torch

from . import reference as _ref
from .packing import SequencePack, pack_sequences  # noqa: F401


import os as _os

# 0: projection and loss as two operators with full-batch logits (A/B measurements; caps the batch at 42 x 1024 tokens)
_LM_HEAD_FUSED = _os.environ.get("PDT_LM_HEAD_FUSED", "1") != "0"


def _hip():
    from . import hip  # imported lazily: loading it maps the kernel library

    return hip


def residual_link(x):
    """Token shared by the first convolution of a residual block and the other consumer of the block input
    ``x`` (the block tail, or the projection convolution of a down-sampling block): on GPU it lets the
    shortcut's gradient be added inside the first convolution's data-gradient kernel instead of in a separate
    pass.  ``None`` (no effect) for CPU tensors."""
    return _hip().residual_link() if x.is_cuda else None


def conv2d_stats(x, weight, stride: int = 1, padding: int = 0, want_stats: bool = True, link=None, link_out=None):
    """Convolution without bias.  Returns ``(y, stats)`` where ``stats`` carries the per-channel
    batch statistics of ``y`` gathered in the kernel epilogue (``None`` on CPU or when not wanted,
    e.g. in inference where BatchNorm uses its running statistics).

    ``link`` / ``link_out`` (see :func:`residual_link`): with ``link`` this convolution's data-gradient kernel
    adds whatever gradient the link carries; with ``link_out`` this convolution hands its input gradient to the
    link instead of returning it to autograd."""
    if x.is_cuda:
        return _hip().conv2d_stats(x, weight, stride, padding, want_stats, link, link_out)
    return _ref.conv2d_stats(x, weight, stride, padding)


def bn_act(y, stats, bn, relu: bool = True):
    """BatchNorm (+ReLU) of a raw convolution output."""
    if y.is_cuda:
        return _hip().bn_act(y, stats, bn, relu)
    return _ref.bn_act(y, stats, bn, relu)


def bn_relu_conv2d(y_prev, stats_prev, bn, weight, stride: int = 1, padding: int = 0):
    """conv(relu(bn(y_prev))) from a raw convolution output and its batch statistics.  On GPU the normalisation is
    applied inside the convolution's kernels for 1x1 consumers with at most 128 input channels (no normalised
    activation is written) and as one streaming pass in front of the convolution otherwise (``ops.hip.FUSE_BN_INTO_1X1``)."""
    if y_prev.is_cuda:
        return _hip().bn_relu_conv2d(y_prev, stats_prev, bn, weight, stride, padding)
    return _ref.bn_relu_conv2d(y_prev, stats_prev, bn, weight, stride, padding)


def bn_add_relu(y, stats, bn, identity, id_stats=None, id_bn=None, link=None):
    """relu(bn(y) + identity), or relu(bn(y) + id_bn(identity)) for a projected shortcut."""
    if y.is_cuda:
        return _hip().bn_add_relu(y, stats, bn, identity, id_stats, id_bn, link)
    return _ref.bn_add_relu(y, stats, bn, identity, id_stats, id_bn)


def bn_relu_maxpool(y, stats, bn):
    """Stem tail: maxpool3x3/2(relu(bn(y)))."""
    if y.is_cuda:
        return _hip().bn_relu_maxpool(y, stats, bn)
    return _ref.bn_relu_maxpool(y, stats, bn)


def global_avgpool(a):
    if a.is_cuda:
        return _hip().global_avgpool(a)
    return _ref.global_avgpool(a)


def skip_link(x):
    """Token shared by the LayerNorm at the head of a pre-norm residual branch and the linear layer that closes
    the branch with ``residual=x``: ``linear(f(layer_norm(x, ..., link=L)), ..., residual=x, link=L)``.  On GPU
    the skip connection's gradient is then added inside the LayerNorm backward kernel instead of by a separate
    element-wise pass.  Both ops must see the same ``x``.  ``None`` (no effect) for CPU tensors."""
    return _hip().skip_link() if x.is_cuda else None


def linear(x, weight, bias=None, activation: Optional[str] = None, residual=None, link=None):
    """act(x W^T + bias) or x W^T + bias + residual (the residual is added in the GEMM epilogue on GPU).
    ``link``: see :func:`skip_link`."""
    if x.is_cuda:
        return _hip().linear(x, weight, bias, activation, residual, link)
    return _ref.linear(x, weight, bias, activation, residual)


def gelu_mlp(x, w1, b1, w2, b2, residual=None, link=None):
    """gelu(x W1^T + b1) W2^T + b2 (+ residual): the transformer feed-forward block.  On GPU every element-wise
    step (bias, GELU, residual, GELU's derivative, bias gradients) runs inside a GEMM epilogue."""
    if x.is_cuda and b1 is not None and b2 is not None and not (w1.shape[0] % 64 or w1.shape[1] % 64 or w2.shape[0] % 64):
        return _hip().gelu_mlp(x, w1, b1, w2, b2, residual, link)
    return linear(linear(x, w1, b1, activation="gelu"), w2, b2, residual=residual, link=link)


def softmax_cross_entropy(logits, labels):
    """Mean cross-entropy over the rows that have a label: -100 leaves its row out, without gradient and not counted (on GPU
    every label that is none of the classes does; on CPU the others are an error).  0 where no row has one."""
    if logits.is_cuda:
        return _hip().softmax_cross_entropy(logits, labels)
    return _ref.softmax_cross_entropy(logits, labels)


def lm_head_loss(x, weight, labels):
    """Mean cross-entropy of the logits ``x W^T`` (no bias) against ``labels``: a language model's tied output
    projection and loss, over the rows whose label lies in the vocabulary (0 without any).  On GPU the rows are processed
    in chunks through one scratch buffer, so the ``[rows, vocabulary]`` logits of the whole batch never exist (see
    ``ops.hip._LMHeadLoss``)."""
    if x.is_cuda and 1024 < weight.shape[0] <= 65536 and _LM_HEAD_FUSED:
        return _hip().lm_head_loss(x, weight, labels)
    logits = linear(x, weight, None)
    if not x.is_cuda:
        labels = _ref.without_others(labels, weight.shape[0])
    return softmax_cross_entropy(logits.reshape(-1, logits.shape[-1]), labels.reshape(-1))


MAX_TEACHER_TOP = 1024  # teacher logits of a row that the distillation losses take


def _check_head(x, weight, what: str) -> None:
    if x.dim() < 1 or weight.dim() != 2 or x.shape[-1] != weight.shape[1]:
        raise ValueError(f"{what}: expected [..., width] and [vocabulary, width], got {tuple(x.shape)} and {tuple(weight.shape)}")
    if not x.is_floating_point() or not weight.is_floating_point():
        raise TypeError(f"{what} takes floating-point tensors")
    if x.device != weight.device:
        raise ValueError(f"{what}: x on {x.device}, weight on {weight.device}")
    if x.is_cuda and weight.shape[1] % 64:
        raise ValueError("in_features must be a multiple of 64")
    if weight.numel() == 0 or weight.shape[0] >= 1 << 22:
        raise ValueError(f"{what}: a vocabulary of 1 to 2^22 - 1 entries, got {weight.shape[0]}")


def _check_targets(lead, ids, device, what: str, name: str) -> None:
    if ids.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"{what}: {name} must be int64 or int32")
    if tuple(ids.shape) != tuple(lead):
        raise ValueError(f"{what}: {name} of shape {tuple(lead)} expected, got {tuple(ids.shape)}")
    if ids.device != device:
        raise ValueError(f"{what}: {name} on {ids.device}, expected on {device}")


def _check_teacher(lead, teacher_logits, teacher_ids, temperature: float, device, what: str) -> float:
    if teacher_ids.dim() != len(lead) + 1:
        raise ValueError(f"{what}: teacher ids of shape {tuple(lead) + ('K',)} expected, got {tuple(teacher_ids.shape)}")
    top = teacher_ids.shape[-1]
    if not 1 <= top <= MAX_TEACHER_TOP:
        raise ValueError(f"{what}: 1 to {MAX_TEACHER_TOP} teacher logits per row, got {top}")
    _check_targets(tuple(lead) + (top,), teacher_ids, device, what, "teacher ids")
    if teacher_logits.shape != teacher_ids.shape or teacher_logits.device != device or not teacher_logits.is_floating_point():
        raise ValueError(f"{what}: teacher logits must be floating-point, of the ids' shape and device")
    if teacher_logits.requires_grad or _ref.any_tangent(teacher_logits):
        raise ValueError(f"{what}: no gradient flows to the teacher; pass its logits detached")
    temperature = float(temperature)
    if not 1e-6 <= temperature <= 1e6:  # (its square and its inverse are fp32 factors)
        raise ValueError(f"a temperature between 1e-6 and 1e6, got {temperature}")
    return temperature


def linear_cross_entropy(x, weight, labels):
    """Mean cross-entropy of the logits ``x W^T`` (``x`` ``[..., width]``, ``weight`` ``[vocabulary, width]``, no bias)
    against ``labels`` ``[...]``, over the rows that have a label: a label outside ``[0, vocabulary)`` (-100, say) leaves
    its row out, without gradient and not counted.  0 where no row has one.  On GPU the vocabulary (below 2^22 entries) is
    worked off in tiles; matrix products take bf16, loss and sums are fp32.  With a gradient one buffer of rows x vocabulary in
    bf16 is held, of ``PDT_VOCAB_CHUNK_MB`` (8192) MB at most: beyond, rows are worked off in pieces; without one, an eighth of
    a byte per entry."""
    _check_head(x, weight, "linear_cross_entropy")
    _check_targets(x.shape[:-1], labels, x.device, "linear_cross_entropy", "labels")
    if x.is_cuda and labels.numel():
        from . import hip_vocab

        return hip_vocab.head_loss(x, weight, _rows(labels, 1, torch.int64), None, 1.0)
    return _ref.linear_cross_entropy(x, weight, labels)


def distillation_loss(logits, teacher_logits, teacher_ids, temperature: float = 1.0):
    """``tau^2 KL(p || q)``, mean over rows, of a student's ``q = softmax(logits / tau)`` (``[..., vocabulary]``) from a
    teacher's top logits: ``p = softmax(teacher_logits / tau)`` over its ``K`` entries ``[..., K]`` at ``teacher_ids``.
    Entries with an id outside the vocabulary are absent; a row without any (or with -inf alone) is left out, without
    gradient and not counted.  An id that occurs twice in a row counts with both its entries."""
    if logits.dim() < 1 or not logits.is_floating_point() or not 1 <= logits.shape[-1] < 1 << 24:
        raise ValueError("distillation_loss: logits are a floating-point tensor [..., vocabulary] of 1 to 2^24 - 1 entries")
    tau = _check_teacher(logits.shape[:-1], teacher_logits, teacher_ids, temperature, logits.device, "distillation_loss")
    if logits.is_cuda and logits.numel():
        from . import hip_vocab

        return hip_vocab.logits_distill(logits, *_teacher_rows(teacher_logits, teacher_ids), tau)
    return _ref.distillation_loss(logits, teacher_logits, teacher_ids, tau)


def linear_distillation_loss(x, weight, teacher_logits, teacher_ids, temperature: float = 1.0):
    """:func:`distillation_loss` of the logits ``x W^T``, on GPU without storing them (see :func:`linear_cross_entropy`)."""
    _check_head(x, weight, "linear_distillation_loss")
    tau = _check_teacher(x.shape[:-1], teacher_logits, teacher_ids, temperature, x.device, "linear_distillation_loss")
    if x.is_cuda and teacher_ids.numel():
        from . import hip_vocab

        return hip_vocab.head_loss(x, weight, *_teacher_rows(teacher_logits, teacher_ids), tau)
    up = torch.promote_types(x.dtype, torch.float32)
    return _ref.distillation_loss(_ref.linear(x.to(up), weight.to(up)), teacher_logits, teacher_ids, tau)


def _rows(x, width: int, dtype):
    """[rows, width] in ``dtype`` without gaps; the tensor itself where it is that (host time counts in small calls)."""
    if x.dim() != 2 or x.shape[1] != width:
        x = x.reshape(-1, width)
    if x.dtype != dtype:
        x = x.to(dtype)
    return x if x.is_contiguous() else x.contiguous()


def _teacher_rows(teacher_logits, teacher_ids):
    top = teacher_ids.shape[-1]
    return _rows(teacher_ids, top, torch.int64), _rows(teacher_logits, top, torch.float32)


def layer_norm(x, weight, bias, eps: float = 1e-5, link=None):
    if x.is_cuda:
        return _hip().layer_norm(x, weight, bias, eps, link)
    return _ref.layer_norm(x, weight, bias, eps)


def gelu(x):
    if x.is_cuda:
        return _hip().gelu(x)
    return _ref.gelu(x)


def attention(q, k, v, causal: bool = False, scale: Optional[float] = None):
    if q.is_cuda:
        return _hip().attention(q, k, v, causal, scale)
    return _ref.attention(q, k, v, causal, scale)


def attention_qkv(qkv, heads: int, causal: bool = False):
    """Self-attention on the packed QKV projection ``[B, S, 3*H*Dh]`` -> ``[B, S, H*Dh]``."""
    if qkv.is_cuda:
        return _hip().attention_qkv(qkv, heads, causal)
    return _ref.attention_qkv(qkv, heads, causal)


def _check_packed(x, pack, name: str) -> None:
    if not isinstance(pack, SequencePack):
        raise TypeError("pack: a SequencePack, made by ops.pack_sequences")
    if x.device != pack.device:
        raise ValueError(f"{name} on {x.device}, pack on {pack.device}")
    if x.shape[0] != pack.rows:
        raise ValueError(f"{name} has {x.shape[0]} rows, the pack {pack.rows}")
    if not x.is_floating_point():
        raise TypeError(f"{name} must be a floating-point tensor")


def _check_scale(scale: Optional[float], head_dim: int) -> float:
    scale = 1.0 / math.sqrt(head_dim) if scale is None else float(scale)
    if not 1e-30 <= scale <= 1e30:  # (an fp32 factor)
        raise ValueError(f"a softmax scale between 1e-30 and 1e30, got {scale}")
    return scale


def attention_packed(q, k, v, pack: SequencePack, causal: bool = True, scale: Optional[float] = None):
    """Attention inside every sequence of a pack, with grouped heads: ``q`` ``[T, H, D]``, ``k`` and ``v`` ``[T, Hk, D]`` ->
    ``[T, H, D]``, query head ``h`` reading head ``h // (H // Hk)``.  A row attends to the rows of its own sequence, up to
    itself if ``causal``; rows outside every sequence give 0 and get no gradient.  ``scale`` defaults to ``1 / sqrt(D)``.
    On GPU: ``D`` of 64 or 128, computed in bf16 (fp32 softmax), any strides with a contiguous last axis."""
    if q.dim() != 3 or k.dim() != 3 or k.shape != v.shape or q.shape[0] != k.shape[0] or q.shape[2] != k.shape[2] or q.shape[2] == 0:
        raise ValueError(f"expected [T, H, D], [T, Hk, D], [T, Hk, D], got {tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}")
    if k.shape[1] == 0 or q.shape[1] == 0 or q.shape[1] % k.shape[1]:
        raise ValueError(f"{q.shape[1]} query heads cannot share {k.shape[1]} key heads")
    for x, name in ((q, "q"), (k, "k"), (v, "v")):
        _check_packed(x, pack, name)
    scale = _check_scale(scale, q.shape[2])
    if q.is_cuda:
        from . import hip_packed

        return hip_packed.attention_packed(q, k, v, pack, causal, scale)
    return _ref.attention_packed(q, k, v, pack.spans, causal, scale)


def attention_packed_qkv(qkv, pack: SequencePack, heads: int, kv_heads: Optional[int] = None, causal: bool = True, scale: Optional[float] = None):
    """:func:`attention_packed` on a joint projection ``[T, (heads + 2 * kv_heads) * D]`` (query heads, key heads, value
    heads) -> ``[T, heads * D]``; on GPU the projection is read in place and its gradient written as one tensor."""
    kv_heads = heads if kv_heads is None else kv_heads
    if heads <= 0 or kv_heads <= 0 or heads % kv_heads:
        raise ValueError(f"{heads} query heads cannot share {kv_heads} key heads")
    if qkv.dim() != 2 or qkv.shape[1] == 0 or qkv.shape[1] % (heads + 2 * kv_heads):
        raise ValueError(f"expected [T, ({heads} + 2 * {kv_heads}) * D], got {tuple(qkv.shape)}")
    _check_packed(qkv, pack, "qkv")
    scale = _check_scale(scale, qkv.shape[1] // (heads + 2 * kv_heads))
    if qkv.is_cuda:
        from . import hip_packed

        return hip_packed.attention_packed_qkv(qkv, pack, heads, kv_heads, causal, scale)
    x = qkv.reshape(qkv.shape[0], heads + 2 * kv_heads, qkv.shape[1] // (heads + 2 * kv_heads))
    out = _ref.attention_packed(x[:, :heads], x[:, heads:heads + kv_heads], x[:, heads + kv_heads:], pack.spans, causal, scale)
    return out.flatten(1)


def embedding(ids, weight):
    if weight.is_cuda:
        return _hip().embedding(ids, weight)
    return _ref.embedding(ids, weight)


def token_position_embedding(ids, wte, wpe, pack: Optional[SequencePack] = None):
    """Input embedding of a language model: ``wte[ids] + wpe[position]`` for ``ids`` of shape ``[B, S]``, or of shape
    ``[rows]`` with ``pack``, where positions count from the start of each sequence (and are 0 outside).  A sequence longer
    than the table is refused where the pack knows its lengths; of one made from offsets on the GPU the tokens behind the
    table's end take its last row, and their gradients go to it."""
    if pack is not None:
        if not isinstance(pack, SequencePack):
            raise TypeError("pack: a SequencePack, made by ops.pack_sequences")
        if ids.dim() != 1 or ids.shape[0] != pack.rows or ids.device != pack.device:
            raise ValueError(f"packed tokens of shape ({pack.rows},) on {pack.device} expected, got {tuple(ids.shape)} on {ids.device}")
        if ids.dtype not in (torch.int64, torch.int32):
            raise TypeError("packed tokens must be int64 or int32")
        if wte.device != ids.device or wpe.device != ids.device:
            raise ValueError(f"tokens on {ids.device}, tables on {wte.device} and {wpe.device}")
        if pack.longest is not None and pack.longest > wpe.shape[0]:
            raise ValueError(f"a sequence of {pack.longest} tokens exceeds the {wpe.shape[0]} positions of the table")
    if wte.is_cuda:
        from . import hip_transformer as ht

        if pack is not None:
            return ht.packed_embedding(ids, pack, wte, wpe)
        return ht.token_position_embedding(ids, wte, wpe)
    if pack is not None:
        return _ref.packed_embedding(ids, pack.positions, wte, wpe)
    return _ref.token_position_embedding(ids, wte, wpe)


def vit_assemble(tok, cls, pos):
    """Vision-transformer token sequence: class token in front of the patch tokens, plus the position table."""
    if tok.is_cuda:
        from . import hip_transformer as ht

        return ht.vit_assemble(tok, cls, pos)
    return _ref.vit_assemble(tok, cls, pos)


def add_bias_residual(x, bias, residual):
    if x.is_cuda:
        return _hip().add_bias_residual(x, bias, residual)
    return _ref.add_bias_residual(x, bias, residual)


def nonfinite_seen(device, clear: bool = True) -> bool:
    """Whether a GPU kernel met non-finite batch statistics since the last call (always False on the CPU path, where
    PyTorch's own operators propagate NaN / Inf into the loss)."""
    if torch.device(device).type == "cuda":
        return _hip().nonfinite_seen(device, clear)
    return False


def set_deterministic(on: bool) -> None:
    """Run-to-run bit-identical GPU results (see ``ops.hip.set_deterministic``; ``PDT_DETERMINISTIC=1`` does the same at
    import).  The CPU path is PyTorch's own operators and is not affected."""
    if torch.cuda.is_available():
        _hip().set_deterministic(on)


def prepare_module(module):
    """One-time per-model setup of the GPU path (no-op for CPU modules): lets weight-gradient kernels
    accumulate directly into ``.grad`` where that is safe."""
    p = next(module.parameters(), None)
    if p is not None and p.is_cuda:
        _hip().enable_grad_sink(module)
    return module


def to_device_layout(x, dtype=torch.bfloat16):
    """NCHW float batch -> compute dtype in the layout the GPU kernels read (NHWC / channels_last)."""
    if x.is_cuda:
        return _hip().to_device_layout(x, dtype)
    return x.to(dtype)


def image_batch_to_device_layout(x, dtype=torch.bfloat16, mean=None, std=None):
    """uint8 ``[N, H, W, 3]`` batch (the form images travel in) -> float batch the models read: normalised
    ``(x / 255 - mean) / std``, logical NCHW.  On GPU one kernel produces bf16 NHWC; on CPU plain PyTorch."""
    if x.is_cuda:
        if dtype != torch.bfloat16:
            raise ValueError("GPU kernels compute in bf16")
        return _hip().u8_to_device_layout(x, mean, std)
    out = x.permute(0, 3, 1, 2).to(torch.float32).contiguous().div_(255.0)  # plain NCHW, as ToTensor + default collation give
    if mean is not None or std is not None:
        m = torch.tensor(mean or (0.0, 0.0, 0.0), dtype=torch.float32).view(1, 3, 1, 1)
        s_ = torch.tensor(std or (1.0, 1.0, 1.0), dtype=torch.float32).view(1, 3, 1, 1)
        out = (out - m) / s_
    return out.to(dtype)
