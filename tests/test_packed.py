"""Packs of sequences and packed attention on the CPU: definitions, gradients and refusals."""
import math

import pytest
import torch

from pytorch_distributed_training_amd import ops


def _pack(offsets, rows):
    return ops.pack_sequences(offsets, rows)


def test_pack_spans_and_positions():
    p = _pack([1, 3, 3, 7], 9)
    assert p.spans.tolist() == [[0, 0], [1, 3], [1, 3]] + [[3, 7]] * 4 + [[0, 0]] * 2
    assert p.positions.tolist() == [0, 0, 1, 0, 1, 2, 3, 0, 0]
    assert _pack(torch.tensor([0], dtype=torch.int32), 2).spans.tolist() == [[0, 0], [0, 0]]
    assert _pack([0, 0], 0).spans.shape == (0, 2)


@pytest.mark.parametrize("offsets,rows", [([0, 5, 4], 8), ([-1, 4], 8), ([0, 9], 8), ([], 8), ([0, 4], -1), ([[0, 4]], 8), ([0.0, 4.0], 8)])
def test_pack_refusals(offsets, rows):
    with pytest.raises(ValueError):
        ops.pack_sequences(torch.tensor(offsets), rows)


def _qkv(t, h, hk, d, dtype=torch.float64):
    g = torch.Generator().manual_seed(t * 31 + h)
    return [torch.randn(t, n, d, generator=g, dtype=dtype, requires_grad=True) for n in (h, hk, hk)]


@pytest.mark.parametrize("causal", [True, False])
def test_matches_masked_softmax(causal):
    q, k, v = _qkv(12, 4, 2, 8)
    pack = _pack([0, 1, 1, 6, 11], 12)
    out = ops.attention_packed(q, k, v, pack, causal=causal)
    row = torch.arange(12)
    seq = torch.tensor([0] + [1] * 5 + [2] * 5 + [-1])
    seen = (seq[:, None] == seq[None]) & (seq[:, None] >= 0)
    if causal:
        seen &= row[:, None] >= row[None]
    s = torch.einsum("ihd,jhd->hij", q, k.repeat_interleave(2, 1)) / math.sqrt(8)
    p = torch.softmax(s.masked_fill(~seen, -1e300), -1) * seen
    ref = torch.einsum("hij,jhd->ihd", p, v.repeat_interleave(2, 1))
    torch.testing.assert_close(out, ref, rtol=1e-12, atol=1e-12)
    assert out[11].abs().max() == 0


def test_gradients_against_differences():
    q, k, v = _qkv(7, 2, 1, 4)
    pack = _pack([0, 3, 6], 7)
    assert torch.autograd.gradcheck(lambda a, b, c: ops.attention_packed(a, b, c, pack, scale=0.3), (q, k, v))
    joint = torch.randn(7, 16, dtype=torch.float64, requires_grad=True)
    assert torch.autograd.gradcheck(lambda x: ops.attention_packed_qkv(x, pack, 2, 1, causal=False), (joint,))


def test_no_sequences():
    q, k, v = _qkv(3, 2, 1, 4)
    out = ops.attention_packed(q, k, v, _pack([0], 3))
    out.sum().backward()
    assert out.abs().max() == 0 and q.grad.abs().max() == 0


def test_attention_refusals():
    q, k, v = _qkv(6, 4, 2, 8)
    pack = _pack([0, 6], 6)
    with pytest.raises(ValueError, match="cannot share"):
        ops.attention_packed(q[:, :3], k, v, pack)
    with pytest.raises(ValueError, match="expected"):
        ops.attention_packed(q, k, v[:, :1], pack)
    with pytest.raises(ValueError, match="expected"):
        ops.attention_packed(q[0], k, v, pack)
    with pytest.raises(ValueError, match="rows"):
        ops.attention_packed(q, k, v, _pack([0, 5], 5))
    with pytest.raises(TypeError, match="pack"):
        ops.attention_packed(q, k, v, torch.tensor([0, 6]))
    with pytest.raises(TypeError, match="floating"):
        ops.attention_packed(q.long(), k.long(), v.long(), pack)
    for scale in (0.0, -1.0, math.inf, math.nan):
        with pytest.raises(ValueError, match="scale"):
            ops.attention_packed(q, k, v, pack, scale=scale)
    with pytest.raises(ValueError, match="expected"):
        ops.attention_packed_qkv(torch.zeros(6, 13), pack, 2, 1)
    with pytest.raises(ValueError, match="cannot share"):
        ops.attention_packed_qkv(torch.zeros(6, 14), pack, 3, 2)


def test_gpt2_on_packed_documents():
    """The packed model against one forward per document: loss and every gradient."""
    from pytorch_distributed_training_amd.models.gpt2 import gpt2_tiny

    torch.manual_seed(0)
    model = gpt2_tiny(vocab_size=97, n_ctx=32)
    lengths = [5, 1, 32, 11]
    docs = [torch.randint(0, 97, (n,)) for n in lengths]
    targets = [torch.cat([d[1:], torch.tensor([-100])]) for d in docs]
    offsets = [0, 5, 6, 38, 49]
    pack = _pack(offsets, 51)
    assert pack.longest == 32
    pad = torch.zeros(2, dtype=torch.int64)
    idx, tgt = torch.cat(docs + [pad]), torch.cat(targets + [pad - 100])
    loss = model(idx, tgt, pack=pack)
    loss.backward()
    got = [p.grad.clone() for p in model.parameters()]
    model.zero_grad()
    count = sum(n - 1 for n in lengths)
    total = 0.0
    for d, t in zip(docs, targets):
        logits = model(d[None])[0]
        total = total + torch.nn.functional.cross_entropy(logits, t, ignore_index=-100, reduction="sum") / count
    total.backward()
    torch.testing.assert_close(loss, total, rtol=1e-5, atol=1e-5)
    for a, p in zip(got, model.parameters()):
        torch.testing.assert_close(a, p.grad, rtol=1e-4, atol=1e-5)
    logits = model(idx, pack=pack)
    t, ids = logits.detach().topk(4, dim=-1)
    t = t + 1.0  # (a shift of the teacher's logits changes nothing)
    loss = model(idx, pack=pack, teacher=(t, ids), temperature=2.0)
    torch.testing.assert_close(loss, ops.distillation_loss(logits, t, ids, 2.0))
    with pytest.raises(ValueError, match="exceeds"):
        model(torch.zeros(40, dtype=torch.int64), pack=_pack([0, 40], 40))
    with pytest.raises(ValueError, match="packed tokens"):
        model(idx[:10], pack=pack)
    with pytest.raises(ValueError, match="not both"):
        model(idx, tgt, pack=pack, teacher=(t, ids))


def test_lists_of_floats_are_refused_and_offsets_of_arrays_taken():
    import numpy as np

    for bad in ([0.0, 4.5], [], [[0, 4]]):
        with pytest.raises(ValueError, match="offsets"):
            ops.pack_sequences(bad, 8)
    assert torch.equal(ops.pack_sequences(np.array([0, 3, 8]), 8).spans, _pack([0, 3, 8], 8).spans)


def test_joint_projection_of_other_strides_and_of_no_rows():
    pack = _pack([0, 4, 6], 6)
    a = torch.randn(6, 32, dtype=torch.float64)
    b = torch.randn(32, 6, dtype=torch.float64).t().copy_(a)
    assert torch.equal(ops.attention_packed_qkv(a, pack, 2, 1), ops.attention_packed_qkv(b, pack, 2, 1))
    assert ops.attention_packed_qkv(a[:0], _pack([0], 0), 2, 1).shape == (0, 16)


def test_sizes_and_factors_out_of_range():
    q, k, v = _qkv(6, 4, 2, 8)
    pack = _pack([0, 6], 6)
    with pytest.raises(ValueError, match="expected"):
        ops.attention_packed(q[..., :0], k[..., :0], v[..., :0], pack)
    for scale in (1e-31, 1e39):
        with pytest.raises(ValueError, match="scale"):
            ops.attention_packed(q, k, v, pack, scale=scale)
    ids, table = torch.zeros(6, dtype=torch.int64), torch.zeros(10, 8)
    with pytest.raises(TypeError, match="SequencePack"):
        ops.token_position_embedding(ids, table, table, torch.tensor([0, 6]))
    with pytest.raises(TypeError, match="int64"):
        ops.token_position_embedding(ids.float(), table, table, pack)
    with pytest.raises(ValueError, match="tables on"):
        ops.token_position_embedding(ids, table.to("meta"), table, pack)
