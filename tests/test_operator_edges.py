"""Limits and bookkeeping of the packed and vocabulary operators that need no GPU."""
import pytest
import torch


def test_padding_is_known_of_the_buffer_itself():
    """What a loss says of its gradient's padding ends with the buffer: another one at the same address says nothing."""
    from pytorch_distributed_training_amd.ops import hip

    def at(memory):
        return torch.frombuffer(memory, dtype=torch.bfloat16).view(6, 64)

    memory = bytearray(6 * 64 * 2)
    buf = hip.zero_padded(at(memory))
    g = buf[:, :50]
    assert hip.padded_form(g, 64).shape == (6, 64) and hip.padded_form(g, 64).data_ptr() == buf.data_ptr()
    assert hip.padded_form(g.reshape(2, 3, 50).reshape(6, 50), 64) is not None  # a view of a view
    assert hip.padded_form(g, 128) is None and hip.padded_form(g[1:], 64) is None and hip.padded_form(g[:, 1:], 64) is None
    total = g + g  # a sum with another loss's gradient is dense, and the buffer goes unused
    assert hip.padded_form(total, 64) is None
    address = buf.data_ptr()
    del buf, g
    later = at(memory)[:, :50]
    assert later.data_ptr() == address and later.stride() == (64, 1)
    assert hip.padded_form(later, 64) is None


def test_no_tangent_of_the_teacher():
    from torch.autograd import forward_ad

    from pytorch_distributed_training_amd import ops

    z, t, ids = torch.randn(3, 5), torch.randn(3, 2), torch.tensor([[0, 1], [2, 3], [4, 0]])
    x, w = torch.randn(3, 8), torch.randn(5, 8)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(t, torch.ones_like(t))
        with pytest.raises(ValueError, match="teacher"):
            ops.distillation_loss(z, dual, ids)
        with pytest.raises(ValueError, match="teacher"):
            ops.linear_distillation_loss(x, w, dual, ids)
        tangent = forward_ad.unpack_dual(ops.distillation_loss(forward_ad.make_dual(z, torch.ones_like(z)), t, ids)).tangent
        assert abs(float(tangent)) < 1e-6  # (a shift of all logits changes nothing)


@pytest.mark.parametrize("labels", [[1, 4, 0], [1, -100, 0], [-1, 5, 2], [-100, -100, -100]])
def test_cross_entropy_over_the_rows_with_a_label(labels):
    from pytorch_distributed_training_amd import ops

    x, w = (torch.randn(*s, generator=torch.Generator().manual_seed(0)).requires_grad_(True) for s in ((3, 64), (5, 64)))
    y = torch.tensor(labels)
    has = (y >= 0) & (y < 5)
    z = (x @ w.t()).detach()
    want = -(torch.log_softmax(z.double(), 1)[torch.arange(3), y.clamp(0, 4)] * has).sum() / has.sum().clamp(min=1)
    loss = ops.lm_head_loss(x, w, y)
    (g,) = torch.autograd.grad(loss, x)
    assert abs(loss.item() - float(want)) < 1e-5 * (1 + float(want)) and bool((g[~has] == 0).all())
    if bool(((y >= 0) | (y == -100)).all() & (y < 5).all()):
        assert abs(ops.softmax_cross_entropy(z, y).item() - float(want)) < 1e-5 * (1 + float(want))
    else:
        with pytest.raises(IndexError):
            ops.softmax_cross_entropy(z, y)


def test_rows_of_a_launch():
    """Rows are rounded up to 64 in the passes over them, with 1024 threads each: 2^22 - 64 rows are the last that stay below 2^32 threads."""
    from pytorch_distributed_training_amd.ops import hip_vocab

    assert hip_vocab.MAX_ROWS == (1 << 22) - 63  # the first that is refused
    for rows, taken in (((1 << 22) - 64, True), ((1 << 22) - 63, False), ((1 << 22) - 1, False), (1 << 22, False)):
        assert (hip_vocab._head_scratch(rows, 1, 50, 64, rows, 0, 1, 1) > 0) == taken
        assert (hip_vocab._distill_scratch(rows, 1) > 0) == taken
    with pytest.raises(ValueError, match="rows at a time"):
        hip_vocab._check_rows((1 << 22) - 63)


def test_rows_of_all_heads_fit_the_tiles_offsets():
    """Inputs whose rows overlap can have more heads than a row's stride: out and its gradient are [T, H, D] without gaps, and the
    offsets of 64 of their rows are 32 bits."""
    import ctypes

    from pytorch_distributed_training_amd.ops import hip_packed

    strides = (ctypes.c_longlong * 12)(*([8] * 12))
    heads = (1 << 24) // 64
    one = 1 << 20  # (an address that is never read: the call is refused)
    assert hip_packed._fwd(one, one, one, one, one, one, one, one, strides, 2, heads, 1, 64, 0.1, 1, None) == -1
    assert hip_packed._bwd(*[one] * 12, 1, one, one, strides, 2, heads, 1, 64, 0.1, 1, None) == -1
