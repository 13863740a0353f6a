"""Losses over a vocabulary on the CPU: definitions, gradients and refusals."""
import math

import pytest
import torch
import torch.nn.functional as F

from pytorch_distributed_training_amd import ops


def _r(*shape, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed), dtype=torch.float64)


def test_cross_entropy_leaves_out_rows_without_a_label():
    x, w = _r(2, 3, 8).requires_grad_(True), _r(11, 8, seed=1).requires_grad_(True)
    y = torch.tensor([[0, -100, 10], [11, 5, -1]])
    loss = ops.linear_cross_entropy(x, w, y)
    keep = torch.tensor([0, 2, 4])
    ref = F.cross_entropy(x.reshape(-1, 8)[keep] @ w.t(), y.reshape(-1)[keep])
    torch.testing.assert_close(loss, ref)
    loss.backward()
    assert x.grad.reshape(-1, 8)[[1, 3, 5]].abs().max() == 0
    assert torch.autograd.gradcheck(lambda a, b: ops.linear_cross_entropy(a, b, y), (x, w))


def test_no_labels_at_all():
    x, w = _r(3, 8).requires_grad_(True), _r(5, 8)
    loss = ops.linear_cross_entropy(x, w, torch.full((3,), -100))
    loss.backward()
    assert float(loss) == 0.0 and x.grad.abs().max() == 0
    assert float(ops.linear_cross_entropy(x[:0], w, torch.zeros(0, dtype=torch.int64))) == 0.0


def _teacher():
    ids = torch.tensor([[3, 1, 4], [0, -1, 2], [-1, 7, -5], [5, 5, 1]])  # absent entries, an empty row, an id twice
    return _r(4, 3, seed=2), ids


@pytest.mark.parametrize("tau", [1.0, 2.5])
def test_distillation_definition(tau):
    z = _r(4, 6, seed=3).requires_grad_(True)
    t, ids = _teacher()
    t[0, 1] = -math.inf  # weight 0
    loss = ops.distillation_loss(z, t, ids, temperature=tau)
    ref = 0.0
    for r, ks in ((0, [0, 2]), (1, [0, 2]), (3, [0, 1, 2])):
        p = torch.softmax(t[r, ks] / tau, 0)
        logq = torch.log_softmax(z[r] / tau, 0)[ids[r, ks]]
        ref = ref + tau ** 2 * (p * (p.log() - logq)).sum() / 3
    torch.testing.assert_close(loss, ref)
    loss.backward()
    assert z.grad[2].abs().max() == 0 and torch.isfinite(z.grad).all()
    assert torch.autograd.gradcheck(lambda a: ops.distillation_loss(a, t, ids, temperature=tau), (z,))
    x, w = _r(4, 8, seed=4).requires_grad_(True), _r(6, 8, seed=5).requires_grad_(True)
    torch.testing.assert_close(ops.linear_distillation_loss(x, w, t, ids, tau), ops.distillation_loss(x @ w.t(), t, ids, tau))
    assert torch.autograd.gradcheck(lambda a, b: ops.linear_distillation_loss(a, b, t, ids, tau), (x, w))


def test_masked_vocabulary_entries():
    """A student that rules entries out (-inf or the type's lowest value) is finite where the teacher does not want them."""
    for low in (-math.inf, torch.finfo(torch.float64).min):
        z = _r(2, 6)
        z[:, 4:] = low
        t, ids = _r(2, 3, seed=1), torch.tensor([[0, 1, 2], [3, 0, 5]])
        t[1, 2] = -math.inf
        z.requires_grad_(True)
        loss = ops.distillation_loss(z, t, ids)
        loss.backward()
        assert math.isfinite(float(loss)) and torch.isfinite(z.grad).all() and z.grad[:, 4:].abs().max() == 0


def test_refusals():
    x, w, y = torch.zeros(3, 8), torch.zeros(5, 8), torch.zeros(3, dtype=torch.int64)
    t, ids = torch.zeros(3, 2), torch.zeros(3, 2, dtype=torch.int64)
    with pytest.raises(ValueError, match="expected"):
        ops.linear_cross_entropy(x, w[:, :4], y)
    with pytest.raises(ValueError, match="labels"):
        ops.linear_cross_entropy(x, w, y[:2])
    with pytest.raises(TypeError, match="labels"):
        ops.linear_cross_entropy(x, w, y.float())
    with pytest.raises(TypeError, match="floating"):
        ops.linear_cross_entropy(x.long(), w, y)
    with pytest.raises(ValueError, match="vocabulary"):
        ops.linear_cross_entropy(x, w[:0], y)
    for bad in (0.0, -1.0, math.inf, math.nan):
        with pytest.raises(ValueError, match="temperature"):
            ops.distillation_loss(x, t, ids, bad)
    with pytest.raises(ValueError, match="teacher ids"):
        ops.distillation_loss(x, t, ids[0])
    with pytest.raises(ValueError, match="teacher ids"):
        ops.linear_distillation_loss(x, w, t, ids[:2])
    with pytest.raises(ValueError, match="teacher logits"):
        ops.distillation_loss(x, t[:, :1], ids)
    with pytest.raises(ValueError, match="per row"):
        ops.distillation_loss(x, torch.zeros(3, 1025), torch.zeros(3, 1025, dtype=torch.int64))
    with pytest.raises(ValueError, match="no gradient flows"):
        ops.distillation_loss(x, t.requires_grad_(True), ids)
    with pytest.raises(TypeError, match="int64"):
        ops.distillation_loss(x, t.detach(), ids.float())


def test_temperatures_out_of_range():
    x, t, ids = torch.zeros(3, 8), torch.zeros(3, 2), torch.zeros(3, 2, dtype=torch.int64)
    for bad in (1e-7, 1e7):
        with pytest.raises(ValueError, match="temperature"):
            ops.distillation_loss(x, t, ids, bad)


def test_head_distillation_is_the_loss_on_the_projection_in_mixed_types_and_without_rows():
    x, w = _r(4, 6).to(torch.bfloat16), _r(9, 6, seed=1).float().requires_grad_(True)
    t, ids = _r(4, 3, seed=2), torch.tensor([[0, 8, 3]] * 4)
    a = ops.linear_distillation_loss(x, w, t, ids, 2.0)
    assert abs(float(a) - float(ops.distillation_loss(x.double() @ w.double().t(), t, ids, 2.0))) < 1e-5
    none = ops.linear_distillation_loss(x[:0], w, t[:0], ids[:0])
    none.backward()
    assert float(none) == 0 and w.grad.abs().max() == 0
