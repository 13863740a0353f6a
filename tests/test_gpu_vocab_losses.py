"""Vocabulary losses on the GPU against the formulas in 64 bits (needs an MI355X).

Tolerances follow from the roundings, element by element, with h = 2^-8 (bf16, half a step).  Behind a projection the
exponentials and q - p are rounded once each, the result once: with a = tau / rows,
    |D - (q - p)| <= h q + h |q - p| =: F,   |dx - ref| <= a F |W| + h |ref|,   |dW - ref| <= a F' |x| + h |ref|.
On given logits only the result is rounded.  Scores in 32 bits: a sum of w products is off by w 2^-24 of their absolute sum
at most, which exponents take over as a relative error of the probabilities (s below); 2e-5 covers exp2 and the sums.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

H = 2.0 ** -8


@pytest.fixture(scope="module")
def ops():
    from pytorch_distributed_training_amd import ops as m

    return m


def _gen(seed):
    return torch.Generator("cuda").manual_seed(seed)


def _head(n, v, w, seed=0):
    g = _gen(seed)
    x = torch.randn(n, w, generator=g, device="cuda").to(torch.bfloat16)
    wt = (torch.randn(v, w, generator=g, device="cuda") * (2.0 / math.sqrt(w))).to(torch.bfloat16)
    return x, wt


def _labels(n, v, seed=0):
    y = torch.randint(0, v, (n,), generator=_gen(seed + 1), device="cuda")
    y[::5] = -100
    if n > 2:
        y[2] = v  # beyond the vocabulary: left out too
    if n > 1:
        y[1] = v - 1
    return y


def _teacher(n, v, k, seed=0):
    g = _gen(seed + 2)
    ids = torch.randint(0, v, (n, k), generator=g, device="cuda")  # repeats among them
    ids[torch.rand(n, k, generator=g, device="cuda") < 0.1] = -1
    t = torch.randn(n, k, generator=g, device="cuda") * 3
    if n > 2:
        ids[2] = -1
    if n > 4:
        t[4] = -math.inf
    if n > 1 and k > 1:
        ids[1, 1] = ids[1, 0] = v - 1
        t[1, 0] = -math.inf
    return t, ids


def _targets(labels, teacher, v, tau):
    """[N, K] ids (clamped), weights p and which rows count, in 64 bits."""
    if teacher is None:
        ids = labels[:, None]
        ok = (ids >= 0) & (ids < v)
        return ids.clamp(0, v - 1), ok.double(), ok[:, 0]
    t, ids = teacher[0].double(), teacher[1]
    t = t.masked_fill((ids < 0) | (ids >= v), -math.inf)
    some = (t > -math.inf).any(1)
    p = torch.softmax(t.masked_fill(~some[:, None], 0.0) / tau, 1) * some[:, None] * (t > -math.inf)
    return ids.clamp(0, v - 1), p, some


def _expected(z, labels, teacher, tau):
    """loss, dz, q and the size of the loss's terms, in 64 bits."""
    ids, p, some = _targets(labels, teacher, z.shape[1], tau)
    count = some.sum().clamp(min=1)
    logq = torch.log_softmax(z / tau, 1)
    taken = torch.where(p > 0, logq.gather(1, ids), 0.0)
    ent = torch.where(p > 0, p * p.clamp(min=1e-300).log(), 0.0)
    loss = tau * tau * (ent - p * taken).sum() / count
    terms = tau * tau * (ent.abs() + p * taken.abs()).sum() / count
    q = logq.exp() * some[:, None]
    target = torch.zeros_like(z).scatter_add_(1, ids, p)
    return loss, (q - target) * (tau / count), q * (tau / count), terms


def _head_check(got, x, w, labels, teacher, tau, factor=1.0):
    x, w = x.double(), w.double()
    z = x @ w.t()
    loss, dz, q, terms = _expected(z, labels, teacher, tau)
    s = x.shape[1] * 2.0 ** -24 * float((x.abs() @ w.abs().t()).max()) / tau + 2e-5
    assert abs(float(got[0]) - float(loss)) <= s * (1 + float(terms)) + tau * tau * s
    f = H * q + H * dz.abs() + s * q
    for name, r, y, e in (("dx", got[1], dz @ w, f @ w.abs()), ("dw", got[2], dz.t() @ x, f.t() @ x.abs())):
        y, e = factor * y, factor * e
        over = (r.double() - y).abs() - 1.05 * (e + H * y.abs() + 1e-30)
        assert r.shape == y.shape and float(over.max()) <= 0, f"{name}: {float(over.max()):.3g} over its bound"


SIZES = [(1, 1, 64), (1, 65, 64), (3, 64, 128), (130, 1000, 192), (257, 5003, 64), (300, 257, 320), (64, 40000, 128)]


@pytest.mark.parametrize("n,v,w", SIZES)
def test_cross_entropy(ops, n, v, w):
    x, wt = _head(n, v, w)
    y = _labels(n, v)
    y[0] = 0
    x.requires_grad_(True), wt.requires_grad_(True)
    loss = ops.linear_cross_entropy(x, wt, y)
    got = (loss.detach(), *torch.autograd.grad(loss, (x, wt)))
    _head_check(got, x.detach(), wt.detach(), y, None, 1.0)
    with torch.no_grad():
        assert torch.equal(ops.linear_cross_entropy(x, wt, y), loss)


@pytest.mark.parametrize("n,v,w", SIZES)
@pytest.mark.parametrize("k,tau", [(1, 1.0), (7, 2.0), (300, 0.5)])
def test_head_distillation(ops, n, v, w, k, tau):
    x, wt = _head(n, v, w, seed=3)
    teacher = _teacher(n, v, k)
    x.requires_grad_(True), wt.requires_grad_(True)
    loss = ops.linear_distillation_loss(x, wt, *teacher, tau)
    got = (loss.detach(), *torch.autograd.grad(loss, (x, wt)))
    _head_check(got, x.detach(), wt.detach(), None, teacher, tau)


def test_chunks_parameters_and_incoming_gradient(ops, monkeypatch):
    """Several chunks of rows, an fp32 parameter (gradient in fp32, into .grad where that is allowed), a factor behind."""
    from pytorch_distributed_training_amd.ops import hip_vocab

    n, v, w = 700, 1300, 128
    x, wt = _head(n, v, w)
    y = _labels(n, v)
    monkeypatch.setattr(hip_vocab, "CHUNK_BYTES", 300 * 2 * 1344)
    param = torch.nn.Parameter(wt.float())
    x.requires_grad_(True)
    (ops.linear_cross_entropy(x.view(7, 100, w), param, y.view(7, 100)) * 3).backward()
    loss = ops.linear_cross_entropy(x, wt, y).detach()
    assert param.grad.dtype == torch.float32 and x.grad.dtype == torch.bfloat16
    _head_check((loss, x.grad, param.grad), x.detach(), wt, y, None, 1.0, factor=3.0)
    once = param.grad.clone()
    param._pdt_sink_ok = True
    (ops.linear_cross_entropy(x, param, y) * 3).backward()
    torch.testing.assert_close(param.grad, 2 * once, rtol=1e-6, atol=1e-9)
    bf = wt.clone().requires_grad_(True)  # a bf16 weight over several chunks
    (g,) = torch.autograd.grad(ops.linear_cross_entropy(x, bf, y), bf)
    _head_check((loss, torch.autograd.grad(ops.linear_cross_entropy(x, wt, y), x)[0], g), x.detach(), wt, y, None, 1.0)


@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_left_out_rows_do_not_show(ops, bad):
    n, v, w = 150, 700, 64
    x, wt = _head(n, v, w)
    y = _labels(n, v)
    keep = (y >= 0) & (y < v)
    x2 = x.clone()
    x2[~keep] = bad
    a, b = x2.requires_grad_(True), wt.requires_grad_(True)
    loss = ops.linear_cross_entropy(a, b, y)
    dx, dw = torch.autograd.grad(loss, (a, b))
    _head_check((loss.detach(), dx, dw), x, wt.detach(), y, None, 1.0)
    assert dx[~keep].abs().max() == 0
    # a NaN in a row that counts is seen
    x2 = x.clone()
    x2[keep.nonzero()[0, 0]] = math.nan
    assert math.isnan(float(ops.linear_cross_entropy(x2, wt.detach(), y)))


def test_no_targets_at_all(ops):
    x, wt = _head(5, 100, 64)
    x.requires_grad_(True), wt.requires_grad_(True)
    loss = ops.linear_cross_entropy(x, wt, torch.full((5,), -100, device="cuda"))
    dx, dw = torch.autograd.grad(loss, (x, wt))
    assert float(loss) == 0 and dx.abs().max() == 0 and dw.abs().max() == 0
    none = torch.zeros(0, dtype=torch.int64, device="cuda")
    assert float(ops.linear_cross_entropy(x[:0], wt, none)) == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n,v,k,tau", [(1, 1, 1, 1.0), (5, 63, 3, 2.0), (40, 1000, 5, 2.0), (33, 1001, 64, 0.5), (17, 50257, 64, 2.0), (3, 70001, 1000, 4.0)])
def test_distillation_on_logits(ops, dtype, n, v, k, tau):
    z = (torch.randn(n, v, generator=_gen(v), device="cuda") * 3).to(dtype)
    if v > 8:
        z[0, 5:8] = -math.inf  # entries the student rules out
        z[-1, 0:2] = torch.finfo(dtype).min
    teacher = _teacher(n, v, k)
    if v > 8:  # (and the teacher does not want)
        teacher[1][0].masked_fill_((teacher[1][0] >= 5) & (teacher[1][0] < 8), -1)
        teacher[1][-1].masked_fill_((teacher[1][-1] < 2), -1)
    z.requires_grad_(True)
    loss = ops.distillation_loss(z, *teacher, tau)
    (g,) = torch.autograd.grad(loss, z)
    ref, dz, q, terms = _expected(z.detach().double(), None, teacher, tau)
    assert abs(float(loss) - float(ref)) <= 2e-5 * (1 + float(terms))
    h = H if dtype == torch.bfloat16 else 2.0 ** -24
    over = (g.double() - dz).abs() - 1.05 * (h * dz.abs() + 2e-5 * (q + (q - dz).abs()) + 1e-38)
    assert g.dtype == dtype and g.shape == z.shape and float(over.max()) <= 0
    # rows with gaps, off 16-byte boundaries, more leading axes, and a factor behind
    wide = torch.zeros(n, 1, v + 3, dtype=dtype, device="cuda")
    wide[:, 0, 1:v + 1] = z.detach()
    view = wide[:, :, 1:v + 1].requires_grad_(True)
    loss2 = ops.distillation_loss(view, teacher[0][:, None], teacher[1][:, None].int(), tau)
    (g2,) = torch.autograd.grad(loss2 * 2, view)
    assert torch.equal(loss2, loss) and torch.equal(g2[:, 0], (g * 2))


def test_gradients_against_differences(ops):
    """Directional differences of the loss itself, in steps the fp32 loss resolves."""
    n, v, w, k = 24, 400, 64, 6
    x, wt = _head(n, v, w, seed=9)
    teacher = _teacher(n, v, k, seed=9)
    y = _labels(n, v, seed=9)
    for f in (lambda a, b: ops.linear_cross_entropy(a, b, y), lambda a, b: ops.linear_distillation_loss(a, b, *teacher, 2.0),
              lambda a, b: ops.distillation_loss((a.float() @ b.float().t()), *teacher, 2.0)):
        a, b = x.clone().requires_grad_(True), wt.clone().requires_grad_(True)
        dx, dw = torch.autograd.grad(f(a, b), (a, b))
        for leaf, grad, mk in ((x, dx, lambda t: (t, wt)), (wt, dw, lambda t: (x, t))):
            u = torch.sign(grad.float())
            step = 2.0 ** -4 * leaf.float().abs().mean()
            hi, lo = (leaf.float() + step * u).to(torch.bfloat16), (leaf.float() - step * u).to(torch.bfloat16)
            with torch.no_grad():
                diff = float(f(*mk(hi))) - float(f(*mk(lo)))
            want = float((grad.double() * (hi.double() - lo.double())).sum())
            # central differences over a relative step of 1/16 leave a third-order term, a few per cent here
            assert abs(diff - want) <= 0.1 * abs(want), (diff, want)


def test_same_bits_every_time_and_on_another_stream(ops):
    x, wt = _head(200, 3001, 128)
    teacher, y = _teacher(200, 3001, 16), _labels(200, 3001)
    x.requires_grad_(True), wt.requires_grad_(True)

    def run():
        a = ops.linear_cross_entropy(x, wt, y)
        b = ops.linear_distillation_loss(x, wt, *teacher, 2.0)
        return (a.detach(), *torch.autograd.grad(a, (x, wt)), b.detach(), *torch.autograd.grad(b, (x, wt)))

    first = run()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        other = run()
    side.synchronize()
    for a, b, c in zip(first, run(), other):
        assert torch.equal(a, b) and torch.equal(a, c)


def test_captured_graph_follows_new_inputs(ops):
    n, v, w, k = 130, 1500, 64, 9
    x, wt = _head(n, v, w)
    y, (t, ids) = _labels(n, v), _teacher(n, v, k)
    z = torch.randn(n, v, device="cuda")
    leaves = [a.requires_grad_(True) for a in (x, wt, z)]

    def run():
        a = ops.linear_cross_entropy(x, wt, y)
        b = ops.linear_distillation_loss(x, wt, t, ids, 2.0)
        c = ops.distillation_loss(z, t, ids, 2.0)
        return (a, *torch.autograd.grad(a, leaves[:2]), b, *torch.autograd.grad(b, leaves[:2]), c, *torch.autograd.grad(c, leaves[2:]))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run()
    for seed in range(4):
        with torch.no_grad():
            for a, b in zip((x, wt, y, t, ids), (*_head(n, v, w, seed), _labels(n, v, seed), *_teacher(n, v, k, seed))):
                a.copy_(b)
            z.normal_()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, run()):
            assert torch.equal(a, b)


def test_backward_runs_once(ops):
    x, wt = _head(4, 100, 64)
    loss = ops.linear_cross_entropy(x.requires_grad_(True), wt, torch.zeros(4, dtype=torch.int64, device="cuda"))
    loss.backward(retain_graph=True)
    with pytest.raises(RuntimeError, match="backward ran twice"):
        loss.backward()


def test_refusals(ops):
    x, wt = _head(4, 100, 64)
    y = torch.zeros(4, dtype=torch.int64, device="cuda")
    with pytest.raises(ValueError, match="multiple of 64"):
        ops.linear_cross_entropy(x[:, :32], wt[:, :32], y)
    with pytest.raises(ValueError, match="weight on"):
        ops.linear_cross_entropy(x, wt.cpu(), y)
    with pytest.raises(ValueError, match="labels on"):
        ops.linear_cross_entropy(x, wt, y.cpu())
    with pytest.raises(ValueError, match="teacher ids on"):
        ops.distillation_loss(x, torch.zeros(4, 2), torch.zeros(4, 2, dtype=torch.int64))
