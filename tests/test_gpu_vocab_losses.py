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


def _sampled_check(got, x, w, labels, cols, scale_sum):
    """A cross-entropy whose matrices are too large for 64 bits at once: every row's loss and dx in pieces of rows, dW at
    some vocabulary entries.  Bounds as in _head_check, with the scores' error from the largest absolute sum."""
    n, v = x.shape[0], w.shape[0]
    ok = (labels >= 0) & (labels < v)
    count = max(int(ok.sum()), 1)
    s = x.shape[1] * 2.0 ** -24 * scale_sum + 2e-5
    loss = torch.zeros((), dtype=torch.float64, device="cuda")
    wc = w[cols].double()
    dw, dwe = torch.zeros_like(wc), torch.zeros_like(wc)
    for r in range(0, n, 512):
        xs, ys, oks = x[r:r + 512].double(), labels[r:r + 512], ok[r:r + 512]
        lse = torch.full((xs.shape[0],), -math.inf, dtype=torch.float64, device="cuda")
        for c in range(0, v, 1 << 18):
            lse = torch.logaddexp(lse, torch.logsumexp(xs @ w[c:c + (1 << 18)].double().t(), 1))
        zy = (xs * w[ys.clamp(0, v - 1)].double()).sum(1)
        loss += torch.where(oks, lse - zy, 0.0).sum() / count
        q = torch.exp(xs @ wc.t() - lse[:, None]) * oks[:, None] / count
        dz = q - ((cols[None] == ys[:, None]) & oks[:, None]).double() / count
        dw += dz.t() @ xs
        dwe += (H * q + H * dz.abs() + s * q).t() @ xs.abs()
    assert abs(float(got[0]) - float(loss)) <= s * (1 + float(loss)) + s
    over = (got[2][cols].double() - dw).abs() - 1.05 * (dwe + H * dw.abs() + 1e-30)
    assert float(over.max()) <= 0, f"dw: {float(over.max()):.3g} over its bound"
    return ok


def test_exponentials_past_32_bits(ops):
    """34 000 rows of 65 537 exponentials (4.5 GB) in one piece."""
    n, v, w = 34000, 65537, 64
    x, wt = _head(n, v, w)
    y = _labels(n, v)
    x.requires_grad_(True), wt.requires_grad_(True)
    loss = ops.linear_cross_entropy(x, wt, y)
    dx, dw = torch.autograd.grad(loss, (x, wt))
    cols = torch.cat([torch.arange(0, 40, device="cuda"), y[(y >= 0) & (y < v)][-60:], torch.arange(v - 40, v, device="cuda")])
    big = float(x.detach().double().abs().sum(1).max()) * float(wt.detach().abs().max())
    ok = _sampled_check((loss.detach(), dx, dw), x.detach(), wt.detach(), y, cols, big)
    # the last rows again by themselves: their share of the whole mean
    last = slice(n - 300, n)
    xs = x.detach()[last].clone().requires_grad_(True)
    (dl,) = torch.autograd.grad(ops.linear_cross_entropy(xs, wt.detach(), y[last]), xs)
    share = int(ok[last].sum()) / int(ok.sum())
    a, b = dx[last].double(), dl.double() * share
    # either side: sum_v (h q + h |q - p|) |W| / rows <= 3 h max |W| / rows, and the result's own rounding
    bound = 2 * (3 * H * float(wt.detach().abs().max()) / int(ok.sum()) + H * float(b.abs().max()))
    assert float((a - b).abs().max()) <= 1.05 * bound


def test_weights_past_32_bits(ops):
    """A vocabulary of 1.1 million entries (4.6 GB of weights), most of a row's blocks empty."""
    n, v, w = 3, 1_100_003, 2112
    g = _gen(0)
    x = torch.randn(n, w, generator=g, device="cuda").to(torch.bfloat16).requires_grad_(True)
    wt = torch.empty(v, w, dtype=torch.bfloat16, device="cuda").normal_(0, 0.03, generator=g).requires_grad_(True)
    y = torch.tensor([v - 1, 5, -100], device="cuda")
    loss = ops.linear_cross_entropy(x, wt, y)
    dx, dw = torch.autograd.grad(loss, (x, wt))
    cols = torch.cat([torch.arange(0, 50, device="cuda"), torch.arange(v - 50, v, device="cuda")])
    big = float(x.detach().double().abs().sum(1).max()) * float(wt.detach().abs().max())
    _sampled_check((loss.detach(), dx, dw), x.detach(), wt.detach(), y, cols, big)
    assert dx[2].abs().max() == 0 and bool(torch.isfinite(dx).all())


@pytest.mark.parametrize("k", [1023, 1024])
def test_as_many_targets_as_there_may_be(ops, k):
    n, v, w = 9, 700, 64  # more targets than entries: every row repeats some
    x, wt = _head(n, v, w)
    t, ids = _teacher(n, v, k)
    x.requires_grad_(True), wt.requires_grad_(True)
    loss = ops.linear_distillation_loss(x, wt, t, ids, 2.0)
    _head_check((loss.detach(), *torch.autograd.grad(loss, (x, wt))), x.detach(), wt.detach(), None, (t, ids), 2.0)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float64])
def test_other_input_types(ops, dtype):
    n, v, w = 20, 300, 64
    x, wt = (a.to(torch.float16).to(torch.bfloat16) for a in _head(n, v, w))  # (values that every type holds)
    y, (t, ids) = _labels(n, v), _teacher(n, v, 5)
    xo, wo = x.to(dtype).requires_grad_(True), wt.to(dtype).requires_grad_(True)
    xb, wb = x.requires_grad_(True), wt.requires_grad_(True)
    a, b = ops.linear_cross_entropy(xo, wo, y.to(torch.int32)), ops.linear_cross_entropy(xb, wb, y)
    assert torch.equal(a, b)
    for p, r in zip(torch.autograd.grad(a, (xo, wo)), torch.autograd.grad(b, (xb, wb))):
        # (rounded to bf16 here, h; to the finer type there, 2^-11, 2^-25 where fp16 is subnormal)
        assert p.dtype == dtype and bool(((p.double() - r.double()).abs() <= 1.2 * H * r.double().abs() + 2.0 ** -24).all())
    z = torch.randn(n, v, generator=_gen(9), device="cuda").to(torch.float16).to(dtype).requires_grad_(True)
    zf = z.detach().float().requires_grad_(True)
    a, b = ops.distillation_loss(z, t.to(dtype), ids.to(torch.int32), 2.0), ops.distillation_loss(zf, t.to(dtype).float(), ids, 2.0)
    assert torch.equal(a, b)
    (p,), (r,) = torch.autograd.grad(a, z), torch.autograd.grad(b, zf)
    assert p.dtype == dtype and torch.equal(p, r.to(dtype))


def test_some_gradients_no_rows_and_views(ops):
    n, v, w = 130, 1000, 64
    x, wt = _head(n, v, w)
    y, (t, ids) = _labels(n, v), _teacher(n, v, 5)
    x.requires_grad_(True), wt.requires_grad_(True)
    for f in (lambda a, b: ops.linear_cross_entropy(a, b, y), lambda a, b: ops.linear_distillation_loss(a, b, t, ids, 2.0)):
        both = torch.autograd.grad(f(x, wt), (x, wt))
        assert torch.equal(torch.autograd.grad(f(x, wt.detach()), x)[0], both[0])
        assert torch.equal(torch.autograd.grad(f(x.detach(), wt), wt)[0], both[1])
        with torch.no_grad():
            assert torch.equal(f(x, wt), f(x.t().contiguous().t(), wt.t().contiguous().t()))
    for loss in (ops.linear_cross_entropy(x[:0], wt, y[:0]), ops.linear_distillation_loss(x[:0], wt, t[:0], ids[:0])):
        dx, dw = torch.autograd.grad(loss, (x, wt))
        assert float(loss) == 0 and dx.abs().max() == 0 and dw.abs().max() == 0
    # logits as a view with gaps, as one row for all, and in three axes with an odd width
    z = torch.randn(6, 7, 331, generator=_gen(4), device="cuda")
    t3, i3 = t[:42].reshape(6, 7, 5), ids[:42].reshape(6, 7, 5) % 101
    view = z[:, :, 230:331].requires_grad_(True)
    copy = view.detach().clone().requires_grad_(True)
    a, b = ops.distillation_loss(view, t3, i3), ops.distillation_loss(copy, t3, i3)
    assert torch.equal(a, b) and torch.equal(torch.autograd.grad(a, view)[0], torch.autograd.grad(b, copy)[0])
    row = z[0, :1, :101]
    a, b = ops.distillation_loss(row.expand(42, 101), t[:42], i3.reshape(42, 5)), ops.distillation_loss(row.repeat(42, 1), t[:42], i3.reshape(42, 5))
    assert torch.equal(a, b)


def test_two_streams_at_once(ops):
    sets = [(_head(1500, 5003, 128, s), _labels(1500, 5003, s), _teacher(1500, 5003, 16, s)) for s in (0, 1)]
    for (x, wt), _, _ in sets:
        x.requires_grad_(True), wt.requires_grad_(True)

    def run(s):
        (x, wt), y, teacher = s
        a, b = ops.linear_cross_entropy(x, wt, y), ops.linear_distillation_loss(x, wt, *teacher, 2.0)
        return (a.detach(), *torch.autograd.grad(a, (x, wt)), b.detach(), *torch.autograd.grad(b, (x, wt)))

    want = [run(s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = [[], []]
    for _ in range(3):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(run(sets[i]))
    torch.cuda.synchronize()
    for a, g in zip(want, got):
        for each in g:
            assert all(torch.equal(p, r) for p, r in zip(a, each))


def test_too_many_rows_are_refused(ops):
    n = 1 << 22
    ids = torch.zeros(n, 1, dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError, match="rows at a time"):
        ops.distillation_loss(torch.zeros(n, 1, dtype=torch.bfloat16, device="cuda"), torch.zeros(n, 1, device="cuda"), ids)
    with pytest.raises(ValueError, match="rows at a time"):
        ops.linear_cross_entropy(torch.zeros(1, 64, dtype=torch.bfloat16, device="cuda").expand(n, 64), torch.zeros(5, 64, dtype=torch.bfloat16, device="cuda"), ids[:, 0])


@pytest.mark.parametrize("n", [1023, 1024, 1025, 3000])
def test_distillation_on_many_rows(ops, n):
    """Rows with a target counted by every workgroup, and by a launch of its own."""
    test_distillation_on_logits(ops, torch.bfloat16, n, 130, 5, 2.0)
