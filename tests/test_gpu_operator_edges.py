"""Packed attention, vocabulary losses and the losses beside them on the GPU, where they meet other parts: the linear layer's
padded gradients, over-long documents, forward-mode derivatives, rows without a label, students close to their teacher,
results far from 1 (needs an MI355X).

h = 2^-8 is half a step of bf16 relative to the value; sums of n products in 32 bits are off by n 2^-24 of their absolute sum.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

H = 2.0 ** -8
U = 2.0 ** -24


@pytest.fixture(scope="module")
def ops():
    from pytorch_distributed_training_amd import ops as m

    return m


def _gen(seed):
    return torch.Generator("cuda").manual_seed(seed)


def _bf16(*shape, seed=0, std=1.0):
    return (torch.randn(*shape, generator=_gen(seed), device="cuda") * std).to(torch.bfloat16)


def _distill_64(z, teacher, ids, tau):
    """Gradient of the logits in 64 bits (every row has a target, no id twice in a row)."""
    p = torch.softmax(teacher.double() / tau, 1)
    dz = torch.softmax(z.double() / tau, 1).scatter_add(1, ids, -p)
    return dz * (tau / len(z))


@pytest.mark.parametrize("vocab", [1000, 2010, 1020])
@pytest.mark.parametrize("left_out", [False, True])
def test_distillation_behind_a_linear_layer(ops, vocab, left_out):
    """Distillation alone behind a projection whose rows are padded, in memory that held NaN, after a step that added
    cross-entropy and distillation on the same logits: the gradient of x against the formula's."""
    n, width, top, tau = 64, 128, 5, 2.0
    weight = torch.nn.Parameter(_bf16(vocab, width, seed=1, std=2.0 / math.sqrt(width)).float())
    x = _bf16(n, width, seed=2)
    ids = (torch.arange(n, device="cuda")[:, None] * 13 + torch.arange(top, device="cuda") * 7) % vocab
    teacher = torch.randn(n, top, generator=_gen(3), device="cuda")
    labels = ids[:, 0].contiguous()
    if left_out:
        ids = ids.clone()
        ids[5] = -1
    pitch = (vocab + 63) // 64 * 64
    for _ in range(3):
        a = x.clone().requires_grad_(True)
        z = ops.linear(a, weight)
        (ops.softmax_cross_entropy(z, labels) + ops.distillation_loss(z, teacher, ids, tau)).backward()
        del z
        for fill in [torch.full((n, pitch), math.nan, dtype=torch.bfloat16, device="cuda") for _ in range(8)]:
            del fill
        b = x.clone().requires_grad_(True)
        z = ops.linear(b, weight)
        ops.distillation_loss(z, teacher, ids, tau).backward()
        dz = _distill_64(z.detach(), teacher, ids.clamp(min=0), tau)
        if left_out:
            dz[5] = 0
            dz *= n / (n - 1)
        w = weight.detach().double()
        want = dz @ w
        # the gradient of the logits rounded once, the result once; the sums in 32 bits, the probabilities to 2e-5
        bound = (H + 2e-5 + vocab * U) * (dz.abs() @ w.abs()) + 2e-5 * tau / n * (torch.softmax(z.detach().double() / tau, 1) @ w.abs()) + H * want.abs()
        assert bool(torch.isfinite(b.grad).all())
        over = (b.grad.double() - want).abs() - 1.05 * bound
        assert float(over.max()) <= 0, float(over.max())
        weight.grad = None


def test_distillation_gradient_is_taken_as_it_is(ops):
    """The rows' padding is written with zeros, left-out rows' too, whatever the memory held."""
    from pytorch_distributed_training_amd.ops import hip_vocab

    for dtype in (torch.bfloat16, torch.float32):
        for vocab in (1000, 1001, 63, 1023):
            n = 7
            pitch = (vocab + 63) // 64 * 64
            z = _bf16(n, vocab, seed=vocab).to(dtype)
            ids = torch.randint(0, vocab, (n, 3), generator=_gen(4), device="cuda")
            ids[2] = -1
            full = torch.full((n, pitch), math.nan, dtype=dtype, device="cuda")
            del full
            _, dz = hip_vocab._distill_forward(z, ids, torch.zeros(n, 3, device="cuda"), 1.0, True)
            assert dz.shape[1] == pitch and bool((dz[:, vocab:] == 0).all()) and bool(torch.isfinite(dz).all())


@pytest.mark.parametrize("deterministic", [False, True])
def test_gradient_of_positions_behind_the_tables_end(ops, deterministic):
    """Tokens behind the position table's end read its last row, so their gradients are its."""
    offsets = torch.tensor([0, 40, 47, 52], device="cuda")
    rows, d = 53, 64
    wte, wpe = torch.randn(30, d, generator=_gen(0), device="cuda"), torch.randn(16, d, generator=_gen(1), device="cuda")
    wte.requires_grad_(True), wpe.requires_grad_(True)
    ids = torch.randint(0, 30, (rows,), generator=_gen(2), device="cuda")
    g = _bf16(rows, d, seed=3)
    pack = ops.pack_sequences(offsets, rows)
    at = pack.positions.clamp(max=15)
    ops.set_deterministic(deterministic)
    try:
        out = ops.token_position_embedding(ids, wte, wpe, pack)
        a, b = torch.autograd.grad(out, (wte, wpe), g)
    finally:
        ops.set_deterministic(False)
    assert torch.equal(out.detach(), (wte[ids] + wpe[at]).to(torch.bfloat16))
    for got, index in ((a, ids), (b, at)):
        want = torch.zeros(got.shape, dtype=torch.float64, device="cuda").index_add_(0, index, g.double())
        terms = torch.zeros(got.shape, dtype=torch.float64, device="cuda").index_add_(0, index, g.double().abs())
        assert bool(((got.double() - want).abs() <= rows * U * terms).all())


def test_forward_mode_derivatives_are_refused(ops):
    """Not dropped: a dual tensor goes the way of a tensor that requires a gradient, and is refused there."""
    from torch.autograd import forward_ad

    q, k, v = _bf16(6, 2, 64), _bf16(6, 2, 64, seed=1), _bf16(6, 2, 64, seed=2)
    pack = ops.pack_sequences([0, 6], 6, device="cuda")
    x, w, z = _bf16(6, 64), _bf16(70, 64, seed=3), _bf16(6, 70, seed=4)
    labels, teacher = torch.arange(6, device="cuda"), torch.randn(6, 2, generator=_gen(5), device="cuda")
    ids = torch.arange(12, device="cuda").view(6, 2)
    calls = {
        "attention": (lambda a, b, c: ops.attention_packed(a, b, c, pack), [q, k, v]),
        "joint": (lambda a: ops.attention_packed_qkv(a, pack, 2), [torch.cat([q, k, v], 1).flatten(1)]),
        "loss": (lambda a, b: ops.linear_cross_entropy(a, b, labels), [x, w]),
        "head distillation": (lambda a, b, t: ops.linear_distillation_loss(a, b, t, ids), [x, w, teacher]),
        "distillation": (lambda a, t: ops.distillation_loss(a, t, ids), [z, teacher]),
    }
    for name, (call, inputs) in calls.items():
        plain = call(*inputs)
        for i in range(len(inputs)):
            for grad in (True, False):
                with forward_ad.dual_level(), torch.set_grad_enabled(grad):
                    with pytest.raises((NotImplementedError, ValueError)):
                        call(*(forward_ad.make_dual(t, torch.ones_like(t)) if i == j else t for j, t in enumerate(inputs)))
                    assert torch.equal(call(*inputs), plain), name


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("classes", [10, 1000, 1032, 5003, 66000])
@pytest.mark.parametrize("labelled", ["all", "some", "none"])
def test_cross_entropy_over_the_rows_with_a_label(ops, dtype, classes, labelled):
    n = 37
    z = _bf16(n, classes, seed=classes, std=2.0).to(dtype).requires_grad_(True)
    y = torch.randint(0, classes, (n,), generator=_gen(6), device="cuda")
    if labelled != "all":
        y[::3] = -100
        y[1], y[2] = classes, -1
    if labelled == "none":
        y[:] = -100
    loss = ops.softmax_cross_entropy(z, y)
    (g,) = torch.autograd.grad(loss * 2, z)
    has = (y >= 0) & (y < classes)
    count = has.sum().clamp(min=1)
    z64 = z.detach().double()
    logp = torch.log_softmax(z64, 1)
    each = -logp.gather(1, y.clamp(0, classes - 1)[:, None])[:, 0] * has
    dz = logp.exp()
    dz[torch.arange(n, device="cuda"), y.clamp(0, classes - 1)] -= 1.0
    dz *= (2.0 * has / count)[:, None]
    # exponentials and sums in 32 bits: 2e-5 of the loss's terms and of the probabilities (their exponents are below 2^6)
    assert abs(float(loss) - float(each.sum() / count)) <= 2e-5 * (1 + float(each.sum() / count))
    # four factors and differences in 32 bits; bf16: rounded once (the longer rows' gradient in the forward pass: doubling it is exact)
    rounding = 4 * U + (H if dtype == torch.bfloat16 else 0)
    assert bool(((g.double() - dz).abs() <= rounding * dz.abs() + 2e-5 * 2.0 * (logp.exp() / count) * has[:, None] + 1e-38).all())
    assert bool((g[~has] == 0).all())


@pytest.mark.parametrize("vocab", [1000, 1100, 66000])
@pytest.mark.parametrize("packed", [False, True])
def test_gpt2_targets_mean_the_same_at_every_vocabulary(ops, vocab, packed):
    """Targets outside the vocabulary do not count, in a batch or packed, on either side of what the fused head takes; the
    gradients agree with the fp32 model on the CPU in direction and size."""
    import copy

    from pytorch_distributed_training_amd.models.gpt2 import gpt2_tiny

    torch.manual_seed(0)
    ref = gpt2_tiny(vocab_size=vocab, n_ctx=32)
    gpu = ops.prepare_module(copy.deepcopy(ref).cuda())
    idx = torch.randint(0, vocab, (2, 32))
    targets = torch.randint(0, vocab, (2, 32))
    targets[0, 5:] = -100
    targets[1, ::2] = -100
    if packed:
        idx, targets = idx.flatten(), targets.flatten()
        a = ref(idx, targets, pack=ops.pack_sequences([0, 32, 64], 64))
        b = gpu(idx.cuda(), targets.cuda(), pack=ops.pack_sequences([0, 32, 64], 64, device="cuda"))
    else:
        a, b = ref(idx, targets), gpu(idx.cuda(), targets.cuda())
    a.backward(), b.backward()
    # bf16 activations through two blocks: each rounds at 2^-8 of the value a dozen times, at random
    assert abs(float(a) - float(b)) < 12 * H
    for (name, p), r in zip(ref.named_parameters(), gpu.parameters()):
        g, w = r.grad.cpu().double().flatten(), p.grad.double().flatten()
        assert float((g - w).norm()) <= 12 * H * float(w.norm()) + 1e-9, (name, float((g - w).norm() / w.norm()))


def test_fused_head_without_any_label(ops):
    x, w = _bf16(8, 64).requires_grad_(True), torch.nn.Parameter(_bf16(2000, 64, seed=1).float())
    loss = ops.lm_head_loss(x, w, torch.full((8,), -100, device="cuda"))
    loss.backward()
    assert float(loss) == 0.0 and bool((x.grad == 0).all()) and bool((w.grad == 0).all())


@pytest.mark.parametrize("near", [0.0, 0.003, 0.03])
def test_students_close_to_their_teacher(ops, near):
    """q - p at the targets is a small difference there: both are formed in 32 bits, and only the difference is rounded."""
    n, vocab, width, top, tau = 70, 4000, 256, 64, 1.0
    # small whole numbers and eighths: every score is exact in 32 bits; the highest share two groups of 64 entries, so that
    # most of them are not the largest of their group
    x = torch.randint(-3, 4, (n, width), generator=_gen(1), device="cuda").to(torch.bfloat16).requires_grad_(True)
    w = torch.randint(-3, 4, (vocab, width), generator=_gen(2), device="cuda").to(torch.bfloat16) / 8
    w[128:] /= 4
    w.requires_grad_(True)
    x64, w64 = x.detach().double(), w.detach().double()
    z = x64 @ w64.t()
    ids = z.topk(top, 1).indices
    teacher = (z.gather(1, ids) + near * torch.randn(n, top, generator=_gen(3), device="cuda")).float()
    loss = ops.linear_distillation_loss(x, w, teacher, ids, tau)
    dx, dw = torch.autograd.grad(loss, (x, w))
    q, p = torch.softmax(z, 1), torch.softmax(teacher.double(), 1)
    dz = q.scatter_add(1, ids, -p) / n
    # q of entries that are no targets: an exponential and its multiple, each rounded; q - p at the targets: rounded once;
    # exponents below 2^6 and sums in 32 bits: 2e-5 of q and p
    others = q.scatter(1, ids, 0.0) / n
    f = 2.01 * H * others + H * (dz - others).abs() + 2e-5 * (q / n).scatter_add(1, ids, p / n)
    for got, want, bound in ((dx, dz @ w64, f @ w64.abs()), (dw, dz.t() @ x64, f.t() @ x64.abs())):
        terms = dz.abs() @ w64.abs() if got is dx else dz.abs().t() @ x64.abs()
        over = (got.double() - want).abs() - 1.05 * (bound + H * want.abs() + vocab * U * terms)
        assert float(over.max()) <= 0, float(over.max())


def _uniform(n_rows, keys, hk, d, seed, value_scale):
    """Documents of `keys` rows (a power of two) whose keys all get the same weight, exactly; their values share a large part,
    so that dS = P (dout.v - dout.out) is a small difference; dout has the sign of what rounding takes from out."""
    base = torch.rand(n_rows // keys, 1, hk, d, generator=_gen(seed), device="cuda") + 1.5
    near = torch.randn(n_rows // keys, keys, hk, d, generator=_gen(seed + 1), device="cuda") * 0.02
    v = ((base + near) * value_scale).to(torch.bfloat16).reshape(n_rows, hk, d)
    out = v.double().reshape(-1, keys, hk, d).mean(1, keepdim=True).expand(-1, keys, hk, d).reshape(n_rows, hk, d)
    taken = out - out.to(torch.bfloat16).double()
    return v, out, taken, torch.where(taken >= 0, 1.0, -1.0).to(torch.bfloat16)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("keys", [2, 8, 32])
@pytest.mark.parametrize("value_scale", [2.0 ** -30, 2.0 ** -14, 1.0, 2.0 ** 20])
@pytest.mark.parametrize("beside_nan", [False, True])
def test_row_terms_from_unrounded_outputs(ops, d, keys, value_scale, beside_nan):
    """The backward pass knows out to an eighth of what its rounding took, whatever the size of the values; rows that share
    tiles with NaN (done one by one) know it too."""
    rows, heads = 256, 2
    v, out, taken, dout = _uniform(rows, keys, heads, d, keys, value_scale)
    other = _bf16(rows, heads, d, seed=9)
    zero = torch.zeros_like(other)
    clean = torch.ones(rows, dtype=torch.bool, device="cuda")
    if beside_nan:
        v = v.clone()
        for first in range(0, rows, 64):
            v[first:first + keys] = math.nan
            clean[first:first + keys] = False
    pack = ops.pack_sequences(list(range(0, rows + 1, keys)), rows, device="cuda")
    scale = d ** -0.5
    v64, g64, o64 = torch.nan_to_num(v.double()), dout.double(), other.double()
    by = lambda x: x.reshape(rows // keys, keys, heads, d).transpose(1, 2)  # [documents, heads, keys, d]
    back = lambda x: x.transpose(1, 2).reshape(rows, heads, d)
    p = 1.0 / keys
    dp = by(g64) @ by(v64).transpose(2, 3)
    ds = p * (dp - (by(g64) * by(out)).sum(-1, keepdim=True))
    # dS rounded once; the row term off by an eighth of what rounding took; sums of d products in 32 bits
    term = (by(g64).abs() * by(taken).abs()).sum(-1, keepdim=True) / 8 + (d + 16) * U * (by(g64).abs() * by(out).abs()).sum(-1, keepdim=True)
    f = H * ds.abs() + p * (term + (d + 16) * U * (by(g64).abs() @ by(v64).abs().transpose(2, 3)))
    for q, k, index in ((zero, other, 0), (other, zero, 1)):  # scores of 0 either way: weights of 1 / keys
        q, k = q.clone().requires_grad_(True), k.clone().requires_grad_(True)
        res = ops.attention_packed(q, k, v, pack, causal=False)
        assert torch.equal(res.detach()[clean], out[clean].to(torch.bfloat16))
        got = torch.autograd.grad(res, (q, k), dout)[index]
        side, ff = (ds, f) if index == 0 else (ds.transpose(2, 3), f.transpose(2, 3))
        want, bound = back(scale * side @ by(o64)), back(scale * ff @ by(o64).abs())
        over = ((got.double() - want).abs() - 1.05 * (bound + H * want.abs() + 1e-37))[clean]
        assert float(over.max()) <= 0, float((over / bound[clean]).max())


def test_second_derivative_of_the_packed_embedding_is_refused(ops):
    wte, wpe = (torch.randn(10, 64, device="cuda", requires_grad=True) for _ in range(2))
    g = torch.ones(6, 64, dtype=torch.bfloat16, device="cuda", requires_grad=True)
    pack = ops.pack_sequences([0, 6], 6, device="cuda")
    out = ops.token_position_embedding(torch.arange(6, device="cuda"), wte, wpe, pack)
    for table in (wte, wpe):
        (d,) = torch.autograd.grad(out, table, g, create_graph=True, retain_graph=True)
        with pytest.raises(RuntimeError, match="once_differentiable"):
            (d * d).sum().backward()


def test_gradients_with_a_graph_are_not_added_on_the_quiet(ops):
    """Under create_graph a parameter whose .grad the kernels may add into gets a gradient that refuses its own derivative."""
    x, ids = _bf16(6, 64).requires_grad_(True), torch.arange(6, device="cuda")
    pack = ops.pack_sequences([0, 6], 6, device="cuda")
    for call in (lambda w: ops.linear_cross_entropy(x, w, ids), lambda w: ops.token_position_embedding(ids, w, w, pack).float().pow(2).sum()):
        plain = torch.nn.Parameter(_bf16(70, 64, seed=1).float())
        call(plain).backward()
        w = torch.nn.Parameter(plain.detach().clone())
        w.grad, w._pdt_sink_ok = torch.zeros_like(w), True
        call(w).backward(create_graph=True)
        assert torch.equal(w.grad.detach(), plain.grad)
        with pytest.raises(RuntimeError, match="once_differentiable"):
            w.grad.pow(2).sum().backward()


def test_derivatives_of_gradients_by_the_inputs_are_refused(ops):
    """Also where the incoming gradient is a constant (a gradient penalty on a loss)."""
    ids, pack = torch.arange(12, device="cuda").view(6, 2), ops.pack_sequences([0, 6], 6, device="cuda")
    x, z, q = (_bf16(*s, seed=i).requires_grad_(True) for i, s in enumerate([(6, 64), (6, 70), (6, 1, 64)]))
    w, do = _bf16(70, 64, seed=4), _bf16(6, 1, 64, seed=5)
    calls = [(x, ops.linear_cross_entropy(x, w, ids[:, 0]), None), (z, ops.distillation_loss(z, torch.zeros(6, 2, device="cuda"), ids), None),
             (q, ops.attention_packed(q, do, do, pack), do), (q, ops.attention_packed_qkv(torch.cat([q, do, do], 1).flatten(1), pack, 1), do.flatten(1))]
    for leaf, out, g in calls:
        (d,) = torch.autograd.grad(out, leaf, g, create_graph=True)
        with pytest.raises(RuntimeError, match="once_differentiable"):
            (leaf.float().sum() + d.float().pow(2).sum()).backward()


def test_as_many_rows_as_there_may_be(ops):
    """2^22 - 64 equal rows: the loss is a row's, the gradients are the row's share of them."""
    n, vocab = (1 << 22) - 64, 50
    row, w = _bf16(1, 64), (_bf16(vocab, 64, seed=1) / 8).requires_grad_(True)
    x = row.repeat(n, 1).requires_grad_(True)
    loss = ops.linear_cross_entropy(x, w, torch.full((n,), 7, device="cuda", dtype=torch.int32))
    dx, dw = torch.autograd.grad(loss, (x, w))
    r, w64 = row.double(), w.detach().double()
    q = torch.softmax(r @ w64.t(), 1)
    want = -torch.log(q[0, 7])
    d = q.clone()
    d[0, 7] -= 1
    # sums over the rows: a term is off by n 2^-24 of the sum at most where it is added one by one; 256 workgroups and 16 terms
    # a product and more share them: 1024 + 256
    sums = (n / 256 / 16 + 256) * U
    assert abs(float(loss) - float(want)) <= (1e-5 + 4096 * U) * float(want)  # (a thread adds 4096 row losses)
    f = 2 * H * q + H * d.abs() + 2e-5 * q
    assert torch.equal(dx[0], dx[-1]) and torch.equal(dx[0], dx[n // 2 + 1])
    assert bool(((dx[:1].double() * n - d @ w64).abs() <= 1.05 * (f @ w64.abs() + H * (d @ w64).abs())).all())
    assert bool(((dw.double() - d.t() @ r).abs() <= 1.05 * (f.t() @ r.abs() + (H + sums) * (d.t() @ r).abs())).all())


def test_backward_pass_alone_is_not_captured(ops, monkeypatch):
    """The losses' gradients lie in the forward pass's buffers and are scaled in place: a graph that holds the backward pass without
    the forward pass would scale them again at every replay, so it is refused (the stream is only said to be captured here)."""
    x, w, z = _bf16(6, 64).requires_grad_(True), _bf16(70, 64, seed=1), _bf16(6, 70, seed=2).requires_grad_(True)
    ids, teacher = torch.arange(12, device="cuda").view(6, 2), torch.zeros(6, 2, device="cuda")
    for leaf, loss in ((x, ops.linear_cross_entropy(x, w, ids[:, 0])), (z, ops.distillation_loss(z, teacher, ids))):
        with monkeypatch.context() as m:
            m.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
            with pytest.raises(RuntimeError, match="captured"):
                torch.autograd.grad(loss, leaf, retain_graph=True)
        (g,) = torch.autograd.grad(loss, leaf)  # nothing was taken
        assert bool(torch.isfinite(g).all())


def test_forward_and_backward_in_a_graph_each(ops):
    """As torch's own graphed callables record them: the forward pass's graph, then the backward pass's, replayed in turn with eager work
    between; every round's gradients are those of its inputs and its factor."""
    x, w = _bf16(40, 64).requires_grad_(True), _bf16(70, 64, seed=1).requires_grad_(True)
    z, t = _bf16(40, 70, seed=2).requires_grad_(True), torch.randn(40, 2, generator=_gen(3), device="cuda")
    ids = torch.randint(0, 70, (40, 2), generator=_gen(4), device="cuda")
    factor = torch.tensor(3.0, device="cuda")
    for call, leaves in ((lambda: ops.linear_cross_entropy(x, w, ids[:, 0]), (x, w)), (lambda: ops.distillation_loss(z, t, ids), (z,))):
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            torch.autograd.grad(call(), leaves, factor)
        torch.cuda.current_stream().wait_stream(side)
        first, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(first):
            loss = call()
        with torch.cuda.graph(second, pool=first.pool()):
            got = torch.autograd.grad(loss, leaves, factor)
        for n in range(3):
            with torch.no_grad():
                for leaf in leaves:
                    leaf.normal_(generator=_gen(10 + n))
                factor.fill_(2.0 + n)
            first.replay()
            second.replay()
            torch.cuda.synchronize()
            kept = [loss.detach().clone()] + [g.clone() for g in got]
            again = call()
            want = [again.detach(), *torch.autograd.grad(again, leaves, factor)]
            assert all(torch.equal(a, b) for a, b in zip(kept, want))
            del again


def test_losses_without_a_gradient_in_pieces(ops, monkeypatch):
    """Rows are worked off in pieces without a gradient too: the row statistics (8 bytes per 64 entries) of one piece at a time."""
    from pytorch_distributed_training_amd.ops import hip_vocab

    n, vocab, width = 2000, 50257, 64
    x, w = _bf16(n, width), _bf16(vocab, width, seed=1)
    y = torch.randint(0, vocab, (n,), generator=_gen(2), device="cuda")
    teacher, ids = torch.randn(n, 3, generator=_gen(3), device="cuda"), torch.randint(0, vocab, (n, 3), generator=_gen(4), device="cuda")
    groups = (vocab + 63) // 64

    def peak(call):
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        return call(), torch.cuda.max_memory_allocated() - before

    for call in (lambda: ops.linear_cross_entropy(x, w, y), lambda: ops.linear_distillation_loss(x, w, teacher, ids, 2.0)):
        whole, much = peak(call)
        with monkeypatch.context() as m:
            m.setattr(hip_vocab, "CHUNK_BYTES", 300 * 8 * groups)
            pieces, little = peak(call)
        assert torch.equal(whole, pieces)
        assert much >= n * 8 * groups and little < 256 * 8 * groups + (1 << 20)


@pytest.mark.parametrize("tau", [1e-3, 0.05])
def test_students_equal_to_their_teacher_at_low_temperatures(ops, tau):
    """Exponents of 10^4 and more: q is formed from differences to the row's maximum, so that it agrees with p to 32 bits."""
    n, vocab, width, top = 40, 700, 128, 8
    x = torch.randint(-3, 4, (n, width), generator=_gen(1), device="cuda").to(torch.bfloat16).requires_grad_(True)
    w = (torch.randint(-3, 4, (vocab, width), generator=_gen(2), device="cuda").to(torch.bfloat16) / 8).requires_grad_(True)
    x64, w64 = x.detach().double(), w.detach().double()
    with torch.no_grad():
        w[1], w[2] = w[0], w[0]  # a few entries that share the maximum
        x.abs_()
        w[:3] = w[:3].abs() + 0.125
    x64, w64 = x.detach().double(), w.detach().double()
    z = x64 @ w64.t()
    ids = z.topk(top, 1).indices
    teacher = z.gather(1, ids).float()
    dx, dw = torch.autograd.grad(ops.linear_distillation_loss(x, w, teacher, ids, tau), (x, w))
    q, p = torch.softmax(z / tau, 1), torch.softmax(teacher.double() / tau, 1)
    dz = q.scatter_add(1, ids, -p) * (tau / n)
    others = q.scatter(1, ids, 0.0) * (tau / n)
    f = 2.01 * H * others + H * (dz - others).abs() + 2e-5 * (tau / n) * q.scatter_add(1, ids, p)
    for got, want, bound in ((dx, dz @ w64, f @ w64.abs()), (dw, dz.t() @ x64, f.t() @ x64.abs())):
        over = (got.double() - want).abs() - 1.05 * (bound + H * want.abs())
        assert float(over.max()) <= 0, float(over.max())
