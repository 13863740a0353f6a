"""Packed attention on the GPU against the formulas in 64 bits (needs an MI355X).

Tolerances follow from the kernel's roundings alone, element by element: probabilities, score gradients and results are
rounded to bf16, off by at most h = 2^-8 of the value each.  With P the exact probabilities,
    |out - ref|  <= h (P |v|) + h |ref|                                                        =: E
    |dv - ref|   <= h (P' |dout|) + h |ref|
    |ds - ref|   <= h |ds| + P (|dout| E)   (the row term dout.out uses the rounded out)       =: F
    |dq - ref|   <= scale (F |k|) + h |ref|,   |dk - ref| <= scale (F' |q|) + h |ref|
Sums in 32 bits, exp2 (1 ulp of a 32-bit exponent of magnitude < 2^6) and second-order terms: 5 % on top, and 2e-5 of the
sums' terms in place of zero.
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


def _inputs(t, h, hk, d, seed=0, std=1.0):
    g = torch.Generator("cuda").manual_seed(seed)
    r = lambda n: (torch.randn(t, n, d, generator=g, device="cuda") * std).to(torch.bfloat16)
    return r(h), r(hk), r(hk), r(h)


def _expected(q, k, v, do, offsets, causal, scale):
    """(values, error bounds) of out, dq, dk, dv in 64 bits, one sequence and head at a time."""
    q, k, v, do = (x.double() for x in (q, k, v, do))
    group = q.shape[1] // k.shape[1]
    val = [torch.zeros_like(x) for x in (q, q, k, v)]
    err = [torch.zeros_like(x) for x in (q, q, k, v)]
    for a, e in zip(offsets[:-1], offsets[1:]):
        for j in range(q.shape[1]):
            qs, ks, vs, ds_ = q[a:e, j], k[a:e, j // group], v[a:e, j // group], do[a:e, j]
            s = qs @ ks.t() * scale
            if causal:
                s = s.masked_fill(torch.ones_like(s, dtype=torch.bool).triu(1), -math.inf)
            p = torch.softmax(s, -1)
            o = p @ vs
            eo = (H + 2e-5) * (p @ vs.abs()) + H * o.abs()
            dp = ds_ @ vs.t()
            ds = p * (dp - (ds_ * o).sum(-1, keepdim=True))
            f = H * ds.abs() + p * ((ds_.abs() * eo).sum(-1, keepdim=True) + 2e-5 * (ds_.abs() @ vs.abs().t()))
            val[0][a:e, j], err[0][a:e, j] = o, eo
            val[1][a:e, j], err[1][a:e, j] = scale * ds @ ks, scale * f @ ks.abs()
            val[2][a:e, j // group] += scale * ds.t() @ qs
            err[2][a:e, j // group] += scale * f.t() @ qs.abs()
            val[3][a:e, j // group] += p.t() @ ds_
            err[3][a:e, j // group] += (H + 2e-5) * p.t() @ ds_.abs()
    return val, [e + (0 if i == 0 else H) * x.abs() for i, (x, e) in enumerate(zip(val, err))]


def _check(got, val, err, what=("out", "dq", "dk", "dv")):
    for name, x, y, e in zip(what, got, val, err):
        assert x.shape == y.shape and bool(torch.isfinite(x).all()), name
        over = (x.double() - y).abs() - 1.05 * e
        assert float(over.max()) <= 0, f"{name}: {float(over.max()):.3g} over its bound at {int(over.argmax())}"


def _offsets(lengths, first=0):
    o = [first]
    for n in lengths:
        o.append(o[-1] + n)
    return o


CASES = [
    # lengths, rows in front, rows behind, H, Hk, D, causal
    ([1], 0, 0, 1, 1, 64, True),
    ([2, 1, 0, 3], 0, 2, 2, 2, 128, True),
    ([63, 64, 65, 1, 127, 129], 0, 3, 4, 2, 64, True),
    ([63, 64, 65, 1, 127, 129], 5, 3, 4, 1, 128, False),
    ([31, 33, 1, 1, 1, 200, 7, 300], 0, 0, 6, 3, 128, True),
    ([1] * 200, 0, 1, 3, 3, 64, True),
    ([1] * 130, 1, 0, 2, 1, 128, False),
    ([700], 0, 0, 8, 1, 64, True),
    ([1000, 24, 513], 0, 0, 5, 5, 64, False),
    ([640, 383], 0, 0, 16, 2, 128, True),
]


@pytest.mark.parametrize("lengths,front,behind,h,hk,d,causal", CASES)
def test_forward_and_gradients(ops, lengths, front, behind, h, hk, d, causal):
    offsets = _offsets(lengths, front)
    t = offsets[-1] + behind
    q, k, v, do = _inputs(t, h, hk, d, seed=t)
    for x in (q, k, v):
        x.requires_grad_(True)
    pack = ops.pack_sequences(torch.tensor(offsets, dtype=torch.int32, device="cuda"), t)
    host = ops.pack_sequences(offsets, t)
    assert torch.equal(pack.spans.cpu(), host.spans) and torch.equal(pack.positions.cpu(), host.positions)
    out = ops.attention_packed(q, k, v, pack, causal=causal)
    got = (out, *torch.autograd.grad(out, (q, k, v), do))
    val, err = _expected(q.detach(), k.detach(), v.detach(), do, offsets, causal, d ** -0.5)
    _check([x.detach() for x in got], val, err)  # (rows outside: values and bounds are zero)


@pytest.mark.parametrize("h,hk,d", [(4, 2, 64), (3, 1, 128)])
def test_joint_projection_views_and_scale(ops, h, hk, d):
    """The joint form, views with gaps, other axis orders and another scale give what separate tensors give."""
    offsets, t = _offsets([70, 3, 130]), 205
    q, k, v, do = _inputs(t, h, hk, d, seed=7)
    pack = ops.pack_sequences(offsets, t, device="cuda")
    val, err = _expected(q, k, v, do, offsets, True, 0.11)
    joint = torch.cat([q, k, v], 1).reshape(t, -1).requires_grad_(True)
    out = ops.attention_packed_qkv(joint, pack, h, hk, scale=0.11)
    (g,) = torch.autograd.grad(out, joint, do.reshape(t, -1))
    g = g.view(t, h + 2 * hk, d)
    a = [out.detach().view(t, h, d), g[:, :h], g[:, h:h + hk], g[:, h + hk:]]
    _check(a, val, err)
    wide = torch.zeros(t, h, d + 8, dtype=torch.bfloat16, device="cuda")
    wide[:, :, :d] = q
    qv = wide[:, :, :d].requires_grad_(True)                              # rows with gaps
    kv = k.transpose(0, 1).contiguous().transpose(0, 1).requires_grad_(True)  # heads outermost
    odd = torch.zeros(v.numel() + 1, dtype=torch.bfloat16, device="cuda")
    vv = odd[1:].view(v.shape).copy_(v).requires_grad_(True)              # not on a 16-byte boundary
    gout = do.transpose(0, 1).contiguous().transpose(0, 1)
    out = ops.attention_packed(qv, kv, vv, pack, scale=0.11)
    b = [out.detach(), *torch.autograd.grad(out, (qv, kv, vv), gout)]
    for x, y in zip(a, b):
        assert torch.equal(x, y)


def test_fp32_inputs_are_computed_in_bf16(ops):
    q, k, v, do = _inputs(40, 2, 2, 64)
    pack = ops.pack_sequences([0, 40], 40, device="cuda")
    ref = ops.attention_packed(q, k, v, pack)
    qf = q.float().requires_grad_(True)
    out = ops.attention_packed(qf, k.float(), v.float(), pack)
    assert torch.equal(out.detach(), ref)
    (g,) = torch.autograd.grad(out, qf, do)
    assert g.dtype == torch.float32


@pytest.mark.parametrize("d", [64, 128])
def test_large_scores_and_rising_maximum(ops, d):
    """Scores far beyond the first keys' (the running maximum has to follow) and far below zero."""
    offsets, t = _offsets([300, 200]), 500
    q, k, v, do = _inputs(t, 2, 1, d, seed=3)
    k[150:300] *= 16  # from the middle of the first sequence on
    k[300:] *= 20
    q[300:] = -k[300:, :1].clone() / 8  # the diagonal is hugely negative
    pack = ops.pack_sequences(offsets, t, device="cuda")
    with torch.no_grad():
        out = ops.attention_packed(q, k, v, pack)
    val, err = _expected(q, k, v, do, offsets, True, d ** -0.5)
    # scores of magnitude s are off by s 2^-23 in 32 bits (products summed in fp32: s 2^-20 over d terms), so are exponents
    s = float((q.double().abs().amax() * k.double().abs().amax()) * d ** 0.5)
    slack = 2 * s * 2.0 ** -20
    assert slack < 0.05
    over = (out.double() - val[0]).abs() - 1.05 * err[0] - slack * v.double().abs().amax()
    assert float(over.max()) <= 0


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_other_sequences_and_later_rows_do_not_show(ops, d, bad):
    """NaN or infinity in one sequence, in rows outside and behind a row leave every other result as it is."""
    offsets, t = [2, 40, 110, 150], 154
    q, k, v, do = _inputs(t, 4, 2, d, seed=11)
    pack = ops.pack_sequences(offsets, t, device="cuda")

    def run(q, k, v, do):
        q, k, v = (x.clone().requires_grad_(True) for x in (q, k, v))
        out = ops.attention_packed(q, k, v, pack)
        return [out.detach(), *torch.autograd.grad(out, (q, k, v), do)]

    val, err = _expected(q, k, v, do, offsets, True, d ** -0.5)
    q2, k2, v2, do2 = (x.clone() for x in (q, k, v, do))
    for x in (q2, k2, v2, do2):
        x[:2] = bad
        x[150:] = bad
        x[60:110] = bad  # the second sequence from its 20th row on
    got = run(q2, k2, v2, do2)
    keep = torch.ones(t, dtype=torch.bool, device="cuda")
    keep[40:110] = False
    _check([x[keep] for x in got], [x[keep] for x in val], [x[keep] for x in err])
    for i in (0, 1):  # rows in front of the bad ones: their outputs and query gradients
        _check([got[i][40:60]], [val[i][40:60]], [err[i][40:60]], [("out", "dq")[i]])
    assert not torch.isfinite(got[0][60:110]).any()


def test_offsets_beyond_the_rows_are_cut(ops):
    q, k, v, _ = _inputs(20, 2, 2, 64)
    far = ops.pack_sequences(torch.tensor([0, 5, 900], device="cuda"), 20)
    cut = ops.pack_sequences([0, 5, 20], 20, device="cuda")
    assert torch.equal(far.spans, cut.spans)
    assert torch.equal(ops.attention_packed(q, k, v, far), ops.attention_packed(q, k, v, cut))


def test_same_bits_every_time_and_on_another_stream(ops):
    offsets, t = _offsets([300, 77, 400]), 777
    q, k, v, do = _inputs(t, 8, 2, 128, seed=5)
    for x in (q, k, v):
        x.requires_grad_(True)
    pack = ops.pack_sequences(offsets, t, device="cuda")

    def run():
        out = ops.attention_packed(q, k, v, pack)
        return (out.detach(), *torch.autograd.grad(out, (q, k, v), do))

    first = run()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        other = run()
    side.synchronize()
    for x, y, z in zip(first, run(), other):
        assert torch.equal(x, y) and torch.equal(x, z)


def test_captured_graph_follows_new_offsets_and_inputs(ops):
    """Everything, the pack included, replayed over inputs and offsets written in place."""
    t, h, hk, d = 260, 4, 2, 64
    q, k, v, do = _inputs(t, h, hk, d)
    offsets = torch.tensor([0, 100, 260], dtype=torch.int32, device="cuda")
    leaves = [x.requires_grad_(True) for x in (q, k, v)]

    def run():
        out = ops.attention_packed(q, k, v, ops.pack_sequences(offsets, t))
        return (out, *torch.autograd.grad(out, leaves, do))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run()
    for i, new in enumerate(([0, 1, 260], [0, 128, 256], [3, 200, 230], [0, 260, 260])):
        offsets.copy_(torch.tensor(new, dtype=torch.int32))
        with torch.no_grad():
            for x, y in zip((q, k, v, do), _inputs(t, h, hk, d, seed=i + 50)):
                x.copy_(y)
        graph.replay()
        torch.cuda.synchronize()
        want = [x.detach().clone() for x in run()]
        for x, y in zip(got, want):
            assert torch.equal(x, y)


def test_refusals(ops):
    q, k, v, _ = _inputs(6, 2, 2, 64)
    pack = ops.pack_sequences([0, 6], 6, device="cuda")
    with pytest.raises(ValueError, match="head_dim"):
        ops.attention_packed(q[..., :32], k[..., :32], v[..., :32], pack)
    with pytest.raises(ValueError, match="pack on"):
        ops.attention_packed(q, k, v, ops.pack_sequences([0, 6], 6))
    with pytest.raises(ValueError, match="offsets on"):
        ops.pack_sequences(torch.tensor([0, 6], device="cuda"), 6, device="cpu")


def test_packed_embedding(ops):
    g = torch.Generator("cuda").manual_seed(0)
    wte, wpe = torch.randn(50, 64, generator=g, device="cuda"), torch.randn(20, 64, generator=g, device="cuda")
    ids = torch.randint(0, 50, (33,), generator=g, device="cuda")
    pack = ops.pack_sequences([0, 20, 20, 31], 33, device="cuda")
    wte.requires_grad_(True), wpe.requires_grad_(True)
    out = ops.token_position_embedding(ids, wte, wpe, pack)
    assert torch.equal(out, (wte[ids] + wpe[pack.positions]).to(torch.bfloat16))  # one rounding of the fp32 sum
    do = torch.randn(33, 64, generator=g, device="cuda").to(torch.bfloat16)
    a, b = torch.autograd.grad(out, (wte, wpe), do)
    ra = torch.zeros_like(wte, dtype=torch.float64).index_add_(0, ids, do.double())
    rb = torch.zeros_like(wpe, dtype=torch.float64).index_add_(0, pack.positions, do.double())
    # fp32 sums of at most 33 terms of magnitude below 8
    assert float((a.double() - ra).abs().max()) < 33 * 33 * 8 * 2.0 ** -24 and float((b.double() - rb).abs().max()) < 33 * 33 * 8 * 2.0 ** -24
    with pytest.raises(ValueError, match="exceeds"):
        ops.token_position_embedding(ids, wte, wpe[:19], pack)
    with pytest.raises(ValueError, match="packed tokens"):
        ops.token_position_embedding(ids.cpu(), wte, wpe, pack)


@pytest.mark.parametrize("with_teacher", [False, True])
def test_gpt2_trains_on_packed_documents(ops, with_teacher):
    """Embedding, attention, projection and loss together: the packed GPU model against the fp32 model on the CPU, with the
    gradients left in .grad by the kernels and an optimizer step behind them."""
    import copy

    from pytorch_distributed_training_amd.models.gpt2 import gpt2_tiny
    from pytorch_distributed_training_amd.optim import build_optimizer

    torch.manual_seed(0)
    ref = gpt2_tiny(vocab_size=2000, n_ctx=64)
    gpu = ops.prepare_module(copy.deepcopy(ref).cuda())
    for p in gpu.parameters():
        p.grad = torch.zeros_like(p)
    offsets, rows = _offsets([60, 1, 33, 64, 5]), 165
    idx = torch.randint(0, 2000, (rows,))
    targets = torch.roll(idx, -1)
    targets[[o - 1 for o in offsets[1:]]] = -100
    targets[163:] = -100
    teacher = (torch.randn(rows, 8) * 3, torch.randint(0, 2000, (rows, 8)))
    cpu_pack, gpu_pack = ops.pack_sequences(offsets, rows), ops.pack_sequences(offsets, rows, device="cuda")
    if with_teacher:
        a = ref(idx, pack=cpu_pack, teacher=teacher, temperature=2.0)
        b = gpu(idx.cuda(), pack=gpu_pack, teacher=tuple(t.cuda() for t in teacher), temperature=2.0)
    else:
        a, b = ref(idx, targets, pack=cpu_pack), gpu(idx.cuda(), targets.cuda(), pack=gpu_pack)
    a.backward(), b.backward()
    # bf16 activations through two blocks: each rounds at 2^-8 of the value a dozen times, at random
    assert abs(float(a) - float(b)) < 12 * 2.0 ** -8
    for (n, x), y in zip(ref.named_parameters(), gpu.parameters()):
        cos = torch.nn.functional.cosine_similarity(x.grad.flatten(), y.grad.cpu().flatten(), dim=0)
        assert cos > 0.99, (n, float(cos))
    before = [p.detach().clone() for p in gpu.parameters()]
    build_optimizer(gpu.parameters(), "adamw", 1e-3, 0.0, 0.9).step()
    again = gpu(idx.cuda(), targets.cuda(), pack=gpu_pack)
    assert torch.isfinite(again) and any(not torch.equal(x, y) for x, y in zip(before, gpu.parameters()))


@pytest.mark.parametrize("d", [64, 128])
def test_offsets_of_64_bits_and_rows_far_apart(ops, d):
    """Row strides that carry the last rows past 2^32 bytes and 2^31 elements; 64-bit offsets past 2^32 are cut off."""
    t, h, hk = 300, 2, 1
    q, k, v, do = _inputs(t, h, hk, d, seed=11)
    room = torch.empty(t, 1 << 23, dtype=torch.bfloat16, device="cuda")
    far = []
    for i, x in enumerate((q, k, v)):
        at = room[:, 1024 * i:1024 * i + x.shape[1] * d].unflatten(1, (x.shape[1], d))
        far.append(at.copy_(x).detach().requires_grad_(True))
    assert far[0].stride(0) * (t - 1) > 1 << 31
    pack = ops.pack_sequences(torch.tensor([0, 100, (1 << 32) + 5], device="cuda"), t)
    same = ops.pack_sequences([0, 100, t], t, device="cuda")
    assert torch.equal(pack.spans, same.spans)
    near = [x.requires_grad_(True) for x in (q, k, v)]
    a, b = ops.attention_packed(*far, pack), ops.attention_packed(*near, same)
    assert torch.equal(a, b)
    for x, y in zip(torch.autograd.grad(a, far, do), torch.autograd.grad(b, near, do)):
        assert torch.equal(x, y)


def test_no_rows_no_sequences_and_some_gradients(ops):
    q, k, v, do = _inputs(70, 4, 2, 64)
    none = ops.pack_sequences(torch.zeros(1, dtype=torch.int64, device="cuda"), 70)
    out = ops.attention_packed(q.requires_grad_(True), k, v, none)
    (dq,) = torch.autograd.grad(out, q, do)
    assert out.abs().max() == 0 and dq.abs().max() == 0
    nothing = ops.pack_sequences([0, 0], 0, device="cuda")
    empty = [x[:0].detach().requires_grad_(True) for x in (q, k, v)]
    out = ops.attention_packed(*empty, nothing)
    assert out.shape == (0, 4, 64) and all(g.shape == x.shape for g, x in zip(torch.autograd.grad(out.sum(), empty), empty))
    assert ops.attention_packed_qkv(torch.zeros(0, 8 * 64, device="cuda"), nothing, 4, 2).shape == (0, 256)
    pack = ops.pack_sequences([0, 33, 70], 70, device="cuda")
    q, k, v = (x.detach().requires_grad_(True) for x in (q, k, v))
    every = torch.autograd.grad(ops.attention_packed(q, k, v, pack), (q, k, v), do)
    for i, name in enumerate("qkv"):
        leaf = (q, k, v)[i]
        (one,) = torch.autograd.grad(ops.attention_packed(*(x if x is leaf else x.detach() for x in (q, k, v)), pack), leaf, do)
        assert torch.equal(one, every[i]), name
    # keys and values given as one head expanded over the key heads
    k1, v1 = (x.detach()[:, :1].expand(-1, 2, -1).requires_grad_(True) for x in (k, v))
    a = ops.attention_packed(q, k1, v1, pack)
    b = ops.attention_packed(q, k1.detach().contiguous(), v1.detach().contiguous(), pack)
    assert torch.equal(a, b)
    # the first pass' graph used twice
    out = ops.attention_packed(q, k, v, pack)
    once, twice = torch.autograd.grad(out, (q, k, v), do, retain_graph=True), torch.autograd.grad(out, (q, k, v), do)
    assert all(torch.equal(x, y) for x, y in zip(once, twice))


@pytest.mark.parametrize("dtype", [torch.float16, torch.float64])
def test_other_input_types(ops, dtype):
    q, k, v, do = (x.to(torch.float16).to(torch.bfloat16) for x in _inputs(40, 2, 1, 128, seed=3))  # (values that every type holds)
    pack = ops.pack_sequences([0, 40], 40, device="cuda")
    other = [x.to(dtype).requires_grad_(True) for x in (q, k, v)]
    own = [x.requires_grad_(True) for x in (q, k, v)]
    a, b = ops.attention_packed(*other, pack), ops.attention_packed(*own, pack)
    assert a.dtype == torch.bfloat16 and torch.equal(a, b)
    for x, y in zip(torch.autograd.grad(a, other, do), torch.autograd.grad(b, own, do)):
        assert x.dtype == dtype and torch.equal(x, y.to(dtype))


def test_two_streams_at_once_with_one_pack(ops):
    t = 3000
    pack = ops.pack_sequences([0, 900, 901, 2990], t, device="cuda")
    sets = [[x.requires_grad_(i < 3) for i, x in enumerate(_inputs(t, 8, 2, d, seed=d))] for d in (64, 128)]

    def run(s):
        out = ops.attention_packed(*s[:3], pack)
        return (out.detach(), *torch.autograd.grad(out, s[:3], s[3]))

    want = [run(s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = [[], []]
    for _ in range(3):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(run(sets[i]))
    torch.cuda.synchronize()
    for w, g in zip(want, got):
        for each in g:
            assert all(torch.equal(x, y) for x, y in zip(w, each))


def test_pack_devices_and_embedding_refusals(ops):
    offsets = torch.tensor([0, 6], device="cuda")
    pack = ops.pack_sequences(offsets, 6, device="cuda")  # any index
    assert pack.device == offsets.device
    table = torch.zeros(10, 64, device="cuda")
    ids = torch.zeros(6, dtype=torch.int64, device="cuda")
    with pytest.raises(ValueError, match="tables on"):
        ops.token_position_embedding(ids.cpu(), table, table, ops.pack_sequences([0, 6], 6))
    with pytest.raises(TypeError, match="float32"):
        ops.token_position_embedding(ids, table.to(torch.bfloat16), table, pack)
    long = ops.pack_sequences(torch.tensor([0, 12], device="cuda"), 12)  # lengths unknown on the host: the table's last row
    wpe = torch.arange(10.0, device="cuda")[:, None].repeat(1, 64)
    got = ops.token_position_embedding(torch.zeros(12, dtype=torch.int64, device="cuda"), table, wpe, long)
    assert got[:, 0].tolist() == [0, 1, 2, 3, 4, 5, 6, 7, 8, 9, 9, 9]


def test_gradients_of_views_that_are_not_dense(ops):
    """Keys and values as slices of wider tensors, one head of several, one row of several: gradients of any layout."""
    t, d = 140, 64
    q, k, v, do = _inputs(t, 4, 2, d, seed=21)
    pack = ops.pack_sequences([0, 75, t], t, device="cuda")
    want = [x.detach().requires_grad_(True) for x in (q, k, v)]
    a = torch.autograd.grad(ops.attention_packed(*want, pack), want, do)
    wide = torch.zeros(2, t, 5, 3 * d, dtype=torch.bfloat16, device="cuda")
    views = [wide[0, :, :4, :d], wide[0, :, 1:3, d:2 * d], wide[1].transpose(0, 1)[3:5, :, 2 * d:].transpose(0, 1)]
    views = [x.copy_(y).detach().requires_grad_(True) for x, y in zip(views, (q, k, v))]
    b = torch.autograd.grad(ops.attention_packed(views[0], views[1], views[2], pack), views, do)
    # (the first two views overlap in nothing but their memory's rows; every gradient is its own tensor)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    one = ops.pack_sequences([0, 1], 1, device="cuda")
    row = [x[5:6].detach().requires_grad_(True) for x in (q, k, v)]
    col = [x.transpose(0, 1).contiguous().transpose(0, 1)[5:6].detach().requires_grad_(True) for x in (q, k, v)]
    for x, y in zip(*(torch.autograd.grad(ops.attention_packed(*r, one), r, do[5:6]) for r in (row, col))):
        assert torch.equal(x, y)
    single = [x[:, 1:2].detach().requires_grad_(True) for x in (q, k, v)]
    dense = [x.detach().contiguous().requires_grad_(True) for x in single]
    for x, y in zip(*(torch.autograd.grad(ops.attention_packed(*r, pack), r, do[:, 1:2]) for r in (single, dense))):
        assert torch.equal(x, y)


def test_captured_training_step_of_packed_gpt2(ops):
    """Forward and backward of the packed model, its pack included, replayed over other documents; gradients land in .grad."""
    from pytorch_distributed_training_amd.models.gpt2 import gpt2_tiny

    torch.manual_seed(0)
    model = ops.prepare_module(gpt2_tiny(vocab_size=2000, n_ctx=64).cuda())
    params = list(model.parameters())
    for p in params:
        p.grad = torch.zeros_like(p)
    rows = 165
    offsets = torch.tensor([0, 60, 124, 160], dtype=torch.int32, device="cuda")
    idx, targets = (torch.randint(0, 2000, (rows,), device="cuda") for _ in range(2))

    def step():
        for p in params:
            p.grad.zero_()
        loss = model(idx, targets, pack=ops.pack_sequences(offsets, rows))
        loss.backward()
        return loss.detach()

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for new in ([0, 1, 2, 66], [0, 64, 64, 128], [5, 50, 110, 165]):
        offsets.copy_(torch.tensor(new, dtype=torch.int32))
        idx.random_(0, 2000)
        targets.random_(0, 2000)
        targets[new[-1]:] = -100
        graph.replay()
        torch.cuda.synchronize()
        loss, grads = float(got), [p.grad.clone() for p in params]
        assert float(step()) == loss
        for g, p in zip(grads, params):
            # sums of up to 165 fp32 terms in another order: 165 x 2^-24 of their absolute sum, ten times the result's size at most
            assert float((g - p.grad).norm()) <= 10 * 165 * 2.0 ** -24 * float(p.grad.norm()) + 1e-12


def test_second_derivatives_are_refused(ops):
    q, k, v, do = _inputs(20, 2, 2, 64)
    pack = ops.pack_sequences([0, 20], 20, device="cuda")
    q.requires_grad_(True)
    do.requires_grad_(True)
    (dq,) = torch.autograd.grad(ops.attention_packed(q, k, v, pack), q, do, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        dq.float().sum().backward()
    x, w = torch.randn(4, 64, device="cuda", requires_grad=True), torch.randn(10, 64, device="cuda")
    (dx,) = torch.autograd.grad(ops.linear_cross_entropy(x, w, torch.zeros(4, dtype=torch.int64, device="cuda")) ** 2, x, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        dx.float().sum().backward()


def _random_lengths(rows, longest, seed):
    g = torch.Generator().manual_seed(seed)
    lengths = []
    while sum(lengths) < rows:
        lengths.append(min(int(torch.randint(0, longest + 1, (1,), generator=g)), rows - sum(lengths)))
    return lengths


@pytest.mark.parametrize("rows,longest", [(3968, 400), (3969, 400), (5000, 300), (65536, 5000), (66000, 60)])
def test_order_of_the_blocks(ops, rows, longest):
    """In the rows' own order, put in order within the launch and by a second one, offsets searched in LDS and in memory."""
    offsets = _offsets(_random_lengths(rows - 212, longest, rows), 5)
    pack = ops.pack_sequences(torch.tensor(offsets, dtype=torch.int32, device="cuda"), rows)
    spans = ops.pack_sequences(offsets, rows).spans
    assert torch.equal(pack.spans.cpu(), spans)
    blocks = -(-rows // 128)
    order = pack.plan[2 * rows:2 * rows + 6 * blocks].cpu().view(torch.int32).view(3, blocks, 4)
    row = torch.arange(0, rows, 128)
    last = (row + 127).clamp(max=rows - 1)
    first = torch.where(spans[row, 1] > 0, spans[row, 0], row)
    end = torch.where(spans[last, 1] > 0, spans[last, 1], last + 1)
    for got, a, b, reverse in zip(order, (first, row, first), (last + 1, end, end), (True, False, False)):
        work = b - a
        if blocks <= 31:
            want = torch.arange(blocks).flip(0) if reverse else torch.arange(blocks)
        else:
            want = torch.sort(-work, stable=True).indices
        assert torch.equal(got.long(), torch.stack([want, a[want], b[want], work[want]], 1))


@pytest.mark.parametrize("h,hk,d", [(2, 1, 64), (2, 2, 128)])
def test_many_blocks(ops, h, hk, d):
    rows = 5000
    offsets = _offsets(_random_lengths(rows - 100, 500, 3), 40)
    q, k, v, do = _inputs(rows, h, hk, d, seed=3)
    leaves = [x.requires_grad_(True) for x in (q, k, v)]
    pack = ops.pack_sequences(torch.tensor(offsets, device="cuda"), rows)
    for causal in (True, False):
        out = ops.attention_packed(*leaves, pack, causal=causal)
        got = (out.detach(), *torch.autograd.grad(out, leaves, do))
        _check(got, *_expected(q.detach(), k.detach(), v.detach(), do, offsets, causal, d ** -0.5))


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("causal", [True, False])
def test_rows_done_one_by_one_are_right(ops, d, causal):
    """One element of one value is NaN: its column of the output is, every other number of the document is as it was (all of
    its rows take the slow path), and its neighbours do not notice."""
    offsets, h, hk = [0, 70, 410, 433], 4, 2
    t = offsets[-1]
    q, k, v, do = _inputs(t, h, hk, d, seed=d)
    val, err = _expected(q, k, v, do, offsets, causal, d ** -0.5)
    bad = v.clone()
    bad[75, 1, 7] = math.nan
    leaves = [x.requires_grad_(True) for x in (q, k, bad)]
    pack = ops.pack_sequences(offsets, t, device="cuda")
    out = ops.attention_packed(*leaves, pack, causal=causal)
    got = [out.detach(), *torch.autograd.grad(out, leaves, do)]
    seen = slice(75, 410) if causal else slice(70, 410)  # rows that attend to it, through the second key head: heads 2 and 3
    assert bool(torch.isnan(got[0][seen, 2:, 7]).all()) and bool(torch.isnan(got[1][seen, 2:]).all())
    # every key that one of those rows attends to gets a NaN, and nothing of dv, which does not depend on v
    assert bool(torch.isnan(got[2][70:410, 1]).all())
    for x, y in ((got[0][seen, 2:, 7], val[0][seen, 2:, 7]), (got[1][seen, 2:], val[1][seen, 2:]), (got[2][70:410, 1], val[2][70:410, 1])):
        x.copy_(y)
    _check([x.double() for x in got], val, [e + H * y.abs() for y, e in zip(val, err)])  # (the copies are rounded to bf16)
