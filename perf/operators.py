"""Speed and accuracy cases of the packed-sequence and vocabulary operators.

Four operators of language-model training are covered, each as a user calls it, with gradients where it trains:

* ``attention``       softmax attention over sequences packed one behind the other, with grouped heads
* ``head_loss``       output projection and mean cross-entropy over a large vocabulary, logits not kept
* ``distill``         divergence of the student's distribution from a teacher's top logits, on given logits
* ``head_distill``    the same with the student's output projection in front, logits not kept

``run`` computes an operator from elementary fp32 operations, or - where ``own`` is true - through the public entry
points of :mod:`pytorch_distributed_training_amd.ops`.  ``exact`` states the same definitions in 64 bits.
"""

import math
import random

import torch

own = False

BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64


def listed():
    return [
        # a handful of short prompts to score: the latency of one call
        attention("attention, few short documents", 200, 96, 16, 16, 64, causal=True, train=False),
        # one training batch of documents cut at the 1024-token context, 16 heads
        attention("attention, documents", 16381, 1024, 16, 16, 64, causal=True, train=True),
        # grouped heads, documents of very different lengths
        attention("attention, grouped heads", 8192, 4096, 32, 8, 128, causal=True, train=True),
        # one long document, grouped heads
        attention("attention, long document", 16384, 16384, 16, 4, 128, causal=True, train=True, lengths=0),
        # images of different sizes as token sequences, every token sees its whole image
        attention("attention, images", 12601, 197, 12, 12, 64, causal=False, train=True),
        # the loss of a few sequences' last tokens: bound by reading the vocabulary's weights
        head_loss("loss, few rows", 64, 50257, 768, train=False),
        # one step of a medium language model
        head_loss("loss, 50k vocabulary", 8192, 50257, 1024, train=True),
        # a large multilingual vocabulary
        head_loss("loss, 130k vocabulary", 8192, 130001, 2048, train=True),
        # an image classifier that learns from a larger one's best five classes
        distill("distillation, 1000 classes", 256, 1000, 5, "bf16"),
        # logits of a language model against stored top-64 logits
        distill("distillation, 50k vocabulary", 8192, 50257, 64, "bf16"),
        # the same from the hidden states, a small and a usual step
        head_distill("head distillation, few rows", 512, 50257, 768, 32),
        head_distill("head distillation, 50k vocabulary", 8192, 50257, 1024, 64),
    ]


def attention(name, rows, longest, heads, kv_heads, head_dim, causal, train, lengths=1):
    """``lengths``: 0 one sequence over all rows, else the seed of the sequence lengths."""
    return dict(name=name, op="attention", rows=rows, longest=longest, heads=heads, kv_heads=kv_heads, head_dim=head_dim,
                causal=causal, train=train, lengths=lengths)


def head_loss(name, rows, vocab, width, train):
    return dict(name=name, op="head_loss", rows=rows, vocab=vocab, width=width, train=train)


def distill(name, rows, vocab, top, dtype):
    return dict(name=name, op="distill", rows=rows, vocab=vocab, top=top, dtype=dtype, temperature=2.0)


def head_distill(name, rows, vocab, width, top):
    return dict(name=name, op="head_distill", rows=rows, vocab=vocab, width=width, top=top, temperature=2.0)


def draw(rng):
    def spread(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["attention", "attention", "head_loss", "distill", "head_distill"])
    if op == "attention":
        rows = spread(100, 12000)
        longest = min(rows, spread(16, 4096))
        kv_heads = rng.choice([1, 2, 3, 4, 8, 12])
        heads = kv_heads * rng.choice([g for g in (1, 2, 4, 8) if kv_heads * g <= 16])
        case = attention("", rows, longest, heads, kv_heads, rng.choice([64, 128]), rng.random() < 0.7, rng.random() < 0.7,
                         rng.randrange(1, 1 << 20))
    elif op == "head_loss":
        case = head_loss("", spread(16, 8000), spread(2000, 130000), 64 * rng.randint(4, 32), rng.random() < 0.7)
    elif op == "distill":
        case = distill("", spread(32, 8000), spread(500, 130000), spread(1, 128), rng.choice(["bf16", "fp32"]))
    else:
        case = head_distill("", spread(64, 8000), spread(2000, 130000), 64 * rng.randint(4, 24), spread(1, 128))
    del case["name"]
    return case


def sequence_lengths(case):
    """Lengths of the packed sequences: documents spread over the logarithm of their length, images (not causal) over a
    factor of four.  Up to 3 rows at the end belong to none."""
    if case["lengths"] == 0:
        return [case["rows"]]
    rng, longest = random.Random(case["lengths"]), case["longest"]
    left, got = case["rows"] - rng.randint(0, 3), []
    while left > 0:
        n = int(round(math.exp(rng.uniform(0.0, math.log(longest))))) if case["causal"] else rng.randint((longest + 3) // 4, longest)
        got.append(min(left, n))
        left -= got[-1]
    return got


def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)

    def normal(*shape, std=1.0, dtype=BF16):
        return torch.randn(*shape, generator=g, device="cuda", dtype=F32).mul_(std).to(dtype)

    st = dict(case)
    if case["op"] == "attention":
        lengths = sequence_lengths(case)
        offsets = [0]
        for n in lengths:
            offsets.append(offsets[-1] + n)
        t, h, hk, d = case["rows"], case["heads"], case["kv_heads"], case["head_dim"]
        st["offsets"] = torch.tensor(offsets, dtype=torch.int32, device="cuda")
        st["bounds"], st["most"] = offsets, max(lengths)
        st["q"], st["k"], st["v"] = normal(t, h, d), normal(t, hk, d), normal(t, hk, d)
        if case["train"]:
            st["dout"] = normal(t, h, d)
        wrt = ("q", "k", "v")
    else:
        n, v = case["rows"], case["vocab"]
        if "width" in case:  # hidden states behind a layer norm, logits of a standard deviation of 2
            st["x"], st["weight"] = normal(n, case["width"]), normal(v, case["width"], std=2.0 / math.sqrt(case["width"]))
            wrt = ("x", "weight")
        else:
            st["logits"] = normal(n, v, std=2.0, dtype=F32 if case["dtype"] == "fp32" else BF16)
            wrt = ("logits",)
        if case["op"] == "head_loss":  # one row in sixteen (the last token of a document, padding) has no label
            labels = torch.randint(0, v, (n,), generator=g, device="cuda")
            st["labels"] = labels.masked_fill_(torch.rand(n, generator=g, device="cuda") < 1 / 16, -100)
        else:  # a teacher's logits in falling order; one entry in sixteen is absent
            k = case["top"]
            first = torch.randint(0, v, (n, 1), generator=g, device="cuda")
            step = torch.randint(1, max(2, v // k), (n, 1), generator=g, device="cuda")
            ids = (first + step * torch.arange(k, device="cuda")) % v
            st["ids"] = ids.masked_fill_(torch.rand(n, k, generator=g, device="cuda") < 1 / 16, -1)
            st["teacher"] = (torch.randn(n, k, generator=g, device="cuda") * 3 + 8).sort(1, descending=True).values
    if case.get("train", True):
        for name in wrt:
            st[name].requires_grad_(True)
    st["wrt"] = wrt
    return st


def run(st):
    if own:
        return run_own(st)
    with torch.no_grad():
        return {"attention": plain_attention, "head_loss": plain_head_loss, "distill": plain_distill, "head_distill": plain_head_distill}[st["op"]](st)


def run_own(st):
    from pytorch_distributed_training_amd import ops

    if st["op"] == "attention":
        pack = ops.pack_sequences(st["offsets"], st["rows"])
        out = ops.attention_packed(st["q"], st["k"], st["v"], pack, causal=st["causal"])
        return (out, *torch.autograd.grad(out, [st[n] for n in st["wrt"]], st["dout"])) if st["train"] else (out,)
    if st["op"] == "head_loss":
        loss = ops.linear_cross_entropy(st["x"], st["weight"], st["labels"])
        if not st["train"]:
            return (loss,)
    elif st["op"] == "distill":
        loss = ops.distillation_loss(st["logits"], st["teacher"], st["ids"], temperature=st["temperature"])
    else:
        loss = ops.linear_distillation_loss(st["x"], st["weight"], st["teacher"], st["ids"], temperature=st["temperature"])
    return (loss, *torch.autograd.grad(loss, [st[n] for n in st["wrt"]]))


# ---- plain forms: elementary operations in 32 bits


def padded(st):
    """[B, longest] row indices of the packed sequences, and which of them exist."""
    off = st["offsets"].long()
    pos = torch.arange(st["most"], device=off.device)
    at = off[:-1, None] + pos
    return at.clamp(max=st["rows"] - 1), at < off[1:, None]


def plain_attention(st):
    t, h, hk, d = st["rows"], st["heads"], st["kv_heads"], st["head_dim"]
    at, there = padded(st)
    b, s = at.shape

    def batched(x, heads):  # [T, heads, d] -> [B, kv heads, (group *) s, d]
        y = x.float()[at] * there[:, :, None, None]
        return y.view(b, s, hk, heads // hk, d).permute(0, 2, 3, 1, 4).reshape(b, hk, heads // hk * s, d)

    def packed(y, heads):
        out = torch.zeros(t, heads, d, device=y.device)
        out[at[there]] = y.view(b, hk, heads // hk, s, d).permute(0, 3, 1, 2, 4).reshape(b, s, heads, d)[there]
        return out.to(BF16)

    scale = 1.0 / math.sqrt(d)
    q, k, v = batched(st["q"], h), batched(st["k"], hk), batched(st["v"], hk)
    seen = there[:, None, :].expand(b, s, s)
    if st["causal"]:
        seen = seen & torch.ones(s, s, dtype=torch.bool, device=q.device).tril_()
    p = (q @ k.transpose(2, 3)).mul_(scale).view(b, hk, h // hk, s, s)
    p.masked_fill_(~seen[:, None, None], -math.inf)
    p = p.sub_(p.amax(-1, keepdim=True)).exp_()
    p = p.div_(p.sum(-1, keepdim=True)).view(b, hk, h // hk * s, s)
    o = p @ v
    if not st["train"]:
        return (packed(o, h),)
    do = batched(st["dout"], h)
    dv = p.transpose(2, 3) @ do
    ds = (do @ v.transpose(2, 3)).sub_((do * o).sum(-1, keepdim=True)).mul_(p).mul_(scale)
    return packed(o, h), packed(ds @ k, h), packed(ds.transpose(2, 3) @ q, hk), packed(dv, hk)


def plain_log_softmax(z):
    z = z - z.amax(-1, keepdim=True)
    return z.sub_(z.exp().sum(-1, keepdim=True).log_())


def plain_head_loss(st):
    x, w, y = st["x"].float(), st["weight"].float(), st["labels"]
    logp = plain_log_softmax(x @ w.t())
    has = y >= 0
    rows, count = torch.arange(len(y), device=y.device), has.sum()
    loss = -(logp[rows, y.clamp(min=0)] * has).sum() / count
    if not st["train"]:
        return (loss,)
    dz = logp.exp_()
    dz[rows, y.clamp(min=0)] -= 1.0
    dz.mul_((has / count)[:, None])
    return loss, (dz @ w).to(BF16), (dz.t() @ x).to(BF16)


def plain_divergence(z, st):
    """Loss and the gradient of the logits ``z``."""
    tau, ids = st["temperature"], st["ids"]
    has = ids >= 0
    at = ids.clamp(min=0)
    logt = plain_log_softmax((st["teacher"] / tau).masked_fill(~has, -math.inf))
    t = logt.exp()
    logp = plain_log_softmax(z / tau)
    some = has.any(1)
    count = some.sum()
    each = torch.where(has & some[:, None], t * (logt - logp.gather(1, at)), 0.0)
    loss = tau * tau * each.sum(dtype=F64) / count
    dz = logp.exp_().scatter_add_(1, at, -torch.where(has, t, 0.0))
    return loss.float(), dz.mul_((some * (tau / count))[:, None])


def plain_distill(st):
    loss, dz = plain_divergence(st["logits"].float(), st)
    return loss, dz.to(st["logits"].dtype)


def plain_head_distill(st):
    x, w = st["x"].float(), st["weight"].float()
    loss, dz = plain_divergence(x @ w.t(), st)
    return loss, (dz @ w).to(BF16), (dz.t() @ x).to(BF16)


# ---- bytes and operations that a pass cannot do without


def work(case):
    if case["op"] == "attention":
        lengths = sequence_lengths(case)
        t, h, hk, d = case["rows"], case["heads"], case["kv_heads"], case["head_dim"]
        pairs = sum(n * (n + 1) // 2 if case["causal"] else n * n for n in lengths)
        q, kv = 2 * t * h * d, 2 * 2 * t * hk * d
        products = 7 if case["train"] else 2
        return {"bytes": (4 * q + 2 * kv) if case["train"] else (2 * q + kv), "flops": 2 * products * pairs * h * d}
    n, v = case["rows"], case["vocab"]
    teacher = n * case.get("top", 0) * 12
    if case["op"] == "distill":
        return {"bytes": 2 * n * v * (4 if case["dtype"] == "fp32" else 2) + teacher, "flops": 5 * n * v}
    w = case["width"]
    once = 2 * (n + v) * w
    train = case.get("train", True)
    return {"bytes": (2 if train else 1) * once + teacher + 8 * n, "flops": (6 if train else 2) * n * v * w}


# ---- the definitions in 64 bits


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] != "attention":
        with torch.no_grad():
            return exact_vocabulary(st)
    t, h, d = st["rows"], st["heads"], st["head_dim"]
    group, scale, train = h // st["kv_heads"], d ** -0.5, st["train"]
    q_, k_, v_ = (st[name].detach() for name in st["wrt"])
    res = [torch.zeros(x.shape, dtype=F64, device="cuda") for x in ([q_, q_, k_, v_] if train else [q_])]
    for a, e in zip(st["bounds"][:-1], st["bounds"][1:]):
        n = e - a
        ahead = torch.full((n, n), -math.inf, dtype=F64, device="cuda").triu_(1) if st["causal"] else 0.0
        for j in range(h):
            q, k, v = (x[a:e, i].double() for x, i in ((q_, j), (k_, j // group), (v_, j // group)))
            p = torch.softmax(q @ k.t() * scale + ahead, -1)
            res[0][a:e, j] = p @ v
            if train:
                do = st["dout"][a:e, j].double()
                dp = do @ v.t()
                ds = p * (dp - (p * dp).sum(-1, keepdim=True)) * scale
                res[1][a:e, j] = ds @ k
                res[2][a:e, j // group] += ds.t() @ q
                res[3][a:e, j // group] += p.t() @ do
    return tuple(res)


def exact_vocabulary(st):
    """Both losses are a weighted sum of -log q at some places of a row, plus the entropy term of the weights."""
    tau = st.get("temperature", 1.0)
    z = st["logits"].double() if "logits" in st else st["x"].double() @ st["weight"].double().t()
    n, v = z.shape
    if st["op"] == "head_loss":
        ids = st["labels"][:, None]
        p = (ids >= 0).double()
    else:
        ids = st["ids"]
        p = torch.where(ids >= 0, torch.exp((st["teacher"].double() - st["teacher"].double().amax(1, keepdim=True)) / tau), 0.0)
        p = p / p.sum(1, keepdim=True).clamp(min=1e-300)
    valid = p.sum(1) > 0
    lse = torch.logsumexp(z / tau, 1)
    at = ids.clamp(min=0)
    taken = z.gather(1, at) / tau
    loss = (p * (torch.log(p.clamp(min=1e-300)) - taken + lse[:, None])).sum() * tau * tau / valid.sum()
    if not st.get("train", True):
        return (loss,)
    dz = torch.exp(z.div_(tau).sub_(lse[:, None]))
    dz.scatter_add_(1, at, -p)
    dz *= (valid * (tau / valid.sum()))[:, None]
    if "logits" in st:
        return loss, dz
    return loss, dz @ st["weight"].double(), dz.t() @ st["x"].double()
