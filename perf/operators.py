"""Measured cases of packed causal attention, token log probabilities and
distillation from a teacher's top logits.

What a program that trains on packed documents against a teacher has these
operators do: attention over sequences of different lengths packed into one
row dimension, with heads that share keys and values; the log probabilities,
entropies and top alternatives of given tokens; and the distillation loss on a
teacher's top logits.  `own` chooses between the framework's operators and
their plain form in elementary torch operations.

`listed()` names the cases, `draw(rng)` gives one more of the same ranges,
`prepare(case, seed)` makes what a program has in hand before the call,
`run(state)` one pass, `work(case)` the bytes and operations a pass cannot do
without, and `exact(case, seed)` the same outputs from the definitions in
64 bits.
"""

import math

import torch

own = False

DEVICE = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
IGNORE = -100


# ------------------------------------------------------------------- cases --
def listed():
    return [
        # three short prompts in one call: latency
        dict(name="attn-fwd-t96", kind="attn", lens="1,30,65", tail=0, n=8, m=2, hn=64, dtype="bf16", train=False),
        # a teacher scoring packed documents, 32 heads of 80 in eight groups
        # (the fp16 stage's head size), an empty one and unused rows among them
        dict(name="attn-fwd-t4000-d80", kind="attn", lens="700,1,1311,0,255,64,129,990,531", tail=19, n=32, m=8,
             hn=80, dtype="fp16", train=False),
        # the benchmark's 16 heads of 128 over a packed micro-batch of 8192 rows
        dict(name="attn-train-t8192-d128", kind="attn",
             lens="2048,311,1500,96,1024,777,2048,33,160,128,67", tail=0, n=16, m=4, hn=128, dtype="bf16",
             train=True),
        # one long document, one key and value head for all queries
        dict(name="attn-train-t16384-d64", kind="attn", lens="16384", tail=0, n=8, m=1, hn=64, dtype="bf16",
             train=True),
        # one row of logits: the last token of a prompt
        dict(name="logp-r1-v50304", kind="logp", rows=1, v=50304, k=5, dtype="bf16", masked=0, ignored=0.0,
             train=False),
        # a teacher's sequence of 2048, the padded columns of the vocabulary masked
        dict(name="logp-r2048-v50304-k20", kind="logp", rows=2048, v=50304, k=20, dtype="bf16", masked=47,
             ignored=0.0, train=False),
        # a policy's log probabilities and entropies with their gradients,
        # a tenth of the rows prompts that are not scored
        dict(name="logp-train-r4096-v50304", kind="logp", rows=4096, v=50304, k=0, dtype="bf16", masked=0,
             ignored=0.1, train=True),
        # fp32 logits of an odd vocabulary, gradients and many alternatives
        dict(name="logp-train-r777-v32001-k64", kind="logp", rows=777, v=32001, k=64, dtype="fp32", masked=0,
             ignored=0.0, train=True),
        # a large vocabulary, the most alternatives
        dict(name="logp-r512-v262144-k128", kind="logp", rows=512, v=262144, k=128, dtype="fp16", masked=0,
             ignored=0.0, train=False),
        # a handful of rows: latency of both passes
        dict(name="distill-r16-v50304-k8", kind="distill", rows=16, v=50304, k=8, dtype="fp16", pad=0, tau=1.0,
             absent=0.0, train=True),
        # odd vocabulary, rows of a padded buffer, some alternatives absent
        dict(name="distill-r1000-v50257-k20", kind="distill", rows=1000, v=50257, k=20, dtype="fp32", pad=47,
             tau=1.0, absent=0.1, train=True),
        # the student's micro-batch of the benchmark's vocabulary
        dict(name="distill-r4096-v50304-k64", kind="distill", rows=4096, v=50304, k=64, dtype="bf16", pad=0, tau=2.0,
             absent=0.0, train=True),
    ]


def _log_uniform(rng, lo, hi):
    return math.exp(rng.uniform(math.log(lo), math.log(hi)))


def draw(rng):
    kind = rng.choice(("attn", "logp", "distill"))
    if kind == "attn":
        m = rng.choice((1, 2, 3, 4, 8))
        n = m * rng.choice((1, 1, 2, 3, 4, 8))
        hn = rng.choice((16, 40, 64, 64, 80, 96, 128, 128))
        while True:
            total = int(_log_uniform(rng, 16, 16384))
            cuts = sorted(rng.randrange(total + 1) for _ in range(int(_log_uniform(rng, 1, 24)) - 1))
            lens = [b - a for a, b in zip([0, *cuts], [*cuts, total])]
            # no dearer than the longest listed document, padded to its longest
            # sequence as the plain form pads, or not
            if len(lens) * max(lens) ** 2 * n <= 16384**2 * 8 and sum(x * x for x in lens) * n * hn <= 16384**2 * 512:
                break
        return dict(kind="attn", lens=",".join(map(str, lens)), tail=rng.choice((0, 0, 1, 40)), n=n, m=m, hn=hn,
                    dtype=rng.choice(("bf16", "fp16")), train=rng.random() < 0.6)
    v = int(_log_uniform(rng, 1000, 262144))
    dtype = rng.choice(("bf16", "bf16", "fp16", "fp32"))
    rows = int(_log_uniform(rng, 1, min(8192, 4096 * 50304 / v / (2 if dtype == "fp32" else 1))))
    if kind == "logp":
        return dict(kind="logp", rows=rows, v=v, k=rng.choice((0, 1, 5, 20, 64, 128)), dtype=dtype,
                    masked=rng.choice((0, 0, 47)), ignored=rng.choice((0.0, 0.0, 0.2)), train=rng.random() < 0.5)
    return dict(kind="distill", rows=rows, v=v, k=rng.choice((1, 8, 20, 64, 128)), dtype=dtype,
                pad=rng.choice((0, 0, 5, 47)), tau=rng.choice((0.5, 1.0, 2.0, 4.0)),
                absent=rng.choice((0.0, 0.0, 0.2)), train=rng.random() < 0.7)


def _lens(case):
    return [int(x) for x in case["lens"].split(",")]


# ----------------------------------------------------------------- prepare --
def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, generator=gen, device=DEVICE)

    dtype = DTYPES[case["dtype"]]
    st = dict(case)
    if case["kind"] == "attn":
        lens = _lens(case)
        n, m, hn, rows = case["n"], case["m"], case["hn"], sum(lens) + case["tail"]
        # the projections of one QKV product, read in place
        mixed = (randn(rows, n + 2 * m, hn) * 1.2).to(dtype)
        st["q"], st["k"], st["v"] = torch.split(mixed, (n, m, m), dim=1)
        st["dout"] = randn(rows, n * hn).to(dtype)
        st["lengths"] = lens
        # what the plain form pads with: where each sequence starts and ends
        ends = torch.tensor(lens, device=DEVICE).cumsum(0)
        st["starts"], st["ends"], st["longest"] = ends - torch.tensor(lens, device=DEVICE), ends, max(lens)
        if own:
            from eth_amd.packed import PackedSequences

            # made once for a batch, shared by all its layers
            st["packed"] = PackedSequences(lens, total=rows, device=DEVICE)
        return st
    rows, v = case["rows"], case["v"]
    # a model's logits: a wide bulk and a few tokens that stand out
    z = randn(rows, v + case.get("pad", 0)) * 2.0
    hot = torch.randint(0, v, (rows, 12), generator=gen, device=DEVICE)
    z.scatter_add_(1, hot, randn(rows, 12).abs() * 5.0)
    if case["kind"] == "logp":
        if case["masked"]:
            z[:, v - case["masked"] :] = -math.inf
        tokens = hot[:, 0].clamp_max(v - 1 - case["masked"])
        drop = torch.rand(rows, generator=gen, device=DEVICE) < case["ignored"]
        st["tokens"] = torch.where(drop, torch.full_like(tokens, IGNORE), tokens).contiguous()
        st["logits"] = z.to(dtype)
        st["dlogprob"], st["dentropy"] = randn(rows), randn(rows) * 0.1
    else:
        teacher = z[:, :v] + randn(rows, v) * 0.7
        top, ids = torch.topk(teacher, case["k"], dim=1)
        drop = torch.rand(rows, case["k"], generator=gen, device=DEVICE) < case["absent"]
        st["teacher_ids"] = torch.where(drop, torch.full_like(ids, -1), ids).contiguous()
        st["teacher_logits"] = top.contiguous()
        st["logits"] = z.to(dtype)[:, :v]
        st["dloss"] = torch.rand(rows, generator=gen, device=DEVICE) + 0.5
    st["bad"] = torch.zeros(1, dtype=torch.int32, device=DEVICE)
    return st


# --------------------------------------------------------------------- run --
def run(st):
    if st["kind"] == "attn":
        return _attn_own(st) if own else _attn_plain(st)
    if st["kind"] == "logp":
        return _logp_own(st) if own else _logp_plain(st)
    return _distill_own(st) if own else _distill_plain(st)


def _attn_own(st):
    from eth_amd.model.functional import PackedCausalAttentionFn

    if not st["train"]:
        with torch.no_grad():
            return PackedCausalAttentionFn.apply(st["q"], st["k"], st["v"], st["packed"])
    q, k, v = (st[x].detach().requires_grad_(True) for x in "qkv")
    out = PackedCausalAttentionFn.apply(q, k, v, st["packed"])
    return (out.detach(), *torch.autograd.grad(out, (q, k, v), st["dout"]))


def _attn_plain(st):
    q, k, v = st["q"], st["k"], st["v"]
    rows, n, hn = q.shape
    m, longest = k.shape[1], st["longest"]
    # every sequence padded to the longest: [sequences, longest] rows
    pos = torch.arange(longest, device=q.device)
    at = st["starts"][:, None] + pos[None, :]
    real = at < st["ends"][:, None]
    at = at.clamp_max(rows - 1)

    def padded(x):  # [rows, heads, hn] -> [sequences, n, longest, hn], shared heads repeated
        x = torch.where(real[:, :, None, None], x[at].float(), torch.zeros((), device=x.device))
        return x.repeat_interleave(n // x.shape[2], dim=2).transpose(1, 2).contiguous()

    def packed(x, heads):  # back, the group of a shared head added up
        x = x.transpose(1, 2).reshape(*at.shape, heads, n // heads, hn).sum(3)
        out = torch.zeros(rows, heads, hn, device=x.device)
        out[at[real]] = x[real]
        return out.to(q.dtype)

    qp, kp, vp = padded(q), padded(k), padded(v)
    hidden = pos[None, :] > pos[:, None]
    s = torch.matmul(qp, kp.transpose(2, 3).contiguous()) * (1.0 / math.sqrt(hn))
    s.masked_fill_(hidden, -math.inf)
    s = (s - s.amax(-1, keepdim=True)).exp_()
    p = s.div_(s.sum(-1, keepdim=True))
    o = torch.matmul(p, vp)
    out = packed(o, n).view(rows, n * hn)
    if not st["train"]:
        return out
    do = padded(st["dout"].view(rows, n, hn))
    dv = torch.matmul(p.transpose(2, 3).contiguous(), do)
    dp = torch.matmul(do, vp.transpose(2, 3).contiguous())
    ds = dp.sub_((do * o).sum(-1, keepdim=True)).mul_(p).mul_(1.0 / math.sqrt(hn))
    dq = torch.matmul(ds, kp)
    dk = torch.matmul(ds.transpose(2, 3).contiguous(), qp)
    return out, packed(dq, n), packed(dk, m), packed(dv, m)


def _logp_own(st):
    from eth_amd.model.functional import TokenLogprobsFn

    if not st["train"]:
        with torch.no_grad():
            return TokenLogprobsFn.apply(st["logits"], st["tokens"], st["k"], st["bad"], IGNORE)
    z = st["logits"].detach().requires_grad_(True)
    logprob, entropy, top, ids = TokenLogprobsFn.apply(z, st["tokens"], st["k"], st["bad"], IGNORE)
    (dz,) = torch.autograd.grad((logprob, entropy), (z,), (st["dlogprob"], st["dentropy"]))
    return logprob.detach(), entropy.detach(), top, ids, dz


def _logp_plain(st):
    z, tokens, k = st["logits"].float(), st["tokens"], st["k"]
    scored = tokens != IGNORE
    t = tokens.clamp_min(0)[:, None]
    top_z = z.amax(1, keepdim=True)
    lse = top_z + (z - top_z).exp().sum(1, keepdim=True).log()
    logp = z - lse
    p = logp.exp()
    plogp = torch.where(p > 0, p * logp, torch.zeros((), device=z.device))
    entropy = -plogp.sum(1)
    logprob = torch.where(scored, logp.gather(1, t)[:, 0], torch.zeros((), device=z.device))
    # the largest, equal ones by the lowest index: whole keys that never tie
    bits = (z + 0.0).view(torch.int32).long()
    order = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits)
    index = torch.arange(z.shape[1], device=z.device)
    ids = torch.topk(order * z.shape[1] - index, k, dim=1)[1]
    top = torch.where(scored[:, None], logp.gather(1, ids), torch.full((), -math.inf, device=z.device))
    ids = torch.where(scored[:, None], ids, torch.full_like(ids, -1))
    out = logprob, torch.where(scored, entropy, torch.zeros_like(entropy)), top, ids
    if not st["train"]:
        return out
    g = torch.where(scored, st["dlogprob"], torch.zeros_like(entropy))[:, None]
    h = torch.where(scored, st["dentropy"], torch.zeros_like(entropy))[:, None]
    dz = -g * p - h * (plogp + p * entropy[:, None])
    dz.scatter_add_(1, t, g)
    return (*out, dz.to(st["logits"].dtype))


def _distill_own(st):
    from eth_amd.model.functional import TopkDistillFn

    args = (st["teacher_ids"], st["teacher_logits"], st["tau"], st["bad"])
    if not st["train"]:
        with torch.no_grad():
            return TopkDistillFn.apply(st["logits"], *args)
    z = st["logits"].detach().requires_grad_(True)
    loss = TopkDistillFn.apply(z, *args)
    return (loss.detach(), *torch.autograd.grad(loss, (z,), st["dloss"]))


def _distill_plain(st):
    z, ids, tau = st["logits"].float() / st["tau"], st["teacher_ids"], st["tau"]
    present = ids >= 0
    t = torch.where(present, st["teacher_logits"] / tau, torch.full((), -math.inf, device=z.device))
    high = t.amax(1, keepdim=True)
    e = torch.where(present, (t - high).exp(), torch.zeros((), device=z.device))
    total = e.sum(1, keepdim=True)
    q = e / total.clamp_min(1e-30)
    logq = torch.where(q > 0, t - high - total.log(), torch.zeros((), device=z.device))
    top_z = z.amax(1, keepdim=True)
    lse = top_z + (z - top_z).exp().sum(1, keepdim=True).log()
    at = ids.clamp_min(0)
    loss = tau * tau * (q * (logq - (z.gather(1, at) - lse))).sum(1)
    if not st["train"]:
        return loss
    g = (st["dloss"] * tau)[:, None]
    dz = (z - lse).exp() * (g * q.sum(1, keepdim=True))
    dz.scatter_add_(1, at, -g * q)
    return loss, dz.to(st["logits"].dtype)


# -------------------------------------------------------------------- work --
def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["kind"] == "attn":
        lens = _lens(case)
        rows, n, m, hn = sum(lens) + case["tail"], case["n"], case["m"], case["hn"]
        flops = 2.0 * n * hn * sum(x * (x + 1) for x in lens)  # QK^T and PV over the causal half
        moved = rows * hn * (2 * n + 2 * m)  # q, k, v, out
        if case["train"]:
            flops *= 3.5  # dP, dV, dQ, dK and S once more
            moved += rows * hn * (2 * n + 2 * m)  # dout, dq, dk, dv
        return {"bytes": float(moved * size), "flops": flops}
    rows, v, k = case["rows"], case["v"], case["k"]
    moved = rows * v * size * (2 if case["train"] else 1)  # the logits, and their gradient
    if case["kind"] == "logp":
        moved += rows * (8 + 4 + 4 + 12 * k + (8 if case["train"] else 0))
    else:
        moved += rows * (12 * k + 4 + (4 if case["train"] else 0))
    return {"bytes": float(moved), "flops": float(rows * v * (10 if case["train"] else 5))}


# ------------------------------------------------------------------- exact --
def exact(case, seed):
    """The outputs from the definitions in 64 bits, a sequence and head (or a
    block of rows) at a time."""
    st = prepare(case, seed)
    if case["kind"] == "attn":
        return _attn_exact(case, st)
    return _rows_exact(case, st)


def _attn_exact(case, st):
    n, m, hn = case["n"], case["m"], case["hn"]
    q, k, v = st["q"], st["k"], st["v"]
    rows = q.shape[0]
    do = st["dout"].view(rows, n, hn)
    f64 = dict(dtype=torch.float64, device=q.device)
    out, dq = torch.zeros(rows, n, hn, **f64), torch.zeros(rows, n, hn, **f64)
    dk, dv = torch.zeros(rows, m, hn, **f64), torch.zeros(rows, m, hn, **f64)
    a = 0
    for length in _lens(case):
        b = a + length
        for h in range(n if length else 0):
            g = h // (n // m)
            qh, kh, vh, dh = q[a:b, h].double(), k[a:b, g].double(), v[a:b, g].double(), do[a:b, h].double()
            logit = (qh @ kh.t() / hn**0.5).tril_()
            logit += torch.full((length, length), -math.inf, **f64).triu_(1)
            prob = torch.softmax(logit, dim=1)
            del logit
            out[a:b, h] = prob @ vh
            if case["train"]:
                dv[a:b, g] += prob.t() @ dh
                grad = dh @ vh.t()
                grad = prob * (grad - (grad * prob).sum(1, keepdim=True)) / hn**0.5
                dq[a:b, h] = grad @ kh
                dk[a:b, g] += grad.t() @ qh
        a = b
    out = out.view(rows, n * hn)
    return (out, dq, dk, dv) if case["train"] else out


def _rows_exact(case, st):
    rows, step = case["rows"], max(1, 2**27 // case["v"])
    parts = [_block_exact(case, st, slice(r, r + step)) for r in range(0, rows, step)]
    if not isinstance(parts[0], tuple):
        return torch.cat(parts)
    return tuple(torch.cat(x) for x in zip(*parts))


def _block_exact(case, st, at):
    z = st["logits"][at].double()
    if case["kind"] == "logp":
        tokens = st["tokens"][at]
        scored = (tokens >= 0).double()
        logp = torch.log_softmax(z, dim=1)
        p = logp.exp()
        finite = logp.masked_fill(p == 0, 0.0)
        entropy = -(p * finite).sum(1)
        best, ids = torch.sort(z, dim=1, descending=True, stable=True)
        ids = ids[:, : case["k"]].clone()
        top = logp.gather(1, ids)
        top[tokens < 0] = -math.inf
        ids[tokens < 0] = -1
        del best
        hit = torch.nn.functional.one_hot(tokens.clamp_min(0), case["v"]) if case["train"] else None
        out = logp.gather(1, tokens.clamp_min(0)[:, None])[:, 0] * scored, entropy * scored, top, ids
        if not case["train"]:
            return out
        g, h = (st[x][at].double() * scored for x in ("dlogprob", "dentropy"))
        return (*out, g[:, None] * (hit - p) - h[:, None] * p * (finite + entropy[:, None]))
    tau, ids = case["tau"], st["teacher_ids"][at]
    t = (st["teacher_logits"][at].double() / tau).masked_fill(ids < 0, -math.inf)
    some = (ids >= 0).any(1, keepdim=True)
    q = torch.softmax(t.masked_fill(~some, 0.0), dim=1) * some
    q = q.masked_fill(ids < 0, 0.0)
    logp = torch.log_softmax(z / tau, dim=1)
    picked = logp.gather(1, ids.clamp_min(0))
    loss = tau**2 * (torch.special.xlogy(q, q) - q * picked).sum(1)
    if not case["train"]:
        return loss
    target = torch.zeros_like(z).scatter_add_(1, ids.clamp_min(0), q)
    g = st["dloss"][at].double()[:, None]
    return loss, g * tau * (logp.exp() * q.sum(1, keepdim=True) - target)
