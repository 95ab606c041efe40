"""The operators for packed documents and for distillation, as workloads that can be timed and compared.

Three operators, each with a plain form in elementary torch operations (``own = False``) and the call that a
user makes of this package (``own = True``):

* ``bounds``: for each row of a packed batch, the first row of its sequence and the row past its last one,
  from sequence offsets or from token ids in which every document starts with BOS;
* ``attention``: causal (and sliding-window) attention inside each sequence of a packed batch with grouped
  heads, its log-sum-exp, and with ``backward`` the gradients of q, k and v;
* ``distill``: the loss against a teacher's top logits (with the hard-label loss mixed in) and its gradient.

Sequence lengths are dealt from the case alone (``deal``), so a case always has the same work; the values of
the tensors come from the seed.
"""
import math
import random

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
# the plain form holds a few [sequences, heads, longest, longest] fp32 tensors: at most 12 GB each
_MOST_SCORES = 3_000_000_000
_MOST_FLOPS = 3.0e12
_EPS = 1e-10  # the package's cross-entropy is -log(p + 1e-10)


# ---------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # a batch of a few short requests: the call is launch latency
        dict(name="bounds_offsets_small", op="bounds", source="offsets", rows=600, tail=37, mean=60, cap=600, deal=1,
             batch=1),
        # one micro-batch of the d512 preset: 128 rows of 2048 tokens, documents of 512 tokens on average
        dict(name="bounds_ids_step", op="bounds", source="ids", rows=128 * 2048, tail=0, mean=512, cap=2048, deal=2,
             batch=128),
        # scoring a handful of short documents with the d512 model's heads: launch latency
        dict(name="attn_fwd_short", op="attention", dtype="bf16", heads=4, kv_heads=4, dim=128, rows=217, tail=0,
             mean=40, cap=96, window=0, backward=False, deal=3, fused=True),
        # ragged prompts, grouped heads of 64, half precision, odd total
        dict(name="attn_fwd_ragged_gqa64", op="attention", dtype="fp16", heads=16, kv_heads=4, dim=64, rows=9001,
             tail=0, mean=300, cap=1500, window=0, backward=False, deal=4, fused=False),
        # one long prompt, causal over its whole length
        dict(name="attn_fwd_long", op="attention", dtype="bf16", heads=8, kv_heads=2, dim=128, rows=16384, tail=0,
             mean=1 << 30, cap=16384, window=0, backward=False, deal=5, fused=False),
        # evaluation of packed documents with the d512 model's heads and its short window
        dict(name="attn_fwd_docs_window", op="attention", dtype="bf16", heads=4, kv_heads=4, dim=128, rows=65536,
             tail=0, mean=512, cap=2048, window=1024, backward=False, deal=6, fused=True),
        # a training layer of the d512 model on packed documents, forward and backward
        dict(name="attn_train_docs", op="attention", dtype="bf16", heads=4, kv_heads=4, dim=128, rows=65536, tail=0,
             mean=512, cap=2048, window=0, backward=True, deal=7, fused=True),
        # a training layer on one long document, grouped heads
        dict(name="attn_train_long_gqa", op="attention", dtype="bf16", heads=16, kv_heads=4, dim=128, rows=8192,
             tail=0, mean=1 << 30, cap=8192, window=0, backward=True, deal=8, fused=False),
        # the reference's default model's heads (4 x 64), documents of a few tokens to a few hundred, padded end
        dict(name="attn_train_ragged64", op="attention", dtype="bf16", heads=4, kv_heads=2, dim=64, rows=5003,
             tail=130, mean=90, cap=512, window=0, backward=True, deal=9, fused=False),
        # a few scored positions with an odd vocabulary: launch latency
        dict(name="distill_small", op="distill", dtype="fp32", rows=7, vocab=1001, top=8, cap=0.0, temperature=1.0,
             alpha=1.0, padded=False),
        # a d512 micro-batch of 16 rows of 2048 tokens: softened teacher mixed with the hard labels
        dict(name="distill_d512", op="distill", dtype="bf16", rows=16 * 2048, vocab=8192, top=32, cap=15.0,
             temperature=2.0, alpha=0.5, padded=True),
        # the d1280 preset's vocabulary, teacher only
        dict(name="distill_d1280", op="distill", dtype="bf16", rows=8191, vocab=65536, top=64, cap=15.0,
             temperature=1.0, alpha=1.0, padded=False),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["bounds", "attention", "attention", "attention", "distill", "distill"])
    deal = rng.randrange(1 << 30)
    if op == "bounds":
        if rng.random() < 0.5:
            rows = _log_int(rng, 1, 1 << 18)
            return dict(op=op, source="offsets", rows=rows, tail=rng.choice([0, rows // 7]),
                        mean=_log_int(rng, 2, 2048), cap=rows, deal=deal, batch=1)
        batch, length = _log_int(rng, 1, 128), _log_int(rng, 16, 2048)
        return dict(op=op, source="ids", rows=batch * length, tail=0, mean=_log_int(rng, 2, 2048), cap=length,
                    deal=deal, batch=batch)
    if op == "attention":
        heads, backward = rng.choice([1, 2, 4, 8, 10, 16]), rng.random() < 0.5
        # with one visible key a row's weights are constant, and dq and dk are exactly zero: nothing to compare
        rows = _log_int(rng, 16 if backward else 1, 32768)
        tail = rng.choice([0, 0, rows // 9])
        case = dict(op=op, dtype=rng.choice(["bf16", "bf16", "fp16"]), heads=heads,
                    kv_heads=rng.choice([d for d in range(1, heads + 1) if heads % d == 0]),
                    dim=rng.choice([64, 128]), rows=rows, tail=tail, mean=_log_int(rng, 6, 8192),
                    cap=_log_int(rng, 64, 16384), window=rng.choice([0, 0, _log_int(rng, 8 if backward else 1, 2048)]),
                    backward=backward, deal=deal, fused=rng.random() < 0.5)
        while _scores(case) > _MOST_SCORES or work(case)["flops"] > _MOST_FLOPS:
            case["rows"] = case["rows"] * 3 // 4
            case["tail"] = min(case["tail"], case["rows"] // 9)
        return case
    vocab = _log_int(rng, 64, 131072)
    alpha = rng.choice([1.0, 1.0, round(rng.uniform(0.05, 0.95), 3)])
    return dict(op=op, dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]),
                rows=_log_int(rng, 1, min(32768, (1 << 28) // vocab)), vocab=vocab,
                top=_log_int(rng, 1, min(128, vocab // 2)), cap=rng.choice([0.0, 15.0]),
                temperature=rng.choice([1.0, 2.0, round(rng.uniform(0.5, 4.0), 3)]), alpha=alpha,
                padded=rng.random() < 0.3)


def _lengths(case):
    """The sequence lengths of a packed batch: exponential around ``mean``, zero among them when short."""
    rng, left, out = random.Random(case["deal"]), case["rows"] - case["tail"], []
    while left > 0:
        n = min(left, case["cap"], int(rng.expovariate(1.0 / case["mean"])))
        out.append(n)
        left -= n
    return out


def _scale(case):
    """The loss is the mean over rows; in half precision it is scaled up by the number of rows, as a scaled loss
    would be, so that the gradients stay normal numbers."""
    return 1.0 if case["dtype"] == "fp16" else 1.0 / case["rows"]


def _scores(case):
    lengths = _lengths(case)
    return len(lengths) * case["heads"] * max(lengths, default=0) ** 2


def _pairs(n, window):
    """(query, key) pairs of a causal sequence of n tokens with a window of keys (0: none)."""
    w = min(window, n) if window else n
    return w * (w + 1) // 2 + (n - w) * w


def work(case):
    if case["op"] == "bounds":
        read = case["rows"] if case["source"] == "ids" else len(_lengths(case)) + 1
        return {"bytes": 4 * (read + 2 * case["rows"]), "flops": 0}
    if case["op"] == "attention":
        n, h, kv, d, e = case["rows"] - case["tail"], case["heads"], case["kv_heads"], case["dim"], 2
        pairs = sum(_pairs(x, case["window"]) for x in _lengths(case)) * h
        tensors = (2 * h + 2 * kv) * d * e * n + 4 * h * n  # q, k, v in; out, lse out
        flops = 4 * d * pairs
        if case["backward"]:  # dout in, dq, dk, dv out; scores again, dP, dV, dQ, dK
            tensors += (2 * h + 2 * kv) * d * e * n
            flops += 10 * d * pairs
        return {"bytes": tensors, "flops": flops}
    m, v, k, e = case["rows"], case["vocab"], case["top"], _BYTES[case["dtype"]]
    return {"bytes": 2 * m * v * e + m * k * 8 + 8 * m, "flops": 0}


# ---------------------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dev = "cuda"
    if case["op"] == "bounds":
        if case["source"] == "offsets":
            # the documents come in another order for another seed
            lengths = _lengths(case)
            random.Random(seed).shuffle(lengths)
            off = torch.tensor([0] + lengths, dtype=torch.int64).cumsum(0).to(torch.int32)
            return dict(case=case, offsets=off.to(dev))
        batch, length, vocab = case["batch"], case["rows"] // case["batch"], 8192
        ids = torch.randint(0, vocab - 1, (batch, length), generator=g, device=dev, dtype=torch.int32)
        ids[torch.rand(batch, length, generator=g, device=dev) < 1.0 / case["mean"]] = vocab - 1
        return dict(case=case, ids=ids, bos=vocab - 1)
    if case["op"] == "attention":
        dt, n, h, kv, d = _DTYPES[case["dtype"]], case["rows"], case["heads"], case["kv_heads"], case["dim"]
        lengths = _lengths(case)
        off = torch.tensor([0] + lengths, dtype=torch.int64).cumsum(0)
        r = lambda *s: torch.randn(*s, generator=g, device=dev)  # noqa: E731
        unit = lambda x: x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + 1e-5)  # noqa: E731  (q and k are normalised)
        q, k, v = unit(r(n, h, d)).to(dt), unit(r(n, kv, d)).to(dt), r(n, kv, d).to(dt)
        if case["fused"]:  # views into one projection buffer, as a fused QKV product leaves them
            qkv = torch.cat([q, k, v], 1)
            q, k, v = qkv[:, :h], qkv[:, h:h + kv], qkv[:, h + kv:]
        # rows behind the last sequence belong to none: [row, row) is their span
        rows = torch.arange(n)
        lo, hi = rows.clone(), rows.clone()
        real = int(off[-1])
        ln = torch.tensor(lengths, dtype=torch.int64)
        lo[:real] = off[:-1].repeat_interleave(ln)
        hi[:real] = off[1:].repeat_interleave(ln)
        s = dict(case=case, q=q, k=k, v=v, offsets=off.to(dev), longest=max(lengths, default=0),
                 start=lo.to(torch.int32).to(dev), end=hi.to(torch.int32).to(dev),
                 out=torch.zeros(n, h, d, device=dev, dtype=dt), lse=torch.zeros(h, n, device=dev))
        if case["backward"]:
            s.update(dout=(0.1 * r(n, h, d)).to(dt), dq=torch.zeros(n, h, d, device=dev, dtype=dt),
                     dk=torch.zeros(n, kv, d, device=dev, dtype=dt), dv=torch.zeros(n, kv, d, device=dev, dtype=dt))
        return s
    dt, m, v, top = _DTYPES[case["dtype"]], case["rows"], case["vocab"], case["top"]
    z = torch.randn(m, v, generator=g, device=dev).mul_(2.0)
    # the teacher's top logits: the student's own score plus noise, the largest of them kept
    val, ids = (z + torch.randn(m, v, generator=g, device=dev)).topk(top, dim=1)
    if case["padded"]:  # some rows keep fewer than `top` of them, some none
        ids[torch.arange(top, device=dev)[None, :] >= torch.randint(0, 2 * top, (m, 1), generator=g, device=dev)] = -1
    if case["cap"]:
        z = torch.tanh(z.div_(case["cap"])).mul_(case["cap"])
    targets = None
    if case["alpha"] < 1.0:
        targets = torch.randint(0, v, (m,), generator=g, device=dev, dtype=torch.int32)
        targets[torch.rand(m, generator=g, device=dev) < 0.05] = -1
    return dict(case=case, logits=z.to(dt), ids=ids.to(torch.int32), teacher=val.float().contiguous(), targets=targets,
                grad=torch.zeros(m, v, device=dev, dtype=dt))


# ---------------------------------------------------------------------------------------------- one pass
def run(state):
    op = state["case"]["op"]
    if op == "bounds":
        return _bounds(state)
    return _attention(state) if op == "attention" else _distill(state)


def _bounds(s):
    case = s["case"]
    if own:
        from bitresearch_b200.ops import packed
        if case["source"] == "offsets":
            start, end = packed.bounds_from_offsets(s["offsets"], case["rows"])
        else:
            start, end = packed.bounds_from_ids(s["ids"], s["bos"])
        return {"start": start, "end": end}
    if case["source"] == "offsets":
        off, rows = s["offsets"], torch.arange(case["rows"], device="cuda", dtype=torch.int32)
        seq = torch.searchsorted(off, rows, right=True)
        inside = seq < off.numel()
        start = torch.where(inside, off[seq - 1], rows)
        end = torch.where(inside, off[seq.clamp(max=off.numel() - 1)], rows)
        return {"start": start.to(torch.int32), "end": end.to(torch.int32)}
    ids = s["ids"]
    batch, length = ids.shape
    rows = torch.arange(batch * length, device="cuda").view(batch, length)
    first = (ids == s["bos"]) | (rows == rows[:, :1])
    start = torch.where(first, rows, -1).cummax(1).values
    after = torch.cat([torch.where(first, rows, batch * length)[:, 1:], rows[:, -1:] + 1], 1)
    end = after.flip(1).cummin(1).values.flip(1)
    return {"start": start.reshape(-1).to(torch.int32), "end": end.reshape(-1).to(torch.int32)}


def _attention(s):
    case = s["case"]
    if own:
        from bitresearch_b200.ops import packed
        out, lse = packed.attention_fwd(s["q"], s["k"], s["v"], s["start"], s["end"], window=case["window"],
                                        out=s["out"], lse=s["lse"])
        if not case["backward"]:
            return {"out": out, "lse": lse}
        dq, dk, dv = packed.attention_bwd(s["q"], s["k"], s["v"], out, lse, s["dout"], s["start"], s["end"],
                                          window=case["window"], dq=s["dq"], dk=s["dk"], dv=s["dv"])
        return {"out": out, "lse": lse, "dq": dq, "dk": dk, "dv": dv}
    # the sequences side by side, padded to the longest: [sequences, heads, longest, dim]
    n, h, kv, d, longest = case["rows"], case["heads"], case["kv_heads"], case["dim"], s["longest"]
    off = s["offsets"]
    real = n - case["tail"]
    place = off[:-1, None] + torch.arange(longest, device="cuda")
    inside = (place < off[1:, None])[:, None, :, None]
    place = place.clamp(max=n - 1)
    wide = lambda x, heads: x.float()[place].transpose(1, 2).repeat_interleave(h // heads, 1)  # noqa: E731
    q, k, v = wide(s["q"], h), wide(s["k"], kv), wide(s["v"], kv)
    rows = torch.arange(real, device="cuda")
    seq = torch.searchsorted(off, rows, right=True) - 1
    flat = seq * longest + rows - off[seq]  # where row i sits in the padded form
    narrow = lambda x: x.transpose(1, 2).reshape(-1, x.shape[1], x.shape[3])[flat]  # noqa: E731
    i = torch.arange(longest, device="cuda")
    seen = i[:, None] >= i[None, :]
    if case["window"]:
        seen &= i[:, None] - i[None, :] < case["window"]
    scale = 1.0 / math.sqrt(d)
    p = (q @ k.transpose(2, 3)).mul_(scale).masked_fill_(~seen, -math.inf)
    top = p.amax(-1, keepdim=True)
    p = p.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    p = p.div_(total)
    o = p @ v
    s["out"][:real] = narrow(o).to(s["out"].dtype)
    s["lse"][:, :real] = narrow(top + total.log())[:, :, 0].t()
    if not case["backward"]:
        return {"out": s["out"], "lse": s["lse"]}
    do = wide(s["dout"], h) * inside
    dv = p.transpose(2, 3) @ do
    ds = (do @ v.transpose(2, 3)).sub_((do * o).sum(-1, keepdim=True)).mul_(p).mul_(scale)
    dq = ds @ k
    dk = ds.transpose(2, 3) @ q
    group = lambda x: x.view(x.shape[0], kv, h // kv, longest, d).sum(2)  # noqa: E731
    s["dq"][:real] = narrow(dq).to(s["dq"].dtype)
    s["dk"][:real] = narrow(group(dk)).to(s["dk"].dtype)
    s["dv"][:real] = narrow(group(dv)).to(s["dv"].dtype)
    return {"out": s["out"], "lse": s["lse"], "dq": s["dq"], "dk": s["dk"], "dv": s["dv"]}


def _distill(s):
    case = s["case"]
    m, cap, t, alpha, scale = case["rows"], case["cap"], case["temperature"], case["alpha"], _scale(case)
    if own:
        from bitresearch_b200.ops import distill
        loss, rows, grad = distill.distill_topk(s["logits"], s["ids"], s["teacher"], s["targets"], cap=cap,
                                                temperature=t, alpha=alpha, scale=scale, grad=s["grad"])
        return {"loss": loss, "rows": rows, "grad": grad}
    logits = s["logits"].float()
    kept = s["ids"] >= 0
    at = s["ids"].long().clamp(min=0)
    any_kept = kept.any(1)
    u = torch.where(kept, s["teacher"] / t, -math.inf)
    u = u - torch.where(any_kept, u.amax(1), torch.zeros_like(u[:, 0]))[:, None]
    logq = u - u.exp().sum(1, keepdim=True).clamp(min=1e-30).log()
    q = torch.where(kept, logq.exp(), torch.zeros_like(logq))
    x = logits / t
    top = x.amax(1, keepdim=True)
    x = x.sub_(top).exp_()
    total = x.sum(1, keepdim=True)
    logp = logits.gather(1, at) / t - top - total.log()
    kl = torch.where(q > 0, q * (logq - logp), torch.zeros_like(q)).sum(1)
    rows = alpha * t * t * kl
    dz = x.div_(total).mul_(any_kept[:, None]).scatter_add_(1, at, -q).mul_(alpha * t)
    if s["targets"] is not None:
        valid = s["targets"] >= 0
        target = s["targets"].long().clamp(min=0)[:, None]
        e = (logits - logits.amax(1, keepdim=True)).exp_()
        e = e.div_(e.sum(1, keepdim=True))
        pt = e.gather(1, target)
        rows = rows + (1 - alpha) * torch.where(valid, -(pt[:, 0] + _EPS).log(), torch.zeros_like(rows))
        r = (1 - alpha) * valid[:, None] * pt / (pt + _EPS)
        dz = dz.add_(e.scatter_add_(1, target, torch.full_like(pt, -1.0)).mul_(r))
    if cap:
        dz = dz.mul_(1 - (logits / cap) ** 2)
    s["grad"].copy_(dz.mul_(scale))
    return {"loss": rows.sum() * scale, "rows": rows, "grad": s["grad"]}


# ---------------------------------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    """The definition, sequence by sequence and head by head (or row block by row block), in fp64."""
    if case["op"] == "bounds":
        return None  # whole numbers
    s = prepare(case, seed)
    return _exact_attention(case, s) if case["op"] == "attention" else _exact_distill(case, s)


def _exact_attention(case, s):
    n, h, kv, d = case["rows"], case["heads"], case["kv_heads"], case["dim"]
    f8 = dict(dtype=torch.float64, device="cuda")
    res = {"out": torch.zeros(n, h, d, **f8), "lse": torch.zeros(h, n, **f8)}
    if case["backward"]:
        res.update(dq=torch.zeros(n, h, d, **f8), dk=torch.zeros(n, kv, d, **f8), dv=torch.zeros(n, kv, d, **f8))
    at = 0
    for length in _lengths(case):
        span = slice(at, at + length)
        at += length
        if not length:
            continue
        for a in range(h):
            b = a // (h // kv)
            q, k, v = s["q"][span, a].double(), s["k"][span, b].double(), s["v"][span, b].double()
            x = torch.mm(q, k.t()) / math.sqrt(d)
            hide = torch.ones_like(x, dtype=torch.bool).triu(1)
            if case["window"]:
                hide |= torch.ones_like(hide).tril(-case["window"])
            x[hide] = -math.inf
            lse = torch.logsumexp(x, 1)
            w = torch.exp(x - lse[:, None])
            o = torch.mm(w, v)
            res["out"][span, a] = o
            res["lse"][a, span] = lse
            if case["backward"]:
                do = s["dout"][span, a].double()
                res["dv"][span, b] += torch.mm(w.t(), do)
                dx = w * (torch.mm(do, v.t()) - torch.sum(do * o, 1)[:, None]) / math.sqrt(d)
                res["dq"][span, a] = torch.mm(dx, k)
                res["dk"][span, b] += torch.mm(dx.t(), q)
    return res


def _exact_distill(case, s):
    m, cap, t, alpha = case["rows"], case["cap"], case["temperature"], case["alpha"]
    rows, grad = torch.zeros(m, dtype=torch.float64, device="cuda"), torch.zeros(m, case["vocab"], device="cuda",
                                                                                 dtype=torch.float64)
    step = max(1, (1 << 26) // case["vocab"])
    for a in range(0, m, step):
        b = slice(a, min(m, a + step))
        z = s["logits"][b].double()
        soft = torch.log_softmax(z / t, 1)
        ids = s["ids"][b].long()
        some = (ids >= 0).any(1, keepdim=True)
        # the teacher's distribution over the whole vocabulary; a padded place has no mass
        spread = torch.full((z.shape[0], z.shape[1] + 1), -math.inf, dtype=torch.float64, device="cuda")
        spread.scatter_(1, torch.where(ids < 0, z.shape[1], ids), s["teacher"][b].double() / t)
        spread = spread[:, :-1]
        logq = torch.where(some, spread - torch.logsumexp(spread, 1, keepdim=True), spread)
        q = logq.exp()
        rows[b] = alpha * t * t * torch.where(q > 0, q * (logq - soft), 0.0).sum(1)
        g = alpha * t * (soft.exp() * some - q)
        if s["targets"] is not None:
            hard = torch.softmax(z, 1)
            goal = s["targets"][b].long()
            on = (goal >= 0).double()
            pt = hard[torch.arange(z.shape[0], device="cuda"), goal.clamp(min=0)]
            rows[b] += (1 - alpha) * on * -torch.log(pt + _EPS)
            one = torch.nn.functional.one_hot(goal.clamp(min=0), z.shape[1]).double()
            g += ((1 - alpha) * on * pt / (pt + _EPS))[:, None] * (hard - one)
        if cap:
            g *= 1 - (z / cap) ** 2
        grad[b] = g * _scale(case)
    return {"loss": rows.sum() * _scale(case), "rows": rows, "grad": grad}
