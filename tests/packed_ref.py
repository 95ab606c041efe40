"""Plain 64-bit forms of packed attention and top-logit distillation, with the error that one rounding of each
16-bit quantity may cause (half a step: ``finfo.eps / 2`` relative)."""
import math

import torch

F32_SLACK = 1e-4  # fp32 sums of up to a few thousand products and the approximate exp2: far below a 16-bit half step
SUBNORMAL = 2.0 ** -25  # half of fp16's smallest step; bf16's is far below fp32's own error


def spans(lengths, rows):
    start, end = list(range(rows)), list(range(rows))
    at = 0
    for n in lengths:
        start[at:at + n], end[at:at + n] = [at] * n, [at + n] * n
        at += n
    return torch.tensor(start, dtype=torch.int32), torch.tensor(end, dtype=torch.int32)


def visible(start, end, window):
    n = start.numel()
    i = torch.arange(n, device=start.device)
    j = i[None, :]
    m = (j >= start[:, None]) & (j <= i[:, None]) & (j < end[:, None])
    return m & (i[:, None] - j < window) if window else m


def attention(q, k, v, start, end, window, scale, dout=None):
    """{name: (value, tolerance)} of out, lse and, with ``dout``, dq, dk, dv; rows of no sequence are zero."""
    eps = torch.finfo(q.dtype).eps / 2
    sub = SUBNORMAL if q.dtype == torch.float16 else 0.0
    n, H, D = q.shape
    KV = k.shape[1]
    f8 = dict(dtype=torch.float64, device=q.device)
    names = {"out": (n, H, D), "lse": (H, n)}
    if dout is not None:
        names.update(dq=(n, H, D), dk=(n, KV, D), dv=(n, KV, D))
    val = {a: torch.zeros(s, **f8) for a, s in names.items()}
    tol = {a: torch.zeros(s, **f8) for a, s in names.items()}
    see = visible(start, end, window)
    has = see.any(1)
    count = see.sum(1).double()
    for h in range(H):
        g = h // (H // KV)
        # a row that is not seen takes no part: what it holds must not matter
        Q, K, V = (torch.where(has[:, None], t.double(), 0.0) for t in (q[:, h], k[:, g], v[:, g]))
        x = (Q @ K.t() * scale).masked_fill(~see, -math.inf)
        lse = torch.where(has, torch.logsumexp(x, 1), 0.0)
        p = torch.where(see, torch.exp(x - lse[:, None]), 0.0)
        o = p @ V
        val["out"][:, h], val["lse"][h] = o, lse
        o_err = (eps + F32_SLACK) * (p @ V.abs()) + sub * count[:, None] * V.abs().amax()
        tol["out"][:, h] = eps * o.abs() + o_err + sub
        tol["lse"][h] = 1e-4 + 1e-6 * lse.abs()
        if dout is None:
            continue
        G = torch.where(has[:, None], dout[:, h].double(), 0.0)
        dp = G @ V.t()
        delta = (G * o).sum(1, keepdim=True)
        ds = torch.where(see, p * (dp - delta), 0.0)
        # dS: its own rounding, the error of delta through the rounded out, the fp32 error of P and dP
        d_err = (G.abs() * (eps * o.abs() + o_err)).sum(1, keepdim=True)
        ds_err = torch.where(see, eps * ds.abs() + p * d_err + F32_SLACK * p * (G.abs() @ V.abs().t() + delta.abs()) + sub,
                             0.0)
        val["dq"][:, h] = scale * ds @ K
        tol["dq"][:, h] = eps * val["dq"][:, h].abs() + scale * ds_err @ K.abs() + sub
        val["dk"][:, g] += scale * ds.t() @ Q
        tol["dk"][:, g] += scale * ds_err.t() @ Q.abs()
        val["dv"][:, g] += p.t() @ G
        tol["dv"][:, g] += (eps + F32_SLACK) * (p.t() @ G.abs()) + sub * see.t().double() @ G.abs()
    if dout is not None:
        for a in ("dk", "dv"):
            tol[a] += eps * val[a].abs() + sub
    return {a: (val[a], tol[a]) for a in names}


def distill(logits, ids, teacher, targets, cap, t, alpha, scale):
    """(rows, grad, tolerance of the rows, tolerance of the gradient), by loops over rows and entries."""
    z = logits.double().cpu()
    M, V = z.shape
    eps = torch.finfo(logits.dtype).eps / 2
    sub = SUBNORMAL if logits.dtype == torch.float16 else 0.0
    rows, grad = torch.zeros(M, dtype=torch.float64), torch.zeros(M, V, dtype=torch.float64)
    row_tol, grad_tol = torch.zeros_like(rows), torch.zeros_like(grad)
    rel = 2e-5  # exp of arguments up to about 60: 60 roundings of 2^-24, and the fp32 sums
    for m in range(M):
        dead = bool((z[m] == -math.inf).all())
        slope = 1 - (z[m] / cap) ** 2 if cap else torch.ones(V, dtype=torch.float64)
        g, terms = torch.zeros(V, dtype=torch.float64), torch.zeros(V, dtype=torch.float64)
        kept = [i for i in range(ids.shape[1]) if 0 <= int(ids[m, i]) < V]
        u = teacher[m].double().cpu()[kept] / t
        if kept and bool((u > -math.inf).any()):
            logq = u - torch.logsumexp(u, 0)
            q = logq.exp()
            logp = torch.full((V,), -math.inf, dtype=torch.float64) if dead else torch.log_softmax(z[m] / t, 0)
            for i, lq, w in zip(kept, logq.tolist(), q.tolist()):
                if w > 0:
                    lp = float(logp[int(ids[m, i])])
                    rows[m] += alpha * t * t * w * (lq - lp)
                    row_tol[m] += alpha * t * t * w * (rel * (abs(lq) + abs(lp)) + rel) if math.isfinite(lp) else 0.0
            if not dead:
                g += alpha * t * logp.exp()
                terms += alpha * t * logp.exp()
                for i, w in zip(kept, q.tolist()):
                    g[int(ids[m, i])] -= alpha * t * w
                    terms[int(ids[m, i])] += alpha * t * w
        y = int(targets[m]) if targets is not None and alpha < 1 else -1
        if 0 <= y < V:
            p = torch.zeros(V, dtype=torch.float64) if dead else torch.softmax(z[m], 0)
            ce = -math.log(float(p[y]) + 1e-10)
            rows[m] += (1 - alpha) * ce
            row_tol[m] += (1 - alpha) * rel * (1 + abs(ce))
            if not dead:
                r = (1 - alpha) * float(p[y]) / (float(p[y]) + 1e-10)
                g += r * p
                g[y] -= r
                terms += r * p
                terms[y] += r
        if not dead:
            grad[m] = scale * g * slope
            grad_tol[m] = eps * grad[m].abs() + abs(scale) * terms * (rel * slope.abs() + 1e-6) + sub
    return rows, grad, row_tol, grad_tol
