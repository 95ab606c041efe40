"""Top-logit distillation where a block takes many rows, one after the other: every row against a vectorised 64-bit form
(the tolerances are those of packed_ref.py's loops)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
BAD_INDEX = 6
REL = 2e-5  # exp of arguments up to about 60: 60 roundings of 2^-24, and the fp32 sums


def _op():
    from bitresearch_b200.ops.distill import distill_topk
    from bitresearch_b200.ops._ext import check_status
    assert check_status() == 0
    return distill_topk, check_status


def reference(z, ids, u, y, cap, t, alpha, scale):
    """(rows, grad, tolerance of the rows, tolerance of the gradient); ids of a row differ, -1 and other ids outside
    the vocabulary are unused places."""
    eps = torch.finfo(z.dtype).eps / 2
    sub = 2.0 ** -25 if z.dtype == torch.float16 else 0.0
    V = z.shape[1]
    out = []
    for a in range(0, z.shape[0], max(1, (1 << 25) // V)):
        b = slice(a, min(z.shape[0], a + max(1, (1 << 25) // V)))
        x, at = z[b].double(), ids[b].long()
        kept = (at >= 0) & (at < V)
        at = torch.where(kept, at, 0)
        some = kept.any(1, keepdim=True)
        logp = torch.log_softmax(x / t, 1)
        logq = torch.where(kept, u[b].double() / t, -math.inf)
        logq = logq - torch.where(some, torch.logsumexp(logq, 1, keepdim=True), 0.0)
        q = logq.exp()
        lp = logp.gather(1, at)
        rows = alpha * t * t * torch.where(q > 0, q * (logq - lp), 0.0).sum(1)
        row_tol = alpha * t * t * torch.where(q > 0, q * REL * (logq.abs() + lp.abs() + 1), 0.0).sum(1)
        mass = torch.zeros_like(x).scatter_add_(1, at, q)
        soft = alpha * t * some * logp.exp()
        g, terms = soft - alpha * t * mass, soft + alpha * t * mass
        if alpha < 1:
            goal = y[b].long()
            on = ((goal >= 0) & (goal < V))[:, None]
            goal = torch.where(on[:, 0], goal, 0)[:, None]
            p = torch.softmax(x, 1)
            py = p.gather(1, goal)
            ce = torch.where(on, -(py + 1e-10).log(), 0.0)[:, 0]
            rows = rows + (1 - alpha) * ce
            row_tol = row_tol + (1 - alpha) * REL * torch.where(on[:, 0], 1 + ce.abs(), 0.0)
            r = torch.where(on, (1 - alpha) * py / (py + 1e-10), 0.0)
            g = (g + r * p).scatter_add_(1, goal, -r)
            terms = (terms + r * p).scatter_add_(1, goal, r)
        slope = 1 - (x / cap) ** 2 if cap else torch.ones_like(x)
        g = scale * g * slope
        out.append((rows, g, row_tol, eps * g.abs() + abs(scale) * terms * (REL * slope.abs() + 1e-6) + sub))
    return [torch.cat(p) for p in zip(*out)]


def inputs(M, V, K, dt, cap, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    z = 3 * r(M, V)
    if cap:
        z = cap * torch.tanh(z / cap)
    # ids of a row are a step through the vocabulary from a place of its own, so they differ
    first = torch.randint(0, V, (M, 1), generator=g, device="cuda")
    ids = (first + torch.arange(K, device="cuda") * max(1, V // K)) % V
    ids[torch.rand(M, K, generator=g, device="cuda") < 0.1] = -1
    y = torch.randint(0, V, (M,), generator=g, device="cuda", dtype=torch.int32)
    y[torch.rand(M, generator=g, device="cuda") < 0.1] = -1
    return z.to(dt), ids.to(torch.int32), 4 * r(M, K), y


# the forms that hold a row in 16, 64 and 128 KB of a block, and in 2, 4 and 8 blocks; several rows for each of them
# on a GPU of 148 SMs
FORMS = [(6007, 1000, torch.bfloat16), (5003, 8192, torch.bfloat16), (4999, 3001, torch.float32), (6007, 77, torch.float16),
         (1001, 20_000, torch.bfloat16), (1003, 9999, torch.float32), (601, 60_001, torch.float16),
         (403, 130_000, torch.bfloat16), (301, 200_003, torch.float16), (101, 150_000, torch.float32)]


@pytest.mark.parametrize("M,V,dt", FORMS, ids=lambda x: str(x).replace("torch.", ""))
@pytest.mark.parametrize("t,alpha,cap", [(1.0, 1.0, 15.0), (1.0, 0.4, 0.0), (2.0, 0.5, 15.0), (1.5, 0.6, 15.0),
                                         (0.7, 0.3, 0.0)])
def test_every_row_of_a_block(cuda, M, V, dt, t, alpha, cap):
    op, check_status = _op()
    z, ids, u, y = inputs(M, V, 16, dt, cap, seed=V)
    args = dict(cap=cap, temperature=t, alpha=alpha, scale=0.5)
    loss, rows, grad = op(z, ids, u, y, **args)
    alone, rows2, none = op(z, ids, u, y, need_grad=False, **args)
    torch.cuda.synchronize()
    assert check_status() == 0 and none is None
    assert torch.equal(rows, rows2) and torch.equal(loss, alone)
    r, g, rt, gt = reference(z, ids, u, y, cap, t, alpha, 0.5)
    err = (rows.double() - r).abs()
    assert (err <= rt).all(), (int((err > rt).sum()), (err - rt).max().item())
    err = (grad.double() - g).abs()
    assert (err <= gt).all(), (int((err > gt).sum()), (err - gt).max().item())
    op(z, ids, u, y, grad=z, **args)
    assert torch.equal(z, grad)


def test_short_rows_in_turn(cuda):
    """Rows of a few values, where a row's time is shortest, many times over: the same bits each time."""
    op, _ = _op()
    z, ids, u, y = inputs(60_000, 40, 4, torch.bfloat16, 0.0, seed=1)
    r, g, rt, gt = reference(z, ids, u, y, 0.0, 1.5, 0.5, 1.0)
    first = None
    for need_grad in (True, False) * 5:
        _, rows, grad = op(z, ids, u, y, cap=0.0, temperature=1.5, alpha=0.5, scale=1.0, need_grad=need_grad)
        first = rows if first is None else first
        assert torch.equal(rows, first)
        assert grad is None or ((grad.double() - g).abs() <= gt).all()
    assert ((first.double() - r).abs() <= rt).all()


@pytest.mark.parametrize("M,V,dt", [FORMS[1], FORMS[4], FORMS[6], FORMS[7]], ids=lambda x: str(x).replace("torch.", ""))
@pytest.mark.parametrize("t,alpha", [(1.0, 1.0), (2.0, 0.5)])
def test_a_bad_id_costs_its_own_entry_alone(cuda, M, V, dt, t, alpha):
    """Ids outside the vocabulary in the first rows, while thousands of waits of the other rows are still to come; and a
    call while the status word still holds the last one's report."""
    op, check_status = _op()
    z, ids, u, y = inputs(M, V, 16, dt, 15.0, seed=V + 1)
    ids[0, 3], ids[1, 0], ids[2] = V, -7, 2 ** 31 - 1
    y[3] = V
    r, g, rt, gt = reference(z, ids, u, y, 15.0, t, alpha, 1.0)
    for _ in range(2):
        _, rows, grad = op(z, ids, u, y, cap=15.0, temperature=t, alpha=alpha, scale=1.0)
        assert ((rows.double() - r).abs() <= rt).all() and ((grad.double() - g).abs() <= gt).all()
    assert check_status() == BAD_INDEX


@pytest.mark.parametrize("V", [1000, 70_000])
def test_a_teacher_of_no_weight_is_not_read_into_the_result(cuda, V):
    """alpha = 0: loss and gradient are those of the hard labels, whatever the teacher's logits hold."""
    op, check_status = _op()
    z, ids, u, y = inputs(50, V, 8, torch.float32, 15.0, seed=2)
    want = op(z, ids, u, y, alpha=0.0)
    for what in (math.nan, math.inf, -math.inf):
        got = op(z, ids, torch.full_like(u, what), y, alpha=0.0)
        assert all(torch.equal(a, b) for a, b in zip(want, got))
    assert torch.isfinite(want[2]).all() and check_status() == 0
