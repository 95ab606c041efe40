"""Top-logit distillation on the GPU against loops in 64 bits (packed_ref.py has the tolerances)."""
import math

import pytest
import torch

from packed_ref import distill as reference

pytestmark = pytest.mark.gpu
BAD_INDEX = 6


def _op():
    from bitresearch_b200.ops.distill import distill_topk
    from bitresearch_b200.ops._ext import check_status
    assert check_status() == 0
    return distill_topk, check_status


def _inputs(M, V, K, dt, cap, seed=0, teacher_dt=torch.float32):
    g = torch.Generator().manual_seed(seed)
    z = 3 * torch.randn(M, V, generator=g)
    if cap:
        z = cap * torch.tanh(z / cap)
    z = z.to(dt).cuda()
    ids = torch.stack([torch.randperm(V, generator=g)[:K] for _ in range(M)]).to(torch.int32).cuda()
    u = (4 * torch.randn(M, K, generator=g)).to(teacher_dt).cuda()
    y = torch.randint(0, V, (M,), generator=g, dtype=torch.int32)
    y[torch.rand(M, generator=g) < 0.2] = -1
    return z, ids, u, y.cuda()


def _check(z, ids, u, y, cap, t, alpha, scale, **kw):
    op, check_status = _op()
    before = z.clone()
    loss, rows, grad = op(z, ids, u, y, cap=cap, temperature=t, alpha=alpha, scale=scale, **kw)
    torch.cuda.synchronize()
    assert check_status() == 0
    r, g, rt, gt = reference(before, ids, u, y, cap, t, alpha, scale)
    assert ((rows.double().cpu() - r).abs() <= rt).all(), ((rows.double().cpu() - r).abs() - rt).max()
    assert abs(loss.item() - scale * r.sum().item()) <= abs(scale) * (rt.sum().item() + 1e-6 * r.abs().sum().item())
    if grad is not None:
        err = (grad.double().cpu() - g).abs()
        assert (err <= gt).all(), (err - gt).max()
    return loss, rows, grad


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16, torch.float16], ids=["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("V", [1, 7, 64, 1000, 1001, 2048, 8192, 9999])
@pytest.mark.parametrize("t,alpha,cap", [(1.0, 1.0, 15.0), (2.0, 0.5, 15.0), (0.7, 1.0, 0.0), (1.0, 0.0, 15.0)])
def test_sizes_and_types(cuda, dt, V, t, alpha, cap):
    z, ids, u, y = _inputs(5, V, min(V, 16), dt, cap, seed=V)
    _check(z, ids, u, y, cap, t, alpha, 0.25)


@pytest.mark.parametrize("V", [16384, 32771, 65536, 131072, 200_003])
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
def test_wide_rows(cuda, V, dt):
    z, ids, u, y = _inputs(2, V, 64, dt, 15.0, seed=V)
    _check(z, ids, u, y, 15.0, 1.5, 0.6, 1.0)
    _check(z, ids, u, y, 15.0, 1.0, 1.0, 1.0, grad=z)


@pytest.mark.parametrize("K", [1, 2, 33, 255, 1024])
@pytest.mark.parametrize("teacher_dt", [torch.float32, torch.bfloat16, torch.float16], ids=["fp32", "bf16", "fp16"])
def test_entries(cuda, K, teacher_dt):
    z, ids, u, y = _inputs(3, 1200, K, torch.bfloat16, 15.0, seed=K, teacher_dt=teacher_dt)
    _check(z, ids, u, y, 15.0, 2.0, 0.9, 1 / 3)


def test_unused_places_repeated_ids_and_empty_rows(cuda):
    z, ids, u, y = _inputs(6, 50, 8, torch.float32, 15.0)
    ids[0, 3:] = -1
    u[0, 3:] = math.nan          # an unused place is not read
    ids[1] = -1                  # no entry at all
    ids[2] = 7                   # one column eight times
    ids[3, :4] = int(y[3]) if int(y[3]) >= 0 else 4  # repeated, and the target's own column
    y[3] = ids[3, 0]
    u[4, 2] = -math.inf          # an entry without mass
    u[5] = -math.inf             # a row whose entries have none
    _check(z, ids, u, y, 15.0, 1.3, 0.5, 1.0)
    _check(z, ids, u, y, 15.0, 1.0, 1.0, 1.0)


def test_masked_logits(cuda):
    """Logits of -inf (a mask), the type's lowest value, and rows that the mask leaves empty."""
    z, ids, u, y = _inputs(5, 40, 4, torch.float32, 0.0)
    y[:] = 1
    z[0, 10:] = -math.inf
    z[1, 10:] = torch.finfo(torch.float32).min
    z[2] = -math.inf
    z[3] = torch.finfo(torch.float32).min
    ids[0] = torch.tensor([0, 1, 2, 3])
    ids[1] = torch.tensor([0, 1, 2, 3])
    _check(z[[0, 3, 4]], ids[[0, 3, 4]], u[[0, 3, 4]], y[[0, 3, 4]], 0.0, 1.0, 0.5, 1.0)
    op, _ = _op()
    loss, rows, grad = op(z, ids, u, y, cap=0.0, alpha=0.5, scale=1.0)
    assert (grad[2] == 0).all() and rows[2].item() == math.inf
    assert torch.isfinite(grad).all() and (grad[0, 10:] == 0).all() and (grad[1, 10:] == 0).all()
    assert torch.isfinite(rows[[0, 1, 3, 4]]).all()


def test_no_numbers_stay_in_their_row(cuda):
    op, _ = _op()
    z, ids, u, y = _inputs(5, 300, 8, torch.bfloat16, 15.0)
    _, want_rows, want = op(z, ids, u, y, alpha=0.5, scale=1.0)
    z[1, 77] = math.nan
    u[3, 2] = math.nan
    _, rows, grad = op(z, ids, u, y, alpha=0.5, scale=1.0)
    keep = [0, 2, 4]
    assert torch.equal(rows[keep], want_rows[keep]) and torch.equal(grad[keep], want[keep])
    assert rows[[1, 3]].isnan().all() and grad[1].isnan().all()
    # a teacher's entry reaches the gradient of the columns that the row's entries name, and no other
    named = torch.zeros(300, dtype=torch.bool, device="cuda")
    named[ids[3].long()] = True
    assert grad[3][named].isnan().all() and torch.isfinite(grad[3][~named]).all()


def test_bad_ids_are_reported_and_skipped(cuda):
    op, check_status = _op()
    big = torch.full((4, 64), 5.0, device="cuda")
    z, ids, u, y = _inputs(4, 60, 4, torch.float32, 15.0)
    y[:] = 3
    want = ids.clone()
    ids[0, 1], ids[2, 0] = 60, -5
    want[0, 1], want[2, 0] = -1, -1
    y2 = y.clone()
    y2[1] = 61
    grad = big[:, :60]
    loss, rows, _ = op(z, ids, u, y2, alpha=0.5, scale=1.0, grad=grad)
    torch.cuda.synchronize()
    assert check_status() == BAD_INDEX
    y[1] = -1
    r, g, rt, gt = reference(z, want, u, y, 15.0, 1.0, 0.5, 1.0)
    assert ((rows.double().cpu() - r).abs() <= rt).all() and ((grad.double().cpu() - g).abs() <= gt).all()
    assert (big[:, 60:] == 5.0).all()


@pytest.mark.parametrize("V", [1000, 1003, 8192, 70_000])
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
def test_strides_alignment_and_place(cuda, V, dt):
    """Rows that start off a 16-byte boundary, different strides in and out, in place, and no gradient."""
    op, _ = _op()
    M, K = 6, 12
    z, ids, u, y = _inputs(M, V, K, dt, 15.0, seed=3)
    args = dict(cap=15.0, temperature=2.0, alpha=0.5, scale=0.5)
    # another alignment cuts the row into other vectors and adds its sums in another order, so the bits may differ: each
    # call is held to the 64-bit form
    r, g, rt, gt = (x.cuda() for x in reference(z, ids, u, y, 15.0, 2.0, 0.5, 0.5))
    near = lambda rows, grad: bool(((rows.double() - r).abs() <= rt).all() and ((grad.double() - g).abs() <= gt).all())  # noqa: E731
    _, rows, _ = op(z, ids, u, y, **args)
    for off, pad in ((0, 5), (1, 0), (3, 8)):
        wide = torch.full((M, V + off + pad), 9.0, device="cuda").to(dt)
        wide[:, off:off + V] = z
        wide_ids = torch.zeros(M, K + 3, dtype=torch.int32, device="cuda")
        wide_ids[:, 1:K + 1] = ids
        out = torch.full((M, V + 2), 9.0, device="cuda").to(dt)
        _, r1, _ = op(wide[:, off:off + V], wide_ids[:, 1:K + 1], u, y, grad=out[:, 1:V + 1], **args)
        assert near(r1, out[:, 1:V + 1])
        assert (out[:, 0] == 9).all() and (out[:, -1] == 9).all()
        _, r2, g2 = op(wide[:, off:off + V], ids, u, y, grad=wide[:, off:off + V], **args)
        assert near(r2, wide[:, off:off + V])
        assert (wide[:, :off] == 9).all() and (wide[:, off + V:] == 9).all()
    l3, r3, none = op(z, ids, u, y, need_grad=False, **args)
    assert none is None and torch.equal(r3, rows)


def test_offsets_past_32_bits(cuda):
    op, _ = _op()
    M, V, K = 34_000, 65_536, 4
    if torch.cuda.get_device_properties(0).total_memory < 30e9:
        pytest.skip("needs 30 GB")
    z = torch.empty(M, V, dtype=torch.bfloat16, device="cuda").normal_(std=3.0)
    ids = torch.randint(0, V, (M, K), device="cuda", dtype=torch.int32)
    u = torch.randn(M, K, device="cuda")
    last = z[-2:].clone()
    _, rows, _ = op(z, ids, u, cap=15.0, scale=1.0, grad=z)
    r, g, rt, gt = reference(last, ids[-2:], u[-2:], None, 15.0, 1.0, 1.0, 1.0)
    assert ((rows[-2:].double().cpu() - r).abs() <= rt).all() and ((z[-2:].double().cpu() - g).abs() <= gt).all()


def test_empty_batch_and_default_scale(cuda):
    op, _ = _op()
    z, ids, u, y = _inputs(4, 100, 8, torch.bfloat16, 15.0)
    loss, rows, grad = op(z[:0], ids[:0], u[:0])
    assert loss.item() == 0.0 and rows.numel() == 0 and grad.shape == (0, 100)
    loss, rows, _ = op(z, ids, u)
    assert abs(loss.item() - rows.double().mean().item()) <= 1e-6 * abs(loss.item())


def test_same_bits_two_streams_and_graph(cuda):
    op, _ = _op()
    sets = [_inputs(300, 2000, 16, torch.bfloat16, 15.0, seed=s) for s in range(2)]
    call = lambda s: op(*s, temperature=2.0, alpha=0.5)  # noqa: E731
    want = [call(s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = []
    for _ in range(4):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got.append((i, call(sets[i])))
    torch.cuda.synchronize()
    for i, r in got:
        assert all(torch.equal(a, b) for a, b in zip(want[i], r))
    graphs = []
    for s in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            r = call(s)
        graphs.append((g, r))
    for _ in range(2):
        for (g, r), st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    for w, (g, r) in zip(want, graphs):
        assert all(torch.equal(a, b) for a, b in zip(w, r))
