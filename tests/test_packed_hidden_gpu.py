"""Values that are no numbers in rows of a row's own sequence that it does not see (later ones, ones outside its
window): its results are what they are without them."""
import math

import pytest
import torch

from packed_ref import attention, spans, visible

pytestmark = pytest.mark.gpu


def _ops():
    from bitresearch_b200.ops import packed
    from bitresearch_b200.ops._ext import check_status
    assert check_status() == 0
    return packed, check_status


def _inputs(n, H, KV, D, dt):
    g = torch.Generator(device="cuda").manual_seed(n + H)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda").to(dt)  # noqa: E731
    return r(n, H, D), r(n, KV, D), r(n, KV, D), r(n, H, D)


def _within(got, ref, rows, what):
    value, tol = (t[rows] for t in ref)
    bad = ~((got[rows].double() - value).abs() <= tol)
    assert not bad.any(), (what, int(bad.sum()), bad.nonzero()[:3].tolist())


@pytest.mark.parametrize("what", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("H,KV,D,dt", [(4, 2, 128, torch.bfloat16), (3, 3, 64, torch.float16), (2, 1, 64, torch.bfloat16)])
@pytest.mark.parametrize("lengths,window", [([1000], 0), ([1000], 200), ([90, 700, 210], 0), ([90, 700, 210], 65)])
@pytest.mark.parametrize("at", [[333], [130, 560, 561], [0], [999]], ids=str)
def test_hidden_rows(cuda, lengths, window, H, KV, D, dt, what, at):
    packed, check_status = _ops()
    n = sum(lengths)
    start, end = (t.cuda() for t in spans(lengths, n))
    see = visible(start, end, window)
    hit = torch.zeros(n, dtype=torch.bool, device="cuda")
    hit[at] = True
    q, k, v, do = _inputs(n, H, KV, D, dt)
    zero = lambda t: torch.where(hit[:, None, None], torch.zeros_like(t), t)  # noqa: E731
    scale = 1 / math.sqrt(D)
    # forward: the rows that see none of them; a row's hidden keys may hold anything
    fwd_ok = ~(see & hit[None, :]).any(1)
    kk, vv = k.clone(), v.clone()
    kk[hit, :, 5] = what
    vv[hit, :, 7] = what
    out, lse = packed.attention_fwd(q, kk, vv, start, end, window=window)
    clean = attention(q, zero(k), zero(v), start, end, window, scale, do)
    _within(out, clean["out"], fwd_ok, "out")
    _within(lse.t(), tuple(t.t() for t in clean["lse"]), fwd_ok, "lse")
    # backward: dq of rows that see none of the keys, from outputs that are right for those rows
    dq, _, _ = packed.attention_bwd(q, kk, vv, out, lse, do, start, end, window=window)
    _within(dq, clean["dq"], fwd_ok, "dq")
    # dk, dv of the keys that no poisoned query sees
    key_ok = ~(see & hit[:, None]).any(0)
    good = packed.attention_fwd(q, k, v, start, end, window=window)
    qq, dd = q.clone(), do.clone()
    qq[hit, :, 3] = what
    dd[hit, 0, 9] = what
    clean = attention(zero(q), k, v, start, end, window, scale, zero(do))
    _, dk, dv = packed.attention_bwd(qq, k, v, *good, dd, start, end, window=window)
    _within(dk, clean["dk"], key_ok, "dk")
    _within(dv, clean["dv"], key_ok, "dv")
    torch.cuda.synchronize()
    assert check_status() == 0


@pytest.mark.parametrize("what", ["v", "v column", "do", "do row", "everything"])
def test_no_numbers_throughout_cost_little(cuda, what):
    """A long sequence in which most rows rightly come out as no numbers does not compute them one by one."""
    packed, check_status = _ops()
    n, H, KV, D = 40_000, 4, 2, 128
    q, k, v, do = _inputs(n, H, KV, D, torch.bfloat16)
    start, end = (t.cuda() for t in spans([n], n))
    if what == "v":
        v[100:] = math.nan
    elif what == "v column":
        v[:, :, 3] = math.nan
    elif what == "do":
        do[:] = math.nan
    elif what == "do row":
        do[n - 50] = math.nan
    else:
        for t in (q, k, v, do):
            t[:] = math.nan

    def run():
        out, lse = packed.attention_fwd(q, k, v, start, end)
        packed.attention_bwd(q, k, v, out, lse, do, start, end)
        return out

    out = run()
    a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    a.record()
    run()
    b.record()
    torch.cuda.synchronize()
    assert check_status() == 0
    if what == "v":
        assert torch.isfinite(out[:100]).all() and out[100:].isnan().all()
    elif what == "v column":
        assert out[:, :, 3].isnan().all() and torch.isfinite(out[:, :, 4:]).all()
    # 30 ms without them; row by row it would be the order of a second
    assert a.elapsed_time(b) < 200, a.elapsed_time(b)


@pytest.mark.parametrize("what", ["v", "v column", "do", "do column"])
def test_infinities_throughout_cost_little(cuda, what):
    """As overflowed half-precision values are: the computation of a row alone ends at the first infinity too."""
    packed, check_status = _ops()
    n, H, KV, D = 40_000, 4, 2, 128
    q, k, v, do = _inputs(n, H, KV, D, torch.float16)
    start, end = (t.cuda() for t in spans([n], n))
    if what == "v":
        v[100:] = math.inf
    elif what == "v column":
        v[:, :, 3] = -math.inf
    elif what == "do":
        do[:] = math.inf
    else:
        do[:, :, 5] = math.inf

    def run():
        out, lse = packed.attention_fwd(q, k, v, start, end)
        return out, *packed.attention_bwd(q, k, v, out, lse, do, start, end)

    run()
    a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    a.record()
    out, dq, dk, dv = run()
    b.record()
    torch.cuda.synchronize()
    assert check_status() == 0
    if what == "v":
        assert torch.isfinite(out[:100]).all() and not torch.isfinite(out[100:]).any()
    elif what == "v column":
        assert not torch.isfinite(out[:, :, 3]).any() and torch.isfinite(out[:, :, 4:]).all()
    elif what == "do column":
        assert not torch.isfinite(dv[:, :, 5]).any() and torch.isfinite(dv[:, :, 6:]).all()
    assert a.elapsed_time(b) < 200, a.elapsed_time(b)


def test_rows_by_themselves_in_a_very_long_sequence(cuda):
    """Some rows at the end of 400,060 are computed alone, which takes seconds: no other warp's wait runs out."""
    packed, check_status = _ops()
    L, H, KV, D = 400_060, 2, 1, 64  # 60 rows share their tile with the next sequence
    n = L + 100
    q, k, v, _ = _inputs(n, H, KV, D, torch.bfloat16)
    start, end = (t.cuda() for t in spans([L, 100], n))
    want = packed.attention_fwd(q, k, v, start, end)
    v[L, 0, 3] = math.nan
    out, lse = packed.attention_fwd(q, k, v, start, end)
    torch.cuda.synchronize()
    assert check_status() == 0
    # computed in another order, in fp32: both are within a rounding of P and of the result
    near = 2.0 ** -8 * want[0][L - 200:L].float().abs() + 2.0 ** -8 * v[:L].float().abs().mean()
    assert ((out[L - 200:L].float() - want[0][L - 200:L].float()).abs() <= near).all()
    assert torch.equal(lse[:, :L], want[1][:, :L]) and torch.equal(out[:L - 1000], want[0][:L - 1000])
