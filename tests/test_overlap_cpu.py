"""Outputs that share memory with another argument are refused, views of one buffer that only lie between each other's
rows are not. The check comes before the first use of a device, so a call that passes it ends at "CUDA device"."""
import random

import pytest
import torch

from bitresearch_b200.ops import distill, packed
from bitresearch_b200.ops._ext import available
from packed_ref import spans

pytestmark = pytest.mark.skipif(not available(), reason="native module not built")


def _view(buf, n, heads, row, head, at):
    return buf.as_strided((n, heads, 64), (row, head, 1), at)


def _places(t):
    """The buffer's elements that a view holds, and whether one stands in it twice."""
    i = torch.arange(t.untyped_storage().nbytes() // t.element_size()).as_strided(t.shape, t.stride(), t.storage_offset())
    s = set(i.flatten().tolist())
    return s, len(s) != i.numel()


def _refused(call):
    try:
        call()
    except ValueError as e:
        assert "CUDA device" in str(e), e
        return False
    except RuntimeError as e:
        assert "memory" in str(e), e
        return True
    raise AssertionError("nothing was raised")


def test_attention_forward_against_all_places():
    rng, seen = random.Random(0), {False: 0, True: 0}
    buf = torch.zeros(1 << 14, dtype=torch.bfloat16)
    for _ in range(600):
        n = rng.choice([1, 2, 3, 7])
        H = rng.choice([1, 2, 4])

        def view():
            head = 64 * rng.choice([1, 1, 2, 3])
            row = max(64, head * H) + 8 * rng.choice([0, 0, 8, 16, 24, 5])
            if rng.random() < 0.3:  # heads outside
                row, head = 64 * rng.choice([1, 2]), 64 * n * rng.choice([1, 2]) + 64 * rng.choice([0, 1])
            return _view(buf, n, H, row, head, 8 * rng.choice([0, 8, 16, 24, 3, 64, 200]))
        q, out = view(), view()
        k = v = torch.zeros(n, H, 64, dtype=torch.bfloat16)
        (a, _), (b, twice) = _places(q), _places(out)
        # rows or heads of the output that interlock are refused as well, whether or not an element stands twice
        counts = sorted(((s, c) for s, c in ((out.stride(0), n), (out.stride(1), H)) if c > 1))
        span, interlock = 64, False
        for step, count in counts:
            interlock |= step < span
            span += step * (count - 1)
        want = bool(a & b) or twice or interlock
        got = _refused(lambda: packed.attention_fwd(q, k, v, *spans([n], n), out=out))
        assert got == want, (n, H, q.stride(), q.storage_offset(), out.stride(), out.storage_offset())
        seen[got] += 1
    assert min(seen.values()) > 50


def test_views_of_one_buffer():
    n, H, KV = 9, 4, 2
    start, end = spans([n], n)
    qkv = torch.zeros(n, H + 2 * KV, 64, dtype=torch.bfloat16)
    q, k, v = qkv[:, :H], qkv[:, H:H + KV], qkv[:, H + KV:]
    o, do, lse = torch.zeros_like(q), torch.zeros_like(q), torch.zeros(H, n)
    d = torch.zeros_like(qkv)
    dq, dk, dv = d[:, :H], d[:, H:H + KV], d[:, H + KV:]
    bwd = lambda **kw: _refused(lambda: packed.attention_bwd(q, k, v, o, lse, do, start, end, **kw))  # noqa: E731
    assert not bwd(dq=dq, dk=dk, dv=dv)
    assert bwd(dq=dq, dk=dk, dv=d[:, H + 1:H + 1 + KV])
    assert bwd(dq=q, dk=dk, dv=dv)
    assert bwd(dk=v, dv=dv)
    big = torch.zeros(packed.bwd_scratch(n, H) + H * n)
    assert not bwd(scratch=big[:packed.bwd_scratch(n, H)])
    lse = big[:H * n].view(H, n)
    assert bwd(scratch=big[:packed.bwd_scratch(n, H)])
    fwd = lambda **kw: _refused(lambda: packed.attention_fwd(q, k, v, start, end, **kw))  # noqa: E731
    assert fwd(out=q) and fwd(out=qkv[:, 1:1 + H]) and not fwd(out=dq)
    both = torch.zeros(n * H * 64 + 2 * H * n, dtype=torch.bfloat16)
    out = both[:n * H * 64].view(n, H, 64)
    assert fwd(out=out, lse=both[:2 * H * n].view(torch.float32).view(H, n))
    assert not fwd(out=out, lse=both[n * H * 64:].view(torch.float32).view(H, n))


def test_bounds():
    ids = torch.zeros(2, 6, dtype=torch.int32)
    s = torch.zeros(24, dtype=torch.int32)
    assert _refused(lambda: packed.bounds_from_ids(ids, 1, s[:12], s[:12]))
    assert _refused(lambda: packed.bounds_from_ids(ids, 1, s[:12], s[11:23]))
    assert _refused(lambda: packed.bounds_from_ids(ids, 1, ids.view(-1), s[:12]))
    assert not _refused(lambda: packed.bounds_from_ids(ids, 1, s[:12], s[12:]))
    assert _refused(lambda: packed.bounds_from_offsets(s[:3], 12, s[2:14]))


def test_distill():
    wide, u = torch.zeros(4, 40), torch.zeros(4, 3)
    ids = torch.zeros(4, 3, dtype=torch.int32)
    call = lambda z, **kw: _refused(lambda: distill.distill_topk(z, ids, u, **kw))  # noqa: E731
    z = wide[:, :16]
    assert not call(z, grad=z) and not call(z, grad=wide[:, 16:32]) and not call(z, grad=wide[:, :16])
    assert call(z, grad=wide[:, 1:17]) and call(z, grad=wide[:, 15:31])
    assert call(z, grad=wide.as_strided((4, 16), (17, 1)))
    one = torch.zeros(1, 40)
    assert not _refused(lambda: distill.distill_topk(one[:, :16], ids[:1], u[:1], grad=one.view(-1)[:16].view(1, 16)))
    assert _refused(lambda: distill.distill_topk(z, ids, wide[:, 30:33], grad=wide[:, 20:36]))
