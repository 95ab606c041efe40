"""Packed attention with several work items for every SM, of either kind of item (two heads, two row tiles), against 64
bits; against the fixed-length kernels on whole rows; and with spans that are none, between guard rows."""
import math
import random

import pytest
import torch

from packed_ref import attention, spans

pytestmark = pytest.mark.gpu


def _ops():
    from bitresearch_b200.ops import packed
    from bitresearch_b200.ops._ext import check_status
    assert check_status() == 0
    return packed, check_status


def _within(got, ref, what):
    value, tol = ref
    bad = ~((got.double() - value).abs() <= tol)
    assert not bad.any(), (what, int(bad.sum()), bad.nonzero()[:3].tolist())


def _by_pieces(lengths, rows):
    """Consecutive sequences of up to ``rows`` rows together: (first row, lengths)."""
    at, piece = 0, []
    for n in lengths:
        if piece and sum(piece) + n > rows:
            yield at, piece
            at, piece = at + sum(piece), []
        piece.append(n)
    yield at, piece


@pytest.mark.parametrize("H,KV", [(8, 2), (4, 4), (6, 2), (3, 1)])
@pytest.mark.parametrize("D,dt", [(64, torch.bfloat16), (128, torch.float16), (64, torch.float16), (128, torch.bfloat16)],
                         ids=lambda x: str(x).replace("torch.", ""))
@pytest.mark.parametrize("window", [0, 300])
def test_every_item_of_a_block(cuda, H, KV, D, dt, window):
    """More work items than a B200 has SMs: blocks take over others. Their two tiles are two heads or two row tiles, whole
    and cut off, with the same key ranges and with others."""
    packed, check_status = _ops()
    rng = random.Random(H * D)
    lengths = [rng.choice([0, 1, 7, 63, 64, 130, 300, 511, 900, 1500]) for _ in range(75)]
    tail = 45
    n = sum(lengths) + tail
    tiles = (n + 127) // 128
    assert (tiles * H // 2 if H // KV % 2 == 0 else (tiles + 1) // 2 * H) > 148
    g = torch.Generator(device="cuda").manual_seed(D + H)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda").to(dt)  # noqa: E731
    qkv, do = r(n, H + 2 * KV, D), r(n, H, D)
    q, k, v = qkv[:, :H], qkv[:, H:H + KV], qkv[:, H + KV:]
    start, end = (t.cuda() for t in spans(lengths, n))
    out, lse = packed.attention_fwd(q, k, v, start, end, window=window)
    dq, dk, dv = packed.attention_bwd(q, k, v, out, lse, do, start, end, window=window)
    torch.cuda.synchronize()
    assert check_status() == 0
    for at, piece in _by_pieces(lengths, 1500):
        b = slice(at, at + sum(piece))
        s, e = (t.cuda() for t in spans(piece, sum(piece)))
        ref = attention(q[b], k[b], v[b], s, e, window, 1 / math.sqrt(D), do[b])
        for name, got in dict(out=out, dq=dq, dk=dk, dv=dv).items():
            _within(got[b], ref[name], name)
        _within(lse[:, b], ref["lse"], "lse")
    assert all((t[sum(lengths):] == 0).all() for t in (out, dq, dk, dv))


@pytest.mark.parametrize("B,T,H,KV,window", [(3, 512, 4, 4, 0), (2, 1024, 8, 2, 0), (5, 640, 4, 2, 256)])
def test_whole_rows_against_the_fixed_length_kernels(cuda, B, T, H, KV, window):
    """Sequences that are the rows of a batch: what attn_fwd_tc and attn_bwd_tc compute there."""
    from bitresearch_b200.ops._ext import ext
    packed, check_status = _ops()
    D, M = 128, B * T
    g = torch.Generator(device="cuda").manual_seed(T)
    qkv = torch.randn(M, (H + 2 * KV) * D, generator=g, device="cuda").to(torch.bfloat16)
    do = torch.randn(M, H * D, generator=g, device="cuda").to(torch.bfloat16)
    o, lse, dqkv = torch.empty_like(do), torch.empty(B, H, T, device="cuda"), torch.empty_like(qkv)
    ext().attn_fwd_tc(qkv, o, lse, B, T, H, KV, D, window or T)
    ext().attn_bwd_tc(qkv, o, do, lse, dqkv, torch.empty(B, H, T, device="cuda"), B, T, H, KV, D, window or T)
    heads = qkv.view(M, H + 2 * KV, D)
    q, k, v = heads[:, :H], heads[:, H:H + KV], heads[:, H + KV:]
    start, end = packed.bounds_from_offsets(torch.arange(0, M + 1, T, dtype=torch.int32, device="cuda"), M)
    out, l2 = packed.attention_fwd(q, k, v, start, end, window=window)
    grads = packed.attention_bwd(q, k, v, out, l2, do.view(M, H, D), start, end, window=window)
    torch.cuda.synchronize()
    assert check_status() == 0
    theirs = dqkv.view(M, H + 2 * KV, D)
    theirs = dict(out=o.view(M, H, D), dq=theirs[:, :H], dk=theirs[:, H:H + KV], dv=theirs[:, H + KV:])
    for at in range(0, M, T):
        b = slice(at, at + T)
        s, e = (t.cuda() for t in spans([T], T))
        ref = attention(q[b], k[b], v[b], s, e, window, 1 / math.sqrt(D), do.view(M, H, D)[b])
        for name, got in zip(("out", "dq", "dk", "dv"), (out, *grads)):
            _within(got[b], ref[name], name)
            value, tol = ref[name]  # both are within the tolerance of the 64-bit value
            _within(got[b], (theirs[name][b].double(), 2 * tol), name + " against the fixed-length kernel")
        _within(l2[:, b], ref["lse"], "lse")


@pytest.mark.parametrize("n", [300, 1000, 129])
@pytest.mark.parametrize("D,dt,window", [(64, torch.bfloat16, 0), (128, torch.float16, 0), (128, torch.bfloat16, 70),
                                         (64, torch.float16, 70)])
@pytest.mark.parametrize("kind", ["random", "reversed", "far", "none"])
def test_bad_spans_write_nothing_outside(cuda, n, D, dt, window, kind):
    """Spans that are none: no error, and the memory around every output and the scratch stays as it was."""
    packed, check_status = _ops()
    H, KV, guard = 4, 2, 40
    g = torch.Generator().manual_seed(n)
    far = 2 ** 31 - 1
    if kind == "random":
        start, end = (torch.randint(-1000, 2 * n, (n,), generator=g, dtype=torch.int32) for _ in range(2))
    elif kind == "reversed":
        start, end = (t.flip(0) for t in spans([n // 3, n - n // 3], n))
    elif kind == "far":
        start = torch.where(torch.rand(n, generator=g) < 0.5, -far, far).to(torch.int32)
        end = torch.where(torch.rand(n, generator=g) < 0.5, -far, far).to(torch.int32)
        start[:n // 2], end[:n // 2] = -far, far
    else:
        start, end = torch.full((n,), far, dtype=torch.int32), torch.full((n,), -far, dtype=torch.int32)
    start, end = start.cuda().contiguous(), end.cuda().contiguous()
    gc = torch.Generator(device="cuda").manual_seed(n)
    r = lambda h: torch.randn(n, h, D, generator=gc, device="cuda").to(dt)  # noqa: E731
    q, k, v, do = r(H), r(KV), r(KV), r(H)
    v[n // 2, :, 1] = math.nan  # also through the rows that are computed alone
    whole = []

    def rows(heads):
        whole.append((torch.full((n + 2 * guard, heads, D), 7.0, device="cuda").to(dt), guard * heads * D, n * heads * D))
        return whole[-1][0][guard:guard + n]

    def flat(count):
        whole.append((torch.full((count + 2 * 64,), 7.0, device="cuda"), 64, count))
        return whole[-1][0][64:64 + count]
    out, lse = rows(H), flat(H * n).view(H, n)
    scratch = flat(packed.bwd_scratch(n, H))
    dq, dk, dv = rows(H), rows(KV), rows(KV)
    packed.attention_fwd(q, k, v, start, end, window=window, out=out, lse=lse)
    packed.attention_bwd(q, k, v, out, lse, do, start, end, window=window, dq=dq, dk=dk, dv=dv, scratch=scratch)
    torch.cuda.synchronize()
    assert check_status() == 0
    for buf, before, count in whole:
        assert (buf.view(-1)[:before] == 7.0).all() and (buf.view(-1)[before + count:] == 7.0).all()
    if kind == "none":
        assert all((t == 7.0).all() for t in (out, lse, dq, dk, dv))


@pytest.mark.parametrize("D,dt", [(64, torch.float16), (128, torch.bfloat16)])
@pytest.mark.parametrize("lengths,tail", [([500, 1, 200], 3), ([1], 0), ([130], 0)])
def test_outputs_of_any_layout(cuda, lengths, tail, D, dt):
    """Outputs stored head by head, or between other columns: the bits of dense ones, and nothing around them written."""
    packed, check_status = _ops()
    H, KV, n = 4, 2, sum(lengths) + tail
    g = torch.Generator(device="cuda").manual_seed(n)
    r = lambda h: torch.randn(n, h, D, generator=g, device="cuda").to(dt)  # noqa: E731
    q, k, v, do = r(H), r(KV), r(KV), r(H)
    start, end = (t.cuda() for t in spans(lengths, n))
    want = packed.attention_fwd(q, k, v, start, end)
    want += packed.attention_bwd(q, k, v, *want, do, start, end)
    whole = lambda *s: torch.full(s, 7.0, device="cuda").to(dt)  # noqa: E731
    for make in (lambda h: (b := whole(h, n, D), b.transpose(0, 1)), lambda h: (b := whole(n, 2 * h + 1, D + 16), b[:, 1:h + 1, 8:D + 8])):
        (ob, out), (qb, dq), (kb, dk), (vb, dv) = make(H), make(H), make(KV), make(KV)
        packed.attention_fwd(q, k, v, start, end, out=out)
        packed.attention_bwd(q, k, v, want[0], want[1], do, start, end, dq=dq, dk=dk, dv=dv)
        for buf, view, right in ((ob, out, want[0]), (qb, dq, want[2]), (kb, dk, want[3]), (vb, dv, want[4])):
            assert torch.equal(view[:n - tail], right[:n - tail])
            view[:n - tail] = 7.0
            assert (buf == 7.0).all()
    assert check_status() == 0
