"""Packed attention and its spans on the GPU against plain 64-bit forms (packed_ref.py has the tolerances)."""
import math

import pytest
import torch

from packed_ref import attention, spans

pytestmark = pytest.mark.gpu
BAD_INDEX = 6


def _ops():
    from bitresearch_b200.ops import packed
    from bitresearch_b200.ops._ext import check_status
    assert check_status() == 0
    return packed, check_status


def _within(got, ref, what):
    value, tol = ref
    bad = ~((got.double() - value).abs() <= tol)
    assert not bad.any(), (what, int(bad.sum()), (got.double() - value).abs()[bad].max().item(), tol[bad].max().item())


def _make(n, H, KV, D, dt, layout="fused", seed=0, spread=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    if layout == "fused":  # views into one projection buffer
        x = (r(n, H + 2 * KV, D) * spread).to(dt)
        return x[:, :H], x[:, H:H + KV], x[:, H + KV:]
    if layout == "heads":  # head-major storage
        return tuple((r(h, n, D) * spread).to(dt).transpose(0, 1) for h in (H, KV, KV))
    return tuple((r(n, h, D) * spread).to(dt) for h in (H, KV, KV))


def _check(lengths, H, KV, D, dt, window=0, tail=0, layout="fused", scale=None, seed=0, spread=1.0, only=None):
    packed, check_status = _ops()
    n = sum(lengths) + tail
    q, k, v = _make(n, H, KV, D, dt, layout, seed, spread)
    do = _make(n, H, KV, D, dt, "plain", seed + 1)[0]
    start, end = (t.cuda() for t in spans(lengths, n))
    kw = dict(window=window) if scale is None else dict(window=window, scale=scale)
    out, lse = packed.attention_fwd(q, k, v, start, end, **kw)
    dq, dk, dv = packed.attention_bwd(q, k, v, out, lse, do, start, end, **kw)
    torch.cuda.synchronize()
    assert check_status() == 0
    ref = attention(q, k, v, start, end, window, 1 / math.sqrt(D) if scale is None else scale, do)
    for name, got in dict(out=out, lse=lse, dq=dq, dk=dk, dv=dv).items():
        _within(got, ref[name], name)


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("lengths", [[1], [2], [0, 1, 0, 5, 0], [64, 64], [127, 1, 128, 129, 1, 0, 2],
                                     [300, 0, 700, 33], [5] * 130, [1] * 300, [257], [256, 256], [255, 2, 600]],
                         ids=lambda x: "-".join(map(str, x[:4])))
def test_lengths(cuda, lengths, D, dt):
    _check(lengths, 2, 1, D, dt)


@pytest.mark.parametrize("window", [1, 2, 31, 128, 129, 500, 10_000])
@pytest.mark.parametrize("D", [64, 128])
def test_windows(cuda, window, D):
    _check([300, 1, 700, 33, 128], 2, 2, D, torch.bfloat16, window=window, tail=5)


@pytest.mark.parametrize("H,KV", [(1, 1), (4, 4), (4, 2), (6, 1), (8, 2), (5, 5), (3, 1)])
@pytest.mark.parametrize("layout", ["fused", "heads", "plain"])
def test_heads_and_layouts(cuda, H, KV, layout):
    _check([90, 200, 3, 310], H, KV, 128 if H % 2 else 64, torch.bfloat16, tail=20, layout=layout)


@pytest.mark.parametrize("scale", [0.01, 1.0])
def test_scales(cuda, scale):
    _check([400, 100], 2, 2, 128, torch.bfloat16, scale=scale, spread=0.6)


def test_many_rows(cuda):
    """More row tiles than the GPU has SMs, sequences of every length up to 300."""
    _check(list(range(0, 90)), 8, 2, 64, torch.bfloat16, tail=1)


@pytest.mark.parametrize("D", [64, 128])
def test_large_scores_stay_finite(cuda, D):
    """Scores of a few hundred: the running maximum moves by far more than one rescale's allowance."""
    packed, check_status = _ops()
    n = 700
    q, k, v = _make(n, 2, 2, D, torch.bfloat16, spread=3.0)
    # a ramp along the keys makes every tile raise the maximum
    k = (k.float() * torch.linspace(0.1, 4, n, device="cuda")[:, None, None]).to(torch.bfloat16)
    start, end = (t.cuda() for t in spans([n], n))
    out, lse = packed.attention_fwd(q, k, v, start, end)
    ref = attention(q, k, v, start, end, 0, 1 / math.sqrt(D))
    # a score of size x carries x * 2^-20 of fp32 error into its weight: sums of 128 products of 2^-24 each
    size = (q.float().abs().transpose(0, 1) @ k.float().abs().permute(1, 2, 0)).amax().item() / math.sqrt(D)
    value, tol = ref["out"]
    assert ((out.double() - value).abs() <= tol + size * 2.0 ** -20 * v.double().abs().amax()).all()
    assert ((lse.double() - ref["lse"][0]).abs() <= size * 2.0 ** -20).all()


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("what", ["nan", "inf"])
def test_nothing_crosses_a_border(cuda, D, what):
    """A sequence of values that are no numbers between others, and padding rows that hold them, in every input: the
    other sequences' results are what they are without them, and padding rows stay as they were."""
    packed, check_status = _ops()
    lengths, tail = [50, 70, 200, 1, 90, 300, 40], 77
    n, H, KV = sum(lengths) + tail, 4, 2
    q, k, v = (t.clone() for t in _make(n, H, KV, D, torch.bfloat16, "plain"))
    do = _make(n, H, KV, D, torch.bfloat16, "plain", 1)[0]
    start, end = (t.cuda() for t in spans(lengths, n))
    poison = torch.zeros(n, dtype=torch.bool, device="cuda")
    poison[50:120] = True    # the second sequence
    poison[411:] = False
    poison[321:411] = True   # the fifth
    poison[sum(lengths):] = True
    good = ~poison
    clean = attention(*(torch.where(poison[:, None, None], torch.zeros_like(t), t) for t in (q, k, v)), start, end, 0,
                      1 / math.sqrt(D), torch.where(poison[:, None, None], torch.zeros_like(do), do))
    for t in (q, k, v, do):
        t[poison] = float(what)
    full = lambda *s: torch.full(s, 7.0, device="cuda", dtype=torch.bfloat16)  # noqa: E731
    out, dq, dk, dv = full(n, H, D), full(n, H, D), full(n, KV, D), full(n, KV, D)
    lse = torch.full((H, n), 7.0, device="cuda")
    packed.attention_fwd(q, k, v, start, end, out=out, lse=lse)
    packed.attention_bwd(q, k, v, out, lse, do, start, end, dq=dq, dk=dk, dv=dv)
    torch.cuda.synchronize()
    assert check_status() == 0
    for name, got in dict(out=out, dq=dq, dk=dk, dv=dv).items():
        value, tol = clean[name]
        _within(got[good], (value[good], tol[good]), name)
        assert (got[sum(lengths):] == 7.0).all(), name
        assert not torch.isfinite(got[50:120].float()).all()
    _within(lse[:, good], tuple(t[:, good] for t in clean["lse"]), "lse")
    assert (lse[:, sum(lengths):] == 7.0).all()


@pytest.mark.parametrize("window", [0, 300])
@pytest.mark.parametrize("H,KV", [(4, 2), (3, 3)])
def test_nothing_crosses_a_border_into_a_long_sequence(cuda, H, KV, window):
    """One value in each input of a short sequence that is no number: every row tile of the long sequence behind it
    starts in the tile that holds it, and the rows at the long one's end share a tile with the next."""
    packed, check_status = _ops()
    lengths, D = [60, 1500, 2, 700], 128
    n = sum(lengths)
    q, k, v = (t.clone() for t in _make(n, H, KV, D, torch.bfloat16, "plain"))
    do = _make(n, H, KV, D, torch.bfloat16, "plain", 1)[0]
    start, end = (t.cuda() for t in spans(lengths, n))
    good = torch.ones(n, dtype=torch.bool, device="cuda")
    good[:60] = False
    good[1560:1562] = False
    clean = attention(*(torch.where(good[:, None, None], t, torch.zeros_like(t)) for t in (q, k, v)), start, end, window,
                      1 / math.sqrt(D), torch.where(good[:, None, None], do, torch.zeros_like(do)))
    for t in (q, k, v, do):
        t[59, :, 5] = math.inf
        t[1561, 0, 100] = math.nan
    out, lse = packed.attention_fwd(q, k, v, start, end, window=window)
    grads = packed.attention_bwd(q, k, v, out, lse, do, start, end, window=window)
    torch.cuda.synchronize()
    assert check_status() == 0
    for name, got in zip(("out", "dq", "dk", "dv"), (out, *grads)):
        value, tol = clean[name]
        _within(got[good], (value[good], tol[good]), name)
    _within(lse[:, good], tuple(t[:, good] for t in clean["lse"]), "lse")


def test_bad_spans_stay_inside(cuda):
    """Spans that are none (negative, reversed, past the end): no fault and no error code, other rows untouched."""
    packed, check_status = _ops()
    n, H, D = 300, 2, 128
    q, k, v = _make(n, H, H, D, torch.bfloat16)
    g = torch.Generator().manual_seed(3)
    start = torch.randint(-1000, 2000, (n,), generator=g, dtype=torch.int32).cuda()
    end = torch.randint(-1000, 2000, (n,), generator=g, dtype=torch.int32).cuda()
    out, lse = packed.attention_fwd(q, k, v, start, end)
    packed.attention_bwd(q, k, v, out, lse, q.clone(), start, end)
    torch.cuda.synchronize()
    assert check_status() == 0


def test_offsets_past_32_bits(cuda):
    """2.4e9 elements of q: the last sequences' results are those of the same rows alone."""
    packed, check_status = _ops()
    n, H, D, length = 300_007, 64, 128, 500
    if torch.cuda.get_device_properties(0).total_memory < 60e9:
        pytest.skip("needs 60 GB")
    lengths = [length] * (n // length) + [n % length]
    off = torch.tensor([0] + lengths).cumsum(0).to(torch.int32).cuda()
    start, end = packed.bounds_from_offsets(off, n)
    q = torch.randn(n, H, D, device="cuda", dtype=torch.bfloat16)
    k, v = (torch.randn(n, 1, D, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    out, lse = packed.attention_fwd(q, k, v, start, end)
    dq, dk, dv = packed.attention_bwd(q, k, v, out, lse, q, start, end)
    torch.cuda.synchronize()
    assert check_status() == 0
    a = n - 7 - 3 * length  # whole tiles lie elsewhere in the slice, so sums are added in another order
    s, e = (t[a:] - a for t in (start, end))
    ref = attention(q[a:], k[a:], v[a:], s, e, 0, 1 / math.sqrt(D), q[a:])
    for name, got in dict(out=out, dq=dq, dk=dk, dv=dv).items():
        _within(got[a:], ref[name], name)
    _within(lse[:, a:], ref["lse"], "lse")


def test_empty(cuda):
    packed, _ = _ops()
    q, k, v = _make(0, 2, 1, 64, torch.bfloat16, "plain")
    start = torch.empty(0, dtype=torch.int32, device="cuda")
    out, lse = packed.attention_fwd(q, k, v, start, start)
    assert out.shape == (0, 2, 64) and lse.shape == (2, 0)
    assert [t.shape[1] for t in packed.attention_bwd(q, k, v, out, lse, q, start, start)] == [2, 1, 1]
    # rows, but no sequence
    q, k, v = _make(40, 2, 1, 64, torch.bfloat16, "plain")
    start = torch.arange(40, dtype=torch.int32, device="cuda")
    out, lse = packed.attention_fwd(q, k, v, start, start)
    dq, dk, dv = packed.attention_bwd(q, k, v, out, lse, q, start, start)
    assert all((t == 0).all() for t in (out, lse, dq, dk, dv))


def test_same_bits_two_streams_and_graph(cuda):
    """Two calls at once on two streams, and a captured call replayed, give the bits of a single call."""
    packed, check_status = _ops()
    lengths = [400, 3, 900, 61]
    n, H, KV, D = sum(lengths), 4, 2, 128
    start, end = (t.cuda() for t in spans(lengths, n))
    sets = []
    for s in range(2):
        q, k, v = _make(n, H, KV, D, torch.bfloat16, seed=s)
        do = _make(n, H, KV, D, torch.bfloat16, "plain", 5 + s)[0]
        sets.append((q, k, v, do))

    def call(q, k, v, do):
        out, lse = packed.attention_fwd(q, k, v, start, end)
        return (out, lse, *packed.attention_bwd(q, k, v, out, lse, do, start, end))

    want = [call(*s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = [[], []]
    for _ in range(4):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(call(*sets[i]))
    torch.cuda.synchronize()
    for w, gs in zip(want, got):
        for g in gs:
            assert all(torch.equal(a, b) for a, b in zip(w, g))
    graphs = []
    for s in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            r = call(*s)
        graphs.append((g, r))
    for _ in range(3):
        for (g, r), st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    for w, (g, r) in zip(want, graphs):
        assert all(torch.equal(a, b) for a, b in zip(w, r))
    assert check_status() == 0


# ---------------------------------------------------------------------------------------------- spans
@pytest.mark.parametrize("lengths,tail", [([1], 0), ([], 9), ([0, 0, 3, 0], 2), ([5, 1, 300, 0, 700], 0), ([1] * 1000, 7),
                                          ([100_000, 3], 11)], ids=lambda x: str(x)[:12])
def test_bounds_from_offsets(cuda, lengths, tail):
    packed, check_status = _ops()
    n = sum(lengths) + tail
    off = torch.tensor([0] + lengths).cumsum(0).to(torch.int32).cuda()
    start, end = packed.bounds_from_offsets(off, n)
    s, e = spans(lengths, n)
    assert torch.equal(start.cpu(), s) and torch.equal(end.cpu(), e) and check_status() == 0


def test_bounds_from_offsets_first_row_not_zero_and_bad_tables(cuda):
    packed, check_status = _ops()
    t = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    start, end = packed.bounds_from_offsets(t(2, 4), 5)
    assert start.tolist() == [0, 1, 2, 2, 4] and end.tolist() == [0, 1, 4, 4, 4] and check_status() == 0
    for bad in (t(0, 9), t(-3, 5), t(0, 4, 2, 5), t(7)):
        start, end = packed.bounds_from_offsets(bad, 5)
        assert check_status() == BAD_INDEX
        rows = torch.arange(5, device="cuda")
        assert ((start >= 0) & (start <= rows) & (end >= rows) & (end <= 5)).all()


@pytest.mark.parametrize("B,T", [(1, 1), (3, 7), (2, 2048), (5, 2049), (2, 9001), (1, 30_000), (128, 100)])
@pytest.mark.parametrize("p", [0.0, 0.0005, 0.05, 0.9])
def test_bounds_from_ids(cuda, B, T, p):
    packed, _ = _ops()
    g = torch.Generator().manual_seed(B * T)
    ids = torch.randint(0, 50, (B, T + 3), generator=g, dtype=torch.int32)
    ids[torch.rand(B, T + 3, generator=g) < p] = 99
    start, end = packed.bounds_from_ids(ids.cuda()[:, :T], 99)
    want_s, want_e = [], []
    for b in range(B):
        cuts = [t for t in range(T) if t == 0 or int(ids[b, t]) == 99] + [T]
        for lo, hi in zip(cuts, cuts[1:]):
            want_s += [b * T + lo] * (hi - lo)
            want_e += [b * T + hi] * (hi - lo)
    assert start.tolist() == want_s and end.tolist() == want_e


def test_bounds_into_given_tensors_and_empty(cuda):
    packed, _ = _ops()
    s, e = (torch.full((6,), -1, dtype=torch.int32, device="cuda") for _ in range(2))
    ids = torch.tensor([[1, 9, 1], [1, 1, 9]], dtype=torch.int32, device="cuda")
    a, b = packed.bounds_from_ids(ids, 9, s, e)
    assert a is s or a.data_ptr() == s.data_ptr()
    assert s.tolist() == [0, 1, 1, 3, 3, 5] and e.tolist() == [1, 3, 3, 5, 5, 6]
    assert packed.bounds_from_ids(ids[:, :0], 9)[0].numel() == 0
    assert packed.bounds_from_offsets(torch.zeros(1, dtype=torch.int32, device="cuda"), 0)[1].numel() == 0
