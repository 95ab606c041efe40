"""The half-precision backward of packed attention where dS and P are far below fp16's smallest normal number (long
sequences, small gradients): the error against 64 bits is that of rounding each of dS, P and the result once."""
import math

import pytest
import torch

from packed_ref import spans

pytestmark = pytest.mark.gpu
HALF_STEP = 2.0 ** -11  # fp16, relative


def _ops():
    from bitresearch_b200.ops import packed
    from bitresearch_b200.ops._ext import check_status
    assert check_status() == 0
    return packed, check_status


def reference(q, k, v, do, lengths, window):
    """{name: (value, size)} in 64 bits, ``size`` the root of the summed squares of the terms whose 16-bit factor is
    rounded before the product."""
    n, H, D = q.shape
    KV, scale = k.shape[1], 1 / math.sqrt(D)
    shape = dict(dq=(n, H, D), dk=(n, KV, D), dv=(n, KV, D))
    val = {a: torch.zeros(s, dtype=torch.float64, device="cuda") for a, s in shape.items()}
    sq = {a: torch.zeros(s, dtype=torch.float64, device="cuda") for a, s in shape.items()}
    at = 0
    for length in lengths:
        b = slice(at, at + length)
        at += length
        i = torch.arange(length, device="cuda")
        hide = i[:, None] < i[None, :]
        if window:
            hide |= i[:, None] - i[None, :] >= window
        for h in range(H):
            g = h // (H // KV)
            Q, K, V, G = (t.double() for t in (q[b, h], k[b, g], v[b, g], do[b, h]))
            p = torch.softmax((Q @ K.t() * scale).masked_fill_(hide, -math.inf), 1)
            ds = (G @ V.t()).sub_((G * (p @ V)).sum(1, keepdim=True)).mul_(p).mul_(scale)
            val["dq"][b, h] = ds @ K
            val["dk"][b, g] += ds.t() @ Q
            val["dv"][b, g] += p.t() @ G
            ds, p = ds.square_(), p.square_()
            sq["dq"][b, h] = ds @ K.square()
            sq["dk"][b, g] += ds.t() @ Q.square()
            sq["dv"][b, g] += p.t() @ G.square()
    return {a: (val[a], sq[a].sqrt()) for a in val}


def check(packed, q, k, v, do, lengths, window=0, rows=slice(None)):
    start, end = (t.cuda() for t in spans(lengths, q.shape[0]))
    out, lse = packed.attention_fwd(q, k, v, start, end, window=window)
    got = dict(zip(("dq", "dk", "dv"), packed.attention_bwd(q, k, v, out, lse, do, start, end, window=window)))
    for name, (value, size) in reference(q, k, v, do, lengths, window).items():
        # the result's rounding as it falls, and independent roundings of the terms' 16-bit factors: each is off by at
        # most half a step, which is sqrt(3) times its root mean square and leaves that much for the fp32 sums
        value, size, have = value[rows], size[rows], got[name][rows]
        alone = (value.half().double() - value).norm()
        err = (have.double() - value).norm()
        assert err <= alone + HALF_STEP * size.norm(), (name, (err / alone).item(), (err / size.norm()).item())


@pytest.mark.parametrize("size", [0.1, 1e-2, 1e-3, 1e-5])
@pytest.mark.parametrize("n,H,KV,D,window", [(1024, 2, 1, 64, 0), (4096, 2, 2, 128, 0), (8192, 2, 1, 128, 0),
                                             (8192, 1, 1, 64, 3000)])
def test_small_gradients_of_long_sequences(cuda, n, H, KV, D, window, size):
    packed, check_status = _ops()
    g = torch.Generator(device="cuda").manual_seed(n + D)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    q, k, v = r(n, H, D).half(), r(n, KV, D).half(), r(n, KV, D).half()
    check(packed, q, k, v, (size * r(n, H, D)).half(), [n], window)
    torch.cuda.synchronize()
    assert check_status() == 0


def test_gradients_of_other_sizes_side_by_side(cuda):
    """Sequences and rows whose gradients differ by factors of a few hundred, one behind the other in the same tiles,
    large values among them: each sequence by itself is as near as it is alone."""
    packed, _ = _ops()
    lengths, H, KV, D = [700, 90, 1300, 30, 900], 4, 2, 64
    n = sum(lengths)
    g = torch.Generator(device="cuda").manual_seed(3)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    q, k, v = r(n, H, D).half(), r(n, KV, D).half(), r(n, KV, D)
    do, at = r(n, H, D), 0
    for length, a, b in zip(lengths, (1e-3, 1.0, 1e-2, 100.0, 2e-3), (1.0, 4.0, 0.1, 10.0, 1.0)):
        do[at:at + length] *= a
        v[at:at + length] *= b
        at += length
    do *= torch.where(torch.rand(n, 1, 1, generator=g, device="cuda") < 0.2, 0.01, 1.0)
    v, do, at = v.half(), do.half(), 0
    for length in lengths:
        check(packed, q, k, v, do, lengths, rows=slice(at, at + length))
        at += length


@pytest.mark.parametrize("lengths", [[300], [1, 2, 297]])
def test_large_gradients_do_not_overflow(cuda, lengths):
    """dS beyond fp16's largest number, as a loss scaled too high makes it, where dq and dk are within it."""
    packed, _ = _ops()
    n, H, D = 300, 2, 128
    g = torch.Generator(device="cuda").manual_seed(4)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    q, k, v = (0.05 * r(n, H, D)).half(), (0.05 * r(n, H, D)).half(), (20 * r(n, H, D)).half()
    check(packed, q, k, v, (1500 * r(n, H, D)).half(), lengths)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("below", [13.7, 17.3, 20.7, 24.6])
def test_weights_far_below_the_largest(cuda, D, below):
    """One key that takes nearly all of the weight, and thousands of others with 2^-below of it each, whose values are the
    only ones: the result is their sum, each weight rounded once."""
    packed, check_status = _ops()
    n, scale = 9000, 1 / math.sqrt(D)
    q = torch.ones(n, 1, D, device="cuda").half()
    k = torch.zeros(n, 1, D, device="cuda").half()
    k[0] = below * math.log(2) / (scale * D)
    v = torch.ones(n, 1, D, device="cuda").half()
    v[0] = 0.0
    start, end = (t.cuda() for t in spans([n], n))
    out, lse = packed.attention_fwd(q, k, v, start, end)
    torch.cuda.synchronize()
    assert check_status() == 0
    x = scale * D * float(k[0, 0, 0].double())
    i = torch.arange(n, dtype=torch.float64, device="cuda")
    want = i / (math.exp(x) + i)
    # a weight's rounding and the result's, the score's fp32 error (2^-20 of it) and the sums'
    tol = want * (2 * HALF_STEP + x * 2.0 ** -20 + 1e-4) + 2.0 ** -25
    assert ((out[:, 0].double() - want[:, None]).abs() <= tol[:, None]).all()
    assert ((lse[0].double() - torch.log(math.exp(x) + i)).abs() <= 1e-4).all()
