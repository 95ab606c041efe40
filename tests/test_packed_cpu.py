"""Packed attention and top-logit distillation without a GPU: the plain forms' gradients against differences, and
what the calls refuse (every check comes before the first use of a device)."""
import math

import pytest
import torch

from bitresearch_b200.ops import distill, packed
from bitresearch_b200.ops._ext import available
from packed_ref import attention, spans
from packed_ref import distill as distill_ref

needs_ext = pytest.mark.skipif(not available(), reason="native module not built")


@pytest.mark.parametrize("lengths,window,H,KV", [([3, 1, 4], 0, 2, 1), ([6], 2, 2, 2), ([0, 2, 3], 3, 3, 1)])
def test_attention_formula_matches_differences(lengths, window, H, KV):
    torch.manual_seed(0)
    n, D = sum(lengths) + 2, 4
    start, end = spans(lengths, n)
    f8 = dict(dtype=torch.float64)
    q, k, v = torch.randn(n, H, D, **f8), torch.randn(n, KV, D, **f8), torch.randn(n, KV, D, **f8)
    do = torch.randn(n, H, D, **f8)
    r = attention(q, k, v, start, end, window, 0.7, do)
    step = 1e-6
    for name, x in (("dq", q), ("dk", k), ("dv", v)):
        for e in range(0, x.numel(), 3):
            side = []
            for s in (step, -step):
                y = x.clone().view(-1)
                y[e] += s
                a = {"q": q, "k": k, "v": v, name[1]: y.view_as(x)}
                side.append((attention(a["q"], a["k"], a["v"], start, end, window, 0.7)["out"][0] * do).sum())
            assert abs((side[0] - side[1]) / (2 * step) - r[name][0].reshape(-1)[e]) < 1e-7


@pytest.mark.parametrize("alpha,t,cap", [(1.0, 1.0, 0.0), (0.3, 2.0, 15.0), (0.0, 1.0, 15.0), (1.0, 0.5, 15.0)])
def test_distill_formula_matches_differences(alpha, t, cap):
    torch.manual_seed(1)
    M, V, K = 4, 9, 3
    z = 3 * torch.randn(M, V, dtype=torch.float64)
    ids = torch.tensor([[0, 4, 8], [2, 2, -1], [-1, -1, -1], [5, 1, 5]], dtype=torch.int32)
    u = torch.randn(M, K, dtype=torch.float64)
    y = torch.tensor([3, -1, 7, 5], dtype=torch.int32)
    capped = lambda a: cap * torch.tanh(a / cap) if cap else a  # noqa: E731
    grad = distill_ref(capped(z), ids, u, y, cap, t, alpha, 0.25)[1]
    for e in range(z.numel()):
        side = []
        for s in (1e-6, -1e-6):
            a = z.clone().view(-1)
            a[e] += s
            side.append(0.25 * distill_ref(capped(a.view_as(z)), ids, u, y, cap, t, alpha, 0.25)[0].sum())
        assert abs((side[0] - side[1]) / 2e-6 - grad.view(-1)[e]) < 1e-7


def _qkv(n=8, H=4, KV=2, D=64, dt=torch.bfloat16):
    return (torch.zeros(n, H, D, dtype=dt), torch.zeros(n, KV, D, dtype=dt), torch.zeros(n, KV, D, dtype=dt),
            *spans([n], n))


@needs_ext
@pytest.mark.parametrize("change,message", [
    (lambda a: a.update(q=a["q"].float()), "bfloat16 or float16"),
    (lambda a: a.update(k=a["k"].half()), "another type"),
    (lambda a: a.update(v=a["v"][:7]), r"v must be \[8, 2, 64\]"),
    (lambda a: a.update(q=a["q"][:, :3]), "cannot share"),
    (lambda a: a.update({x: a[x][..., :32] for x in "qkv"}), "64 or 128"),
    (lambda a: a.update(q=torch.zeros(8, 64, 4, dtype=torch.bfloat16).transpose(1, 2)), "contiguous heads"),
    (lambda a: a.update(q=torch.zeros(8, 4, 68, dtype=torch.bfloat16)[..., :64]), "multiples of 8"),
    (lambda a: a.update(k=torch.zeros(8, 1, 64, dtype=torch.bfloat16).expand(8, 2, 64)), "at least 64"),
    (lambda a: a.update(q=torch.zeros(8 * 4 * 64 + 1, dtype=torch.bfloat16)[1:].view(8, 4, 64)), "16-byte"),
    (lambda a: a.update(start=a["start"].long()), "start and end"),
    (lambda a: a.update(end=a["end"][:4]), "start and end"),
    (lambda a: a.update(window=-1), "window"),
    (lambda a: a.update(scale=0.0), "scale"),
    (lambda a: a.update(scale=math.nan), "scale"),
    (lambda a: a.update(out=torch.zeros(8, 4, 64)), "out has another type"),
    (lambda a: a.update(lse=torch.zeros(8, 4)), "lse must be"),
    (lambda a: None, "CUDA device"),
])
def test_attention_fwd_refuses(change, message):
    q, k, v, start, end = _qkv()
    a = dict(q=q, k=k, v=v, start=start, end=end)
    change(a)
    with pytest.raises(ValueError, match=message):
        packed.attention_fwd(**a)


@needs_ext
@pytest.mark.parametrize("change,message", [
    (lambda a: a.update(dout=a["dout"].float()), "dout has another type"),
    (lambda a: a.update(out=a["out"][:, :2]), "out must be"),
    (lambda a: a.update(lse=a["lse"].double()), "lse must be"),
    (lambda a: a.update(dq=a["k"].clone()), "dq must be"),
    (lambda a: a.update(scratch=torch.zeros(2 * 4 * 128 - 1)), "scratch must be"),
    (lambda a: a.update(scratch=torch.zeros(packed.bwd_scratch(8, 4)).half()), "scratch must be"),
    (lambda a: None, "CUDA device"),
])
def test_attention_bwd_refuses(change, message):
    q, k, v, start, end = _qkv()
    a = dict(q=q, k=k, v=v, out=torch.zeros_like(q), lse=torch.zeros(4, 8), dout=torch.zeros_like(q), start=start, end=end)
    change(a)
    with pytest.raises(ValueError, match=message):
        packed.attention_bwd(**a)


@needs_ext
def test_attention_refuses_outputs_over_its_inputs():
    q, k, v, start, end = _qkv()
    with pytest.raises(RuntimeError, match="memory"):
        packed.attention_fwd(q, k, v, start, end, out=q)
    with pytest.raises(RuntimeError, match="memory"):
        packed.attention_bwd(q, k, v, torch.zeros_like(q), torch.zeros(4, 8), torch.zeros_like(q), start, end, dk=k)


@needs_ext
def test_bounds_refuse():
    off = torch.tensor([0, 3, 5], dtype=torch.int32)
    ids = torch.zeros(2, 8, dtype=torch.int32)
    for call, message in (
            (lambda: packed.bounds_from_offsets(off.long(), 5), "int32"),
            (lambda: packed.bounds_from_offsets(off[:0], 5), "at least one"),
            (lambda: packed.bounds_from_offsets(off, -1), "rows"),
            (lambda: packed.bounds_from_offsets(off, 5, start=torch.zeros(4, dtype=torch.int32)), "start must be"),
            (lambda: packed.bounds_from_offsets(off, 5), "CUDA device"),
            (lambda: packed.bounds_from_ids(ids.long(), 0), "int32"),
            (lambda: packed.bounds_from_ids(ids[0], 0), "int32"),
            (lambda: packed.bounds_from_ids(ids.t(), 0), "contiguous rows"),
            (lambda: packed.bounds_from_ids(ids, 1 << 40), "bos"),
            (lambda: packed.bounds_from_ids(ids, 0), "CUDA device")):
        with pytest.raises(ValueError, match=message):
            call()


@needs_ext
@pytest.mark.parametrize("change,message", [
    (lambda a: a.update(logits=a["logits"].double()), "logits must be"),
    (lambda a: a.update(logits=torch.zeros(9, 4).t()), "contiguous rows"),
    (lambda a: a.update(logits=torch.zeros(4, (1 << 18) + 1)), "up to 1 MB"),
    (lambda a: a.update(logits=torch.zeros(1, 9).expand(4, 9)), "overlap"),
    (lambda a: a.update(teacher_ids=a["teacher_ids"].long()), "teacher_ids must be int32"),
    (lambda a: a.update(teacher_ids=a["teacher_ids"][:3]), "teacher_ids must be int32"),
    (lambda a: a.update(teacher_ids=a["teacher_ids"][:, :0], teacher_logits=a["teacher_logits"][:, :0]), "entries per row"),
    (lambda a: a.update(teacher_ids=torch.zeros(4, 1025, dtype=torch.int32), teacher_logits=torch.zeros(4, 1025)), "entries"),
    (lambda a: a.update(teacher_logits=a["teacher_logits"][:, :2]), "teacher_logits must be"),
    (lambda a: a.update(alpha=0.5), "needs targets"),
    (lambda a: a.update(alpha=1.5), "alpha"),
    (lambda a: a.update(temperature=0.0), "temperature"),
    (lambda a: a.update(cap=-1.0), "cap"),
    (lambda a: a.update(scale=math.inf), "scale"),
    (lambda a: a.update(targets=torch.zeros(4)), "targets must be"),
    (lambda a: a.update(grad=torch.zeros(4, 8)), "grad must be"),
    (lambda a: a.update(grad=torch.zeros(4, 9), need_grad=False), "not wanted"),
    (lambda a: None, "CUDA device"),
])
def test_distill_refuses(change, message):
    a = dict(logits=torch.zeros(4, 9), teacher_ids=torch.zeros(4, 3, dtype=torch.int32), teacher_logits=torch.zeros(4, 3))
    change(a)
    with pytest.raises(ValueError, match=message):
        distill.distill_topk(**a)
