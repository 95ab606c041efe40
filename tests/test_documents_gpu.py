"""The engine on packed documents, with and without a teacher, against the eager fp32 model: spans, attention inside
documents, the distillation loss and every gradient together, as training uses them."""
from collections import OrderedDict

import pytest
import torch

pytestmark = pytest.mark.gpu


def _engine(cuda, n_head, n_kv, T, pattern="SL"):
    from bitresearch_b200.config import GPTConfig
    from bitresearch_b200.models.engine import FusedGPTEngine
    from bitresearch_b200.models.gpt import GPT
    cfg = GPTConfig(sequence_len=T, vocab_size=512, n_layer=2, n_head=n_head, n_kv_head=n_kv, n_embd=256,
                    window_pattern=pattern)
    m = GPT(cfg, init="normal", seed=0, device=cuda)
    g = torch.Generator(device="cpu").manual_seed(1)
    with torch.no_grad():
        for n, p in m.named().items():
            if n.endswith("_proj") or n.endswith("_ve_gate"):
                p.copy_((torch.randn(p.shape, generator=g) * 0.05).to(cuda))
    m.document_bos = 511
    flat = torch.zeros(m.num_params(), device=cuda)
    views, o = OrderedDict(), 0
    for n, p in m.named().items():
        views[n] = flat[o:o + p.numel()].view_as(p)
        o += p.numel()
    B = 2
    idx = torch.randint(0, 511, (B, T), generator=g, dtype=torch.int32)
    idx[torch.rand(B, T, generator=g) < 0.02] = 511
    tgt = torch.randint(0, 512, (B, T), generator=g, dtype=torch.int32)
    tgt[0, :5] = -1
    return cfg, m, FusedGPTEngine(m, views, B, T, flat_grad=flat), views, idx.to(cuda), tgt.to(cuda)


def _teacher_loss(logits, tgt, teacher):
    """The mean of alpha t^2 KL + (1 - alpha) CE over all positions, from the eager model's softcapped logits."""
    t, a = teacher.temperature, teacher.alpha
    z = logits.reshape(-1, logits.shape[-1])
    ids, u = teacher.ids.reshape(z.shape[0], -1).long(), teacher.logits.reshape(z.shape[0], -1).float()
    logq = torch.log_softmax(u / t, 1)
    kl = (logq.exp() * (logq - torch.log_softmax(z / t, 1).gather(1, ids))).sum(1)
    y = tgt.reshape(-1).long()
    ce = -torch.log(torch.softmax(z, 1) + 1e-10).gather(1, y.clamp(min=0)[:, None])[:, 0]
    return (a * t * t * kl + (1 - a) * torch.where(y >= 0, ce, 0.0)).mean()


@pytest.mark.parametrize("with_teacher", [False, True])
@pytest.mark.parametrize("n_head,n_kv,T", [(2, 2, 256), (2, 1, 200), (4, 2, 256)])
def test_engine_matches_eager_inside_documents(cuda, n_head, n_kv, T, with_teacher):
    from bitresearch_b200.ops.distill import Teacher
    cfg, m, eng, views, idx, tgt = _engine(cuda, n_head, n_kv, T)
    teacher = None
    if with_teacher:
        g = torch.Generator().manual_seed(2)
        ids = torch.stack([torch.randperm(512, generator=g)[:16] for _ in range(2 * T)]).view(2, T, 16)
        teacher = Teacher(ids.to(torch.int32).to(cuda), (2 * torch.randn(2, T, 16, generator=g)).to(cuda), 2.0, 0.7)
    loss = eng.forward_backward(idx, tgt, teacher=teacher)
    torch.cuda.synchronize()
    assert eng.status() == 0
    if with_teacher:
        ref_loss = _teacher_loss(m.forward_torch(idx.long()), tgt, teacher)
    else:
        ref_loss = m.forward_torch(idx.long(), tgt.long())
    ref_loss.backward()
    # the tolerances of the engine's other comparisons with the eager fp32 model (bf16 operands throughout)
    assert abs(loss.item() - ref_loss.item()) < 2e-2 * abs(ref_loss.item())
    for n, p in m.named().items():
        err, scale = (views[n] - p.grad).abs().max().item(), p.grad.abs().max().item() + 1e-8
        assert err <= 0.08 * scale, (n, err, scale)
    nats = eng.per_token_nats(idx, tgt)
    assert (nats - m.forward_torch(idx.long(), tgt.long(), reduction="none")).abs().max().item() < 0.05


def test_documents_change_the_result(cuda):
    cfg, m, eng, views, idx, tgt = _engine(cuda, 2, 2, 256)
    inside = eng.per_token_nats(idx, tgt)
    m.document_bos = None
    across = m.forward_torch(idx.long(), tgt.long(), reduction="none")
    assert (inside - across).abs().max().item() > 0.05
