"""Attention inside documents on the eager path: a document's logits are what they are when it stands alone."""
import pytest
import torch

from bitresearch_b200.config import GPTConfig, preset
from bitresearch_b200.models.gpt import GPT


def _model(pattern, n_kv=2):
    cfg = GPTConfig(sequence_len=32, vocab_size=64, n_layer=3, n_head=2, n_kv_head=n_kv, n_embd=64, window_pattern=pattern)
    m = GPT(cfg, init="normal", seed=3)
    g = torch.Generator().manual_seed(4)
    with torch.no_grad():
        for n, p in m.named().items():
            if n.endswith("_proj") or n.endswith("_ve_gate"):
                p.copy_(torch.randn(p.shape, generator=g) * 0.1)
    return cfg, m


@pytest.mark.parametrize("pattern,n_kv", [("L", 2), ("SL", 1)])
def test_a_document_reads_nothing_of_the_others(pattern, n_kv):
    cfg, m = _model(pattern, n_kv)
    bos = cfg.vocab_size - 1
    g = torch.Generator().manual_seed(0)
    idx = torch.randint(0, bos, (2, 32), generator=g)
    idx[0, 0], idx[0, 9], idx[0, 10] = bos, bos, bos
    idx[1, 20] = bos  # the row's first document has no BOS of its own
    m.document_bos = bos
    whole = m.forward_torch(idx)
    for row, cuts in ((0, (0, 9, 10, 32)), (1, (0, 20, 32))):
        for lo, hi in zip(cuts, cuts[1:]):
            # rotary positions are relative: the document may start anywhere
            alone = m.forward_torch(idx[row:row + 1, lo:hi])
            assert (whole[row, lo:hi] - alone[0]).abs().max() < 2e-4
    m.document_bos = None
    assert (m.forward_torch(idx)[0, 12] - whole[0, 12]).abs().max() > 1e-3


def test_flex_attention_is_refused():
    cfg, m = _model("L")
    m.document_bos, m.attn_impl = 63, "flex"
    with pytest.raises(ValueError, match="inside documents"):
        m.forward_torch(torch.zeros(1, 32, dtype=torch.long))


@pytest.mark.parametrize("changes,message", [(dict(torch_compile=True), "torch_compile"), (dict(data="tokens"), "bos_token_id")])
def test_trainer_refuses(changes, message):
    from bitresearch_b200.train import Trainer
    cfg = preset("tiny-cpu")
    cfg.document_mask = True
    for k, v in changes.items():
        setattr(cfg, k, v)
    with pytest.raises(ValueError, match=message):
        Trainer(cfg).initialize()


def test_trainer_trains_inside_documents():
    from bitresearch_b200.train import Trainer
    cfg = preset("tiny-cpu")
    cfg.document_mask, cfg.comm, cfg.total_batch_tokens = True, "nccl", 4 * 128
    t = Trainer(cfg)
    t.initialize()
    assert t.model.document_bos == cfg.model.vocab_size - 1
    assert t.train_step() > 0
