"""A kernel that finds an error on record returns with its whole block and leaves its outputs; once the word has been read
the next launch works, with the same bits."""
import pytest
import torch

pytestmark = pytest.mark.gpu
BAD_INDEX = 6


def test_gemm_and_attention_return_and_come_back(cuda):
    from bitresearch_b200.ops import gemm, packed
    from bitresearch_b200.ops._ext import check_status, ext
    E = ext()
    assert check_status() == 0
    g = torch.Generator(device="cuda").manual_seed(0)
    B, T, H, KV, D = 2, 512, 4, 2, 128
    M = B * T
    r = lambda *s: torch.randn(*s, generator=g, device="cuda").to(torch.bfloat16)  # noqa: E731
    a, w, qkv, do = r(M, 256), r(256, 384), r(M, (H + 2 * KV) * D), r(M, H * D)
    outs = lambda fill: (torch.full((M, 384), fill, device="cuda").to(torch.bfloat16), torch.full_like(do, fill),  # noqa: E731
                         torch.full((B, H, T), fill, device="cuda"), torch.full_like(qkv, fill))

    def run(c, o, lse, dqkv, right=None):
        gemm.matmul(a, w, out=c)
        E.attn_fwd_tc(qkv, o, lse, B, T, H, KV, D, T)
        o, lse = right or (o, lse)
        E.attn_bwd_tc(qkv, o, do, lse, dqkv, torch.empty(B, H, T, device="cuda"), B, T, H, KV, D, T)

    want, new = outs(7.0), outs(7.0)
    E.gemm_set_pair(0)  # single blocks: pairs go on and meet their cluster barriers
    try:
        run(*want)
        packed.bounds_from_offsets(torch.tensor([0, 9], dtype=torch.int32, device="cuda"), 5)  # reported
        run(*new, right=want[1:3])
        torch.cuda.synchronize()
        assert all((t == 7.0).all() for t in new)
        assert check_status() == BAD_INDEX
        run(*new)
        torch.cuda.synchronize()
        assert check_status() == 0 and all(torch.equal(x, y) for x, y in zip(want, new))
    finally:
        E.gemm_set_pair(1)
