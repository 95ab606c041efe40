"""What the device status word means to packed attention."""
import pytest
import torch

from packed_ref import spans

pytestmark = pytest.mark.gpu
BAD_INDEX = 6


@pytest.mark.parametrize("D,dt", [(64, torch.bfloat16), (128, torch.float16)])
def test_an_error_on_record_leaves_outputs_alone(cuda, D, dt):
    """Every block of the three kernels returns as a whole; after the word has been read calls work again."""
    from bitresearch_b200.ops import packed
    from bitresearch_b200.ops._ext import check_status
    assert check_status() == 0
    n, H, KV = 5000, 4, 2
    g = torch.Generator(device="cuda").manual_seed(0)
    q, do = (torch.randn(n, H, D, generator=g, device="cuda").to(dt) for _ in range(2))
    k, v = (torch.randn(n, KV, D, generator=g, device="cuda").to(dt) for _ in range(2))
    start, end = (t.cuda() for t in spans([1500, 3, 3400], n))
    want = packed.attention_fwd(q, k, v, start, end)
    want += packed.attention_bwd(q, k, v, *want, do, start, end)
    new = [torch.full_like(t, 7.0) for t in want]
    call = lambda: (packed.attention_fwd(q, k, v, start, end, out=new[0], lse=new[1]),  # noqa: E731
                    packed.attention_bwd(q, k, v, want[0], want[1], do, start, end, dq=new[2], dk=new[3], dv=new[4]))
    packed.bounds_from_offsets(torch.tensor([0, n + 1], dtype=torch.int32, device="cuda"), n)  # reported
    call()
    torch.cuda.synchronize()
    assert all((t == 7.0).all() for t in new)
    assert check_status() == BAD_INDEX
    for t in new:
        t.zero_()
    call()
    torch.cuda.synchronize()
    assert check_status() == 0
    assert all(torch.equal(a, b) for a, b in zip(want, new))
