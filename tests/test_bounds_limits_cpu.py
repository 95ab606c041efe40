"""How many tokens bounds_from_ids takes: as many as the attention, refused before anything is allocated."""
import pytest
import torch

from bitresearch_b200.ops import packed
from bitresearch_b200.ops._ext import available

pytestmark = pytest.mark.skipif(not available(), reason="native module not built")


def test_too_many_tokens_are_refused():
    one = torch.zeros(1, 1 << 16, dtype=torch.int32)
    for rows in (1 << 14, (1 << 15) - 1):  # views of one row: 2^30 tokens and just below 2^31
        with pytest.raises(ValueError, match="too many tokens"):
            packed.bounds_from_ids(one.expand(rows, -1), 0)
