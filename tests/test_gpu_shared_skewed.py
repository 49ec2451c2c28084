"""Attention below shared prefixes where one group has most of the sequences (GPU)."""
import pytest

from test_gpu_kvcache import BF16, F16, F32, random_mask
from test_gpu_shared_attn import Shared, check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,dim,tokens", [(F32, 128, 1), (F32, 256, 2), (F32, 64, 4), (BF16, 128, 1), (F16, 256, 3), (BF16, 64, 9)])
@pytest.mark.parametrize("large", [0, 9, 19])
def test_one_large_group_among_small_ones(cuda, dtype, dim, tokens, large):
    """45 sequences in one group, 19 in groups of their own, first, in the middle and last: tiles are chosen by the rows of an average one."""
    groups, at = [], 0
    for i in range(20):
        members, pages = (45, 40) if i == large else (1, 1 + i % 4)
        groups.append((at, members, pages, pages * 16))
        at += members
    check(Shared([(b * 13) % 70 for b in range(at)], groups, 2, 2, dim, 16, "head", dtype, tokens), random_mask(at, tokens, 6))
