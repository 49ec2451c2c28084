"""How long a SharedPrefix and what is kept of it live (GPU)."""
import pytest
import torch

from technograd_b200 import kvcache
from test_gpu_kvcache import BF16
from test_gpu_shared_attn import Shared

pytestmark = pytest.mark.gpu


def test_dropped_while_another_stream_has_yet_to_read_it(cuda):
    """The prefix is made on one stream and used on another, whose kernels wait; its memory may not be given to what comes next on the first."""
    c = Shared([40, 20, 10, 30], [(0, 2, 20, 320), (2, 2, 30, 480)], 2, 2, 64, 16, "head", BF16, 3)
    args = c.q.cuda(), c.kn.cuda(), c.vn.cuda()
    groups, size = c.prefix.groups, c.prefix._held.numel()
    want = kvcache.shared_attention(c.cache, c.prefix, *args)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for _ in range(3):
        prefix = kvcache.SharedPrefix(c.cache, groups, max_own=40, always=True)
        with torch.cuda.stream(side):
            torch.cuda._sleep(100_000_000)
            got = kvcache.shared_attention(c.cache, prefix, *args)
        c.cache._plans.clear()
        del prefix
        others = [torch.full((size,), 3, dtype=torch.int32, device="cuda") for _ in range(50)]  # as large, at once
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, want)) and len(others) == 50
