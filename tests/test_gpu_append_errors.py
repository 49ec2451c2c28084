"""Appends whose rows find no place (GPU)."""
import pytest
import torch

from technograd_b200 import kvcache
from test_gpu_kvcache import BF16, F32, Case, reported

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("part", [16, 6])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_a_pool_of_no_pages(cuda, dtype, part):
    """Whose pointers are NULL: nothing can be written, which is reported like any page that is not there."""
    k, x = torch.zeros(0, 1, 8, 16, dtype=dtype, device="cuda"), torch.ones(2, 3, 1, 16, dtype=dtype, device="cuda")
    cache = kvcache.PagedKV(k, k, torch.zeros(2, 2, dtype=torch.int32, device="cuda"), torch.tensor([0, 15], dtype=torch.int32, device="cuda"))
    lens, _, kr = kvcache.append(cache, x, x, rotary=kvcache.Rotary(16, theta=1e4, part=part), keys=True)
    good = Case([5], 1, 1, 64, 16, "head", F32, 1)
    said = reported(lambda: kvcache.tree_attention(good.cache, good.q.cuda(), good.kn.cuda(), good.vn.cuda()))
    assert "page number" in said and "past the table" in said
    assert lens.tolist() == [3, 18] and torch.isfinite(kr.float()).all()
