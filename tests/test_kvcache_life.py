"""What the paged cache's calls keep between them (CPU)."""
import gc
import weakref

import pytest

torch = pytest.importorskip("torch")
from technograd_b200 import kvcache  # noqa: E402
from test_kvcache_host import drafted, library  # noqa: E402, F401
from test_shared_attn_abi import fake  # noqa: E402


def test_prefixes_of_batches_that_are_gone_are_not_kept(library):  # noqa: F811
    """A cache that lives through many batches, its lengths changed in place."""
    c, args, seen = fake(), drafted(), []
    for i in range(300):
        x = kvcache.SharedPrefix(c, [(0, 2, 16)], max_own=i)
        kvcache.shared_attention(c, x, *args)
        seen.append(weakref.ref(x._held))
        del x
    gc.collect()
    assert not any(r() is not None for r in seen) and len(c._plans) <= 64


def test_the_size_of_the_scratch_is_asked_for_once(library):  # noqa: F811
    """Prefixes of the same numbers share the answer; any other number asks again."""
    c, args = fake(), drafted()
    asked = lambda: sum(n == "tg_cuda_shared_attn_workspace" for n, _ in library.calls)  # noqa: E731
    for _ in range(3):
        kvcache.shared_attention(c, kvcache.SharedPrefix(c, [(0, 2, 16)], max_own=5), *args)
    assert asked() == 1
    for i, (groups, kw) in enumerate((([(0, 2, 17)], {}), ([(0, 1, 16), (1, 1, 16)], {}), ([(0, 2, 16)], dict(max_own=6)), ([(0, 2, 16)], dict(always=True)))):
        kvcache.shared_attention(c, kvcache.SharedPrefix(c, groups, **{"max_own": 5, **kw}), *args)
        assert asked() == 2 + i
