"""The paged cache's calls and autograd, up to the library's entry points (CPU)."""
import pytest

torch = pytest.importorskip("torch")
from torch.autograd import forward_ad  # noqa: E402

from technograd_b200 import kvcache  # noqa: E402
from test_kvcache_host import BF16, cache, drafted, library  # noqa: E402, F401


@pytest.mark.parametrize("which", ["q_norm", "k_norm"])
def test_a_gradient_of_norms_through_append_is_an_error(library, which):  # noqa: F811
    """... and not left out in silence, where only the weights learn."""
    q, k, v = drafted()
    norms = dict(q_norm=torch.ones(64), k_norm=torch.ones(64))
    norms[which].requires_grad_()
    _, qr, kr = kvcache.append(cache(), k, v, q=q, keys=True, **norms)
    for y in (qr, kr):
        with pytest.raises(RuntimeError, match="append has no backward"):
            y.float().sum().backward(retain_graph=True)
    with torch.no_grad():
        assert not any(y.requires_grad for y in kvcache.append(cache(), k, v, q=q, keys=True, **norms))


def test_frequencies_that_learn_are_refused():
    with pytest.raises(ValueError, match="gradient"):
        kvcache.Rotary(64, torch.ones(32, dtype=torch.float64, requires_grad=True))


def test_tangents_through_the_calls_are_an_error(library):  # noqa: F811
    """The results would have none: derivatives of zero. Nothing has been launched by then."""
    c = cache(device=torch.device("cpu"), table=torch.zeros(2, 4, dtype=torch.int32))
    prefix = kvcache.SharedPrefix(c, [(0, 2, 16)])
    norm = torch.ones(64)
    with forward_ad.dual_level():
        for which in range(3):
            q, k, v = (forward_ad.make_dual(x, torch.ones_like(x)) if i == which else x for i, x in enumerate(drafted()))
            for name, call in (("tree_attention", lambda: kvcache.tree_attention(c, q, k, v)), ("shared_attention", lambda: kvcache.shared_attention(c, prefix, q, k, v)),
                               ("append", lambda: kvcache.append(c, k, v, q=q))):
                with pytest.raises(RuntimeError, match=f"{name} has no forward-mode"):
                    call()
        q, k, v = drafted()
        for kw in (dict(q_norm=forward_ad.make_dual(norm, norm)), dict(k_norm=forward_ad.make_dual(norm, norm))):
            with pytest.raises(RuntimeError, match="append has no forward-mode"):
                kvcache.append(c, k, v, q=q, **kw)
        assert not library.calls
        kvcache.tree_attention(c, q, k, v), kvcache.shared_attention(c, prefix, q, k, v), kvcache.append(c, k, v, q_norm=None, k_norm=norm)
    assert len(library.calls) == 5


def test_pages_that_are_written_have_a_new_version(library):  # noqa: F811
    """A pool saved for a backward pass is not what it was after an append, a commit or an eviction into it."""
    table, lens = torch.zeros(2, 4, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)

    def paged():
        k, v = torch.zeros(8, 2, 16, 64, dtype=BF16), torch.zeros(8, 2, 16, 64, dtype=BF16)
        c = kvcache.PagedKV.__new__(kvcache.PagedKV)
        vars(c).update(vars(cache(k=k, v=v, table=table, lens=lens)))
        c._versioned = kvcache._versions(k, v)
        return c, k, v

    q, k, v = drafted()
    count, acc = torch.ones(2, dtype=torch.int32), torch.zeros(2, 2, 40)
    for write in (lambda c: kvcache.append(c, k, v, q=q), lambda c: kvcache.commit(c, k, v, count), lambda c: kvcache.evict(cache(), c, acc, 8)):
        for pool in range(2):
            c, *pools = paged()
            w = torch.ones(pools[pool].shape, dtype=BF16, requires_grad=True)
            y = (pools[pool] * w).sum()
            write(c)
            with pytest.raises(RuntimeError, match="inplace operation"):
                y.backward()
    w = torch.ones(acc.shape, requires_grad=True)
    y = (acc * w).sum()
    kvcache.commit(paged()[0], k, v, count, new=torch.zeros(2, 2, 3), acc=acc)
    with pytest.raises(RuntimeError, match="inplace operation"):
        y.backward()
    with torch.inference_mode():
        c, *_ = paged()
        kvcache.append(c, k, v)
