"""The paged cache's calls and autograd, up to the library's entry points (CPU)."""
import pytest

torch = pytest.importorskip("torch")
from technograd_b200 import kvcache  # noqa: E402
from test_kvcache_host import cache, drafted, library  # noqa: E402, F401


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
