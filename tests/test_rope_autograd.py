"""rope and autograd, with a stand-in that rotates on the CPU and, as the library does, writes through the pointer (CPU)."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
from technograd_b200 import kvcache  # noqa: E402


class Rotation:
    """What rope's autograd reads of a Rotary."""
    def __init__(self):
        self.freq = torch.tensor([1.0, 0.25], dtype=torch.float64)


def turned(x, freq, pos, inverse):
    angle = (torch.arange(x.shape[1]) if pos is None else pos).double()[..., None, None] * freq
    c, s = angle.cos().float(), angle.sin().float() * (-1 if inverse else 1)
    half = len(freq)
    a, b = x[..., :half], x[..., half:]
    return torch.cat([a * c - b * s, a * s + b * c], -1)


@pytest.fixture
def calls(monkeypatch):
    """The rows that reached the library; as there, they have to be contiguous and on 16-byte boundaries."""
    seen = []

    def turn(x, rotary, pos, inverse, out):
        assert x.data_ptr() % 16 == 0 and x.stride(3) == 1 and all(s * x.element_size() % 16 == 0 for s in x.stride()[:3])
        seen.append(x)
        out = torch.empty_like(x) if out is None else out
        np.copyto(out.detach().numpy(), turned(x.detach(), rotary.freq, pos, inverse).numpy())  # behind autograd's back
        return out
    monkeypatch.setattr(kvcache, "_turn", turn)
    return seen


def rows(seed=0):
    return torch.randn(2, 5, 3, 4, generator=torch.Generator().manual_seed(seed))


@pytest.mark.parametrize("before", [0, 1, 3, 4])
def test_a_gradient_that_begins_off_a_boundary(calls, before):
    """Behind a cat of a few elements a gradient is a contiguous view that begins at any of them."""
    r, x, w = Rotation(), rows(1).requires_grad_(), torch.randn(before + 2 * 5 * 3 * 4)
    (torch.cat([torch.zeros(before), kvcache.rope(x, r).flatten()]) * w).sum().backward()
    assert torch.equal(x.grad, turned(w[before:].view(x.shape), r.freq, None, True))
