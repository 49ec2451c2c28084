"""rope and autograd, with a stand-in that rotates on the CPU and, as the library does, writes through the pointer (CPU)."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
from torch.autograd import forward_ad  # noqa: E402

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


@pytest.mark.parametrize("learns", [False, True])
@pytest.mark.parametrize("inverse", [False, True])
@pytest.mark.parametrize("pos", [None, torch.tensor([3, 1, 4, 1, 5], dtype=torch.int32)])
def test_a_tangent_is_rotated(calls, learns, inverse, pos):
    """The rotation is linear: the result's tangent is the tangent rotated, whether or not x requires a gradient too."""
    r, x, t = Rotation(), rows(1).requires_grad_(learns), rows(2)
    with forward_ad.dual_level():
        y = forward_ad.unpack_dual(kvcache.rope(forward_ad.make_dual(x, t), r, pos, inverse))
        assert torch.equal(y.primal, turned(x, r.freq, pos, inverse)) and torch.equal(y.tangent, turned(t, r.freq, pos, inverse))
        plain = kvcache.rope(rows(1), r, pos, inverse)
        assert forward_ad.unpack_dual(plain).tangent is None
        with torch.no_grad():  # which forward mode does not ask
            y = forward_ad.unpack_dual(kvcache.rope(forward_ad.make_dual(rows(1), t), r, pos, inverse))
            assert torch.equal(y.tangent, turned(t, r.freq, pos, inverse))


def test_a_tangent_of_any_layout(calls):
    r, x = Rotation(), rows(1)
    wide, off = torch.randn(2, 5, 4, 3).transpose(2, 3), torch.randn(1 + 2 * 5 * 3 * 4)[1:].view(2, 5, 3, 4)
    for t in (wide, off, torch.ones(1).expand(2, 5, 3, 4)):
        with forward_ad.dual_level():
            assert torch.equal(forward_ad.unpack_dual(kvcache.rope(forward_ad.make_dual(x, t), r)).tangent, turned(t, r.freq, None, False))


def test_a_tangent_of_a_gradient(calls):
    """Forward over backward: the derivative of 2 R^T R x along t is 2 t."""
    r, x, t = Rotation(), rows(1).requires_grad_(), rows(2)
    with forward_ad.dual_level():
        d = forward_ad.make_dual(x, t)
        g, = torch.autograd.grad(kvcache.rope(d, r).square().sum(), d, create_graph=True)
        h = forward_ad.unpack_dual(g).tangent
    # each rotation: cos, sin and the two products and their sum of elements of up to |t| sqrt(2), five roundings of 2^-24
    assert (h - 2 * t).abs().max() < 2 * 2 * 5 * 2.0 ** -24 * 2 ** 0.5 * 2 * t.abs().max()


def test_transforms_of_the_call_are_refused(calls):
    """torch.func's wrapped tensors have no memory of their own: an error, and no result without its derivative."""
    r, x, t = Rotation(), rows(1), rows(2)
    for f in (lambda: torch.func.jvp(lambda z: kvcache.rope(z, r), (x,), (t,)), lambda: torch.func.grad(lambda z: kvcache.rope(z, r).sum())(x)):
        with pytest.raises(RuntimeError):
            f()


def test_a_tangent_and_out(calls):
    r, x = Rotation(), rows(1)
    with forward_ad.dual_level():
        d = forward_ad.make_dual(x, rows(2))
        for kw in (dict(x=d, out=rows(3)), dict(x=d, out=d), dict(x=x, out=d)):
            with pytest.raises(ValueError, match="out"):
                kvcache.rope(rotary=r, **kw)
    assert not calls


def test_what_is_saved_does_not_change_unnoticed(calls):
    """torch's own error where a tensor saved for a backward pass, or a view of one, was rotated in place."""
    r, w = Rotation(), torch.randn(2, 5, 3, 4, requires_grad=True)
    for view in (lambda x: x, lambda x: x[:1], lambda x: x[:, :, 1:2]):
        x = rows(1)
        y = (x * w).sum()
        kvcache.rope(view(x), r, out=view(x))
        with pytest.raises(RuntimeError, match="inplace operation"):
            y.backward()
    x, out = rows(1), rows(2)
    y = (out * w).sum() + (x * w).sum()
    kvcache.rope(x, r, out=out)
    with pytest.raises(RuntimeError, match="inplace operation"):
        y.backward()
    (x * w).sum().backward()  # x itself was only read
    assert torch.equal(w.grad, x)


def test_out_that_requires_a_gradient_is_refused(calls):
    r, x = Rotation(), rows(1)
    leaf = rows(2).requires_grad_()
    for out in (leaf, leaf * 1):
        with pytest.raises(ValueError, match="out"):
            kvcache.rope(x, r, out=out)
    assert not calls
    with torch.no_grad():  # as torch's own in-place operations
        version = leaf._version
        assert kvcache.rope(x, r, out=leaf) is leaf and torch.equal(leaf, turned(x, r.freq, None, False)) and leaf._version == version + 1


def test_out_in_inference_mode(calls):
    r = Rotation()
    with torch.inference_mode():
        x = rows(1)
        want = turned(x, r.freq, None, False)
        assert torch.equal(kvcache.rope(x, r, out=x), want)


def test_positions_and_frequencies_stay_until_the_backward_pass(calls):
    """Other ones would give another rotation's gradient."""
    for given in (None, torch.arange(5, dtype=torch.int32)):
        for change in [lambda r: r.freq.mul_(2)] + ([] if given is None else [lambda r: given.add_(1)]):
            r, x = Rotation(), rows(1).requires_grad_()
            y = kvcache.rope(x, r, given)
            change(r)
            with pytest.raises(RuntimeError, match="inplace operation"):
                y.sum().backward()
            assert x.grad is None


def test_frequencies_made_in_inference_mode(calls):
    with torch.inference_mode():
        r = Rotation()
    x = rows(1).requires_grad_()
    kvcache.rope(x, r).sum().backward()
    assert torch.equal(x.grad, turned(torch.ones_like(x), r.freq, None, True))
