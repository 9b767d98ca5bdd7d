"""What the tests of the state space block share: inputs, and how far a result may be from the definition in 64 bits.

A result is within half a step of its own type of what 32 bits gave, and that within `count` roundings of 2^-24 of the sum of its terms' absolute
values (the oracle's magnitudes): |got - ref| <= eps(type) / 2 |ref| (1 + small) + count 2^-24 magnitude.  Inputs are rounded to their type before either side sees them."""
import torch

U = 2.0 ** -24


def close(name, got, ref, magnitude, count):
    got, ref, magnitude = got.detach().cpu(), ref.detach().double(), magnitude.detach().double()
    assert got.shape == ref.shape, f"{name}: {tuple(got.shape)} instead of {tuple(ref.shape)}"
    assert torch.isfinite(got).all(), f"{name}: not finite"
    half = torch.finfo(got.dtype).eps / 2
    near = count * U * magnitude
    tiny = torch.finfo(got.dtype).tiny
    allowed = half * (ref.abs() + near) + near + tiny
    off = (got.double() - ref).abs()
    assert (off <= allowed).all(), f"{name}: off by {(off / allowed).max().item():.3g} of what roundings can be (element {int((off / allowed).argmax())})"


def rounded(t, dtype):
    """As the operator sees it, and as a float64 leaf."""
    low = t.to(dtype)
    return low, low.double().requires_grad_()


def cuts(T, inner):
    return torch.tensor([0] + list(inner) + [T])
