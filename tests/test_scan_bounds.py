"""The bounds that the scan is held to (oracle.scan_bounds) admit 32 bits and nothing less: the definition evaluated in fp32 keeps them, with one operand rounded to bf16 it does not."""
import functools

import pytest
import torch

from oracle import state_space_oracle as O
from state_space_util import U, close

NAMES = ("x", "dt", "A", "B", "C", "D", "z", "bias", "h0")
SHAPES = [(1, 1, 16, 16, 1), (2, 40, 9, 8, 1), (1, 300, 12, 16, 2), (1, 1500, 16, 16, 1), (1, 700, 8, 33, 2)]


def inputs(seed, nb, T, d, S, G):
    g = torch.Generator().manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=g)
    v = dict(x=rn(nb, T, d), dt=0.5 * rn(nb, T, d) - 2, A=-torch.exp(rn(d, S)), B=rn(nb, T, G, S), C=rn(nb, T, G, S), D=rn(d), z=rn(nb, T, d), bias=0.5 * rn(d), h0=rn(nb, d, S))
    return v, rn(nb, T, d), rn(nb, d, S)


def results(v, dy, dh, dtype):
    v = {k: t.to(dtype).requires_grad_() for k, t in v.items()}
    y, ht = O.scan(*[v[k] for k in NAMES[:8]], True, v["h0"])
    return dict(zip(("y", "ht") + NAMES, (y, ht) + torch.autograd.grad([y, ht], [v[k] for k in NAMES], [dy.to(dtype), dh.to(dtype)])))


@functools.lru_cache(None)
def of(shape):
    """Inputs, what they give in 64 bits, and the bounds."""
    v, dy, dh = inputs(sum(shape), *shape)
    return v, dy, dh, results(v, dy, dh, torch.float64), O.scan_bounds(*[v[k] for k in NAMES[:8]], True, v["h0"], None, dy, dh)


@pytest.mark.parametrize("shape", SHAPES)
def test_the_definition_in_32_bits_keeps_them(shape):
    v, dy, dh, ref, b = of(shape)
    low = results(v, dy, dh, torch.float32)
    for k in ref:
        close(k, low[k], ref[k], b[k] / U, 1)


@pytest.mark.parametrize("wrong", ["x", "dt", "A", "B", "C", "D", "z", "h0", "bias", "dy", "dh"])
@pytest.mark.parametrize("shape", SHAPES[1:])
def test_an_operand_in_16_bits_does_not(shape, wrong):
    v, dy, dh, ref, b = of(shape)
    given = dict(v, dy=dy, dh=dh)
    given[wrong] = given[wrong].bfloat16().float()
    low = results({k: given[k] for k in NAMES}, given["dy"], given["dh"], torch.float64)
    seen = {k for k in ref if ((low[k].detach() - ref[k].detach()).abs() > b[k] + U * ref[k].detach().abs()).any()}
    # (a gradient is linear in dy; the last state's reaches as far back as a state lasts)
    want = {"dy": {"x", "dt", "z", "B", "C", "A", "D"}, "dh": {"x", "dt", "B"}, "dt": {"y", "ht", "x", "dt", "B", "C"}, "A": {"y", "ht", "x", "dt", "B", "C"}, "B": {"y", "ht", "x", "dt", "C"},
            "x": {"y", "ht", "B", "C", "D"}, "bias": {"y", "ht", "x", "dt", "B", "C"}}.get(wrong, {"y"})
    assert want <= seen, (wrong, want - seen)
