"""A decay of minus infinity beside a step size of zero: a token that the scan passes over leaves a state as it is, and the single-token call does the same."""
import pytest
import torch

from hdla_hip import state_space_scan, state_space_step

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("softplus", [True, False])
@pytest.mark.parametrize("low", [-float("inf"), torch.finfo(torch.float32).min, -1e30])
@pytest.mark.parametrize("adtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("nb,d,S", [(3, 16, 16), (2, 5, 3), (260, 260, 64), (1, 7, 20)])
def test_step_is_the_scan_of_one_token(nb, d, S, adtype, low, softplus):
    g = torch.Generator().manual_seed(nb + d)
    rn = lambda *s: torch.randn(*s, generator=g).to(DEV)
    x, dt, B, C, h0 = rn(nb, d), rn(nb, d).abs(), rn(nb, S), rn(nb, S), rn(nb, d, S)
    dt[:, ::2] = -1e4 if softplus else 0.0                                   # (softplus of -10000 is zero)
    A = -torch.exp(rn(d, S))
    A[:, ::3] = low
    A = A.to(adtype)
    y, h = state_space_step(x, dt, A, B, C, h0, dt_softplus=softplus)
    ys, hs = state_space_scan(x[:, None], dt[:, None], A, B[:, None], C[:, None], dt_softplus=softplus, initial_state=h0, output_final_state=True)
    assert torch.isfinite(y).all() and torch.isfinite(h).all()
    # a step size of zero: the state stays, to the bit
    assert torch.equal(h[:, ::2], h0[:, ::2]) and torch.equal(hs[:, ::2], h0[:, ::2])
    # an infinite decay and any other step size: what the token adds
    delta = torch.nn.functional.softplus(dt.double(), threshold=1e4) if softplus else dt.double()
    add = (delta * x.double())[:, 1::2, None] * B.double()[:, None, ::3]
    for state in (h, hs):
        # four roundings of the step size, one of each product
        assert ((state[:, 1::2, ::3].double() - add).abs() <= 8 * 2.0 ** -24 * add.abs() + 1e-37).all()
    # scan and step: the decay's exponent and a sum over the states may be rounded in another order
    assert ((y - ys[:, 0]).abs() <= (S + 64) * 2.0 ** -23 * ((h.abs() + hs.abs()) * C.abs()[:, None]).sum(-1) + 1e-37).all()
