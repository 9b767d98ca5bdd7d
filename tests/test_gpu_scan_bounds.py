"""The selective state space scan held to what 32 bits can be off by, element by element (oracle.scan_bounds): bounds that a single operand rounded to 16 bits breaks, at any length
(test_scan_bounds.py shows it of the definition)."""
import pytest
import torch

from oracle import state_space_oracle as O
from state_space_util import U, close, cuts
from test_gpu_state_space import DEV, NAMES, call, make, put

pytestmark = pytest.mark.gpu


def compare(low, ref, dy, dh, softplus=True, cu=None):
    v = put(low)
    y, ht = call(v, softplus, True, cu)
    yr, hr = O.scan(*[ref[k] for k in NAMES[:8]], softplus, ref["h0"], cu)
    names = [k for k in NAMES if ref[k] is not None]
    got = torch.autograd.grad([y, ht], [v[k] for k in names], [dy.to(DEV), dh.to(DEV)])
    want = torch.autograd.grad([yr, hr], [ref[k] for k in names], [dy.double(), dh.double()])
    b = O.scan_bounds(*[ref[k] for k in NAMES[:8]], softplus, ref["h0"], cu, dy, dh)
    for k, a, r in zip(["y", "ht"] + names, (y, ht) + got, (yr, hr) + want):
        close(k, a, r, b[k] / U, 1)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("nb,T,d,S,G", [(1, 1, 16, 16, 1), (2, 7, 5, 3, 1), (1, 65, 20, 12, 4), (3, 130, 24, 32, 1), (1, 129, 9, 64, 3), (1, 70, 6, 1, 2), (1, 90, 12, 20, 1), (2, 257, 33, 8, 1),
                                        (20, 40, 33, 16, 1)])
def test_short_sequences(nb, T, d, S, G, dtype):
    compare(*make(T * 7 + d, nb, T, d, S, G, dtype))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("nb,T,d,S,G,state", [(1, 1500, 16, 16, 1, True), (2, 1030, 9, 8, 1, False), (1, 1281, 8, 33, 2, True), (1, 900, 12, 20, 1, True)])
def test_segments(nb, T, d, S, G, state, dtype):
    compare(*make(T + 3 * d, nb, T, d, S, G, dtype, state=state))


def test_a_whole_sequence_of_many_channels():
    """As many workgroups as leave no room for segments: one chain over all tokens."""
    compare(*make(77, 1, 500, 8192, 8, 1, torch.float32))


@pytest.mark.parametrize("inner", [(3, 700, 701), (256, 512, 1024), (0, 0, 1)])
def test_packed_sequences(inner):
    cu = cuts(1501, inner)
    compare(*make(sum(inner) + 5, 1, 1501, 16, 16, 1, torch.float32, N=len(inner) + 1), cu=cu)


@pytest.mark.parametrize("gate,skip,bias,state,softplus", [(False, False, False, False, False), (True, False, False, True, True), (False, True, True, False, True)])
def test_what_may_be_left_out(gate, skip, bias, state, softplus):
    low, ref, dy, dh = make(6, 2, 300, 24, 16, 1, torch.float32, gate, skip, bias, state)
    if not softplus:
        low["dt"] = torch.nn.functional.softplus(low["dt"])
        ref["dt"] = low["dt"].double().requires_grad_()
    compare(low, ref, dy, dh, softplus)


@pytest.mark.parametrize("T", [80, 1300])
def test_extreme_step_sizes(T):
    """A state that is forgotten at once, one that is kept, and softplus at both ends."""
    low, ref, dy, dh = make(15 + T, 1, T, 16, 16, 1, torch.float32)
    low["dt"][:, ::3] = -40.0
    low["dt"][:, 1::3] = 60.0
    ref["dt"] = low["dt"].double().requires_grad_()
    compare(low, ref, dy, dh)


@pytest.mark.parametrize("d,T", [(20, 11), (20, 100), (8, 3001)])
def test_states_that_decay_at_once(d, T):
    """A = -inf: a state is what its last token adds, and nothing comes back through it.  In 64 bits -1e30 is as much (every step size is above 1e-6), and has derivatives."""
    low, ref, dy, dh = make(42 + T, 1, T, d, 8, 1, torch.float32)
    low["A"][:, ::3] = -float("inf")
    ref["A"].data[:, ::3] = -1e30
    assert O.step_sizes(ref["dt"], ref["bias"], True).min() > 1e-6
    compare(low, ref, dy, dh)
