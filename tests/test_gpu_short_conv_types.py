"""A convolution's state of another type than its input: it is not rounded to x's type on the way in, and results are rounded once."""
import pytest
import torch

from hdla_hip import short_conv, short_conv_step
from oracle import state_space_oracle as O
from state_space_util import close, rounded
import test_gpu_short_conv as conv

pytestmark = pytest.mark.gpu
DEV = "cuda"
MIXED = [(torch.bfloat16, torch.float32), (torch.bfloat16, torch.float16), (torch.float32, torch.bfloat16), (torch.float16, torch.float32), (torch.float16, torch.bfloat16)]


def with_state(seed, nb, T, d, W, dtype, other):
    low, ref, dy, _ = conv.make(seed, nb, T, d, W, dtype)
    g = torch.Generator().manual_seed(seed + 1)
    low["state"], ref["state"] = rounded(torch.randn(nb, W - 1, d, generator=g), other)
    return low, ref, dy, torch.randn(nb, W - 1, d, generator=g).to(dtype)


@pytest.mark.parametrize("act", [True, False])
@pytest.mark.parametrize("T", [1, 2, 40])
@pytest.mark.parametrize("dtype,other", MIXED)
def test_state_of_another_type(dtype, other, T, act):
    low, ref, dy, dl = with_state(31 + T, 2, T, 24, 4, dtype, other)
    v = {k: t.to(DEV).requires_grad_() for k, t in low.items()}
    y, last = short_conv(v["x"], v["w"], v["bias"], activation="silu" if act else None, initial_state=v["state"], output_final_state=True)
    yr, lr = O.short_conv(ref["x"], ref["w"], ref["bias"], ref["state"], act)
    m = conv.magnitudes(ref, act, None, dy, dl)
    one, many = 4 + 12, 4 + 12 + 2 * T
    assert y.dtype == last.dtype == dtype
    close("y", y, yr, m["y"], one)
    close("last", last, lr, lr.abs(), 0)                                     # (rounded once, to x's type, as said of it)
    names = ("x", "w", "bias", "state")
    got = torch.autograd.grad([y, last], [v[k] for k in names], [dy.to(DEV), dl.to(DEV)])
    want = torch.autograd.grad([yr, lr], [ref[k] for k in names], [dy.double(), dl.double()])
    for k, a, b in zip(names, got, want):
        assert a.dtype == low[k].dtype, k
        close("d" + k, a, b, m[k], many if k in ("w", "bias") else 2 * one)


@pytest.mark.parametrize("dtype,other", MIXED)
def test_step_with_a_state_of_another_type(dtype, other):
    low, ref, dy, dl = with_state(51, 3, 1, 24, 4, dtype, other)
    v = {k: t.to(DEV) for k, t in low.items()}
    yr, lr = O.short_conv(ref["x"], ref["w"], ref["bias"], ref["state"], True)
    m = conv.magnitudes(ref, True, None, dy, dl)
    before = v["state"].clone()
    y, s = short_conv_step(v["x"][:, 0], v["state"], v["w"], v["bias"], activation="silu")
    assert y.dtype == s.dtype == dtype and torch.equal(v["state"], before)
    close("y", y, yr[:, 0], m["y"][:, 0], 4 + 12)
    close("s", s, lr, lr.abs(), 0)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_a_state_in_fp32_goes_on_in_place_and_loses_nothing(dtype):
    low, ref, _, _ = with_state(61, 3, 1, 24, 4, dtype, torch.float32)
    v = {k: t.to(DEV) for k, t in low.items()}
    y0, _ = short_conv_step(v["x"][:, 0], v["state"], v["w"], v["bias"], activation="silu")
    want = torch.cat([v["state"][:, 1:], v["x"].float()], 1)
    y, s = short_conv_step(v["x"][:, 0], v["state"], v["w"], v["bias"], activation="silu", inplace=True)
    assert s is v["state"] and torch.equal(s, want) and torch.equal(y, y0)


def test_a_narrower_state_is_refused_in_place():
    x, w = torch.randn(2, 8, device=DEV), torch.randn(8, 4, device=DEV)
    for dtype in (torch.bfloat16, torch.float16):
        with pytest.raises(ValueError, match="in place"):
            short_conv_step(x, torch.zeros(2, 3, 8, dtype=dtype, device=DEV), w, inplace=True)
