"""The short causal convolution against its definition in 64 bits: outputs, states and every gradient, and its single-token form."""
import pytest
import torch

from hdla_hip import short_conv, short_conv_step
from oracle import state_space_oracle as O
from state_space_util import close, cuts, rounded

pytestmark = pytest.mark.gpu
DEV = "cuda"


def make(seed, nb, T, d, W, dtype, bias=True, state=True, N=None, pdtype=None):
    g = torch.Generator().manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=g)
    N = nb if N is None else N
    pdtype = dtype if pdtype is None else pdtype
    low, ref = {}, {}
    for k, t, ty in (("x", rn(nb, T, d), dtype), ("w", rn(d, W), pdtype), ("bias", rn(d) if bias else None, pdtype), ("state", rn(N, W - 1, d) if state else None, dtype)):
        low[k], ref[k] = (None, None) if t is None else rounded(t, ty)
    return low, ref, rn(nb, T, d).to(dtype), rn(N, W - 1, d).to(dtype)


def magnitudes(ref, act, cu, dy, dl):
    """Each output with its terms by their absolute values: the operator without silu is linear in either factor, silu' is at most 1.1 and its slope at most 0.5."""
    a = {k: None if t is None else t.detach().abs().requires_grad_() for k, t in ref.items()}
    y, last = O.short_conv(a["x"], a["w"], a["bias"], a["state"], False, cu)
    names = [k for k in a if a[k] is not None]
    size = 1.1 * dy.double().abs()
    if act:
        size = size + 0.5 * dy.double().abs() * y.detach()                  # g moves with p
    g = torch.autograd.grad([y, last], [a[k] for k in names], [size, dl.double().abs()], allow_unused=True)
    m = {k: torch.zeros_like(a[k]) if t is None else t for k, t in zip(names, g)}
    return {**m, "y": 1.2 * y.detach()}


def compare(low, ref, dy, dl, act, cu=None, v=None):
    v = {k: None if t is None else t.to(DEV).requires_grad_() for k, t in low.items()} if v is None else v
    y, last = short_conv(v["x"], v["w"], v["bias"], activation="silu" if act else None, initial_state=v["state"], output_final_state=True, cu_seqlens=cu)
    yr, lr = O.short_conv(ref["x"], ref["w"], ref["bias"], ref["state"], act, cu)
    m = magnitudes(ref, act, cu, dy, dl)
    T, W = ref["x"].shape[1], ref["w"].shape[1]
    one, many = W + 12, W + 12 + ref["x"].shape[0] * T                       # roundings of a sum over taps; over all tokens
    assert y.dtype == low["x"].dtype
    close("y", y, yr, m["y"], one)
    assert torch.equal(last.cpu().double(), lr.detach())
    names = [k for k in ("x", "w", "bias", "state") if ref[k] is not None]
    got = torch.autograd.grad([y, last], [v[k] for k in names], [dy.to(DEV), dl.to(DEV)])
    want = torch.autograd.grad([yr, lr], [ref[k] for k in names], [dy.double(), dl.double()], allow_unused=True)
    for k, a, b in zip(names, got, want):
        assert a.dtype == low[k].dtype, k
        close("d" + k, a, torch.zeros_like(ref[k]) if b is None else b, m[k], many if k in ("w", "bias") else 2 * one)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("nb,T,d,W,act", [(1, 1, 8, 4, True), (2, 2, 5, 4, False), (1, 3, 64, 3, True), (3, 16, 33, 2, True), (2, 17, 16, 4, True), (1, 31, 7, 3, False),
                                          (1, 64, 96, 4, True), (2, 129, 24, 4, True), (1, 300, 1, 4, False)])
def test_convolution_and_gradients(nb, T, d, W, act, dtype):
    compare(*make(T + d, nb, T, d, W, dtype), act)


@pytest.mark.parametrize("bias,state", [(False, False), (True, False), (False, True)])
def test_what_may_be_left_out(bias, state):
    compare(*make(3, 2, 40, 16, 4, torch.bfloat16, bias, state), True)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("inner", [(17, 17, 18), (1, 2, 4), (15, 16, 99), (0, 5, 100), (32, 64, 96)])
@pytest.mark.parametrize("W", [3, 4])
def test_packed_sequences_of_any_length(inner, W, dtype):
    cu = cuts(100, inner)
    compare(*make(sum(inner), 1, 100, 24, W, dtype, N=len(inner) + 1), True, cu)


def test_many_packed_sequences_of_few_tokens():
    cu = torch.arange(0, 151, 2)
    cu = torch.cat([cu[:40], cu[39:40], cu[40:]])                            # (one of them empty)
    compare(*make(4, 1, 150, 8, 4, torch.float32, N=len(cu) - 1), True, cu)


def test_a_table_on_the_device_that_leaves_tokens_out():
    low, ref, dy, dl = make(8, 1, 100, 16, 4, torch.bfloat16, N=2)
    cu = torch.tensor([3, 40, 90])
    v = {k: t.to(DEV).requires_grad_() for k, t in low.items()}
    y, last = short_conv(v["x"], v["w"], v["bias"], activation="silu", initial_state=v["state"], output_final_state=True, cu_seqlens=cu.to(DEV))
    dx = torch.autograd.grad([y, last], v["x"], [dy.to(DEV), dl.to(DEV)])[0]
    for t in (y, dx):
        assert not t[:, :3].any() and not t[:, 90:].any() and t[:, 3:90].any()
    yr, _ = O.short_conv(ref["x"], ref["w"], ref["bias"], ref["state"], True, cu)
    close("y", y, yr, magnitudes(ref, True, cu, dy, dl)["y"], 16)


def test_a_decreasing_table_touches_nothing_outside():
    low, _, dy, dl = make(9, 1, 100, 16, 4, torch.bfloat16, N=3)
    v = {k: t.to(DEV).requires_grad_() for k, t in low.items()}
    y, last = short_conv(v["x"], v["w"], v["bias"], initial_state=v["state"], output_final_state=True, cu_seqlens=torch.tensor([-5, 60, 20, 1000], device=DEV))
    g = torch.autograd.grad([y, last], list(v.values()), [dy.to(DEV), dl.to(DEV)])
    torch.cuda.synchronize()
    assert torch.isfinite(y).all() and all(torch.isfinite(t).all() for t in g)


@pytest.mark.parametrize("offset", [0, 3])
def test_half_of_a_projection(offset):
    low, ref, dy, dl = make(5, 2, 70, 32, 4, torch.bfloat16)
    wide = torch.randn(2, 70, 64 + offset).bfloat16().to(DEV)
    wide[..., offset:offset + 32] = low["x"].to(DEV)
    v = {k: t.to(DEV).requires_grad_() for k, t in low.items()}
    v["x"] = wide[..., offset:offset + 32].detach().requires_grad_()
    assert not v["x"].is_contiguous()
    compare(low, ref, dy, dl, True, v=v)


def test_other_orders_and_types():
    low, ref, dy, dl = make(6, 2, 50, 16, 4, torch.bfloat16, pdtype=torch.float32)
    v = {k: t.to(DEV).requires_grad_() for k, t in low.items()}
    v["x"] = low["x"].transpose(1, 2).contiguous().to(DEV).transpose(1, 2).detach().requires_grad_()
    v["w"] = low["w"].t().contiguous().to(DEV).t().detach().requires_grad_()
    compare(low, ref, dy, dl, True, v=v)
    compare(*make(7, 1, 20, 8, 4, torch.float16), True)


def test_no_tokens_hand_the_state_on():
    low, _, _, dl = make(10, 2, 0, 16, 4, torch.bfloat16)
    v = {k: t.to(DEV).requires_grad_() for k, t in low.items()}
    y, last = short_conv(v["x"], v["w"], v["bias"], initial_state=v["state"], output_final_state=True)
    assert y.shape == (2, 0, 16) and torch.equal(last, v["state"])
    g = torch.autograd.grad(last, [v["state"], v["w"]], dl.to(DEV))
    assert torch.equal(g[0].cpu(), dl) and not g[1].any()


def test_values_that_are_not_finite_stay_near():
    low, _, _, _ = make(11, 1, 40, 16, 4, torch.float32)
    v = {k: t.to(DEV) for k, t in low.items()}
    y0, _ = short_conv(v["x"], v["w"], v["bias"])
    v["x"][0, 20, 3] = float("nan")
    y, _ = short_conv(v["x"], v["w"], v["bias"])
    bad = torch.isnan(y)
    assert bad[0, 20:24, 3].all() and bad.sum() == 4 and torch.equal(y[~bad], y0[~bad])


def test_a_sequence_in_pieces_is_the_sequence():
    low, _, _, _ = make(12, 2, 60, 24, 4, torch.bfloat16)
    v = {k: t.to(DEV) for k, t in low.items()}
    y, last = short_conv(v["x"], v["w"], v["bias"], activation="silu", initial_state=v["state"], output_final_state=True)
    s, ys = v["state"], []
    for a, b in ((0, 1), (1, 3), (3, 20), (20, 60)):
        yp, s = short_conv(v["x"][:, a:b], v["w"], v["bias"], activation="silu", initial_state=s, output_final_state=True)
        ys.append(yp)
    assert torch.equal(torch.cat(ys, 1), y) and torch.equal(s, last)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("nb,d,W", [(1, 8, 4), (3, 5, 2), (7, 64, 3), (2, 2048, 4)])
def test_step_is_the_call_of_one_token(nb, d, W, dtype):
    low, ref, dy, dl = make(nb + d, nb, 1, d, W, dtype)
    v = {k: t.to(DEV) for k, t in low.items()}
    yr, lr = O.short_conv(ref["x"], ref["w"], ref["bias"], ref["state"], True)
    before = v["state"].clone()
    y, s = short_conv_step(v["x"][:, 0], v["state"], v["w"], v["bias"], activation="silu")
    assert torch.equal(v["state"], before) and torch.equal(s.cpu().double(), lr.detach()) and y.dtype == s.dtype == dtype
    close("y", y, yr[:, 0], magnitudes(ref, True, None, dy, dl)["y"][:, 0], W + 12)
    if dtype != torch.float16:
        y2, s2 = short_conv_step(v["x"][:, 0], before, v["w"], v["bias"], activation="silu", inplace=True)
        assert s2 is before and torch.equal(s2, s) and torch.equal(y2, y)


def test_the_same_bits_every_time():
    low, _, dy, dl = make(13, 3, 500, 72, 4, torch.bfloat16)
    v = {k: t.to(DEV).requires_grad_() for k, t in low.items()}
    runs = []
    for _ in range(3):
        y, last = short_conv(v["x"], v["w"], v["bias"], activation="silu", initial_state=v["state"], output_final_state=True)
        runs.append([y] + list(torch.autograd.grad([y, last], list(v.values()), [dy.to(DEV), dl.to(DEV)])))
    assert all(torch.equal(a, b) for r in runs[1:] for a, b in zip(r, runs[0]))
