"""The selective state space scan against its definition in 64 bits: outputs, states and every gradient, and its single-token form."""
import pytest
import torch

from hdla_hip import state_space_scan, state_space_step
from oracle import state_space_oracle as O
from state_space_util import close, cuts, rounded

pytestmark = pytest.mark.gpu
DEV = "cuda"
NAMES = ("x", "dt", "A", "B", "C", "D", "z", "bias", "h0")


def make(seed, nb, T, d, S, G, dtype, gate=True, skip=True, bias=True, state=True, N=None, pdtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=g)
    N = nb if N is None else N
    raw = dict(x=rn(nb, T, d), dt=0.5 * rn(nb, T, d) - 2, A=-torch.exp(rn(d, S)), B=rn(nb, T, G, S), C=rn(nb, T, G, S),
               D=rn(d) if skip else None, z=rn(nb, T, d) if gate else None, bias=0.5 * rn(d) if bias else None, h0=rn(N, d, S) if state else None)
    kind = dict(A=pdtype, D=pdtype, bias=pdtype, h0=torch.float32)
    low, ref = {}, {}
    for k, t in raw.items():
        low[k], ref[k] = (None, None) if t is None else rounded(t, kind.get(k, dtype))
    return low, ref, rn(nb, T, d).to(dtype), rn(N, d, S)


def put(low, grad=True):
    return {k: None if t is None else t.to(DEV).requires_grad_(grad) for k, t in low.items()}


def call(v, softplus, want=True, cu=None):
    return state_space_scan(v["x"], v["dt"], v["A"], v["B"], v["C"], v["D"], v["z"], dt_bias=v["bias"], dt_softplus=softplus, initial_state=v["h0"],
                            output_final_state=want, cu_seqlens=cu)


def compare(low, ref, dy, dh, softplus, cu=None, v=None):
    v = put(low) if v is None else v
    y, ht = call(v, softplus, True, cu)
    yr, hr = O.scan(*[ref[k] for k in NAMES[:8]], softplus, ref["h0"], cu)
    m, count = O.scan_magnitudes(*[ref[k] for k in NAMES[:8]], softplus, ref["h0"], cu, dy.double(), dh.double())
    assert y.dtype == low["x"].dtype and ht.dtype == torch.float32
    close("y", y, yr, m["y"], count)
    close("ht", ht, hr, m["ht"], count)
    names = [k for k in NAMES if ref[k] is not None]
    got = torch.autograd.grad([y, ht], [v[k] for k in names], [dy.to(DEV), dh.to(DEV)])
    want = torch.autograd.grad([yr, hr], [ref[k] for k in names], [dy.double(), dh.double()])
    for k, a, b in zip(names, got, want):
        assert a.dtype == low[k].dtype, k
        close("d" + k, a, b, m[k], count)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("nb,T,d,S,G", [(1, 1, 16, 16, 1), (2, 7, 5, 3, 1), (1, 8, 64, 8, 1), (1, 63, 33, 16, 1), (2, 64, 16, 16, 2), (1, 65, 20, 12, 4),
                                        (3, 130, 24, 32, 1), (1, 300, 40, 16, 1), (1, 129, 9, 64, 3), (1, 70, 6, 1, 2), (1, 90, 12, 20, 1), (1, 257, 7, 33, 1)])
def test_scan_and_gradients(nb, T, d, S, G, dtype):
    low, ref, dy, dh = make(T * 100 + d, nb, T, d, S, G, dtype)
    compare(low, ref, dy, dh, True)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("nb,T,d,S,G,state", [(1, 1500, 16, 16, 1, True), (2, 1030, 9, 8, 1, False), (1, 1281, 8, 33, 2, True), (1, 900, 12, 20, 1, True)])
def test_long_sequences_of_few_channels(nb, T, d, S, G, state, dtype):
    """Cut into segments that run side by side."""
    low, ref, dy, dh = make(T + d, nb, T, d, S, G, dtype, state=state)
    compare(low, ref, dy, dh, True)


@pytest.mark.parametrize("nb,T,d,S,G,dtype", [(130, 35, 64, 16, 1, torch.bfloat16), (130, 33, 31, 8, 1, torch.float32), (20, 3, 2048, 16, 1, torch.bfloat16),
                                              (65, 40, 64, 30, 2, torch.bfloat16), (140, 9, 15, 64, 1, torch.float32)])
def test_many_sequences(nb, T, d, S, G, dtype):
    """More workgroups than compute units; more sequences than workgroups side by side."""
    low, ref, dy, dh = make(nb + T, nb, T, d, S, G, dtype)
    compare(low, ref, dy, dh, True)


def test_many_packed_sequences_of_few_tokens():
    cu = torch.arange(0, 1042, 2)
    cu[100:110] = cu[100]                                                    # (some of them empty)
    low, ref, dy, dh = make(25, 1, 1040, 16, 16, 1, torch.bfloat16, N=len(cu) - 1)
    compare(low, ref, dy, dh, True, cu)


@pytest.mark.parametrize("inner", [(3, 700, 701), (256, 512, 1024), (1400, 1499, 1500), (0, 0, 1)])
def test_long_packed_sequences_of_few_channels(inner):
    T = 1501
    cu = cuts(T, inner)
    low, ref, dy, dh = make(sum(inner), 1, T, 16, 16, 1, torch.float32, N=len(inner) + 1)
    compare(low, ref, dy, dh, True, cu)
    v = put(low)
    v2 = put(low)
    for a, b in zip(call(v, True, True, cu), call(v2, True, True, cu.to(DEV))):
        assert torch.equal(a, b)


def test_long_tables_that_leave_tokens_out_or_decrease():
    low, ref, dy, dh = make(24, 1, 1500, 16, 16, 1, torch.float32, N=3)
    v = put(low)
    cu = torch.tensor([300, 301, 1100, 1400])
    y, ht = call(v, True, True, cu.to(DEV))
    g = torch.autograd.grad([y, ht], [v["x"], v["B"], v["C"]], [dy.to(DEV), dh.to(DEV)])
    yr, hr = O.scan(*[ref[k] for k in NAMES[:8]], True, ref["h0"], cu)
    m, count = O.scan_magnitudes(*[ref[k] for k in NAMES[:8]], True, ref["h0"], cu, dy.double(), dh.double())
    close("y", y, yr, m["y"], count)
    close("ht", ht, hr, m["ht"], count)
    for k, a, b in zip(("x", "B", "C"), g, torch.autograd.grad([yr, hr], [ref["x"], ref["B"], ref["C"]], [dy.double(), dh.double()])):
        close("d" + k, a, b, m[k], count)
    y, ht = call(v, True, True, torch.tensor([-7, 1300, 200, 5000], device=DEV))
    g = torch.autograd.grad(y, [v[k] for k in NAMES], dy.to(DEV))
    torch.cuda.synchronize()
    assert torch.isfinite(y).all() and all(torch.isfinite(t).all() for t in g)


@pytest.mark.parametrize("gate,skip,bias,state,softplus", [(False, False, False, False, False), (True, False, False, True, True), (False, True, True, False, True),
                                                           (True, True, False, False, False)])
def test_what_may_be_left_out(gate, skip, bias, state, softplus):
    low, ref, dy, dh = make(5, 2, 100, 24, 16, 1, torch.bfloat16, gate, skip, bias, state)
    if not softplus:
        low["dt"] = torch.nn.functional.softplus(low["dt"].float()).bfloat16()
        ref["dt"] = low["dt"].double().requires_grad_()
    compare(low, ref, dy, dh, softplus)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("inner", [(17, 17, 18), (1, 64, 128), (63, 64, 199), (0, 5, 200)])
def test_packed_sequences_of_any_length(inner, dtype):
    T = 200
    cu = cuts(T, inner)
    low, ref, dy, dh = make(sum(inner), 1, T, 24, 16, 1, dtype, N=len(inner) + 1)
    compare(low, ref, dy, dh, True, cu)


def test_a_table_on_the_device_that_leaves_tokens_out():
    cu = torch.tensor([3, 40, 90])
    low, ref, dy, dh = make(8, 1, 100, 16, 16, 1, torch.bfloat16, N=2)
    v = put(low)
    y, ht = call(v, True, True, cu.to(DEV))
    grads = torch.autograd.grad([y, ht], [v["x"], v["dt"], v["z"], v["B"], v["C"]], [dy.to(DEV), dh.to(DEV)])
    for t in (y,) + grads:
        assert not t[:, :3].any() and not t[:, 90:].any() and t[:, 3:90].any()
    yr, _ = O.scan(*[ref[k] for k in NAMES[:8]], True, ref["h0"], cu)
    m, count = O.scan_magnitudes(*[ref[k] for k in NAMES[:8]], True, ref["h0"], cu)
    close("y", y, yr, m["y"], count)


def test_a_decreasing_table_touches_nothing_outside():
    cu = torch.tensor([-5, 60, 20, 1000], device=DEV)
    low, _, dy, dh = make(9, 1, 100, 16, 16, 1, torch.bfloat16, N=3)
    v = put(low)
    y, ht = call(v, True, True, cu)
    grads = torch.autograd.grad([y, ht], [v[k] for k in NAMES], [dy.to(DEV), dh.to(DEV)])
    torch.cuda.synchronize()
    assert torch.isfinite(y).all() and all(torch.isfinite(t).all() for t in grads)


@pytest.mark.parametrize("offset", [0, 1, 4])
def test_views_of_projections(offset):
    """x, z of one tensor; dt, B, C of another: aligned, and at any element."""
    low, ref, dy, dh = make(11, 2, 90, 32, 16, 1, torch.bfloat16)
    nb, T, d = low["x"].shape
    xz = torch.zeros(nb, T, 2 * d + offset)
    xz[..., offset:offset + d], xz[..., offset + d:] = low["x"].float(), low["z"].float()
    pr = torch.zeros(nb, T, offset + d + 32)
    pr[..., offset:offset + d], pr[..., offset + d:offset + d + 16], pr[..., offset + d + 16:] = low["dt"].float(), low["B"][:, :, 0].float(), low["C"][:, :, 0].float()
    xz, pr = xz.bfloat16().to(DEV), pr.bfloat16().to(DEV)
    v = put(low)
    cut = lambda t, a, n: t[..., a:a + n].detach().requires_grad_()
    v.update(x=cut(xz, offset, d), z=cut(xz, offset + d, d), dt=cut(pr, offset, d), B=cut(pr, offset + d, 16).unsqueeze(2).detach().requires_grad_(),
             C=cut(pr, offset + d + 16, 16).unsqueeze(2).detach().requires_grad_())
    assert not v["x"].is_contiguous()
    compare(low, ref, dy, dh, True, v=v)


def test_channels_first_and_expanded_inputs():
    """Last dimensions that are not contiguous are copied; one token's B for all of them is read as it is."""
    low, ref, dy, dh = make(12, 2, 50, 16, 16, 1, torch.float32)
    low["B"] = low["B"][:, :1].expand(2, 50, 1, 16)
    ref["B"] = low["B"].double().requires_grad_()
    v = put(low)
    v["B"] = low["B"][:, :1].contiguous().to(DEV).expand(2, 50, 1, 16).detach().requires_grad_()
    v["x"] = low["x"].transpose(1, 2).contiguous().to(DEV).transpose(1, 2).detach().requires_grad_()
    compare(low, ref, dy, dh, True, v=v)


def test_strides_of_dimensions_of_one_and_tokens_far_apart():
    low, ref, dy, dh = make(23, 1, 3, 16, 16, 1, torch.bfloat16)
    v = put(low)
    far = torch.zeros(2 * ((1 << 24) + 8) + 16, dtype=torch.bfloat16, device=DEV).as_strided((1, 3, 16), (0, (1 << 24) + 8, 1))
    far.copy_(low["x"])
    v["x"] = far.detach().requires_grad_()
    v["dt"] = torch.empty(1, dtype=torch.bfloat16, device=DEV).expand(1 << 24).new_zeros(3 * 16).as_strided((1, 3, 16), (5, 16, 1)).copy_(low["dt"]).detach().requires_grad_()
    compare(low, ref, dy, dh, True, v=v)


def test_bf16_parameters_and_mixed_types():
    low, ref, dy, dh = make(13, 1, 70, 16, 16, 1, torch.bfloat16, pdtype=torch.bfloat16)
    compare(low, ref, dy, dh, True)
    v = put(low, False)
    v["dt"] = v["dt"].float()
    y, _ = call(v, True)
    assert y.dtype == torch.bfloat16
    yr, _ = O.scan(*[ref[k] for k in NAMES[:8]], True, ref["h0"])
    m, count = O.scan_magnitudes(*[ref[k] for k in NAMES[:8]], True, ref["h0"])
    close("y", y, yr, m["y"], count)


def test_half_precision_is_computed_in_fp32():
    low, ref, dy, dh = make(14, 1, 40, 16, 16, 1, torch.float16)
    compare(low, ref, dy, dh, True)


def test_extreme_step_sizes():
    """A state that is forgotten at once, one that is kept, and softplus at both ends."""
    low, ref, dy, dh = make(15, 1, 80, 16, 16, 1, torch.float32)
    low["dt"][:, ::3] = -40.0
    low["dt"][:, 1::3] = 60.0
    ref["dt"] = low["dt"].double().requires_grad_()
    compare(low, ref, dy, dh, True)


@pytest.mark.parametrize("d,T", [(20, 11), (20, 100), (8, 3001)])
def test_states_that_decay_at_once(d, T):
    # A = -inf: a state is what its last token adds
    low, ref, dy, dh = make(41 + T, 1, T, d, 8, 1, torch.float32)
    low["A"][:, ::3] = ref["A"].data[:, ::3] = -float("inf")
    v = put(low)
    y, ht = call(v, True)
    yr, hr = O.scan(*[ref[k].detach() for k in NAMES[:8]], True, ref["h0"].detach())
    finite = {k: t.detach().clone() for k, t in ref.items()}
    finite["A"][:, ::3] = -1e30
    m, count = O.scan_magnitudes(*[finite[k].requires_grad_() for k in NAMES[:8]], True, finite["h0"].requires_grad_(), None, dy.double(), dh.double())
    close("y", y, yr, m["y"], count)
    close("ht", ht, hr, m["ht"], count)
    grads = torch.autograd.grad([y, ht], list(v.values()), [dy.to(DEV), dh.to(DEV)])
    assert all(torch.isfinite(t).all() for t in grads) and (grads[2][:, ::3] == 0).all() and (grads[8][:, :, ::3] == 0).all()


def test_inputs_that_are_not_finite_stay_in_their_channel_and_sequence():
    low, _, _, _ = make(16, 2, 70, 16, 16, 1, torch.float32)
    clean, _ = call(put(low, False), True)
    low["x"][0, 10, 3] = float("nan")
    low["x"][0, 20, 5] = float("inf")
    y, _ = call(put(low, False), True)
    other = [i for i in range(16) if i not in (3, 5)]
    assert torch.equal(y[:, :, other], clean[:, :, other]) and torch.equal(y[1], clean[1]) and torch.equal(y[0, :10], clean[0, :10])
    assert torch.isnan(y[0, 10:, 3]).all()


def test_no_tokens():
    low, _, _, _ = make(17, 2, 0, 16, 16, 1, torch.bfloat16)
    v = put(low)
    y, ht = call(v, True)
    assert y.shape == (2, 0, 16) and torch.equal(ht, v["h0"])
    g = torch.autograd.grad(ht.sum(), [v["h0"], v["A"]])
    assert torch.equal(g[0], torch.ones_like(g[0])) and not g[1].any()


def test_a_prompt_in_pieces_is_the_prompt():
    low, ref, _, _ = make(18, 2, 150, 32, 16, 1, torch.float32)
    v = put(low, False)
    y, ht = call(v, True)
    m, count = O.scan_magnitudes(*[ref[k] for k in NAMES[:8]], True, ref["h0"])
    h, ys = v["h0"], []
    for a, b in ((0, 1), (1, 71), (71, 150)):
        part = {k: (t[:, a:b] if k in ("x", "dt", "B", "C", "z") else t) for k, t in v.items()}
        part["h0"] = h
        yp, h = call(part, True)
        ys.append(yp)
    # (either side is within `count` roundings of the definition)
    close("y", torch.cat(ys, 1), y.double().cpu(), m["y"], 2 * count)
    close("ht", h, ht.double().cpu(), m["ht"], 2 * count)


def test_the_same_bits_every_time_and_without_gradients():
    low, _, dy, dh = make(19, 2, 333, 48, 16, 1, torch.bfloat16)
    v = put(low)
    runs = []
    for _ in range(3):
        y, ht = call(v, True)
        runs.append([y.detach(), ht.detach()] + list(torch.autograd.grad([y, ht], [v[k] for k in NAMES], [dy.to(DEV), dh.to(DEV)])))
    for r in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(r, runs[0]))
    with torch.no_grad():
        y, ht = call(v, True)
    assert torch.equal(y, runs[0][0]) and torch.equal(ht, runs[0][1])


def test_gradients_of_one_output_alone():
    low, ref, dy, dh = make(20, 1, 70, 16, 16, 1, torch.float32)
    v = put(low)
    y, ht = call(v, True)
    yr, hr = O.scan(*[ref[k] for k in NAMES[:8]], True, ref["h0"])
    zero = torch.zeros_like(dy), torch.zeros_like(dh)
    for got, want, go, mags in ((y, yr, dy, (dy, zero[1])), (ht, hr, dh, (zero[0], dh))):
        m, count = O.scan_magnitudes(*[ref[k] for k in NAMES[:8]], True, ref["h0"], None, *[t.double() for t in mags])
        for k, a, b in zip(NAMES, torch.autograd.grad(got, [v[k] for k in NAMES], go.to(DEV), retain_graph=True, allow_unused=True),
                           torch.autograd.grad(want, [ref[k] for k in NAMES], go.double(), retain_graph=True, allow_unused=True)):
            close("d" + k, a, torch.zeros_like(ref[k]) if b is None else b, m[k], count)


def test_gradients_against_differences():
    """A directional derivative of the kernel's own outputs: a central difference of step h is off by h^2 / 6 of the third derivative and by the outputs'
    roundings over h; with h = 2^-7 either is far below the bound of 2 %."""
    low, _, dy, _ = make(21, 1, 66, 16, 16, 1, torch.float32)
    v = put(low)
    y, _ = call(v, True)
    w = dy.to(DEV).double()
    grads = torch.autograd.grad(y, [v[k] for k in NAMES], dy.to(DEV))
    for i, k in enumerate(NAMES):
        step = torch.randn(v[k].shape, generator=torch.Generator().manual_seed(i)).to(DEV)
        ends = []
        for s in (2.0 ** -7, -2.0 ** -7):
            moved = {n: t.detach() for n, t in v.items()}
            moved[k] = moved[k] + s * step
            ends.append((call(moved, True)[0].double() * w).sum())
        slope, want = (ends[0] - ends[1]) / 2.0 ** -6, (grads[i].double() * step.double()).sum()
        size = (grads[i].double() * step.double()).norm()
        assert abs(slope - want) <= 2e-2 * max(size, abs(want)), (k, slope.item(), want.item())


def test_another_stream_and_two_calls_at_once():
    low, _, _, _ = make(22, 2, 700, 64, 16, 1, torch.bfloat16)
    v = put(low, False)
    y0, h0 = call(v, True)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            outs.append([call(v, True) for _ in range(4)])
    torch.cuda.synchronize()
    for runs in outs:
        for y, h in runs:
            assert torch.equal(y, y0) and torch.equal(h, h0)


# ---- one token -------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("nb,d,S,G", [(1, 16, 16, 1), (3, 5, 3, 1), (2, 64, 8, 2), (7, 33, 12, 3), (1, 7, 64, 1), (2, 24, 20, 2), (61, 2048, 16, 1), (258, 520, 15, 2)])
def test_step(nb, d, S, G, dtype):
    low, ref, _, _ = make(nb * 10 + d, nb, 1, d, S, G, dtype)
    v = put(low, False)
    yr, hr = O.scan(*[ref[k] for k in NAMES[:8]], True, ref["h0"])
    m, count = O.scan_magnitudes(*[ref[k] for k in NAMES[:8]], True, ref["h0"])
    one = {k: (t[:, 0] if k in ("x", "dt", "B", "C", "z") else t) for k, t in v.items()}
    step = lambda state, **kw: state_space_step(one["x"], one["dt"], one["A"], one["B"], one["C"], state, one["D"], one["z"], dt_bias=one["bias"], dt_softplus=True, **kw)
    before = one["h0"].clone()
    y, h = step(one["h0"])
    assert torch.equal(one["h0"], before) and y.dtype == dtype
    close("y", y, yr[:, 0], m["y"][:, 0], count)
    close("h", h, hr, m["ht"], count)
    y2, h2 = step(before, inplace=True)
    assert h2 is before and torch.equal(h2, h) and torch.equal(y2, y)


def test_step_without_its_optional_inputs_and_of_rows_of_a_wider_tensor():
    low, ref, _, _ = make(31, 4, 1, 32, 16, 1, torch.bfloat16, gate=False, skip=False, bias=False)
    wide = torch.randn(4, 3, 50).bfloat16().to(DEV)
    wide[:, 1, 7:39] = low["x"][:, 0].to(DEV)
    v = put(low, False)
    y, h = state_space_step(wide[:, 1, 7:39], v["dt"][:, 0], v["A"], v["B"][:, 0, 0], v["C"][:, 0, 0], v["h0"], dt_softplus=True)
    yr, hr = O.scan(*[ref[k] for k in NAMES[:8]], True, ref["h0"])
    m, count = O.scan_magnitudes(*[ref[k] for k in NAMES[:8]], True, ref["h0"])
    close("y", y, yr[:, 0], m["y"][:, 0], count)
    close("h", h, hr, m["ht"], count)


def test_step_refuses_gradients():
    low, _, _, _ = make(32, 1, 1, 16, 16, 1, torch.float32)
    v = put(low)
    one = [v["x"][:, 0], v["dt"][:, 0], v["A"], v["B"][:, 0], v["C"][:, 0], v["h0"]]
    y, _ = state_space_step(*one)
    with pytest.raises(NotImplementedError, match="state_space_scan"):
        y.sum().backward()
    with pytest.raises(NotImplementedError, match="for inference"):
        state_space_step(*one, inplace=True)
