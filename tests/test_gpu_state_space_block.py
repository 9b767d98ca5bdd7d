"""The operators of a state space block as they are used together: a block with its norms, trained, prompted and stepped; captured in graphs; through the native
host path and through the Python code."""
import pytest
import torch

from hdla_hip import _lib, block_norm, short_conv, short_conv_step, state_space_scan, state_space_step
from oracle import state_space_oracle as O
from state_space_util import U

pytestmark = pytest.mark.gpu
DEV = "cuda"
E, D, S, R, W = 48, 96, 16, 6, 4


def parameters(seed, dtype):
    g = torch.Generator().manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=g)
    p = dict(w_in=rn(2 * D, E) / E ** 0.5, conv_w=rn(D, W) / 2, conv_b=0.1 * rn(D), w_x=rn(R + 2 * S, D) / D ** 0.5, w_dt=rn(D, R) / R ** 0.5, dt_b=rn(D) - 2,
             A=-torch.exp(0.3 * rn(D, S)), skip=1 + 0.1 * rn(D), w_out=rn(E, D) / D ** 0.5, pre=1 + 0.1 * rn(E), post=1 + 0.1 * rn(E), scale=0.5 + 0.1 * rn(E), w_gate=rn(E, E) / E ** 0.5)
    return {k: v.to(torch.float32 if k in ("A", "dt_b", "skip", "pre", "post", "scale") else dtype) for k, v in p.items()}


def mixer(p, n, conv, scan):
    """norm's output -> what the block gives; conv and scan take what is between the projections."""
    xz = n @ p["w_in"].t()
    x, z = xz[..., :D], xz[..., D:]
    x = conv(x)
    pr = x @ p["w_x"].t()
    return scan(x, pr[..., :R] @ p["w_dt"].t(), pr[..., R:R + S], pr[..., R + S:], z) @ p["w_out"].t()


def ours(p, h, states=None, cu=None):
    """A block over [B, T, E]; returns what the next one reads, the stream, and the states."""
    left = {}
    n, h = block_norm(h, None, p["pre"])

    def conv(x):
        y, left["conv"] = short_conv(x, p["conv_w"], p["conv_b"], activation="silu", initial_state=None if states is None else states["conv"], output_final_state=True, cu_seqlens=cu)
        return y

    def scan(x, dt, B, C, z):
        y, left["scan"] = state_space_scan(x, dt, p["A"], B, C, p["skip"], z, dt_bias=p["dt_b"], dt_softplus=True,
                                           initial_state=None if states is None else states["scan"], output_final_state=True, cu_seqlens=cu)
        return y

    o = mixer(p, n, conv, scan)
    y, r = block_norm(o, h, p["pre"], post_weight=p["post"], gate=n @ p["w_gate"].t(), residual_scale=p["scale"])
    return y, r, left


def step(p, h, states, inplace=False):
    """The same for one token [B, E]."""
    new = {}
    n, h = block_norm(h, None, p["pre"])

    def conv(x):
        y, new["conv"] = short_conv_step(x, states["conv"], p["conv_w"], p["conv_b"], activation="silu", inplace=inplace)
        return y

    def scan(x, dt, B, C, z):
        y, new["scan"] = state_space_step(x, dt, p["A"], B, C, states["scan"], p["skip"], z, dt_bias=p["dt_b"], dt_softplus=True, inplace=inplace)
        return y

    o = mixer(p, n, conv, scan)
    y, r = block_norm(o, h, p["pre"], post_weight=p["post"], gate=n @ p["w_gate"].t(), residual_scale=p["scale"])
    return y, r, new


def definition(p, h, cu=None):
    n, h = O.block_norm(h, None, p["pre"])
    o = mixer(p, n, lambda x: O.short_conv(x, p["conv_w"], p["conv_b"], None, True, cu)[0],
              lambda x, dt, B, C, z: O.scan(x, dt, p["A"], B.unsqueeze(2), C.unsqueeze(2), p["skip"], z, p["dt_b"], True, None, cu)[0])
    return O.block_norm(o, h, p["pre"], post_weight=p["post"], gate=n @ p["w_gate"].t(), scale=p["scale"])


@pytest.mark.parametrize("cu", [None, [0, 13, 14, 60]])
def test_a_block_and_its_gradients(cu):
    """fp32: a chain of some twelve operations, none of which takes more than E + D + T roundings of sums whose terms are at most a hundred times their result."""
    p = parameters(1, torch.float32)
    g = torch.Generator().manual_seed(2)
    h = torch.randn(1 if cu else 2, 60, E, generator=g)
    go = [torch.randn(h.shape, generator=g) for _ in range(2)]
    ref = {k: v.double().requires_grad_() for k, v in p.items()}
    hr = h.double().requires_grad_()
    want = definition(ref, hr, cu)
    wg = torch.autograd.grad(want, [hr] + list(ref.values()), [t.double() for t in go])
    q = {k: v.to(DEV).requires_grad_() for k, v in p.items()}
    hq = h.to(DEV).requires_grad_()
    y, r, _ = ours(q, hq, cu=None if cu is None else torch.tensor(cu))
    gg = torch.autograd.grad([y, r], [hq] + list(q.values()), [t.to(DEV) for t in go])
    bound = 12 * (E + D + 60) * 100 * U
    for name, a, b in [("y", y, want[0]), ("r", r, want[1])] + list(zip(["h"] + list(p), gg, wg)):
        off = (a.detach().cpu().double() - b.detach()).norm() / b.detach().norm()
        assert off <= bound, (name, off.item(), bound)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_prompt_then_tokens_is_the_whole_sequence(dtype):
    """The states of a prompt go on in single steps.  fp32: either way within the bound above of the definition; bf16: a value that one way rounds up and the other down is a step apart
    at each of the seven places where a tensor is rounded, and what a step is of the whole is at most eps."""
    p = {k: v.to(DEV) for k, v in parameters(3, dtype).items()}
    h = torch.randn(3, 40, E, generator=torch.Generator().manual_seed(4)).to(dtype).to(DEV)
    with torch.no_grad():
        y, r, last = ours(p, h)
        yp, _, states = ours(p, h[:, :33])
        outs = [yp]
        for t in range(33, 40):
            yt, rt, states = step(p, h[:, t].contiguous(), states)
            outs.append(yt[:, None])
    bound = 2 * 12 * (E + D + 40) * 100 * U if dtype == torch.float32 else 7 * torch.finfo(dtype).eps
    for a, b in ((torch.cat(outs, 1), y), (rt, r[:, -1]), (states["conv"], last["conv"]), (states["scan"], last["scan"])):
        assert (a.double() - b.double()).norm() <= bound * b.double().norm()


def test_decode_steps_in_a_graph_carry_the_states_in_place():
    p = {k: v.to(DEV) for k, v in parameters(5, torch.bfloat16).items()}
    x = torch.zeros(4, E, dtype=torch.bfloat16, device=DEV)
    states = dict(conv=torch.zeros(4, W - 1, D, dtype=torch.bfloat16, device=DEV), scan=torch.zeros(4, D, S, device=DEV))
    other = {k: v.clone() for k, v in states.items()}
    with torch.no_grad():
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            step(p, x, states, True)
        torch.cuda.current_stream().wait_stream(s)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y, r, new = step(p, x, states, True)
        assert new["conv"] is states["conv"] and new["scan"] is states["scan"]
        for v in states.values():
            v.zero_()
        for i in range(5):
            x.copy_(torch.randn(4, E, generator=torch.Generator().manual_seed(i)))
            graph.replay()
            torch.cuda.synchronize()
            want = step(p, x, other)
            other = want[2]
            assert torch.equal(y, want[0]) and torch.equal(r, want[1]), i
            assert all(torch.equal(states[k], other[k]) for k in states), i


@pytest.mark.parametrize("T,d,cu", [(90, 64, None), (1500, 16, None), (1200, 16, [0, 500, 501, 1200])])
def test_forward_and_backward_replay(T, d, cu):
    """Scan (long ones in segments), convolution and norm captured with their backward passes: every replay gives the eager call's bits."""
    table = None if cu is None else torch.tensor(cu, device=DEV)
    N = 1 if cu is None else len(cu) - 1
    def fresh(i):
        g = torch.Generator().manual_seed(100 + i)
        rn = lambda *s: torch.randn(*s, generator=g)
        low = [rn(1, T, d), rn(1, T, d) - 2, rn(1, T, S), rn(1, T, S), rn(1, T, d), rn(d, W), rn(1, T, d)]
        return [t.bfloat16().to(DEV) for t in low] + [t.to(DEV) for t in (-torch.exp(rn(d, S)), rn(d), rn(N, d, S), 1 + 0.1 * rn(d))]

    def run(x, dt, B, C, z, w, dy, A, skip, h0, norm):
        leaves = [t.detach().requires_grad_() for t in (x, dt, B, C, z, w, A, skip, h0, norm)]
        x, dt, B, C, z, w, A, skip, h0, norm = leaves
        u, _ = short_conv(x, w, activation="silu", cu_seqlens=table)
        y, ht = state_space_scan(u, dt, A, B, C, skip, z, dt_softplus=True, initial_state=h0, output_final_state=True, cu_seqlens=table)
        o, r = block_norm(y, x, norm, gate=z, residual_scale=skip)
        return [o.detach(), r.detach(), ht.detach()] + list(torch.autograd.grad([o, r, ht], leaves, [dy, dy, torch.ones_like(ht)]))

    static = fresh(99)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(2):
            run(*static)
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(*static)
    for i in range(4):
        new = fresh(i)
        for a, b in zip(static, new):
            a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        want = run(*new)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), i


def test_the_python_code_gives_the_same_bits(monkeypatch):
    p = {k: v.to(DEV).requires_grad_() for k, v in parameters(6, torch.bfloat16).items()}
    h = torch.randn(2, 70, E, generator=torch.Generator().manual_seed(7)).bfloat16().to(DEV)
    results = []
    for native in (True, False):
        if not native:
            monkeypatch.setattr(_lib, "_native", _lib._NoNative())
        hq = h.detach().requires_grad_()
        y, r, last = ours(p, hq)
        grads = torch.autograd.grad([y, r, last["scan"]], [hq] + list(p.values()), [torch.ones_like(y), torch.ones_like(r), torch.ones_like(last["scan"])])
        with torch.no_grad():
            ys, rs, new = step(p, h[:, 0].contiguous(), {k: v.detach() for k, v in last.items()})
        results.append([y, r, last["conv"], last["scan"], ys, rs, new["conv"], new["scan"]] + list(grads))
    assert all(torch.equal(a, b) for a, b in zip(*results))


@pytest.mark.parametrize("native", [True, False])
def test_differentiating_twice_is_refused(native, monkeypatch):
    if not native:
        monkeypatch.setattr(_lib, "_native", _lib._NoNative())
    x = torch.randn(1, 8, 16, device=DEV, requires_grad=True)
    w = torch.randn(16, 4, device=DEV, requires_grad=True)
    for y in (short_conv(x, w)[0], block_norm(x)[0], state_space_scan(x, x, -torch.ones(16, 4, device=DEV), x[..., :4], x[..., :4])[0]):
        g, = torch.autograd.grad(y.square().sum(), x, create_graph=True)
        with pytest.raises(RuntimeError, match="twice"):
            g.sum().backward()


def test_calls_on_two_streams_do_not_meet():
    p = {k: v.to(DEV) for k, v in parameters(8, torch.bfloat16).items()}
    h = torch.randn(2, 300, E, generator=torch.Generator().manual_seed(9)).bfloat16().to(DEV)
    with torch.no_grad():
        want = ours(p, h)
        torch.cuda.synchronize()
        outs = []
        for s in [torch.cuda.Stream() for _ in range(3)]:
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                outs += [ours(p, h) for _ in range(3)]
        torch.cuda.synchronize()
    for y, r, left in outs:
        assert torch.equal(y, want[0]) and torch.equal(r, want[1]) and torch.equal(left["scan"], want[2]["scan"])


@pytest.mark.parametrize("native", [True, False])
def test_a_state_that_a_graph_keeps_is_not_written_over_unnoticed(native, monkeypatch):
    if not native:
        monkeypatch.setattr(_lib, "_native", _lib._NoNative())
    g = torch.Generator().manual_seed(5)
    rn = lambda *s: torch.randn(*s, generator=g).to(DEV)
    x, w, A, B = rn(2, 9, 16).requires_grad_(), rn(16, 4), -torch.exp(rn(16, 8)), rn(2, 9, 8)
    near, far = rn(2, 3, 16), rn(2, 16, 8)
    y, _ = short_conv(x, w, initial_state=near)
    short_conv_step(rn(2, 16), near, w, inplace=True)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    out = []
    for write in (False, True):                           # (of the scan's state the backward pass needs nothing)
        v = x.detach().requires_grad_()
        y, _ = state_space_scan(v, v, A, B, B, dt_softplus=True, initial_state=far)
        if write:
            before = far._version
            state_space_step(rn(2, 16), rn(2, 16), A, B[:, 0], B[:, 0], far, inplace=True)
            assert far._version > before
        out.append(torch.autograd.grad(y.sum(), v)[0])
    assert torch.equal(*out)
    with torch.inference_mode():                          # (whose tensors no graph keeps)
        near = rn(2, 3, 16)
        short_conv_step(rn(2, 16), near, w, inplace=True)
    torch.cuda.synchronize()


def test_offsets_past_32_bits():
    # 2^31 elements and more, of which the last rows are compared with a call on these alone; a convolution's and a norm's bits do not depend on the rest
    T, d, tail = 2 ** 22 + 77, 512, 300
    g = torch.Generator(device=DEV).manual_seed(12)
    rn = lambda *s: torch.randn(*s, generator=g, device=DEV, dtype=torch.bfloat16)
    x = rn(1, T, d)
    assert x.numel() > 2 ** 31
    end = lambda t: t[:, T - tail:].contiguous()
    w, b = rn(d, 4), rn(d)
    xe = x.detach().requires_grad_()
    y, _ = short_conv(xe, w, b, activation="silu")
    dx, = torch.autograd.grad(y, xe, x)
    ye, _ = short_conv(end(x), w, b, activation="silu", initial_state=x[:, T - tail - 3:T - tail].contiguous())
    assert torch.equal(y[:, T - tail:].detach(), ye)
    xs = x[:, T - tail - 3:].contiguous().requires_grad_()
    ds, = torch.autograd.grad(short_conv(xs, w, b, activation="silu")[0], xs, x[:, T - tail - 3:].contiguous())
    assert torch.equal(dx[:, T - tail:], ds[:, 3:])
    del y, dx, ds

    n, r = block_norm(x, x, w[:, 0].contiguous(), post_norm=True, gate=x)
    ne, re = block_norm(end(x), end(x), w[:, 0].contiguous(), post_norm=True, gate=end(x))
    assert torch.equal(n[:, T - tail:], ne) and torch.equal(r[:, T - tail:], re)
    del n, r

    # half a step of each side's rounding to bf16, and of sums whose terms' absolute values stay below 2^10 some 2^7 roundings of 2^-24
    close = lambda a, b: ((a.double() - b.double()).abs() <= 2.0 ** -8 * (a.double().abs() + b.double().abs()) + 2.0 ** -7).all()
    A, BC = -0.5 - torch.rand(d, 4, generator=g, device=DEV), rn(1, T, 4)
    grads = lambda x, BC, h0: torch.autograd.grad(state_space_scan(x, x.detach(), A, BC, BC, dt_softplus=True, initial_state=h0)[0], x, x.detach())[0]
    _, h = state_space_scan(x[:, :T - tail], x[:, :T - tail], A, BC[:, :T - tail], BC[:, :T - tail], dt_softplus=True, output_final_state=True)
    y, hT = state_space_scan(x, x, A, BC, BC, dt_softplus=True, output_final_state=True)
    ye, he = state_space_scan(end(x), end(x), A, end(BC), end(BC), dt_softplus=True, initial_state=h, output_final_state=True)
    assert close(y[:, T - tail:], ye) and close(hT, he)
    del y
    assert close(grads(xe, BC, None)[:, T - tail:], grads(end(x).requires_grad_(), end(BC), h))
