"""The norms around a block with gate and residual against their definition in 64 bits: outputs and every gradient."""
import pytest
import torch

from hdla_hip import block_norm
from oracle import state_space_oracle as O
from state_space_util import close, rounded

pytestmark = pytest.mark.gpu
DEV = "cuda"
NAMES = ("x", "residual", "weight", "post_weight", "gate", "scale")


def make(seed, shape, dtype, stream, residual=True, weight=True, post=True, gate=True, scale=True, pdtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=g)
    E = shape[-1]
    raw = dict(x=(rn(*shape), dtype), residual=(2 * rn(*shape), stream) if residual else None, weight=(1 + 0.2 * rn(E), pdtype) if weight else None,
               post_weight=(1 + 0.2 * rn(E), pdtype) if post else None, gate=(rn(*shape), dtype) if gate else None, scale=(rn(E), pdtype) if scale else None)
    low, ref = {}, {}
    for k, t in raw.items():
        low[k], ref[k] = (None, None) if t is None else rounded(*t)
    return low, ref, rn(*shape).to(dtype), rn(*shape).to(stream if residual else dtype)


def compare(low, ref, dy, dr, act="sigmoid", post_norm=False, factor=0.7, eps=1e-5, v=None):
    v = {k: None if t is None else t.to(DEV).requires_grad_() for k, t in low.items()} if v is None else v
    s = factor if ref["scale"] is None else ref["scale"]
    kw = dict(residual=ref["residual"], weight=ref["weight"], post_norm=post_norm, post_weight=ref["post_weight"], gate=ref["gate"], act=act, scale=s, eps=eps)
    y, r = block_norm(v["x"], v["residual"], v["weight"], post_norm=post_norm, post_weight=v["post_weight"], gate=v["gate"], gate_act=act,
                      residual_scale=factor if v["scale"] is None else v["scale"], eps=eps)
    yr, rr = O.block_norm(ref["x"], **kw)
    m, count = O.block_norm_magnitudes(ref["x"], **kw, dy=dy, dr=dr)
    assert y.dtype == low["x"].dtype and r.dtype == dr.dtype
    close("y", y, yr, m["y"], count)
    close("r", r, rr, m["r"], count)
    names = [k for k in NAMES if ref[k] is not None]
    got = torch.autograd.grad([y, r], [v[k] for k in names], [dy.to(DEV), dr.to(DEV)])
    want = torch.autograd.grad([yr, rr], [ref[k] for k in names], [dy.double(), dr.double()])
    for k, a, b in zip(names, got, want):
        assert a.dtype == low[k].dtype, k
        close("d" + k, a, b, m[k], count)


BOTH = [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32)]


@pytest.mark.parametrize("dtype,stream", BOTH)
@pytest.mark.parametrize("rows,E", [(1, 1), (3, 7), (5, 8), (1, 64), (9, 100), (4, 256), (6, 260), (2, 512), (7, 513), (130, 520), (3, 1024), (2, 1025), (4, 2048), (2, 2056), (1, 4095),
                                    (3, 4096)])
def test_norms_and_gradients(rows, E, dtype, stream):
    compare(*make(rows * E, (rows, E), dtype, stream))


@pytest.mark.parametrize("residual,weight,post,gate,scale,post_norm", [(True, True, False, False, False, False), (False, False, False, False, False, False),
                                                                      (True, True, False, True, False, True), (False, True, True, False, True, False),
                                                                      (True, False, False, False, True, True)])
def test_what_may_be_left_out(residual, weight, post, gate, scale, post_norm):
    compare(*make(5, (2, 9, 136), torch.bfloat16, torch.bfloat16, residual, weight, post, gate, scale), post_norm=post_norm)


@pytest.mark.parametrize("act", ["sigmoid", "silu", None])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gates(act, dtype):
    compare(*make(6, (11, 96), dtype, dtype), act=act)


def test_more_rows_than_workgroups():
    compare(*make(7, (4 * 1024 + 37, 40), torch.float32, torch.float32))
    compare(*make(8, (1100, 520), torch.bfloat16, torch.bfloat16))


def test_other_types_orders_and_addresses():
    low, ref, dy, dr = make(9, (6, 72), torch.bfloat16, torch.bfloat16, pdtype=torch.bfloat16)
    compare(low, ref, dy, dr)
    v = {k: t.to(DEV).requires_grad_() for k, t in low.items()}
    v["x"] = low["x"].t().contiguous().to(DEV).t().detach().requires_grad_()
    shifted = torch.zeros(6 * 72 + 1, dtype=torch.bfloat16, device=DEV)
    shifted[1:] = low["residual"].flatten().to(DEV)
    v["residual"] = shifted[1:].view(6, 72).detach().requires_grad_()
    compare(low, ref, dy, dr, v=v)
    compare(*make(10, (5, 64), torch.float16, torch.float16))
    compare(*make(11, (5, 64), torch.float16, torch.float32))
    compare(*make(12, (5, 64), torch.float32, torch.bfloat16))


def test_a_row_of_zeros_and_large_values():
    low, ref, dy, dr = make(13, (4, 64), torch.float32, torch.float32)
    for t in (low, ref):
        with torch.no_grad():
            t["x"][1] = 0
            t["residual"][1] = 0
            t["x"][2] *= 1e4
            t["residual"][3] *= 1e4
    compare(low, ref, dy, dr)


def test_rows_do_not_meet():
    low, _, _, _ = make(14, (8, 520), torch.bfloat16, torch.bfloat16)
    v = {k: t.to(DEV) for k, t in low.items()}
    args = lambda v: dict(residual=v["residual"], weight=v["weight"], post_weight=v["post_weight"], gate=v["gate"], residual_scale=v["scale"])
    y0, r0 = block_norm(v["x"], **args(v))
    v["x"][3, 5], v["gate"][5, 1] = float("nan"), float("inf")
    y, r = block_norm(v["x"], **args(v))
    keep = [0, 1, 2, 4, 6, 7]
    assert torch.equal(y[keep], y0[keep]) and torch.equal(r[keep], r0[keep]) and torch.isnan(y[3]).all()


def test_no_rows():
    low, _, _, _ = make(15, (0, 64), torch.bfloat16, torch.bfloat16)
    v = {k: t.to(DEV).requires_grad_() for k, t in low.items()}
    y, r = block_norm(v["x"], v["residual"], v["weight"], post_weight=v["post_weight"], gate=v["gate"], residual_scale=v["scale"])
    g = torch.autograd.grad([y.sum() + r.sum()], [v["weight"], v["scale"], v["x"]])
    assert y.shape == (0, 64) and not g[0].any() and not g[1].any() and g[2].shape == (0, 64)


def test_gradient_of_one_output_alone():
    low, ref, dy, dr = make(16, (9, 128), torch.float32, torch.float32)
    for which in (0, 1):
        v = {k: t.to(DEV).requires_grad_() for k, t in low.items()}
        outs = block_norm(v["x"], v["residual"], v["weight"], post_weight=v["post_weight"], gate=v["gate"], residual_scale=v["scale"])
        want = O.block_norm(ref["x"], ref["residual"], ref["weight"], False, ref["post_weight"], ref["gate"], "sigmoid", ref["scale"])
        go = (dy, dr)[which]
        m, count = O.block_norm_magnitudes(ref["x"], ref["residual"], ref["weight"], False, ref["post_weight"], ref["gate"], "sigmoid", ref["scale"],
                                           dy=dy if which == 0 else None, dr=dr if which else None)
        got = torch.autograd.grad(outs[which], [v[k] for k in NAMES], go.to(DEV), allow_unused=True)
        ref_g = torch.autograd.grad(want[which], [ref[k] for k in NAMES], go.double(), allow_unused=True)
        for k, a, b in zip(NAMES, got, ref_g):
            close("d" + k, a, torch.zeros_like(ref[k]) if b is None else b, m[k], count)


def test_the_same_bits_every_time():
    low, _, dy, dr = make(17, (3000, 264), torch.bfloat16, torch.float32)
    v = {k: t.to(DEV).requires_grad_() for k, t in low.items()}
    runs = []
    for _ in range(3):
        y, r = block_norm(v["x"], v["residual"], v["weight"], post_weight=v["post_weight"], gate=v["gate"], residual_scale=v["scale"])
        runs.append([y, r] + list(torch.autograd.grad([y, r], [v[k] for k in NAMES], [dy.to(DEV), dr.to(DEV)])))
    assert all(torch.equal(a, b) for x in runs[1:] for a, b in zip(x, runs[0]))
