"""A whole block in fp32 against its definition in 64 bits, as near as the definition itself comes when it is evaluated in fp32.

Both are fp32 evaluations of one formula, in other orders and with other forms of the exponential, the reciprocal and the root.  An operation of ours has up to four roundings where the plain
one has one or two (state_space_oracle.scan_bounds counts them), and the shorter sums lose less: a norm of errors of eight times the plain one's is more than either allows.  Results that the
plain form happens to hit are given four roundings.  An operand rounded to bf16 is off by 2^-9, a hundred times that: shown of the definition, without a GPU."""
import pytest
import torch

from state_space_util import U
from test_gpu_state_space_block import DEV, E, definition, ours, parameters

CU = [None, [0, 13, 14, 60]]


def given(cu):
    p = parameters(11, torch.float32)
    g = torch.Generator().manual_seed(12)
    h = torch.randn(1 if cu else 2, 60, E, generator=g)
    return p, h, [torch.randn(h.shape, generator=g) for _ in range(2)]


def evaluated(p, h, go, cu, dtype):
    q, hq = {k: v.to(dtype).requires_grad_() for k, v in p.items()}, h.to(dtype).requires_grad_()
    out = definition(q, hq, cu)
    return [t.double() for t in list(out) + list(torch.autograd.grad(out, [hq] + list(q.values()), [t.to(dtype) for t in go]))]


def allowed(p, h, go, cu):
    """Names, the definition in 64 bits, and how far from it a result may be in norm."""
    want, plain = evaluated(p, h, go, cu, torch.float64), evaluated(p, h, go, cu, torch.float32)
    return ["y", "r", "dh"] + ["d" + k for k in p], want, [8 * max((a - b).norm(), 4 * U * b.norm()) for a, b in zip(plain, want)]


@pytest.mark.gpu
@pytest.mark.parametrize("cu", CU)
def test_a_block_and_its_gradients(cu):
    p, h, go = given(cu)
    q, hq = {k: v.to(DEV).requires_grad_() for k, v in p.items()}, h.to(DEV).requires_grad_()
    y, r, _ = ours(q, hq, cu=None if cu is None else torch.tensor(cu))
    got = [y, r] + list(torch.autograd.grad([y, r], [hq] + list(q.values()), [t.to(DEV) for t in go]))
    names, want, most = allowed(p, h, go, cu)
    for name, a, b, m in zip(names, got, want, most):
        off = (a.detach().cpu().double() - b.detach()).norm()
        assert off <= m, (name, (off / b.norm()).item(), (m / b.norm()).item())


@pytest.mark.parametrize("wrong", ["conv_w", "A", "skip", "scale", "w_x", "post"])
@pytest.mark.parametrize("cu", CU)
def test_what_an_operand_in_16_bits_does(cu, wrong):
    p, h, go = given(cu)
    names, want, most = allowed(p, h, go, cu)
    low = evaluated(dict(p, **{wrong: p[wrong].bfloat16().float()}), h, go, cu, torch.float64)
    seen = [n for n, a, b, m in zip(names, low, want, most) if (a - b).norm() > m]
    assert {"y", "r", "dh"} <= set(seen), (wrong, seen)
