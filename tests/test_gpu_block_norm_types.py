"""A gate of another type than what it opens: it is not rounded to x's type on the way in, and results are rounded once."""
import pytest
import torch

from hdla_hip import block_norm
from state_space_util import rounded
from test_gpu_block_norm import compare, make

pytestmark = pytest.mark.gpu
DEV = "cuda"
MIXED = [(torch.bfloat16, torch.float32), (torch.bfloat16, torch.float16), (torch.float32, torch.bfloat16), (torch.float16, torch.float32), (torch.float16, torch.bfloat16)]


@pytest.mark.parametrize("act", ["sigmoid", "silu", None])
@pytest.mark.parametrize("stream", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dtype,other", MIXED)
def test_gate_of_another_type(dtype, other, stream, act):
    low, ref, dy, dr = make(21, (7, 136), dtype, stream)
    low["gate"], ref["gate"] = rounded(3 * torch.randn(7, 136, generator=torch.Generator().manual_seed(22)), other)
    compare(low, ref, dy, dr, act=act)


def test_a_gate_is_not_rounded():
    """x is a power of two and the gate multiplies as it is: the stream in fp32 is the gate to the bit."""
    x = torch.full((3, 64), 2.0, dtype=torch.bfloat16, device=DEV)
    gate = torch.randn(3, 64, device=DEV)
    _, r = block_norm(x, torch.zeros(3, 64, device=DEV), gate=gate, gate_act=None, residual_scale=0.5)
    assert r.dtype == torch.float32 and torch.equal(r, gate)
