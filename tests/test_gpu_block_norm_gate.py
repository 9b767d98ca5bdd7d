"""Gates that are wide open or shut: the gate's gradient is small there, and as exact as anywhere."""
import pytest
import torch

from state_space_util import rounded
from test_gpu_block_norm import BOTH, compare, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("act", ["sigmoid", "silu"])
@pytest.mark.parametrize("dtype,stream", BOTH)
@pytest.mark.parametrize("size", [4.0, 20.0, 60.0])
def test_gradient_of_saturated_gates(size, dtype, stream, act):
    low, ref, dy, dr = make(71, (9, 264), dtype, stream)
    low["gate"], ref["gate"] = rounded(size * (2 * torch.rand(9, 264, generator=torch.Generator().manual_seed(72)) - 1), dtype)
    compare(low, ref, dy, dr, act=act)
