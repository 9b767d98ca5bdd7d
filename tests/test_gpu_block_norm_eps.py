"""``block_norm`` with eps = 0, where a row that is not there must not be divided by its root: results and every gradient for row counts that leave places of a workgroup without a row."""
import pytest
import torch

from test_gpu_block_norm import BOTH, compare, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,stream", BOTH)
@pytest.mark.parametrize("post", [True, False])
@pytest.mark.parametrize("rows,E", [(1, 64), (3, 64), (5, 64), (8, 64), (1, 520), (3, 520), (5, 7), (1, 1500), (3201, 40)])
def test_no_eps(rows, E, post, dtype, stream):
    compare(*make(rows + E, (rows, E), dtype, stream, post=post), eps=0.0)


def test_one_row_without_eps_as_without_the_rows_beside_it():
    """The gradients of the weights of one row are its own to the bit, whatever eps makes of places without a row."""
    low, ref, dy, dr = make(3, (1, 64), torch.float32, torch.float32, gate=False)
    compare(low, ref, dy, dr, post_norm=True, eps=0.0)
    compare(low, ref, dy, dr, post_norm=True, eps=2.0 ** -149)
