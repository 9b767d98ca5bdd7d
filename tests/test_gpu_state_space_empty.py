"""A batch of no sequences: results of no rows, and gradients of parameters that are zero."""
import pytest
import torch

from hdla_hip import _lib, block_norm, short_conv, short_conv_step, state_space_scan, state_space_step

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(params=[True, False], ids=["native", "python"], autouse=True)
def path(request, monkeypatch):
    if not request.param:
        monkeypatch.setattr(_lib, "_native", _lib._NoNative())


def leaf(*shape, dtype=torch.float32):
    return torch.randn(*shape, device=DEV).to(dtype).requires_grad_()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T", [0, 1, 70])
def test_calls_over_tokens(T, dtype):
    x, w, b, s = leaf(0, T, 16, dtype=dtype), leaf(16, 4), leaf(16), leaf(0, 3, 16, dtype=dtype)
    y, last = short_conv(x, w, b, activation="silu", initial_state=s, output_final_state=True)
    assert y.shape == x.shape and last.shape == s.shape and y.dtype == last.dtype == dtype
    dx, dw, db, ds = torch.autograd.grad([y, last], [x, w, b, s], [y.detach(), last.detach()])
    assert dx.shape == x.shape and ds.shape == s.shape and not dw.any() and not db.any()
    A, B, h0 = leaf(16, 8), leaf(0, T, 2, 8, dtype=dtype), leaf(0, 16, 8)
    y, h = state_space_scan(x, x.detach(), A, B, B.detach(), b, x.detach(), dt_bias=b.detach(), dt_softplus=True, initial_state=h0, output_final_state=True)
    assert y.shape == x.shape and h.shape == h0.shape
    dx, dA, dB, dD, dh = torch.autograd.grad([y, h], [x, A, B, b, h0], [y.detach(), h.detach()])
    assert dx.shape == x.shape and dB.shape == B.shape and dh.shape == h0.shape and not dA.any() and not dD.any()


@pytest.mark.parametrize("inplace", [False, True])
def test_single_tokens(inplace):
    x, w, s = torch.randn(0, 16, device=DEV), torch.randn(16, 4, device=DEV), torch.randn(0, 3, 16, device=DEV)
    y, new = short_conv_step(x, s, w, inplace=inplace)
    assert y.shape == x.shape and new.shape == s.shape and (new is s) == inplace
    A, B, h = torch.randn(16, 8, device=DEV), torch.randn(0, 8, device=DEV), torch.randn(0, 16, 8, device=DEV)
    y, new = state_space_step(x, x, A, B, B, h, inplace=inplace)
    assert y.shape == x.shape and new.shape == h.shape and (new is h) == inplace


def test_norm():
    x, w = leaf(0, 5, 64), leaf(64)
    y, r = block_norm(x, None, w)
    dx, dw = torch.autograd.grad([y, r], [x, w], [y.detach(), r.detach()])
    assert y.shape == r.shape == dx.shape == x.shape and not dw.any()
