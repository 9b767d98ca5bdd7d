"""What the operators of a state space block refuse, and how: on the CPU, before anything is launched."""
import ctypes
import hashlib
import os
import re

import pytest
import torch

import hdla_hip
from hdla_hip import _lib, block_norm, short_conv, short_conv_step, state_space_scan, state_space_step

HEADER = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "hdla_state_space.h")
# the declarations of each number, without comments and white space: a change of them takes the next number and a line here
DECLARED = {1: "dcb9c70b5ad9866a", 2: "c4ab95f61548d8a0"}


def test_the_number_is_of_these_declarations():
    text = re.sub(r"/\*.*?\*/|//[^\n]*", " ", open(HEADER).read(), flags=re.S)
    number = int(re.search(r"#define HDLA_STATE_SPACE_VERSION (\d+)", text).group(1))
    text = re.sub(r"#define HDLA_STATE_SPACE_VERSION \d+", "", text)
    assert number == max(DECLARED) == _lib.STATE_SPACE_VERSION == _lib.load().hdla_state_space_version()
    assert DECLARED[number] == hashlib.sha256("".join(text.split()).encode()).hexdigest()[:16], "the header declares something else than under this number"


def test_a_library_without_the_operators_is_refused_by_name(monkeypatch):
    monkeypatch.setattr(_lib, "_lib", None)
    monkeypatch.setattr(_lib, "STATE_SPACE_VERSION", _lib.STATE_SPACE_VERSION + 1)
    with pytest.raises(_lib.HdlaError, match="rebuild the library"):
        _lib.load()


def test_exports():
    for name in ("short_conv", "short_conv_step", "state_space_scan", "state_space_step", "block_norm"):
        assert name in hdla_hip.__all__ and callable(getattr(hdla_hip, name))


def r(*s):
    return torch.randn(*s)


@pytest.mark.parametrize("kw,error,match", [
    (dict(x=r(4, 8)), ValueError, "x must be"), (dict(weight=r(9, 4)), ValueError, "weight must be"), (dict(weight=r(8, 5)), NotImplementedError, "5 taps"),
    (dict(weight=r(8, 1)), NotImplementedError, "1 taps"), (dict(bias=r(9)), ValueError, "bias must be"), (dict(activation="relu"), NotImplementedError, "activation"),
    (dict(initial_state=r(2, 4, 8)), ValueError, "initial_state"), (dict(cu_seqlens=torch.tensor([0, 4])), ValueError, "batch size"),
    (dict(x=r(1, 6, 8), cu_seqlens=torch.tensor([0, 4])), ValueError, "end at"), (dict(x=r(1, 6, 8), cu_seqlens=torch.tensor([0, 4, 3, 6])), ValueError, "never decrease"),
    (dict(), _lib.HdlaError, "GPU only")])
def test_short_conv(kw, error, match):
    args = dict(x=r(2, 6, 8), weight=r(8, 4))
    args.update(kw)
    with pytest.raises(error, match=match):
        short_conv(**args)


@pytest.mark.parametrize("kw,error,match", [
    (dict(x=r(2, 1, 8)), ValueError, "x must be"), (dict(state=r(2, 8, 3)), ValueError, "state must be"), (dict(weight=r(8, 6)), NotImplementedError, "taps"),
    (dict(), _lib.HdlaError, "GPU only")])
def test_short_conv_step(kw, error, match):
    args = dict(x=r(2, 8), state=r(2, 3, 8), weight=r(8, 4))
    args.update(kw)
    with pytest.raises(error, match=match):
        short_conv_step(**args)


@pytest.mark.parametrize("kw,error,match", [
    (dict(x=r(6, 8)), ValueError, "x must be"), (dict(dt=r(2, 6, 9)), ValueError, "dt and z"), (dict(z=r(2, 5, 8)), ValueError, "dt and z"),
    (dict(A=r(9, 4)), ValueError, "A must be"), (dict(A=r(8, 65), B=r(2, 6, 65), C=r(2, 6, 65)), NotImplementedError, "65 states"),
    (dict(B=r(2, 6, 5)), ValueError, "B and C"), (dict(B=r(2, 6, 3, 4), C=r(2, 6, 3, 4)), ValueError, "3 groups"), (dict(C=r(2, 6, 2, 4)), ValueError, "B and C"),
    (dict(D=r(4)), ValueError, "D must be"), (dict(dt_bias=r(8, 1)), ValueError, "dt_bias"), (dict(initial_state=r(2, 4, 8)), ValueError, "initial_state"),
    (dict(cu_seqlens=torch.tensor([0, 6])), ValueError, "batch size"), (dict(), _lib.HdlaError, "GPU only")])
def test_state_space_scan(kw, error, match):
    args = dict(x=r(2, 6, 8), dt=r(2, 6, 8), A=r(8, 4), B=r(2, 6, 4), C=r(2, 6, 4))
    args.update(kw)
    with pytest.raises(error, match=match):
        state_space_scan(**args)


@pytest.mark.parametrize("kw,error,match", [
    (dict(x=r(2, 1, 8)), ValueError, "x must be"), (dict(state=r(2, 4, 8)), ValueError, "state must be"), (dict(B=r(2, 3)), ValueError, "B and C"), (dict(), _lib.HdlaError, "GPU only")])
def test_state_space_step(kw, error, match):
    args = dict(x=r(2, 8), dt=r(2, 8), A=r(8, 4), B=r(2, 4), C=r(2, 4), state=r(2, 8, 4))
    args.update(kw)
    with pytest.raises(error, match=match):
        state_space_step(**args)


def test_sizes_that_32_bits_do_not_hold():
    one, many = torch.zeros(1), 2 ** 31
    for shape in ((1, many, 8), (1, 2 ** 32 + 4, 8), (3, 2 ** 30, 8), (many, 1, 8), (1, 2, 2 ** 24 + 8)):
        x, S = one.expand(shape), one.expand(shape[:2] + (4,))
        with pytest.raises(NotImplementedError, match="is not built"):
            short_conv(x, one.expand(shape[-1], 4))
        with pytest.raises(NotImplementedError, match="is not built"):
            state_space_scan(x, x, one.expand(shape[-1], 4), S, S)
    for shape in ((many, 8), (2 ** 32 + 1, 8), (2, 2 ** 24 + 8)):
        x, S = one.expand(shape), one.expand(shape[0], 4)
        with pytest.raises(NotImplementedError, match="is not built"):
            short_conv_step(x, one.expand(shape[0], 3, shape[1]), one.expand(shape[1], 4))
        with pytest.raises(NotImplementedError, match="is not built"):
            state_space_step(x, x, one.expand(shape[1], 4), S, S, one.expand(shape + (4,)))


@pytest.mark.parametrize("kw,error,match", [
    (dict(x=r(3, 4097), residual=None), NotImplementedError, "4097 channels"), (dict(residual=r(3, 7)), ValueError, "residual"), (dict(gate=r(8)), ValueError, "gate"),
    (dict(weight=r(3, 8)), ValueError, "weight must be"), (dict(post_weight=r(7)), ValueError, "post_weight"), (dict(residual_scale=r(1)), ValueError, "residual_scale"),
    (dict(gate_act="tanh"), NotImplementedError, "gate_act"), (dict(x=torch.tensor(1.0), residual=None), ValueError, "x must be"), (dict(), _lib.HdlaError, "GPU only")])
def test_block_norm(kw, error, match):
    args = dict(x=r(3, 8), residual=r(3, 8))
    args.update(kw)
    with pytest.raises(error, match=match):
        block_norm(**args)


def test_c_entry_points_answer_wrong_dimensions_with_codes():
    lib, by = _lib.load(), ctypes.byref
    conv = dict(B=1, T=4, D=8, W=4, N=1, dtype=0, weight_dtype=0, bias_dtype=0, silu=0, x_batch=32, x_row=8)
    assert lib.hdla_short_conv_workspace_bytes(by(_lib.HdlaConvDims(**conv))) > 0
    for wrong, rc in ((dict(W=5), -2), (dict(W=1), -2), (dict(D=0), -2), (dict(dtype=7), -4), (dict(N=2), -7), (dict(T=-1), -2)):
        d = _lib.HdlaConvDims(**dict(conv, **wrong))
        assert lib.hdla_short_conv_workspace_bytes(by(d)) == 0
        assert lib.hdla_short_conv_fwd(by(d), *[None] * 7) == rc
        assert lib.hdla_short_conv_step(by(d), *[None] * 7) == rc
        assert lib.hdla_short_conv_bwd(by(d), *[None] * 11, 0, None) == rc
    assert lib.hdla_short_conv_fwd(by(_lib.HdlaConvDims(**conv)), *[None] * 7) == -1 and lib.hdla_short_conv_fwd(None, *[None] * 7) == -1
    scan = dict(B=1, T=4, D=8, S=16, G=1, N=1, dtype=0, A_dtype=1, D_dtype=1, bias_dtype=1, softplus=1)
    assert lib.hdla_scan_workspace_bytes(by(_lib.HdlaScanDims(**scan))) > 0 and lib.hdla_scan_states_bytes(by(_lib.HdlaScanDims(**scan))) > 0
    for wrong, rc in ((dict(S=65), -2), (dict(S=0), -2), (dict(G=3), -2), (dict(A_dtype=9), -4), (dict(N=3), -7), (dict(B=0), -2)):
        d = _lib.HdlaScanDims(**dict(scan, **wrong))
        assert lib.hdla_scan_workspace_bytes(by(d)) == 0 and lib.hdla_scan_states_bytes(by(d)) == 0
        assert lib.hdla_scan_fwd(by(d), *[None] * 12, 0, None, 0, None) == rc
        assert lib.hdla_scan_bwd(by(d), *[None] * 11, 0, *[None] * 10, 0, None) == rc
        assert lib.hdla_scan_step(by(d), *[None] * 12) == rc
    assert lib.hdla_scan_step(by(_lib.HdlaScanDims(**scan)), *[None] * 12) == -2              # one token
    assert lib.hdla_scan_fwd(by(_lib.HdlaScanDims(**dict(scan, T=0))), *[None] * 12, 0, None, 0, None) == -1      # A is read where there are no tokens, too
    norm = dict(rows=4, E=8, dtype=0, residual_dtype=0, weight_dtype=1, post_dtype=1, scale_dtype=1, act=1, post_norm=1, factor=1.0, eps=1e-5)
    assert lib.hdla_block_norm_workspace_bytes(by(_lib.HdlaBlockNormDims(**norm))) > 0
    for wrong, rc in ((dict(E=4097), -2), (dict(E=0), -2), (dict(act=3), -2), (dict(dtype=1), -4), (dict(rows=-1), -2), (dict(eps=float("nan")), -2)):
        d = _lib.HdlaBlockNormDims(**dict(norm, **wrong))
        assert lib.hdla_block_norm_workspace_bytes(by(d)) == 0
        assert lib.hdla_block_norm_fwd(by(d), *[None] * 9) == rc
        assert lib.hdla_block_norm_bwd(by(d), *[None] * 15, 0, None) == rc


def test_c_entry_points_answer_small_and_misaligned_buffers_with_codes():
    lib, by = _lib.load(), ctypes.byref
    p = lambda a: ctypes.c_void_p(a)
    scan = _lib.HdlaScanDims(B=1, T=100, D=8, S=16, G=1, N=1, dtype=0, A_dtype=1, D_dtype=1, bias_dtype=1, softplus=1)
    ok = p(4096)
    args = lambda y, states, n: [ok] * 5 + [None] * 4 + [y, None, states, n, None, 0, None]
    assert lib.hdla_scan_fwd(by(scan), *args(p(4100), None, 0)) == -6
    assert lib.hdla_scan_fwd(by(scan), *args(ok, ok, 16)) == -5
    assert lib.hdla_scan_bwd(by(scan), *[ok] * 11, 1 << 40, *[ok] * 10, 16, None) == -5
    conv = _lib.HdlaConvDims(B=1, T=4, D=8, W=4, N=1, dtype=0, weight_dtype=0, bias_dtype=0, silu=0, x_batch=32, x_row=8)
    assert lib.hdla_short_conv_fwd(by(conv), ok, ok, None, p(4098), ok, None, None) == -6
    assert lib.hdla_short_conv_bwd(by(conv), ok, ok, None, None, ok, None, ok, ok, None, None, ok, 4, None) == -5
    norm = _lib.HdlaBlockNormDims(rows=4, E=8, dtype=0, residual_dtype=0, weight_dtype=1, post_dtype=1, scale_dtype=1, act=1, post_norm=1, factor=1.0, eps=1e-5)
    assert lib.hdla_block_norm_fwd(by(norm), p(4104), *[ok] * 7, None) == -6
    assert lib.hdla_block_norm_bwd(by(norm), *[ok] * 14, ok, 4, None) == -5
