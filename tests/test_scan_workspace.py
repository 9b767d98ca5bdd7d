"""The scan's workspaces stay near the size of what they work for: the sums of dB and dC over channels, whose parts grow with the square of the states, are bounded."""
import ctypes

import pytest

from hdla_hip import _lib

GIB = 1 << 30


def sizes(B, T, D, S, G=1, N=None, packed=False, dtype=0):
    d = _lib.HdlaScanDims(B=B, T=T, D=D, S=S, G=G, N=B if N is None else N, dtype=dtype, A_dtype=1, D_dtype=1, bias_dtype=1, softplus=1, x_row=D, dt_row=D, z_row=D, B_row=G * S,
                          C_row=G * S, cu_seqlens=4096 if packed else None)
    lib = _lib.load()
    return [f(ctypes.byref(d)) for f in (lib.hdla_scan_states_bytes, lib.hdla_scan_fwd_workspace_bytes, lib.hdla_scan_workspace_bytes)]


@pytest.mark.parametrize("B,T,D,S,G,N,packed", [(4, 2048, 4096, 64, 1, 4, False), (16, 2048, 4096, 64, 1, 16, False), (4, 8192, 8192, 64, 1, 4, False), (1, 65536, 4096, 64, 1, 1, False),
                                                (1, 65536, 4096, 33, 8, 1, False), (1, 100001, 8192, 32, 1, 37, True), (1, 1 << 20, 2048, 64, 2, 1000, True), (64, 4096, 1000, 20, 5, 64, False)])
def test_backward(B, T, D, S, G, N, packed):
    rows = B * T
    states, forward, backward = sizes(B, T, D, S, G, N, packed)
    # two GiB of parts of dB and dC, or two of them where one of dB and dC in fp32 is as large; a part of dA, dD and d bias for each of at most 2048 workgroups of a block of channels;
    # the segments' ends, of which no more are made than keep the device busy
    one = 8 * rows * G * S
    assert backward <= max(2 * GIB, 2 * one) + 2 * (4 * rows * D) + GIB, (backward / GIB)
    assert forward <= GIB // 4
    # a state every 32 or 64 tokens, of whole lanes of four states and whole waves of channels
    lanes = 2 if S <= 8 else 4 if S <= 16 else 8 if S <= 32 else 16
    assert states <= G * -(-(D // G) // (64 // lanes)) * 1024 * (rows // 32 + N + 1)


def test_what_fits_is_in_one_piece():
    # 128 blocks of 16 channels, 8192 rows of 16 states twice, fp32; then 16 parts of dA (16), dD and d bias of 4 x 2048 tokens
    assert sizes(4, 2048, 2048, 16)[2] == 128 * 2 * 8192 * 16 * 4 + 4 * 2048 * 18 * 4
