"""Batches of no sequences at the C entry points: accepted where nothing is asked of the device, and still refused where batch and sequences disagree."""
import ctypes

from hdla_hip import _lib


def test_dimensions_of_no_sequences():
    lib, by = _lib.load(), ctypes.byref
    conv = dict(B=0, T=4, D=8, W=4, N=0, dtype=0, weight_dtype=0, bias_dtype=0, silu=0, x_batch=32, x_row=8)
    scan = dict(B=0, T=4000, D=8, S=16, G=1, N=0, dtype=0, A_dtype=1, D_dtype=1, bias_dtype=1, softplus=1)
    some = ctypes.c_void_p(4096)
    c, s = _lib.HdlaConvDims(**conv), _lib.HdlaScanDims(**scan)
    assert lib.hdla_short_conv_fwd(by(c), None, some, *[None] * 5) == 0
    assert lib.hdla_scan_fwd(by(s), None, None, some, *[None] * 9, 0, None, 0, None) == 0
    assert lib.hdla_short_conv_workspace_bytes(by(c)) == 16 and lib.hdla_scan_workspace_bytes(by(s)) == 16
    assert lib.hdla_scan_states_bytes(by(s)) == 0 and lib.hdla_scan_fwd_workspace_bytes(by(s)) == 0
    one, first = dict(conv, T=1), dict(scan, T=1)
    assert lib.hdla_short_conv_step(by(_lib.HdlaConvDims(**one)), *[None] * 7) == 0
    assert lib.hdla_scan_step(by(_lib.HdlaScanDims(**first)), *[None] * 12) == 0
    for wrong, rc in ((dict(N=1), -2), (dict(B=2), -2), (dict(B=-1, N=-1), -2), (dict(cu_seqlens=4096), -7)):
        assert lib.hdla_short_conv_fwd(by(_lib.HdlaConvDims(**dict(conv, **wrong))), *[None] * 7) == rc
        assert lib.hdla_scan_fwd(by(_lib.HdlaScanDims(**dict(scan, **wrong))), *[None] * 12, 0, None, 0, None) == rc
