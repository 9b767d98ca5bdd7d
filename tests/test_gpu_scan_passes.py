"""The scan's backward pass where the parts of dB and dC are more than one pass keeps: the same sums in the same order, to the bit, as those of the blocks of channels by themselves.

A block of 64 states is four channels.  A call on one block leaves its part as dB and dC: added one after the other in fp32 they have to be the whole call's, whatever its passes are."""
import ctypes

import pytest
import torch

from hdla_hip import _lib, state_space_scan

pytestmark = pytest.mark.gpu
DEV = "cuda"
S, FOUR = 64, 4


def passes(nb, T, d, G, N, packed=False):
    """More than one: the workspace is smaller than all parts."""
    dims = _lib.HdlaScanDims(B=nb, T=T, D=d, S=S, G=G, N=N, dtype=1, A_dtype=1, D_dtype=1, bias_dtype=1, softplus=0, x_row=d, dt_row=d, z_row=d, B_row=G * S, C_row=G * S,
                             cu_seqlens=4096 if packed else None)
    return _lib.load().hdla_scan_workspace_bytes(ctypes.byref(dims)) < d // G // FOUR * 2 * nb * T * G * S * 4


def gradients(v, dy, channels, G, cu=None):
    """Of the channels `channels` (of each group as many) by themselves."""
    cut = {k: v[k][..., channels].contiguous() for k in ("x", "dt", "z", "D")}
    leaves = [t.detach().requires_grad_() for t in (cut["x"], cut["dt"], v["A"][channels].contiguous(), v["B"], v["C"], cut["D"], cut["z"])]
    x, dt, A, B, C, D, z = leaves
    y, _ = state_space_scan(x, dt, A, B, C, D, z, cu_seqlens=cu)
    return torch.autograd.grad(y, leaves, dy[..., channels].contiguous())


def inputs(seed, nb, T, d, G):
    g = torch.Generator(device=DEV).manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=g, device=DEV)
    return dict(x=rn(nb, T, d), dt=0.01 + 0.2 * torch.rand(nb, T, d, generator=g, device=DEV), A=-torch.exp(rn(d, S)), B=rn(nb, T, G, S), C=rn(nb, T, G, S), D=rn(d), z=rn(nb, T, d)), rn(nb, T, d)


def compare(v, dy, G, cu=None):
    d = v["x"].shape[-1]
    every = torch.arange(d, device=DEV)
    whole = gradients(v, dy, every, G, cu)
    sums = None
    for i in range(d // G // FOUR):
        mine = torch.cat([every[g * (d // G) + FOUR * i:][:FOUR] for g in range(G)])
        dx, ddt, _, dB, dC, _, dz = gradients(v, dy, mine, G, cu)
        for name, a, b in (("x", whole[0], dx), ("dt", whole[1], ddt), ("z", whole[6], dz)):
            assert torch.equal(a[..., mine], b), (name, i)
        sums = [dB, dC] if sums is None else [sums[0] + dB, sums[1] + dC]
    assert torch.equal(whole[3], sums[0]) and torch.equal(whole[4], sums[1])
    return whole


def test_many_sequences():
    nb, T, d = 1024, 32, 520
    assert passes(nb, T, d, 1, nb)
    v, dy = inputs(1, nb, T, d, 1)
    compare(v, dy, 1)
    # of one sequence alone the sums over tokens do not depend on how the others are dealt out
    for n in (0, 31, 1023):
        only = torch.zeros_like(dy)
        only[n] = dy[n]
        whole = gradients(v, only, torch.arange(d, device=DEV), 1)
        for i in (0, 1, 64, 65, 66, 129):                                    # (the first and the last blocks of each pass)
            mine = torch.arange(FOUR * i, FOUR * i + FOUR, device=DEV)
            own = gradients(v, only, mine, 1)
            assert torch.equal(whole[2][mine], own[2]) and torch.equal(whole[5][mine], own[5]) and own[2].any() and own[5].any()


def forget(v, starts):
    """Every 128 tokens of a sequence a step that leaves nothing of the state: how it is cut into segments, at multiples of 128 tokens, does not show in any bit."""
    for a, b in starts:
        v["dt"][:, a:b:128] = 1e5
        v["x"][:, a:b:128] *= 1e-5


def test_segments():
    T, d = 33000, 520
    assert passes(1, T, d, 1, 1)
    v, dy = inputs(2, 1, T, d, 1)
    forget(v, [(0, T)])
    whole = compare(v, dy, 1)
    for h in (slice(0, 260), slice(260, 520)):                               # (a half: one pass, whose segments are the same)
        half = gradients(v, dy, torch.arange(d, device=DEV)[h], 1)
        assert torch.equal(whole[2][h], half[2]) and torch.equal(whole[5][h], half[5])


def test_packed_sequences_of_two_groups():
    T, d, table = 33000, 520, [100, 9000, 9000, 30001, 32950]
    assert passes(1, T, d, 2, 4, True)
    v, dy = inputs(3, 1, T, d, 2)
    forget(v, list(zip(table, table[1:])))
    whole = compare(v, dy, 2, torch.tensor(table, device=DEV))
    for t in (whole[0], whole[1], whole[3], whole[4], whole[6]):
        assert not t[:, :100].any() and not t[:, 32950:].any() and t[:, 100:32950].any()
