"""The selective state space scan and the short causal convolution in front of it, for prompts and training and for single tokens.

* ``short_conv``         W taps over the tokens of each channel, optionally followed by silu; ``short_conv_step`` for one token
* ``state_space_scan``   ``h_t = exp(delta_t A) h_{t-1} + delta_t x_t B_t``, ``y_t = (C_t . h_t + D x_t) silu(z_t)``; ``state_space_step`` for one token

They stand beside the delta-rule operators: a state per sequence goes in and comes out, packed batches are given by ``cu_seqlens``, gradients of every
input come from one backward call, sums and states are fp32.  x, dt, z, B and C may be views (a projection's output, split): nothing is copied as long as their
last dimension is contiguous.  Tensors must live on the GPU.
"""
import ctypes
from typing import Optional, Tuple

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .chunk import _require_gpu
from .utils import autocast_custom_bwd, autocast_custom_fwd

_NATIVE = (torch.bfloat16, torch.float32)
CONV_WIDTHS, MAX_STATES = (2, 3, 4), 64
ROW_MOST, TOKENS_MOST, COUNT_MOST = 1 << 24, 1 << 30, (1 << 31) - 1


def on_one_gpu(x, *others):
    _require_gpu(x, *others)
    for t in others:
        if t is not None and t.device != x.device:
            raise ValueError(f"all tensors must be on one device, got {x.device} and {t.device}")


def rows(t: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    """A tensor whose last dimension is contiguous and whose tokens are no further apart than the kernels reach: itself, or a copy."""
    if t is None or ((t.shape[-1] == 1 or t.stride(-1) == 1) and step(t, 1) <= ROW_MOST):
        return t
    return t.contiguous()


def step(t, dim):
    """Elements from one index of a dimension to the next, where there is a next."""
    return t.stride(dim) if t.shape[dim] > 1 else 0


def whole(t: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    """A contiguous tensor that starts on 16 bytes: itself, or a copy."""
    if t is None:
        return None
    t = t.contiguous()
    return t.clone() if t.data_ptr() % 16 else t


def param(t: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    return t if t is None or t.dtype in _NATIVE else t.float()


def code(t: Optional[torch.Tensor]) -> int:
    return _lib.HDLA_FP32 if t is None else _lib.dtype_code(t.dtype)


def _sequences(x, cu_seqlens, state, what):
    """Number of sequences, and the table on x's device."""
    if cu_seqlens is None:
        n = x.shape[0]
    else:
        if x.shape[0] != 1:
            raise ValueError(f"The batch size is expected to be 1 rather than {x.shape[0]} when using `cu_seqlens`."
                             f"Please flatten variable-length inputs before processing.")
        _lib.check_cu_seqlens(cu_seqlens, x.shape[1])
        n = cu_seqlens.numel() - 1
        cu_seqlens = cu_seqlens.to(device=x.device, dtype=torch.int64).contiguous()
    if state is not None and tuple(state.shape) != (n,) + what:
        raise ValueError(f"initial_state must be {(n,) + what}, one for each sequence, got {tuple(state.shape)}")
    return n, cu_seqlens


def _within_reach(x, n):
    """The kernels count rows and sequences in 32 bits."""
    tokens = x.shape[1] if x.dim() == 3 else 1
    if tokens > TOKENS_MOST or x.shape[0] * tokens > COUNT_MOST or n > COUNT_MOST or x.shape[-1] > ROW_MOST:
        raise NotImplementedError(f"x {tuple(x.shape)} of {n} sequences is not built: at most 2^30 tokens a sequence, 2^31 - 1 tokens and sequences, 2^24 channels")


def _not_trained(name):
    return NotImplementedError(f"Backward pass for {name} is not implemented: it is for inference. For training, please use "
                               f"`{name.replace('_step', '' if 'conv' in name else '_scan')}`.")


# ---- the short convolution -------------------------------------------------------------------------------------------
def _conv_dims(x, weight, bias, silu, n, cu):
    b, t = (x.shape[0], x.shape[1]) if x.dim() == 3 else (x.shape[0], 1)
    return _lib.HdlaConvDims(b, t, x.shape[-1], weight.shape[1], n, _lib.dtype_code(x.dtype), code(weight), code(bias), int(silu),
                             step(x, 0), step(x, 1) if x.dim() == 3 else 0, None if cu is None else cu.data_ptr())


def _own(dtype, state):
    """What is computed in: x's type if the state has it too, else fp32, which holds what each of them says."""
    return dtype if dtype in _NATIVE and (state is None or state.dtype == dtype) else torch.float32


def _conv_args(x, weight, bias, activation):
    """Checks of what both calls share."""
    if weight.dim() != 2 or weight.shape[0] != x.shape[-1]:
        raise ValueError(f"weight must be [D, W] with D = {x.shape[-1]} channels, got {tuple(weight.shape)}")
    if weight.shape[1] not in CONV_WIDTHS:
        raise NotImplementedError(f"{weight.shape[1]} taps are not built (2, 3 or 4)")
    if bias is not None and tuple(bias.shape) != (x.shape[-1],):
        raise ValueError(f"bias must be [{x.shape[-1]}], got {tuple(bias.shape)}")
    if activation not in (None, "silu", "swish"):
        raise NotImplementedError(f"activation = {activation!r}: None and 'silu' are built")
    return activation is not None


class ShortConvFunction(torch.autograd.Function):
    """What is kept between the passes: the inputs."""

    @staticmethod
    @autocast_custom_fwd
    def forward(ctx, x, weight, bias, state, silu, want_last, n, cu):
        lib = _lib.load()
        with torch.cuda.device(x.device):
            dims = _conv_dims(x, weight, bias, silu, n, cu)
            y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
            last = torch.empty(n, weight.shape[1] - 1, x.shape[-1], dtype=x.dtype, device=x.device) if want_last else None
            _lib.check(lib.hdla_short_conv_fwd(ctypes.byref(dims), _lib.ptr(x), _lib.ptr(weight), _lib.ptr(bias), _lib.ptr(state), _lib.ptr(y),
                                               _lib.ptr(last), _lib.current_stream(x.device)), "hdla_short_conv_fwd")
        ctx.save_for_backward(x, weight, bias, state, cu)
        ctx.cfg = (silu, n)
        ctx.set_materialize_grads(False)
        return y, last

    @staticmethod
    @once_differentiable
    @autocast_custom_bwd
    def backward(ctx, dy, dlast):
        x, weight, bias, state, cu = ctx.saved_tensors
        silu, n = ctx.cfg
        lib = _lib.load()
        with torch.cuda.device(x.device):
            dims = _conv_dims(x, weight, bias, silu, n, cu)
            dy = torch.zeros(x.shape, dtype=x.dtype, device=x.device) if dy is None else whole(dy.to(x.dtype))
            dlast = None if dlast is None else whole(dlast.to(x.dtype))
            dx = torch.empty_like(dy)
            dw, db = torch.empty_like(weight), None if bias is None else torch.empty_like(bias)
            dstate = None if state is None else torch.empty_like(state)
            ws = torch.empty(lib.hdla_short_conv_workspace_bytes(ctypes.byref(dims)), dtype=torch.uint8, device=x.device)
            _lib.check(lib.hdla_short_conv_bwd(ctypes.byref(dims), _lib.ptr(x), _lib.ptr(weight), _lib.ptr(bias), _lib.ptr(state), _lib.ptr(dy), _lib.ptr(dlast),
                                               _lib.ptr(dx), _lib.ptr(dw), _lib.ptr(db), _lib.ptr(dstate), _lib.ptr(ws), ws.numel(),
                                               _lib.current_stream(x.device)), "hdla_short_conv_bwd")
        return dx, dw, db, dstate, None, None, None, None


@torch.compiler.disable
def short_conv(
    x: torch.Tensor,                                  # [B, T, D]
    weight: torch.Tensor,                             # [D, W]
    bias: Optional[torch.Tensor] = None,              # [D]
    *,
    activation: Optional[str] = None,
    initial_state: Optional[torch.Tensor] = None,     # [N, W - 1, D]
    output_final_state: bool = False,
    cu_seqlens: Optional[torch.Tensor] = None,
) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """Causal convolution of each channel over its tokens: ``p_t = bias + sum_j weight[:, j] x_{t-W+1+j}``, ``y_t = p_t`` or
    (``activation="silu"``) ``p_t sigmoid(p_t)``.  W is 2, 3 or 4.

    ``initial_state`` holds the W - 1 inputs before each sequence (zeros without it), the returned ``final_state`` its last W - 1, both oldest first;
    ``cu_seqlens`` packs N sequences into a batch of one.  Returns ``(y, final_state)``, both in x's dtype; an ``initial_state`` of another dtype is
    computed with in fp32."""
    out = _lib.native().short_conv(x, weight, bias, activation, initial_state, output_final_state, cu_seqlens)
    if out is not None:
        return out
    if x.dim() != 3:
        raise ValueError(f"x must be [B, T, D], got {tuple(x.shape)}")
    silu = _conv_args(x, weight, bias, activation)
    n, cu = _sequences(x, cu_seqlens, initial_state, (weight.shape[1] - 1, x.shape[-1]))
    _within_reach(x, n)
    on_one_gpu(x, weight, bias, initial_state)
    out_dtype = x.dtype
    if out_dtype not in _NATIVE + (torch.float16,):
        raise TypeError(f"unsupported dtype {out_dtype}")
    x = x.to(_own(out_dtype, initial_state))
    state = None if initial_state is None else whole(initial_state.to(x.dtype))
    w, b = param(weight).contiguous(), None if bias is None else param(bias).contiguous()
    y, last = ShortConvFunction.apply(rows(x), w, b, state, silu, bool(output_final_state), n, cu)
    return y.to(out_dtype), None if last is None else last.to(out_dtype)


class _Step(torch.autograd.Function):
    """A call whose gradient is refused where it is asked for."""

    @staticmethod
    def forward(ctx, name, fn, *tensors):
        ctx.name = name
        return fn(*(t.detach() if t is not None else None for t in tensors))

    @staticmethod
    def backward(ctx, *grads):
        raise _not_trained(ctx.name)


def _run_step(name, fn, tensors, inplace):
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        if inplace:
            raise _not_trained(name)
        return _Step.apply(name, fn, *tensors)
    return fn(*tensors)


def _written(state):
    """A state that a kernel has written in place: a graph that kept it notices, as with torch's own operations."""
    if state is not None and not state.is_inference():
        torch.autograd.graph.increment_version(state)


def _new_state(state, inplace, dtype):
    """Where the next state goes: the state's own place, which has to be as the kernels want it."""
    if not inplace:
        return None
    if state.dtype != dtype or not state.is_contiguous() or state.data_ptr() % 16:
        raise ValueError(f"a state that is updated in place must be contiguous, 16-byte aligned and {dtype}")
    return state


@torch.compiler.disable
def short_conv_step(
    x: torch.Tensor,                                  # [B, D]
    state: torch.Tensor,                              # [B, W - 1, D]
    weight: torch.Tensor,                             # [D, W]
    bias: Optional[torch.Tensor] = None,              # [D]
    *,
    activation: Optional[str] = None,
    inplace: bool = False,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """``short_conv`` for one token of each sequence: returns ``(y [B, D], new_state)``, both in x's dtype.  ``inplace=True`` writes the new state where
    ``state`` is, as a loop of decode steps or a captured graph wants it: of x's dtype, or fp32.  No gradients."""
    out = _lib.native().short_conv_step(x, state, weight, bias, activation, inplace)
    if out is not None:
        return out
    if x.dim() != 2:
        raise ValueError(f"x must be [B, D], got {tuple(x.shape)}")
    silu = _conv_args(x, weight, bias, activation)
    if tuple(state.shape) != (x.shape[0], weight.shape[1] - 1, x.shape[1]):
        raise ValueError(f"state must be {(x.shape[0], weight.shape[1] - 1, x.shape[1])}, got {tuple(state.shape)}")
    _within_reach(x, x.shape[0])
    on_one_gpu(x, state, weight, bias)
    out_dtype = x.dtype
    if out_dtype not in _NATIVE + (torch.float16,):
        raise TypeError(f"unsupported dtype {out_dtype}")
    own = _own(out_dtype, state)
    to = _new_state(state, inplace, own)

    def call(x, state, weight, bias):
        xs, s = rows(x.to(own)), whole(state.to(own))
        w, b = param(weight).contiguous(), None if bias is None else param(bias).contiguous()
        with torch.cuda.device(x.device):
            dims = _conv_dims(xs, w, b, silu, x.shape[0], None)
            y, new = torch.empty(x.shape, dtype=own, device=x.device), torch.empty_like(s) if to is None else to
            _lib.check(_lib.load().hdla_short_conv_step(ctypes.byref(dims), _lib.ptr(xs), _lib.ptr(w), _lib.ptr(b), _lib.ptr(s), _lib.ptr(y), _lib.ptr(new),
                                                        _lib.current_stream(x.device)), "hdla_short_conv_step")
            _written(to)
        return y.to(out_dtype), new if to is not None else new.to(out_dtype)

    return _run_step("short_conv_step", call, (x, state, weight, bias), inplace)


# ---- the scan --------------------------------------------------------------------------------------------------------
def _scan_dims(x, dt, A, B, C, D, z, bias, softplus, n, cu):
    one = x.dim() == 2
    st = lambda t: (0, 0) if t is None else (step(t, 0), 0 if one else step(t, 1))
    return _lib.HdlaScanDims(x.shape[0], 1 if one else x.shape[1], x.shape[-1], A.shape[1], B.shape[-2], n, _lib.dtype_code(x.dtype), code(A), code(D), code(bias),
                             int(softplus), *st(x), *st(dt), *st(z), *st(B), step(B, -2), *st(C), step(C, -2), None if cu is None else cu.data_ptr())


def _scan_args(x, dt, A, B, C, D, z, dt_bias):
    """Checks of what both calls share; B and C with their groups."""
    d = x.shape[-1]
    if dt.shape != x.shape or (z is not None and z.shape != x.shape):
        raise ValueError(f"dt and z must have the shape of x {tuple(x.shape)}, got {tuple(dt.shape)}" + ("" if z is None else f" and {tuple(z.shape)}"))
    if A.dim() != 2 or A.shape[0] != d or A.shape[1] < 1:
        raise ValueError(f"A must be [D, S] with D = {d} channels, got {tuple(A.shape)}")
    if A.shape[1] > MAX_STATES:
        raise NotImplementedError(f"{A.shape[1]} states a channel are not built (at most {MAX_STATES})")
    lead = tuple(x.shape[:-1])
    if B.dim() == x.dim():
        B = B.unsqueeze(-2)
    if C.dim() == x.dim():
        C = C.unsqueeze(-2)
    if B.shape != C.shape or tuple(B.shape[:-2]) != lead or B.shape[-1] != A.shape[1]:
        raise ValueError(f"B and C must be {lead + ('G', A.shape[1])} or {lead + (A.shape[1],)}, got {tuple(B.shape)} and {tuple(C.shape)}")
    if B.shape[-2] < 1 or d % B.shape[-2]:
        raise ValueError(f"{d} channels do not divide into {B.shape[-2]} groups")
    for name, t in (("D", D), ("dt_bias", dt_bias)):
        if t is not None and tuple(t.shape) != (d,):
            raise ValueError(f"{name} must be [{d}], got {tuple(t.shape)}")
    return B, C


def _common(x, *others):
    """x, dt, B, C and z in one type: x's where all have it, else fp32, which holds what each of them says."""
    if x.dtype not in _NATIVE + (torch.float16,):
        raise TypeError(f"unsupported dtype {x.dtype}")
    if x.dtype in _NATIVE and all(t is None or t.dtype == x.dtype for t in others):
        return (x,) + others
    return tuple(None if t is None else t.float() for t in (x,) + others)


class StateSpaceScanFunction(torch.autograd.Function):
    """What is kept between the passes: the inputs, and the state that enters every 64th token (32nd where there are many sequences and
    channels), fp32."""

    @staticmethod
    @autocast_custom_fwd
    def forward(ctx, x, dt, A, B, C, D, z, bias, h0, softplus, want_ht, n, cu):
        lib = _lib.load()
        with torch.cuda.device(x.device):
            dims = _scan_dims(x, dt, A, B, C, D, z, bias, softplus, n, cu)
            y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
            ht = torch.empty(n, x.shape[-1], A.shape[1], dtype=torch.float32, device=x.device) if want_ht else None
            left = None
            if any(ctx.needs_input_grad):
                left = torch.empty(lib.hdla_scan_states_bytes(ctypes.byref(dims)), dtype=torch.uint8, device=x.device)
            ws = torch.empty(lib.hdla_scan_fwd_workspace_bytes(ctypes.byref(dims)), dtype=torch.uint8, device=x.device)
            _lib.check(lib.hdla_scan_fwd(ctypes.byref(dims), _lib.ptr(x), _lib.ptr(dt), _lib.ptr(A), _lib.ptr(B), _lib.ptr(C), _lib.ptr(D), _lib.ptr(z), _lib.ptr(bias),
                                         _lib.ptr(h0), _lib.ptr(y), _lib.ptr(ht), _lib.ptr(left), 0 if left is None else left.numel(), _lib.ptr(ws), ws.numel(),
                                         _lib.current_stream(x.device)), "hdla_scan_fwd")
        ctx.save_for_backward(x, dt, A, B, C, D, z, bias, cu, left)      # (the initial state's part in them is in `left`)
        ctx.cfg = (softplus, n, h0 is not None)
        ctx.set_materialize_grads(False)
        return y, ht

    @staticmethod
    @once_differentiable
    @autocast_custom_bwd
    def backward(ctx, dy, dht):
        x, dt, A, B, C, D, z, bias, cu, left = ctx.saved_tensors
        softplus, n, want_dh0 = ctx.cfg
        lib = _lib.load()
        new = lambda t: None if t is None else torch.empty(t.shape, dtype=t.dtype, device=t.device)
        with torch.cuda.device(x.device):
            dims = _scan_dims(x, dt, A, B, C, D, z, bias, softplus, n, cu)
            dy = torch.zeros(x.shape, dtype=x.dtype, device=x.device) if dy is None else whole(dy.to(x.dtype))
            dht = None if dht is None else whole(dht.float())
            dx, ddt, dA, dB, dC, dD, dz, dbias = (new(t) for t in (x, dt, A, B, C, D, z, bias))
            dh0 = torch.empty(n, x.shape[-1], A.shape[1], dtype=torch.float32, device=x.device) if want_dh0 else None
            ws = torch.empty(lib.hdla_scan_workspace_bytes(ctypes.byref(dims)), dtype=torch.uint8, device=x.device)
            _lib.check(lib.hdla_scan_bwd(ctypes.byref(dims), _lib.ptr(x), _lib.ptr(dt), _lib.ptr(A), _lib.ptr(B), _lib.ptr(C), _lib.ptr(D), _lib.ptr(z), _lib.ptr(bias),
                                         _lib.ptr(dy), _lib.ptr(dht), _lib.ptr(left), left.numel(), _lib.ptr(dx), _lib.ptr(ddt), _lib.ptr(dA), _lib.ptr(dB),
                                         _lib.ptr(dC), _lib.ptr(dD), _lib.ptr(dz), _lib.ptr(dbias), _lib.ptr(dh0), _lib.ptr(ws), ws.numel(),
                                         _lib.current_stream(x.device)), "hdla_scan_bwd")
        return dx, ddt, dA, dB, dC, dD, dz, dbias, dh0, None, None, None, None


@torch.compiler.disable
def state_space_scan(
    x: torch.Tensor,                                  # [B, T, D]
    dt: torch.Tensor,                                 # [B, T, D]
    A: torch.Tensor,                                  # [D, S]
    B: torch.Tensor,                                  # [B, T, G, S] or [B, T, S]
    C: torch.Tensor,                                  # as B
    D: Optional[torch.Tensor] = None,                 # [D]
    z: Optional[torch.Tensor] = None,                 # [B, T, D]
    *,
    dt_bias: Optional[torch.Tensor] = None,           # [D]
    dt_softplus: bool = False,
    initial_state: Optional[torch.Tensor] = None,     # [N, D, S]
    output_final_state: bool = False,
    cu_seqlens: Optional[torch.Tensor] = None,
) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """Per channel with S states (at most 64), of a group of D / G neighbouring channels that share B and C:

        delta_t = softplus(dt_t + dt_bias)     (``dt_softplus``; else without it)
        h_t = exp(delta_t A) h_{t-1} + delta_t x_t B_t,     y_t = (C_t . h_t + D x_t) silu(z_t)

    ``A`` is what stands in the exponent: negative where states decay; one that lets them grow must not do so by more than 2^127 over a call;
    minus infinity forgets a state at every step size but zero, which leaves it as it is.  Returns ``(y [B, T, D] in x's dtype, final_state [N, D, S] fp32 or None)``;
    ``cu_seqlens`` packs N sequences into a batch of one.  x, dt, B, C and z of different types are computed in fp32."""
    out = _lib.native().state_space_scan(x, dt, A, B, C, D, z, dt_bias, dt_softplus, initial_state, output_final_state, cu_seqlens)
    if out is not None:
        return out
    if x.dim() != 3:
        raise ValueError(f"x must be [B, T, D], got {tuple(x.shape)}")
    B, C = _scan_args(x, dt, A, B, C, D, z, dt_bias)
    n, cu = _sequences(x, cu_seqlens, initial_state, tuple(A.shape))
    _within_reach(x, n)
    on_one_gpu(x, dt, A, B, C, D, z, dt_bias, initial_state)
    out_dtype = x.dtype
    x, dt, B, C, z = (rows(t) for t in _common(x, dt, B, C, z))
    A, D, dt_bias = (None if t is None else param(t).contiguous() for t in (A, D, dt_bias))
    h0 = None if initial_state is None else whole(initial_state.float())
    y, ht = StateSpaceScanFunction.apply(x, dt, A, B, C, D, z, dt_bias, h0, bool(dt_softplus), bool(output_final_state), n, cu)
    return y.to(out_dtype), ht


@torch.compiler.disable
def state_space_step(
    x: torch.Tensor,                                  # [B, D]
    dt: torch.Tensor,                                 # [B, D]
    A: torch.Tensor,                                  # [D, S]
    B: torch.Tensor,                                  # [B, G, S] or [B, S]
    C: torch.Tensor,                                  # as B
    state: torch.Tensor,                              # [B, D, S]
    D: Optional[torch.Tensor] = None,                 # [D]
    z: Optional[torch.Tensor] = None,                 # [B, D]
    *,
    dt_bias: Optional[torch.Tensor] = None,           # [D]
    dt_softplus: bool = False,
    inplace: bool = False,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """``state_space_scan`` for one token of each sequence: returns ``(y [B, D], new_state [B, D, S] fp32)``.  ``inplace=True`` writes the new state where
    ``state`` is, as a loop of decode steps or a captured graph wants it.  No gradients."""
    out = _lib.native().state_space_step(x, dt, A, B, C, D, z, dt_bias, dt_softplus, state, inplace)
    if out is not None:
        return out
    if x.dim() != 2:
        raise ValueError(f"x must be [B, D], got {tuple(x.shape)}")
    B, C = _scan_args(x, dt, A, B, C, D, z, dt_bias)
    if tuple(state.shape) != (x.shape[0],) + tuple(A.shape):
        raise ValueError(f"state must be {(x.shape[0],) + tuple(A.shape)}, got {tuple(state.shape)}")
    _within_reach(x, x.shape[0])
    on_one_gpu(x, dt, A, B, C, state, D, z, dt_bias)
    out_dtype, to = x.dtype, _new_state(state, inplace, torch.float32)

    def call(x, dt, A, B, C, state, D, z, dt_bias):
        xs, dts, Bs, Cs, zs = (rows(t) for t in _common(x, dt, B, C, z))
        A, D, dt_bias = (None if t is None else param(t).contiguous() for t in (A, D, dt_bias))
        s = whole(state.float())
        with torch.cuda.device(x.device):
            dims = _scan_dims(xs, dts, A, Bs, Cs, D, zs, dt_bias, bool(dt_softplus), x.shape[0], None)
            y, new = torch.empty(x.shape, dtype=xs.dtype, device=x.device), torch.empty_like(s) if to is None else to
            _lib.check(_lib.load().hdla_scan_step(ctypes.byref(dims), _lib.ptr(xs), _lib.ptr(dts), _lib.ptr(A), _lib.ptr(Bs), _lib.ptr(Cs), _lib.ptr(D), _lib.ptr(zs),
                                                  _lib.ptr(dt_bias), _lib.ptr(s), _lib.ptr(y), _lib.ptr(new), _lib.current_stream(x.device)), "hdla_scan_step")
            _written(to)
        return y.to(out_dtype), new

    return _run_step("state_space_step", call, (x, dt, A, B, C, state, D, z, dt_bias), inplace)
