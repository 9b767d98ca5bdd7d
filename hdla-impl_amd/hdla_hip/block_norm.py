"""The norms around a block, fused with its gate, its residual scale and the sum with the residual stream.

``block_norm`` stands beside ``normalize_fn``, which knows no residual: it takes what a block gave and the stream, and returns what the next block reads and
the new stream.  One kernel each way; sums and the stream's sum are fp32, results are rounded once.  Tensors must live on the GPU.
"""
import ctypes
from typing import Optional, Tuple, Union

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .state_space import _NATIVE, code, on_one_gpu, param, whole
from .utils import autocast_custom_bwd, autocast_custom_fwd

_ACTS = {None: 0, "none": 0, "sigmoid": 1, "silu": 2, "swish": 2}
MAX_CHANNELS = 4096


def _dims(x, stream, weight, post, scale, act, post_norm, factor, eps):
    return _lib.HdlaBlockNormDims(x.numel() // x.shape[-1], x.shape[-1], _lib.dtype_code(x.dtype), _lib.dtype_code(stream), code(weight), code(post), code(scale),
                                  act, int(post_norm), float(factor), float(eps))


class BlockNormFunction(torch.autograd.Function):
    """What is kept between the passes: the inputs."""

    @staticmethod
    @autocast_custom_fwd
    def forward(ctx, x, residual, weight, post, gate, scale, act, post_norm, factor, eps):
        lib = _lib.load()
        stream = x.dtype if residual is None else residual.dtype
        with torch.cuda.device(x.device):
            dims = _dims(x, stream, weight, post, scale, act, post_norm, factor, eps)
            y, r = torch.empty_like(x), torch.empty(x.shape, dtype=stream, device=x.device)
            _lib.check(lib.hdla_block_norm_fwd(ctypes.byref(dims), _lib.ptr(x), _lib.ptr(residual), _lib.ptr(weight), _lib.ptr(post), _lib.ptr(gate), _lib.ptr(scale),
                                               _lib.ptr(y), _lib.ptr(r), _lib.current_stream(x.device)), "hdla_block_norm_fwd")
        ctx.save_for_backward(x, residual, weight, post, gate, scale)
        ctx.cfg = (stream, act, post_norm, factor, eps)
        ctx.set_materialize_grads(False)
        return y, r

    @staticmethod
    @once_differentiable
    @autocast_custom_bwd
    def backward(ctx, dy, dr):
        x, residual, weight, post, gate, scale = ctx.saved_tensors
        stream, act, post_norm, factor, eps = ctx.cfg
        lib = _lib.load()
        new = lambda t: None if t is None else torch.empty_like(t)
        with torch.cuda.device(x.device):
            dims = _dims(x, stream, weight, post, scale, act, post_norm, factor, eps)
            dy, dr = None if dy is None else whole(dy.to(x.dtype)), None if dr is None else whole(dr.to(stream))
            dx, dres, dw, dpost, dgate, dscale = (new(t) for t in (x, residual, weight, post, gate, scale))
            ws = torch.empty(lib.hdla_block_norm_workspace_bytes(ctypes.byref(dims)), dtype=torch.uint8, device=x.device)
            _lib.check(lib.hdla_block_norm_bwd(ctypes.byref(dims), _lib.ptr(x), _lib.ptr(residual), _lib.ptr(weight), _lib.ptr(post), _lib.ptr(gate), _lib.ptr(scale),
                                               _lib.ptr(dy), _lib.ptr(dr), _lib.ptr(dx), _lib.ptr(dres), _lib.ptr(dw), _lib.ptr(dpost), _lib.ptr(dgate), _lib.ptr(dscale),
                                               _lib.ptr(ws), ws.numel(), _lib.current_stream(x.device)), "hdla_block_norm_bwd")
        return dx, dres, dw, dpost, dgate, dscale, None, None, None, None


@torch.compiler.disable
def block_norm(
    x: torch.Tensor,                                  # [..., E]: what the block gave
    residual: Optional[torch.Tensor] = None,          # [..., E]: the stream
    weight: Optional[torch.Tensor] = None,            # [E]: of the norm before the next block
    *,
    post_norm: bool = False,
    post_weight: Optional[torch.Tensor] = None,       # [E]: of the norm behind this one
    gate: Optional[torch.Tensor] = None,              # [..., E]
    gate_act: Optional[str] = "sigmoid",
    residual_scale: Union[float, torch.Tensor] = 1.0,
    eps: float = 1e-5,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """``p = x / rms(x) * post_weight`` (with ``post_norm`` or a ``post_weight``, else x), ``u = p * act(gate)``, ``r = residual + residual_scale * u``,
    ``y = r / rms(r) * weight``, with ``rms(v) = sqrt(mean(v^2) + eps)`` over the last dimension.  Returns ``(y in x's dtype, r in residual's)``.

    ``gate_act``: "sigmoid", "silu" or None (the gate multiplies as it is).  ``residual_scale``: a number, or a tensor [E] (learned).  The stream may be fp32 beside
    bf16 blocks; other mixtures of types, and fp16, are computed in fp32.  E is at most 4096.  ``y`` is formed from the sum before that is rounded to the stream's type."""
    out = _lib.native().block_norm(x, residual, weight, post_norm, post_weight, gate, gate_act, residual_scale, eps)
    if out is not None:
        return out
    E = x.shape[-1] if x.dim() else 0
    if E < 1:
        raise ValueError(f"x must be [..., E], got {tuple(x.shape)}")
    if E > MAX_CHANNELS:
        raise NotImplementedError(f"{E} channels are not built (at most {MAX_CHANNELS})")
    for name, t in (("residual", residual), ("gate", gate)):
        if t is not None and t.shape != x.shape:
            raise ValueError(f"{name} {tuple(t.shape)} must have the shape of x {tuple(x.shape)}")
    scale = residual_scale if isinstance(residual_scale, torch.Tensor) else None
    for name, t in (("weight", weight), ("post_weight", post_weight), ("residual_scale", scale)):
        if t is not None and tuple(t.shape) != (E,):
            raise ValueError(f"{name} must be [{E}], got {tuple(t.shape)}")
    if gate_act not in _ACTS:
        raise NotImplementedError(f"gate_act = {gate_act!r}: 'sigmoid', 'silu' and None are built")
    on_one_gpu(x, residual, weight, post_weight, gate, scale)
    out_dtype, stream = x.dtype, x.dtype if residual is None else residual.dtype
    for t in (x, residual):
        if t is not None and t.dtype not in _NATIVE + (torch.float16,):
            raise TypeError(f"unsupported dtype {t.dtype}")
    # fp32, which holds what each of them says, but where the kernels take the types as they are: one of all, or an fp32 stream beside bf16
    if out_dtype == torch.float16 or stream == torch.float16 or (out_dtype == torch.float32 and stream != torch.float32) or (gate is not None and gate.dtype != out_dtype):
        x, residual, gate = (None if t is None else t.float() for t in (x, residual, gate))
    weight, post_weight, scale = (None if t is None else param(t).contiguous() for t in (weight, post_weight, scale))
    y, r = BlockNormFunction.apply(whole(x), whole(residual), weight, post_weight, whole(gate), scale, _ACTS[gate_act], bool(post_norm) or post_weight is not None,
                                   1.0 if scale is not None else float(residual_scale), float(eps))
    return y.to(out_dtype), r.to(stream)
