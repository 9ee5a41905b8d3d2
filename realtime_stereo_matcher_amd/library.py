"""The engine's operators as PyTorch custom ops (``torch.ops.stereocv.*``) with fake kernels.

The reference networks are traced by ``torch.onnx.export`` (tools/convert.py:18-26) and by
thop / fvcore (tools/profiler.py:11-26).  A ctypes call is opaque to a tracer: ``torch.jit.trace``
would bake the call's output in as a constant and ``torch.export`` / ``torch.compile`` could
not see through it.  Registered here with ``torch.library.custom_op``, each operator is one node
of the traced graph: ``functional`` routes a call through ``torch.ops.stereocv.<name>`` whenever
it runs under ``torch.jit.trace`` or a compiler (dynamo / export), the fake kernel gives
FakeTensor tracing the output's shape, dtype and device, and the real kernel is the same
libstereocv call as the eager path (no CPU fallback).  The cost-volume ops are forward-only like
the rest of that engine: their backward raises ``NotImplementedError``.  The matching-transformer
ops have their gradients, as ops of their own.
"""
from __future__ import annotations

import threading
from typing import Optional

import torch

from . import functional as F

_state = threading.local()


def tracing() -> bool:
    """True when a functional call should go through torch.ops.stereocv (a tracer or compiler
    is recording, and the call is not already the body of one of these ops)."""
    if not (torch.compiler.is_compiling() or torch.jit.is_tracing()):
        return False
    return not getattr(_state, "inside", False)


class _Inside:
    def __enter__(self):
        self.prev = getattr(_state, "inside", False)
        _state.inside = True

    def __exit__(self, *exc):
        _state.inside = self.prev


def _forward_only(ctx, *grads):
    raise NotImplementedError(
        "realtime_stereo_matcher_amd cost-volume kernels are forward/inference-only; "
        "backward is not implemented")


def _no_ctx(ctx, inputs, output):
    return None


def _register(name, impl, fake):
    op = torch.library.custom_op(f"stereocv::{name}", mutates_args=())(impl)
    op.register_fake(fake)
    torch.library.register_autograd(f"stereocv::{name}", _forward_only, setup_context=_no_ctx)
    return op


def _empty(shape, like, dtype=None):
    return like.new_empty(shape, dtype=dtype if dtype is not None else like.dtype)


# ------------------------------------------------------------------------------------- ops
def _inner_product(left: torch.Tensor, right: torch.Tensor, max_disparity: int,
                   algo: str) -> torch.Tensor:
    with _Inside():
        return F.inner_product_volume(left, right, max_disparity, algo=algo)


def _inner_product_fake(left, right, max_disparity, algo):
    n, _, h, w = left.shape
    return _empty((n, max_disparity, h, w), left)


def _correlation(left: torch.Tensor, right: torch.Tensor, max_disp: int,
                 algo: str = "auto") -> torch.Tensor:
    with _Inside():
        return F.correlation_volume(left, right, max_disp, algo=algo)


def _correlation_fake(left, right, max_disp, algo="auto"):
    n, _, h, w = left.shape
    return _empty((n, max_disp, h, w), left)


def _groupwise(left: torch.Tensor, right: torch.Tensor, n_groups: int,
               max_disparity: int) -> torch.Tensor:
    with _Inside():
        return F.groupwise_volume(left, right, n_groups, max_disparity)


def _groupwise_fake(left, right, n_groups, max_disparity):
    n, _, h, w = left.shape
    return _empty((n, n_groups, h, w, max_disparity), left, torch.float32)


def _concat(left: torch.Tensor, right: torch.Tensor, max_disparity: int) -> torch.Tensor:
    with _Inside():
        return F.concat_volume(left, right, max_disparity)


def _concat_fake(left, right, max_disparity):
    n, c, h, w = left.shape
    return _empty((n, 2 * c, h, w, max_disparity), left)


def _interweave(left: torch.Tensor, right: torch.Tensor) -> torch.Tensor:
    with _Inside():
        return F.interweave(left, right)


def _interweave_fake(left, right):
    n, c, h, w = left.shape
    return _empty((n, 2 * c, h, w), left)


def _interweave_volume(left: torch.Tensor, right: torch.Tensor, max_disparity: int) -> torch.Tensor:
    with _Inside():
        return F.interweave_volume(left, right, max_disparity)


def _interweave_volume_fake(left, right, max_disparity):
    n, c, h, w = left.shape
    return _empty((n, 2 * c, max_disparity, h, w), left)


def _difference(left: torch.Tensor, right: torch.Tensor, max_disp: int) -> torch.Tensor:
    with _Inside():
        return F.difference_volume(left, right, max_disp)


def _difference_fake(left, right, max_disp):
    n, c, h, w = left.shape
    return _empty((n, c, max_disp, h, w), left)


def _regress_dtype(volume, f32):
    # the autocast rule of functional._regress, decided when the graph was traced (f32: an
    # fp16 / bf16 volume under autocast gives fp32)
    return torch.float32 if f32 else volume.dtype


def _soft_argmin(volume: torch.Tensor, f32: bool = False) -> torch.Tensor:
    with _Inside(), F._F32Decided(f32):
        return F.soft_argmin(volume, keepdim=False)


def _soft_argmin_fake(volume, f32=False):
    n, _, h, w = volume.shape
    return _empty((n, h, w), volume, _regress_dtype(volume, f32))


def _presoftmax(prob: torch.Tensor, f32: bool = False) -> torch.Tensor:
    with _Inside(), F._F32Decided(f32):
        return F.regression_presoftmax(prob)


def _presoftmax_fake(prob, f32=False):
    n, _, h, w = prob.shape
    return _empty((n, h, w), prob, _regress_dtype(prob, f32))


def _argext_fake(volume):
    n, _, h, w = volume.shape
    return _empty((n, h, w), volume, torch.int64)


def _hard_argmin(volume: torch.Tensor) -> torch.Tensor:
    with _Inside():
        return F.hard_argmin(volume)


def _hard_argmax(volume: torch.Tensor) -> torch.Tensor:
    with _Inside():
        return F.hard_argmax(volume)


def _fused(left: torch.Tensor, right: torch.Tensor, max_disparity: int, mean: bool,
           f32: bool = False, exact: bool = False) -> tuple[torch.Tensor, torch.Tensor]:
    with _Inside(), F._F32Decided(f32):
        return F.inner_product_soft_argmin(left, right, max_disparity, mean=mean, keep_volume=True,
                                           exact_accumulators=exact)


def _fused_disp_dtype(left, f32):
    # autocast with half features (decided when the graph was traced): fp32 disparities
    return torch.float32 if f32 else left.dtype


def _fused_fake(left, right, max_disparity, mean, f32=False, exact=False):
    n, _, h, w = left.shape
    return (_empty((n, max_disparity, h, w), left),
            _empty((n, 1, h, w), left, _fused_disp_dtype(left, f32)))


def _fused_novolume(left: torch.Tensor, right: torch.Tensor, max_disparity: int, mean: bool,
                    f32: bool = False, exact: bool = False) -> torch.Tensor:
    with _Inside(), F._F32Decided(f32):
        return F.inner_product_soft_argmin(left, right, max_disparity, mean=mean,
                                           keep_volume=False, exact_accumulators=exact)[1]


def _fused_novolume_fake(left, right, max_disparity, mean, f32=False, exact=False):
    n, _, h, w = left.shape
    return _empty((n, 1, h, w), left, _fused_disp_dtype(left, f32))


def _warp(image: torch.Tensor, flow: torch.Tensor, f32: bool = False) -> torch.Tensor:
    with _Inside(), F._F32Decided(f32):
        return F.warp_by_flow_map(image, flow)


def _warp_fake(image, flow, f32=False):
    # the output dtype rule of functional.warp_by_flow_map: fp32 under autocast (grid_sample is
    # an autocast fp32 op; decided when the graph was traced), else the image dtype (fp32 for an
    # fp32 image)
    n, _, h, w = flow.shape
    odt = torch.float32 if f32 else image.dtype
    return _empty((n, image.shape[1], h, w), image, odt)


def _v4(featL: torch.Tensor, featR: torch.Tensor, w1: torch.Tensor, b1: torch.Tensor,
        w2: torch.Tensor, b2: torch.Tensor, w3: torch.Tensor, b3: torch.Tensor, w4: torch.Tensor,
        b4: torch.Tensor, volume_size: int) -> torch.Tensor:
    with _Inside():
        return F.v4_volume(featL, featR, w1, b1, w2, b2, w3, b3, w4, b4, volume_size)


def _v4_fake(featL, featR, w1, b1, w2, b2, w3, b3, w4, b4, volume_size):
    n, _, h, w = featL.shape
    return _empty((n, volume_size, h, w), featL, torch.float32)


inner_product_volume = _register("inner_product_volume", _inner_product, _inner_product_fake)
correlation_volume = _register("correlation_volume", _correlation, _correlation_fake)
groupwise_volume = _register("groupwise_volume", _groupwise, _groupwise_fake)
concat_volume = _register("concat_volume", _concat, _concat_fake)
interweave = _register("interweave", _interweave, _interweave_fake)
interweave_volume = _register("interweave_volume", _interweave_volume, _interweave_volume_fake)
difference_volume = _register("difference_volume", _difference, _difference_fake)
soft_argmin = _register("soft_argmin", _soft_argmin, _soft_argmin_fake)
regression_presoftmax = _register("regression_presoftmax", _presoftmax, _presoftmax_fake)
hard_argmin = _register("hard_argmin", _hard_argmin, _argext_fake)
hard_argmax = _register("hard_argmax", _hard_argmax, _argext_fake)
inner_product_soft_argmin = _register("inner_product_soft_argmin", _fused, _fused_fake)
inner_product_soft_argmin_novolume = _register("inner_product_soft_argmin_novolume",
                                               _fused_novolume, _fused_novolume_fake)
warp_by_flow_map = _register("warp_by_flow_map", _warp, _warp_fake)
v4_volume = _register("v4_volume", _v4, _v4_fake)


# ----------------------------------------------------------------- matching by attention
def _register_with_grad(name, impl, fake, setup, backward):
    op = torch.library.custom_op(f"stereocv::{name}", mutates_args=())(impl)
    op.register_fake(fake)
    torch.library.register_autograd(f"stereocv::{name}", backward, setup_context=setup)
    return op


def _attn(query: torch.Tensor, key: torch.Tensor, value: torch.Tensor,
          key_lengths: Optional[torch.Tensor] = None, key_mask: Optional[torch.Tensor] = None,
          scale: Optional[float] = None,
          max_disparity: Optional[int] = None) -> tuple[torch.Tensor, torch.Tensor]:
    index, scale, band, lengths, mask = F._attention_checks(query, key, value, scale, max_disparity,
                                                            key_lengths, key_mask)
    return F._attention_forward(index, query, key, value, lengths, mask, scale, band, True)


def _attn_fake(query, key, value, key_lengths=None, key_mask=None, scale=None, max_disparity=None):
    b, lq, h, _ = query.shape
    kv = key.shape[2]
    return (_empty(query.shape, query),
            _empty((b, kv, lq * (h // kv)) if kv else (b, 0, 0), query, torch.float32))


def _attn_setup(ctx, inputs, output):
    q, k, v, lengths, mask, scale, max_disparity = inputs
    ctx.save_for_backward(q, k, v, *output, lengths, mask)
    ctx.mark_non_differentiable(output[1])  # lse is a constant, as in an eager call
    ctx.scale, ctx.max_disparity = scale, max_disparity


def _attn_grad(ctx, dout, _):
    q, k, v, out, lse, lengths, mask = ctx.saved_tensors
    dq, dk, dv = torch.ops.stereocv.cross_attention_backward(
        q, k, v, out, lse, dout, lengths, mask, ctx.scale, ctx.max_disparity)
    return dq, dk, dv, None, None, None, None


def _attn_backward(query: torch.Tensor, key: torch.Tensor, value: torch.Tensor, out: torch.Tensor,
                   lse: torch.Tensor, dout: torch.Tensor,
                   key_lengths: Optional[torch.Tensor] = None,
                   key_mask: Optional[torch.Tensor] = None, scale: Optional[float] = None,
                   max_disparity: Optional[int] = None) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    index, scale, band, lengths, mask = F._attention_checks(query, key, value, scale, max_disparity,
                                                            key_lengths, key_mask)
    if out.shape != query.shape or dout.shape != query.shape or out.dtype != query.dtype \
            or dout.dtype != query.dtype or not out.is_contiguous():
        raise RuntimeError("cross_attention_backward: out and dout must have the query's shape and "
                           "type, and out must be contiguous")
    kv = key.shape[2]
    rows = query.shape[1] * (query.shape[2] // kv if kv else 0)
    if tuple(lse.shape) != (query.shape[0], kv, rows) or lse.dtype != torch.float32 or not lse.is_contiguous():
        raise RuntimeError("cross_attention_backward: lse must be the forward call's")
    F._device_check(query, out, lse, dout)
    return F._attention_backward(index, query, key, value, out, lse, dout, lengths, mask, scale, band)


def _attn_backward_fake(query, key, value, out, lse, dout, key_lengths=None, key_mask=None, scale=None,
                        max_disparity=None):
    return _empty(query.shape, query), _empty(key.shape, key), _empty(key.shape, key)


def _rot(x: torch.Tensor, positions: torch.Tensor, frequencies: torch.Tensor, layout: str = "half",
         amplitude: float = 1.0, inverse: bool = False) -> torch.Tensor:
    index, positions, frequencies = F._rotary_checks(x, positions, frequencies, layout)
    return F._rotary_run(index, x, positions, frequencies, layout == "interleaved", amplitude, inverse)


def _rot_fake(x, positions, frequencies, layout="half", amplitude=1.0, inverse=False):
    return _empty(x.shape, x)


def _rot_setup(ctx, inputs, output):
    _, positions, frequencies, ctx.layout, ctx.amplitude, ctx.inverse = inputs
    ctx.save_for_backward(positions, frequencies)


def _rot_grad(ctx, dy):
    positions, frequencies = ctx.saved_tensors
    dx = torch.ops.stereocv.rotary(dy, positions, frequencies, ctx.layout, ctx.amplitude, not ctx.inverse)
    return dx, None, None, None, None, None


def _norm(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6) -> torch.Tensor:
    with _Inside(), torch.no_grad():
        return F.rms_norm(x, weight, None, eps)


def _norm_fake(x, weight, eps=1e-6):
    return _empty(x.shape, x)


def _norm_setup(ctx, inputs, output):
    x, weight, ctx.eps = inputs
    ctx.save_for_backward(x, weight)


def _norm_grad(ctx, dy):
    x, weight = ctx.saved_tensors
    dx, _, dw = torch.ops.stereocv.rms_norm_backward(x, weight, dy, None, ctx.eps)
    return dx, dw, None


def _add_norm(x: torch.Tensor, weight: torch.Tensor, residual: torch.Tensor,
              eps: float = 1e-6) -> tuple[torch.Tensor, torch.Tensor]:
    with _Inside(), torch.no_grad():
        return F.rms_norm(x, weight, residual, eps)


def _add_norm_fake(x, weight, residual, eps=1e-6):
    return _empty(x.shape, x), _empty(x.shape, residual)


def _add_norm_setup(ctx, inputs, output):
    x, weight, _, ctx.eps = inputs
    ctx.save_for_backward(output[1], weight)


def _add_norm_grad(ctx, dy, dsummed):
    summed, weight = ctx.saved_tensors
    dx, dres, dw = torch.ops.stereocv.rms_norm_backward(summed, weight, dy, dsummed, ctx.eps)
    return dx, dw, dx if summed.dtype == dy.dtype else dres, None


def _norm_backward(summed: torch.Tensor, weight: torch.Tensor, dy: torch.Tensor,
                   dsummed: Optional[torch.Tensor] = None,
                   eps: float = 1e-6) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    index = F._norm_checks("rms_norm_backward", dy, weight, summed, eps)
    if dsummed is not None:
        if dsummed.shape != summed.shape or dsummed.dtype != summed.dtype:
            raise RuntimeError("rms_norm_backward: dsummed must have summed's shape and type")
        F._one_device(summed, dsummed)
    dx, dres, dw = F._norm_backward(index, summed, weight, dy, dsummed, dy.dtype, eps)
    return dx, dx.new_empty(0, dtype=summed.dtype) if dres is None else dres, dw


def _norm_backward_fake(summed, weight, dy, dsummed=None, eps=1e-6):
    same = summed.dtype == dy.dtype
    return (_empty(dy.shape, dy), _empty((0,) if same else summed.shape, summed),
            _empty(weight.shape, weight))


def _norm8_shape(x, group):
    return (*x.shape[:-1], -(-x.shape[-1] // group) if group else 1)


def _norm8(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6,
           group: int = 0) -> tuple[torch.Tensor, torch.Tensor]:
    with _Inside(), torch.no_grad():
        return F.rms_norm_e4m3(x, weight, None, eps, group or None)


def _norm8_fake(x, weight, eps=1e-6, group=0):
    return _empty(x.shape, x, torch.float8_e4m3fn), _empty(_norm8_shape(x, group), x, torch.float32)


def _add_norm8(x: torch.Tensor, weight: torch.Tensor, residual: torch.Tensor, eps: float = 1e-6,
               group: int = 0) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    with _Inside(), torch.no_grad():
        return F.rms_norm_e4m3(x, weight, residual, eps, group or None)


def _add_norm8_fake(x, weight, residual, eps=1e-6, group=0):
    return (*_norm8_fake(x, weight, eps, group), _empty(x.shape, residual))


def _plain_op(name, impl, fake):
    op = torch.library.custom_op(f"stereocv::{name}", mutates_args=())(impl)
    op.register_fake(fake)
    return op


cross_attention = _register_with_grad("cross_attention", _attn, _attn_fake, _attn_setup, _attn_grad)
cross_attention_backward = _plain_op("cross_attention_backward", _attn_backward, _attn_backward_fake)
rotary = _register_with_grad("rotary", _rot, _rot_fake, _rot_setup, _rot_grad)
rms_norm = _register_with_grad("rms_norm", _norm, _norm_fake, _norm_setup, _norm_grad)
add_rms_norm = _register_with_grad("add_rms_norm", _add_norm, _add_norm_fake, _add_norm_setup,
                                   _add_norm_grad)
rms_norm_backward = _plain_op("rms_norm_backward", _norm_backward, _norm_backward_fake)
rms_norm_e4m3 = _register("rms_norm_e4m3", _norm8, _norm8_fake)
add_rms_norm_e4m3 = _register("add_rms_norm_e4m3", _add_norm8, _add_norm8_fake)
