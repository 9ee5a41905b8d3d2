"""Functional front-end of the MI355X stereo cost-volume engine.

Every function validates its arguments the way the reference does, allocates the output
with the caching allocator on the input's device and enqueues ONE libstereocv kernel on
the current HIP stream (no host sync).  There is no CPU / eager fallback: tensors must live
on a HIP device and the native library must load, otherwise the call raises.

Reference operators mirrored (babiking/realtime_stereo_matcher):
  inner_product_volume   cost_volume/inner_product.py:11-42
  groupwise_volume       cost_volume/groupwise.py:24-56
  concat_volume          cost_volume/concatenate.py:11-41
  interweave             cost_volume/interweave.py:10-22, model/mobile_stereo_net_v4.py:17-23
  interweave_volume      model/mobile_stereo_net_v4.py:443-461 (shifted interweave, materialised)
  difference_volume      model/mobile_stereo_net.py:8-27 (+ _v2.py:8-27, _v3.py:9-28)
  correlation_volume     model/mobile_disp_net_c.py:188-205
  inner_product_soft_argmin  either volume fused with soft_argmin
  soft_argmin            model/mobile_disp_net_c.py:208-220, model/mobile_stereo_net.py:144-147
  regression_presoftmax  model/mobile_stereo_net_v4.py:10-14
  hard_argmin/argmax     build-defined
  warp_by_flow_map       tools/warp.py:5-42, model/mobile_stereo_net_v2.py:59-96

Matching by attention instead of a cost volume (no operator of the reference; differentiable):
  rms_norm, rms_norm_e4m3         norm of the token stream, with the residual's addition
  rotary, rotary_frequencies      rotary positions of queries and keys
  cross_attention                 left tokens to the right view's, whose number may differ
"""
from __future__ import annotations

import math
import numpy as np
import threading

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib

# float64 (round 6): the cost volumes and the regressions in fp64 (csrc/f64.hip), as torch
# computes an fp64 input; the warp and the V4 volume stay float32 / 16-bit
_DTYPES = {torch.float32: _lib.SM_F32, torch.float16: _lib.SM_F16, torch.bfloat16: _lib.SM_BF16,
           torch.float64: _lib.SM_F64}
_WARP_DTYPES = (torch.float32, torch.float16, torch.bfloat16)
_ALGOS = {"auto": _lib.SM_IP_AUTO, "valu": _lib.SM_IP_VALU, "mfma": _lib.SM_IP_MFMA_F32,
          "f32": _lib.SM_IP_MFMA_F32, "h2": _lib.SM_IP_MFMA_H2, "h2db": _lib.SM_IP_MFMA_H2DB,
          "rs": _lib.SM_IP_MFMA_RS, "sl": _lib.SM_IP_MFMA_SL}


# ----------------------------------------------------------------------------------- plumbing
_tracing = None  # library.tracing, once imported (library.py imports this module)


def _traced():
    """Under torch.jit.trace or a compiler the call is routed through torch.ops.stereocv, so the
    traced graph holds the operator instead of its output as a constant (library.py)."""
    global _tracing
    if _tracing is None:
        from . import library
        _tracing = library.tracing
    return _tracing()


def _ops():
    from . import library  # noqa: F401  (registers the ops)
    return torch.ops.stereocv

def _device_check(*ts):
    dev = ts[0].device
    for t in ts:
        if t.device.type != "cuda":
            raise RuntimeError(
                "realtime_stereo_matcher_amd runs on HIP devices only (got a tensor on "
                f"'{t.device}'); there is no CPU fallback -- move the features with .cuda()")
        if t.device != dev:
            raise RuntimeError(f"tensors on different devices: {dev} vs {t.device}")
    return dev


def _dtype_code(t):
    code = _DTYPES.get(t.dtype)
    if code is None:
        raise TypeError(f"unsupported dtype {t.dtype}; expected float32, float16, bfloat16 or float64")
    return code


def _rows_contiguous(t):
    """The C ABI needs unit W stride; any other stride pattern is passed through."""
    return t if (t.dim() == 0 or t.stride(-1) == 1 or t.size(-1) <= 1) else t.contiguous()


def _stride_ok(t):
    # size-1 W can carry any stride in torch; normalise so the ABI sees 1
    if t.size(-1) <= 1 and t.stride(-1) != 1:
        t = t.contiguous()
    return t


def _pair(left, right, what):
    if not isinstance(left, torch.Tensor) or not isinstance(right, torch.Tensor):
        raise TypeError(f"{what}: left and right must be tensors")
    if left.dim() != 4 or right.dim() != 4:
        raise RuntimeError(f"{what}: expected 4-D (N, C, H, W) features, got {tuple(left.shape)} "
                           f"and {tuple(right.shape)}")
    if left.shape != right.shape:
        raise RuntimeError(f"{what}: left/right shape mismatch {tuple(left.shape)} vs "
                           f"{tuple(right.shape)}")
    if left.dtype != right.dtype:
        raise RuntimeError(f"{what}: left/right dtype mismatch {left.dtype} vs {right.dtype}")
    code = _dtype_code(left)
    dev = _device_check(left, right)
    left = _stride_ok(_rows_contiguous(left))
    right = _stride_ok(_rows_contiguous(right))
    return left, right, dev, code


def _stream(dev):
    return torch.cuda.current_stream(dev).cuda_stream


def _disp(max_disparity, what):
    d = int(max_disparity)
    if d < 0:
        raise RuntimeError(f"{what}: max disparity must be non-negative, got {d}")
    return d


class _ForwardOnly(torch.autograd.Function):
    """Marks outputs as produced by a forward-only native kernel (no autograd support yet)."""

    @staticmethod
    def forward(ctx, fn, *tensors):
        return fn()

    @staticmethod
    def backward(ctx, *grads):
        raise NotImplementedError(
            "realtime_stereo_matcher_amd cost-volume kernels are forward/inference-only; "
            "backward is not implemented")


def _run(fn, *inputs):
    # the entry points size persistent grids and set kernel attributes on the CURRENT HIP
    # device: make it the inputs' device for the call
    with torch.cuda.device(inputs[0].device):
        if torch.is_grad_enabled() and any(t.requires_grad for t in inputs):
            return _ForwardOnly.apply(fn, *inputs)
        return fn()


def _ptr(t):
    return t.data_ptr()


# the current stream's handle by device index: torch's own raw accessor where it has one, since
# building a Stream object costs more than the smallest kernels' launch
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)


_HALF = (torch.float16, torch.bfloat16)


def _autocast_fp32(*ts):
    """True when torch autocast is active on the tensors' device and one of them is fp16 / bf16.

    The reference evaluates under ``torch.cuda.amp.autocast`` (``mixed_precision`` defaults to
    True: evaluate_stereo.py:48,124,182,231,320; test_stereo.py:117).  Its Conv3d outputs are
    then fp16, but ``F.softmax``, ``torch.sum`` and ``F.grid_sample`` are autocast fp32 ops, so
    the soft-argmin (mobile_stereo_net.py:144-147, mobile_disp_net_c.py:208-220) returns an fp32
    disparity from an fp16 volume and the RefineNet warp (tools/warp.py:39) samples in fp32.
    The engine follows: under autocast these ops return fp32 (one rounding, from fp64 / fp32
    arithmetic), never the volume's reduced dtype.
    """
    ov = getattr(_decided, "f32", None)
    if ov is not None:  # the body of a torch.ops.stereocv op: the decision made at trace time
        return ov
    return any(t.dtype in _HALF for t in ts) and torch.is_autocast_enabled(ts[0].device.type)


_decided = threading.local()


class _F32Decided:
    """Inside a torch.ops.stereocv op (library.py) the fp32-output decision is an op argument
    taken when the graph was traced, not the autocast state at run time: a compiled graph may run
    its ops after the compiler removed the autocast regions."""

    def __init__(self, value):
        self.value = bool(value)

    def __enter__(self):
        self.prev = getattr(_decided, "f32", None)
        _decided.f32 = self.value

    def __exit__(self, *exc):
        _decided.f32 = self.prev


# ----------------------------------------------------------------------------- a-1, a-6, a-2
def inner_product_volume(left, right, max_disparity, algo="auto"):
    """(N,C,H,W) x2 -> (N,D,H,W): sum_c L*R(x-d) for x >= d, 0 elsewhere (left dtype/device)."""
    if _traced():
        return _ops().inner_product_volume(left, right, int(max_disparity), algo)
    left, right, dev, code = _pair(left, right, "inner_product_volume")
    D = _disp(max_disparity, "inner_product_volume")
    if algo not in _ALGOS:
        raise ValueError(f"algo must be one of {sorted(_ALGOS)}")
    n, c, h, w = left.shape

    def fn():
        out = torch.empty((n, D, h, w), dtype=left.dtype, device=dev)
        if out.numel():
            lib = _lib.load()
            _lib.check(lib.sm_cv_inner_product_ex(
                _ptr(left), _ptr(right), _ptr(out), code, n, c, h, w, D,
                _lib.strides_arg(left), _lib.strides_arg(right), _ALGOS[algo], _stream(dev)),
                "sm_cv_inner_product")
        return out

    return _run(fn, left, right)


def correlation_volume(l_fmap, r_fmap, max_disp, algo="auto"):
    """(N,C,H,W) x2 -> (N,D,H,W): mean_c L*R(x-d) for x >= d, 0 elsewhere (``algo``: the band
    kernel, as for inner_product_volume)."""
    if algo not in _ALGOS:
        raise ValueError(f"algo must be one of {sorted(_ALGOS)}")
    if _traced():
        return _ops().correlation_volume(l_fmap, r_fmap, int(max_disp), algo)
    left, right, dev, code = _pair(l_fmap, r_fmap, "correlation_volume")
    D = _disp(max_disp, "correlation_volume")
    n, c, h, w = left.shape

    def fn():
        out = torch.empty((n, D, h, w), dtype=left.dtype, device=dev)
        if out.numel():
            lib = _lib.load()
            _lib.check(lib.sm_cv_correlation_mean_ex(
                _ptr(left), _ptr(right), _ptr(out), code, n, c, h, w, D,
                _lib.strides_arg(left), _lib.strides_arg(right), _ALGOS[algo], _stream(dev)),
                "sm_cv_correlation_mean_ex")
        return out

    return _run(fn, left, right)


def inner_product_soft_argmin(left, right, max_disparity, mean=False, keep_volume=True,
                              exact_accumulators=False):
    """Cost volume + soft-argmin in one kernel pass.

    The inner-product volume (cost_volume/inner_product.py:11-42; ``mean=True``: the
    correlation volume of model/mobile_disp_net_c.py:188-205) and its disparity regression
    sum_d d * softmax_d(volume) (model/mobile_disp_net_c.py:208-220, = the inline soft-argmin of
    model/mobile_stereo_net.py:144-147).  Returns ``(volume, disparity)``: the (N,D,H,W) volume
    (``None`` with ``keep_volume=False``: it is then never written) and the (N,1,H,W) disparity.

    Precision, per the reference's two calls:
    - fp32 features: the volume and the disparity are fp32.  For D <= 192 the disparity does
      not depend on ``keep_volume`` (one kernel folds the same accumulators either way; on the
      sliding-window kernel the fold scales the raw accumulators inside the exponent's FMA
      rather than reading the stored cells, so it is within 1e-4 of the soft-argmin of the
      volume returned, not bit-equal to it).  For C = 16 and D > 192 the volume-kept call runs
      the volume kernel and the regression kernel, the volume-free call one two-pass fold: the
      two disparities agree within 1e-4.
    - fp16 / bf16 features outside autocast: both in the feature dtype.
    - fp16 / bf16 features under ``torch.autocast`` (the reference's default eval,
      evaluate_stereo.py:48): the volume keeps the feature dtype and the disparity is fp32, the
      soft-argmin of the volume's cells as rounded to the feature dtype -- what the reference's
      ``disparity_regression(corr_volume)`` regresses -- on every shape.  ``exact_accumulators=
      True`` regresses the fp32 accumulators of the exact products instead (no rounding), on the
      shapes the fused kernel takes (4-element aligned rows; D <= 192 with the volume kept);
      the other shapes regress the rounded volume either way.

    fp32 features (W >= 4) run one fused band kernel for D <= 192 and, without the volume, for
    C = 16 and D <= 256 (two D passes per segment merged in registers) or other D > 192 (passes
    of <= 192 disparities whose partial softmax states a second kernel merges, in a workspace
    allocated here); other shapes run the volume and the regression kernels back to back.
    """
    if _traced():
        f32, ex = _autocast_fp32(left), bool(exact_accumulators)
        if keep_volume:
            return _ops().inner_product_soft_argmin(left, right, int(max_disparity), bool(mean), f32, ex)
        return None, _ops().inner_product_soft_argmin_novolume(left, right, int(max_disparity),
                                                               bool(mean), f32, ex)
    left, right, dev, code = _pair(left, right, "inner_product_soft_argmin")
    D = _disp(max_disparity, "inner_product_soft_argmin")
    n, c, h, w = left.shape
    mode = 1 if mean else 0
    # autocast eval with fp16 / bf16 features: the volume keeps the feature dtype (the reference
    # assigns into zeros of left.dtype) and the soft-argmin returns fp32 -- the fused kernel's
    # fp32-disparity mode, which rounds each cell to the feature dtype before the fold (the
    # volume the reference regresses); SM_FUSED_EXACT_ACC folds the fp32 accumulators instead
    f32disp = _autocast_fp32(left)
    if f32disp:
        mode |= _lib.SM_FUSED_DISP_F32
        if exact_accumulators:
            mode |= _lib.SM_FUSED_EXACT_ACC

    def call(vol, disp, ws=None, nws=0):
        lib = _lib.load()
        return lib.sm_cv_inner_product_softargmin_ws(
            _ptr(left), _ptr(right), None if vol is None else _ptr(vol), _ptr(disp), code,
            n, c, h, w, D, _lib.strides_arg(left), _lib.strides_arg(right), mode,
            None if ws is None else _ptr(ws), nws, _stream(dev))

    def fn(keep):
        vol = torch.empty((n, D, h, w), dtype=left.dtype, device=dev) if keep else None
        disp = torch.empty((n, 1, h, w), dtype=torch.float32 if f32disp else left.dtype, device=dev)
        if disp.numel():
            # first without a workspace: the volume-free shapes band_sl takes (C = 16, D <= 256)
            # merge their D passes in registers and need none (the cfg4 launch used
            # to allocate 2.6 GB it never read)
            rc = call(vol, disp)
            if rc == _lib.SM_EUNSUPPORTED and vol is None and (code == _lib.SM_F32 or f32disp):
                # several D passes on band_h2: their partial softmax states go to a workspace
                nws = int(_lib.load().sm_cv_inner_product_softargmin_workspace_bytes(n, h, w, D))
                if nws > 0:
                    rc = call(None, disp, torch.empty(nws, dtype=torch.uint8, device=dev), nws)
            if rc == _lib.SM_EUNSUPPORTED and vol is None:
                # not a fused shape: the two-kernel path needs the volume in HBM for a moment
                rc = call(torch.empty((n, D, h, w), dtype=left.dtype, device=dev), disp)
            _lib.check(rc, "sm_cv_inner_product_softargmin")
        return vol, disp

    if keep_volume:
        return _run(lambda: fn(True), left, right)
    return None, _run(lambda: fn(False)[1], left, right)


def groupwise_volume(left, right, n_groups, max_disparity):
    """(N,C,H,W) x2 -> (N,G,H,W,D) float32: per-group mean of L*R(x-d), 0 for x < d.

    Deviation (documented): the reference allocates its output on the CPU regardless of the
    input device (cost_volume/groupwise.py:39); this engine returns it on the input device.
    """
    if _traced():
        return _ops().groupwise_volume(left, right, int(n_groups), int(max_disparity))
    G = int(n_groups)
    D = _disp(max_disparity, "groupwise_volume")
    if isinstance(left, torch.Tensor) and left.dim() == 4 and D > 0:
        # the reference asserts inside groupwise(), reached once per disparity (groupwise.py:15-17)
        c = left.shape[1]
        assert c % G == 0, f"groupwise cost channel ({c}) % #groups ({G}) != 0."
    left, right, dev, code = _pair(left, right, "groupwise_volume")
    n, c, h, w = left.shape

    def fn():
        out = torch.empty((n, G, h, w, D), dtype=torch.float32, device=dev)
        if out.numel():
            lib = _lib.load()
            _lib.check(lib.sm_cv_groupwise(
                _ptr(left), _ptr(right), _ptr(out), code, n, c, h, w, D, G,
                _lib.strides_arg(left), _lib.strides_arg(right), _stream(dev)),
                "sm_cv_groupwise")
        return out

    return _run(fn, left, right)


# ----------------------------------------------------------------------------- a-3, a-4, a-5
def concat_volume(left, right, max_disparity):
    """(N,C,H,W) x2 -> (N,2C,H,W,D): [:C]=L, [C:]=R(x-d) for x >= d, 0 elsewhere (bit-exact)."""
    if _traced():
        return _ops().concat_volume(left, right, int(max_disparity))
    left, right, dev, code = _pair(left, right, "concat_volume")
    D = _disp(max_disparity, "concat_volume")
    n, c, h, w = left.shape

    def fn():
        out = torch.empty((n, 2 * c, h, w, D), dtype=left.dtype, device=dev)
        if out.numel():
            lib = _lib.load()
            _lib.check(lib.sm_cv_concat(
                _ptr(left), _ptr(right), _ptr(out), code, n, c, h, w, D,
                _lib.strides_arg(left), _lib.strides_arg(right), _stream(dev)), "sm_cv_concat")
        return out

    return _run(fn, left, right)


def interweave(left, right):
    """(N,C,H,W) x2 -> (N,2C,H,W): even channels L, odd channels R (bit-exact)."""
    if _traced():
        return _ops().interweave(left, right)
    left, right, dev, code = _pair(left, right, "interweave")
    n, c, h, w = left.shape

    def fn():
        out = torch.empty((n, 2 * c, h, w), dtype=left.dtype, device=dev)
        if out.numel():
            lib = _lib.load()
            _lib.check(lib.sm_cv_interweave(
                _ptr(left), _ptr(right), _ptr(out), code, n, c, h, w,
                _lib.strides_arg(left), _lib.strides_arg(right), _stream(dev)), "sm_cv_interweave")
        return out

    return _run(fn, left, right)


def interweave_volume(left, right, max_disparity):
    """(N,C,H,W) x2 -> (N,2C,D,H,W): the v4 per-disparity interweave, 0 for x < d (bit-exact)."""
    if _traced():
        return _ops().interweave_volume(left, right, int(max_disparity))
    left, right, dev, code = _pair(left, right, "interweave_volume")
    D = _disp(max_disparity, "interweave_volume")
    n, c, h, w = left.shape

    def fn():
        out = torch.empty((n, 2 * c, D, h, w), dtype=left.dtype, device=dev)
        if out.numel():
            lib = _lib.load()
            _lib.check(lib.sm_cv_interweave_shifted(
                _ptr(left), _ptr(right), _ptr(out), code, n, c, h, w, D,
                _lib.strides_arg(left), _lib.strides_arg(right), _stream(dev)),
                "sm_cv_interweave_shifted")
        return out

    return _run(fn, left, right)


def v4_volume(featL, featR, w1, b1, w2, b2, w3, b3, w4, b4, volume_size=48):
    """MobileStereoNetV4's cost volume (model/mobile_stereo_net_v4.py:443-461):
    (N,32,H,W) fp32 x2 -> (N,D,H,W) fp32, slice i = volume11(conv3d(interweave(L[..., i:],
    R[..., :-i]))) at x >= i, 0 elsewhere, from eval-mode-folded weights
    (``model.mobile_stereo_net_v4.fold_v4_weights``)."""
    if _traced():
        return _ops().v4_volume(featL, featR, w1, b1, w2, b2, w3, b3, w4, b4, int(volume_size))
    left, right, dev, code = _pair(featL, featR, "v4_volume")
    if code != _lib.SM_F32:
        raise TypeError("v4_volume: float32 features only")
    D = _disp(volume_size, "v4_volume")
    n, c, h, w = left.shape
    ws = [t.detach().to(device=dev, dtype=torch.float32).contiguous() for t in (w1, b1, w2, b2, w3, b3, w4, b4)]
    shapes = [(16, 8, 3, 3), (16,), (32, 16, 4, 3, 3), (32,), (16, 32, 2, 3, 3), (16,), (16,), (1,)]
    for t, shp in zip(ws, shapes):
        if t.numel() != int(np.prod(shp)):
            raise ValueError(f"v4_volume: weight of {t.numel()} elements, expected shape {shp}")

    def fn():
        out = torch.empty((n, D, h, w), dtype=torch.float32, device=dev)
        if out.numel():
            lib = _lib.load()
            nbytes = int(lib.sm_v4_volume_workspace_bytes(n, h, w))
            scratch = torch.empty(nbytes, dtype=torch.uint8, device=dev)
            _lib.check(lib.sm_v4_volume(
                _ptr(left), _ptr(right), _ptr(out), code, n, c, h, w, D,
                _lib.strides_arg(left), _lib.strides_arg(right), *[_ptr(t) for t in ws],
                _ptr(scratch), nbytes, _stream(dev)), "sm_v4_volume")
        return out

    return _run(fn, left, right)


def difference_volume(left, right, max_disp):
    """(N,C,H,W) x2 -> (N,C,D,H,W): L - R(x-d) for x >= d, 1.0 elsewhere (bit-exact)."""
    if _traced():
        return _ops().difference_volume(left, right, int(max_disp))
    left, right, dev, code = _pair(left, right, "difference_volume")
    D = _disp(max_disp, "difference_volume")
    n, c, h, w = left.shape

    def fn():
        out = torch.empty((n, c, D, h, w), dtype=left.dtype, device=dev)
        if out.numel():
            lib = _lib.load()
            _lib.check(lib.sm_cv_diff(
                _ptr(left), _ptr(right), _ptr(out), code, n, c, h, w, D,
                _lib.strides_arg(left), _lib.strides_arg(right), _stream(dev)), "sm_cv_diff")
        return out

    return _run(fn, left, right)


# ----------------------------------------------------------------------------- a-7, a-8
def _volume(volume, what):
    if not isinstance(volume, torch.Tensor):
        raise TypeError(f"{what}: volume must be a tensor")
    if volume.dim() != 4:
        raise RuntimeError(f"{what}: expected a 4-D (N, D, H, W) volume, got {tuple(volume.shape)}")
    code = _dtype_code(volume)
    dev = _device_check(volume)
    return _stride_ok(_rows_contiguous(volume)), dev, code


def _regress(volume, flags, what):
    vol, dev, code = _volume(volume, what)
    n, d, h, w = vol.shape
    odt = vol.dtype
    if _autocast_fp32(vol):  # autocast: F.softmax / torch.sum run in fp32 (see _autocast_fp32)
        flags |= _lib.SM_REGRESS_OUT_F32
        odt = torch.float32

    def fn():
        out = torch.empty((n, h, w), dtype=odt, device=dev)
        if out.numel():
            lib = _lib.load()
            _lib.check(lib.sm_regress_softargmin(
                _ptr(vol), _ptr(out), code, n, d, h, w, flags, _lib.strides_arg(vol), _stream(dev)),
                "sm_regress_softargmin")
        return out

    return _run(fn, vol)


def soft_argmin(volume, keepdim=True):
    """sum_d d * softmax_d(volume) -> (N,1,H,W) (keepdim) or (N,H,W); fp64 accumulation.
    The output has the volume's dtype; under torch autocast an fp16 / bf16 volume gives fp32
    (the reference's autocast F.softmax + torch.sum)."""
    if _traced():
        out = _ops().soft_argmin(volume, _autocast_fp32(volume))
        return out.unsqueeze(1) if keepdim else out
    out = _regress(volume, _lib.SM_REGRESS_SOFTMAX, "soft_argmin")
    return out.unsqueeze(1) if keepdim else out


def regression_presoftmax(prob):
    """sum_d d * prob[:, d] over an already-softmaxed (N,D,H,W) volume -> (N,H,W) (fp32 under
    autocast for an fp16 / bf16 input, the reference's autocast torch.sum)."""
    if _traced():
        return _ops().regression_presoftmax(prob, _autocast_fp32(prob))
    return _regress(prob, _lib.SM_REGRESS_PRESOFTMAXED, "regression_presoftmax")


def _argext(volume, mode, what):
    vol, dev, code = _volume(volume, what)
    n, d, h, w = vol.shape
    if d == 0 and n * h * w > 0:
        raise IndexError(f"{what}: cannot reduce over an empty disparity axis")
    out = torch.empty((n, h, w), dtype=torch.int64, device=dev)
    if out.numel():
        lib = _lib.load()
        _lib.check(lib.sm_regress_argext(_ptr(vol), _ptr(out), code, n, d, h, w, mode,
                                         _lib.strides_arg(vol), _stream(dev)), "sm_regress_argext")
    return out


def hard_argmin(volume):
    """First index of the minimum over D -> (N,H,W) int64 (ties -> lowest d, NaN wins)."""
    if _traced():
        return _ops().hard_argmin(volume)
    return _argext(volume, _lib.SM_ARGMIN, "hard_argmin")


def hard_argmax(volume):
    """First index of the maximum over D -> (N,H,W) int64 (ties -> lowest d, NaN wins)."""
    if _traced():
        return _ops().hard_argmax(volume)
    return _argext(volume, _lib.SM_ARGMAX, "hard_argmax")


# ------------------------------------------------------------------------------ §8f-4 warp
def warp_by_flow_map(image, flow):
    """Warp ``image`` (N,C,Hi,Wi) by a disparity / flow map ``flow`` (N,1|2,H,W) -> (N,C,H,W).

    Mirrors ``warp_by_flow_map`` (tools/warp.py:5-42, model/mobile_stereo_net_v2.py:59-96,
    _v3.py:60-97): grid (x - fx, y - fy) normalised by (w - 1, h - 1), bilinear grid_sample with
    zero padding and align_corners=False, evaluated by ONE HIP kernel (csrc/warp.hip) in fp32;
    the same AssertionError as the reference for a flow with 3+ channels.

    Dtypes: float32 image and flow as they are.  fp16 / bf16 are read as fp32 and sampled in
    fp32: under torch autocast (grid_sample is an autocast fp32 op, so the reference's RefineNet
    warps an fp16 v3 feature map by an fp32 disparity and gets fp32) the output is fp32; without
    autocast image and flow must share one dtype (as grid_sample requires) and the fp32 result is
    rounded once to it.
    """
    if not isinstance(image, torch.Tensor) or not isinstance(flow, torch.Tensor):
        raise TypeError("warp_by_flow_map: image and flow must be tensors")
    if _traced():
        return _ops().warp_by_flow_map(image, flow, _autocast_fp32(image, flow))
    if flow.dim() != 4:
        raise ValueError(f"warp_by_flow_map: expected a 4-D flow map, got {tuple(flow.shape)}")
    n, c, h, w = flow.shape
    assert c == 1 or c == 2, f"invalid flow map dimension 1 or 2 ({c})!"  # tools/warp.py:18
    if image.dim() != 4:
        raise RuntimeError(f"warp_by_flow_map: expected a 4-D image, got {tuple(image.shape)}")
    if image.shape[0] != n:
        raise RuntimeError(f"warp_by_flow_map: image batch {image.shape[0]} != flow batch {n}")
    for t in (image, flow):
        if t.dtype not in _WARP_DTYPES:
            raise TypeError(f"warp_by_flow_map: unsupported dtype {t.dtype}; expected float32, "
                            "float16 or bfloat16")
    dev = _device_check(image, flow)
    if _autocast_fp32(image, flow):
        odt = torch.float32
    elif image.dtype != flow.dtype:
        raise RuntimeError(f"warp_by_flow_map: image ({image.dtype}) and flow ({flow.dtype}) must "
                           "have the same dtype outside autocast (grid_sample's rule)")
    else:
        odt = image.dtype
    # reduced-precision inputs are widened once on the device (exact); the kernel samples fp32
    image = image.float() if image.dtype != torch.float32 else image
    flow = flow.float() if flow.dtype != torch.float32 else flow
    image = _stride_ok(_rows_contiguous(image))
    flow = _stride_ok(_rows_contiguous(flow))
    N, C, Hi, Wi = image.shape
    out = torch.empty((N, C, h, w), dtype=torch.float32, device=dev)
    if out.numel():
        lib = _lib.load()
        # two-channel flows sample a channel-last copy of the image (csrc/warp.hip)
        nws = int(lib.sm_warp_by_flow_workspace_bytes(N, C, Hi, Wi, c))
        ws = torch.empty(nws, dtype=torch.uint8, device=dev) if nws > 0 else None
        _lib.check(lib.sm_warp_by_flow_ws(_ptr(image), _ptr(flow), _ptr(out), _lib.SM_F32, N, C, Hi,
                                          Wi, h, w, c, _lib.strides_arg(image),
                                          _lib.strides_arg(flow), _ptr(ws) if ws is not None else None,
                                          nws, _stream(dev)), "sm_warp_by_flow_ws")
    return out if odt == torch.float32 else out.to(odt)


# ------------------------------------------------------------------- matching by attention
_POSITIONS = (torch.int32, torch.int64)
_TOKEN_DTYPES = {torch.float32: _lib.SM_F32, torch.float16: _lib.SM_F16, torch.bfloat16: _lib.SM_BF16}


def _token_dtype(t, what, name):
    code = _TOKEN_DTYPES.get(t.dtype)
    if code is None:
        raise TypeError(f"{what}: unsupported dtype {t.dtype} of {name}; expected float32, float16 or "
                        "bfloat16")
    return code


def _tensors(what, *named):
    for i in range(1, len(named), 2):
        if not isinstance(named[i], torch.Tensor):
            raise TypeError(f"{what}: {named[i - 1]} must be a tensor")


def _one_device(*ts):
    """The index of the tensors' HIP device; _device_check's errors."""
    index = ts[0].get_device()
    for t in ts:
        if t.get_device() != index or index < 0:
            _device_check(*ts)
    return index


def _on_device(fn):
    """Run ``fn(index, ...)`` with device ``index`` the current one (where its launches go)."""
    def run(index, *args):
        if torch.cuda.current_device() == index:
            return fn(index, *args)
        with torch.cuda.device(index):
            return fn(index, *args)
    return run


def _token_ready(t, group=1):
    """(tensor, its (batch, token, head) strides): unit stride of the values, the others and the
    address multiples of 16 bytes, 64 rows of ``group`` heads within 2^31 bytes -- a copy where they
    are not."""
    if group == 1 and t.data_ptr() % 16 == 0 and t.is_contiguous():
        return t, None
    per = 16 // t.element_size()
    st = tuple(0 if n == 1 else s for n, s in zip(t.shape[:3], t.stride()))
    if ((t.stride(3) == 1 or t.shape[3] == 1) and t.data_ptr() % 16 == 0
            and st[0] % per == 0 and st[1] % per == 0 and st[2] % per == 0
            and st[1] < (1 << 24) // t.element_size() and (group == 1 or st[2] * group < (1 << 27))):
        return t, _lib.int64s(*st)
    return t.clone(memory_format=torch.contiguous_format), None


def _no_tangents(what, *ts):
    """Refuse tensors with a tangent: the launch would drop it without a word."""
    if forward_ad._current_level >= 0:
        for t in ts:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise NotImplementedError(f"{what}: no forward-mode derivatives, reverse mode only")


def _first_order(fn):
    """once_differentiable, without its cost where no second derivative can follow."""
    with_graph = once_differentiable(fn)

    def backward(ctx, *grads):
        _no_tangents("backward", *grads)
        return with_graph(ctx, *grads) if torch.is_grad_enabled() else fn(ctx, *grads)
    return backward


def _grads_wanted(*ts):
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in ts)


@_on_device
def _attention_forward(index, q, k, v, lengths, mask, scale, band, want_lse):
    b, lq, h, d = q.shape
    lk, kv = k.shape[1], k.shape[2]
    out = q.new_empty((b, lq, h, d))
    lse = q.new_empty((b, kv, lq * (h // kv)) if kv else (b, 0, 0), dtype=torch.float32) if want_lse else None
    if out.numel():
        lib = _lib.load()
        q, qs = _token_ready(q)
        k, ks = _token_ready(k)
        v, vs = _token_ready(v)
        nws = lib.sm_cross_attention_workspace_bytes(b, lq, lk, h, kv, d)
        ws = q.new_empty(nws, dtype=torch.uint8) if nws else None
        _lib.check(lib.sm_cross_attention(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), lse.data_ptr() if want_lse else None,
            _TOKEN_DTYPES[q.dtype], b, lq, lk, h, kv, d, qs, ks, vs, scale, band,
            None if lengths is None else lengths.data_ptr(), None if mask is None else mask.data_ptr(),
            ws.data_ptr() if nws else None, nws, _raw_stream(index)), "sm_cross_attention")
    return out, lse


@_on_device
def _attention_backward(index, q, k, v, out, lse, dout, lengths, mask, scale, band):
    b, lq, h, d = q.shape
    lk, kv = k.shape[1], k.shape[2]
    dq = q.new_empty((b, lq, h, d))
    dk = q.new_empty((b, lk, kv, d))
    dv = q.new_empty((b, lk, kv, d))
    if dq.numel() or dk.numel():
        lib = _lib.load()
        group = h // kv if kv else 1
        q, qs = _token_ready(q, group)
        k, ks = _token_ready(k)
        v, vs = _token_ready(v)
        dout, gs = _token_ready(dout, group)
        nws = lib.sm_cross_attention_backward_workspace_bytes(b, lq, h, kv)
        ws = q.new_empty(nws, dtype=torch.uint8) if nws else None
        _lib.check(lib.sm_cross_attention_backward(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), lse.data_ptr(), dout.data_ptr(),
            dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), _TOKEN_DTYPES[q.dtype], b, lq, lk, h, kv, d, qs, ks,
            vs, gs, scale, band, None if lengths is None else lengths.data_ptr(),
            None if mask is None else mask.data_ptr(), ws.data_ptr() if nws else None, nws,
            _raw_stream(index)), "sm_cross_attention_backward")
    return dq, dk, dv


class _CrossAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, lengths, mask, scale, band):
        out, lse = _attention_forward(q.get_device(), q, k, v, lengths, mask, scale, band, True)
        ctx.save_for_backward(q, k, v, out, lse, lengths, mask)
        ctx.scale, ctx.band = scale, band
        ctx.mark_non_differentiable(lse)
        return out, lse

    @staticmethod
    @_first_order
    def backward(ctx, dout, _):
        q, k, v, out, lse, lengths, mask = ctx.saved_tensors
        return (*_attention_backward(q.get_device(), q, k, v, out, lse, dout, lengths, mask, ctx.scale, ctx.band),
                None, None, None, None)


def _attention_checks(query, key, value, scale, max_disparity, key_lengths, key_mask):
    what = "cross_attention"
    _tensors(what, "query", query, "key", key, "value", value)
    qshape, kshape = query.shape, key.shape
    if len(qshape) != 4 or len(kshape) != 4:
        raise RuntimeError(f"{what}: expected (B, L, heads, D) tokens, got {tuple(qshape)} and "
                           f"{tuple(kshape)}")
    if kshape != value.shape:
        raise RuntimeError(f"{what}: key/value shape mismatch {tuple(kshape)} vs {tuple(value.shape)}")
    b, lq, h, d = qshape
    kb, lk, kv, kd = kshape
    if kb != b or kd != d:
        raise RuntimeError(f"{what}: query {tuple(query.shape)} and key {tuple(key.shape)} differ in batch "
                           "or head width")
    if (h % kv if kv else h) != 0:
        raise RuntimeError(f"{what}: {h} query heads are not a multiple of {kv} key heads")
    if d % 8 != 0 or not 8 <= d <= 128:
        raise RuntimeError(f"{what}: the head width must be a multiple of 8, 8 to 128, got {d}")
    if key.dtype != query.dtype or value.dtype != query.dtype:
        raise RuntimeError(f"{what}: dtype mismatch {query.dtype}, {key.dtype}, {value.dtype}")
    _token_dtype(query, what, "query")
    scale = d ** -0.5 if scale is None else float(scale)
    if not 0.0 < scale < 3.4e38:
        raise ValueError(f"{what}: the scale must be positive and finite, got {scale}")
    band = 0
    if max_disparity is not None:
        band = int(max_disparity)
        if not 1 <= band < 1 << 30:
            raise ValueError(f"{what}: max_disparity must be positive, got {band}")
    if key_lengths is not None:
        _tensors(what, "key_lengths", key_lengths)
        if key_lengths.shape != (b,) or key_lengths.dtype not in (torch.int32, torch.int64):
            raise RuntimeError(f"{what}: key_lengths must be {b} int32 or int64 values, got "
                               f"{tuple(key_lengths.shape)} {key_lengths.dtype}")
    if key_mask is not None:
        _tensors(what, "key_mask", key_mask)
        if key_mask.shape != (b, lk) or key_mask.dtype != torch.bool:
            raise RuntimeError(f"{what}: key_mask must be ({b}, {lk}) truth values, got "
                               f"{tuple(key_mask.shape)} {key_mask.dtype}")
    _no_tangents(what, query, key, value)
    index = _one_device(query, key, value)
    if key_lengths is not None:
        _one_device(query, key_lengths)
        if key_lengths.dtype == torch.int64:
            key_lengths = key_lengths.clamp(0, lk).to(torch.int32)
        key_lengths = key_lengths.contiguous()
    if key_mask is not None:
        _one_device(query, key_mask)
        key_mask = key_mask.contiguous()
    return index, scale, band, key_lengths, key_mask


def cross_attention(query, key, value, scale=None, max_disparity=None, key_lengths=None,
                    key_mask=None, return_lse=False):
    """Attention of one view's tokens to another's: (B,Lq,H,D), (B,Lk,KV,D) x2 -> (B,Lq,H,D).

    ``out[b,i,h] = sum_j p_ij value[b,j,kv]`` with ``p_i`` the softmax of ``scale * query[b,i,h] .
    key[b,j,kv]`` over the allowed keys j, and ``kv = h // (H // KV)``: KV divides H, and query heads
    share key heads.  ``scale``: D ** -0.5 by default.  Key j is allowed for token i where

    - ``j < key_lengths[b]`` ((B,) int32 / int64, taken into 0 .. Lk): states padded to Lk,
    - ``key_mask[b, j]`` ((B, Lk) bool): holes, e.g. invalid columns, and
    - ``0 <= i - j < max_disparity``: the band of candidates of a cost volume's row.

    A row without an allowed key gives 0.  Keys and values at positions past the length or masked are
    never read, whatever they hold (NaN included); those inside, and queries and gradients, have to be
    finite where the band separates them from some of their 128 neighbours.  A row of a channels-last
    feature map is one sequence: ``feat.permute(0, 2, 3, 1).reshape(N * H, W, heads, C // heads)`` is a
    view, and with ``max_disparity`` the call is the inner-product volume, its softmax over disparities
    and a weighted sum of values in one pass.

    D is a multiple of 8 up to 128; any strides (a copy is made where the values are not contiguous
    or rows not 16-byte aligned).  fp32, fp16 or bf16 with scores, statistics and sums in fp32; the
    weights enter the second product rounded to the inputs' type.  Differentiable once, in reverse mode,
    in query, key and value, with the same bits on every run.  ``return_lse``: also the (B,Lq,H) fp32
    logarithm of the softmax's sum (-inf for an empty row; not differentiable), which joins parts of the
    keys.
    """
    if _traced():
        out, lse = _ops().cross_attention(query, key, value, key_lengths, key_mask, scale, max_disparity)
    else:
        index, scale, band, lengths, mask = _attention_checks(query, key, value, scale, max_disparity,
                                                              key_lengths, key_mask)
        if _grads_wanted(query, key, value):
            out, lse = _CrossAttention.apply(query, key, value, lengths, mask, scale, band)
        else:
            out, lse = _attention_forward(index, query, key, value, lengths, mask, scale, band, return_lse)
    if not return_lse:
        return out
    b, lq, h, _ = query.shape
    kv = key.shape[2]
    lse = lse.view(b, kv, lq, h // kv).permute(0, 2, 1, 3).reshape(b, lq, h) if kv else lse.reshape(b, lq, 0)
    return out, lse


# ------------------------------------------------------------------------------ rotary positions
def rotary_frequencies(dim, base=10000.0, scaling=None, factor=1.0, original_length=None, low=1.0,
                       high=32.0, device=None):
    """The ``dim // 2`` frequencies (radians a position, float64) that ``rotary`` turns ``dim`` values
    by: ``base ** (-2 n / dim)``, scaled for contexts ``factor`` times longer than was trained for:

    - ``None``: not at all;
    - ``"linear"``: all divided by ``factor`` (positions are interpolated);
    - ``"base"``: of the larger base ``base * factor ** (dim / (dim - 2))``, which divides the lowest
      by ``factor`` and leaves the highest;
    - ``"parts"``: divided by ``factor`` where a pair makes fewer than ``low`` turns over
      ``original_length`` positions, left where it makes more than ``high``, in between in proportion.
    """
    dim = int(dim)
    if dim < 2 or dim % 2:
        raise ValueError(f"rotary_frequencies: dim must be even and positive, got {dim}")
    if not (math.isfinite(base) and base > 0 and math.isfinite(factor) and factor > 0):
        raise ValueError("rotary_frequencies: base and factor must be positive and finite")
    if scaling not in (None, "linear", "base", "parts"):
        raise ValueError("rotary_frequencies: scaling must be None, 'linear', 'base' or 'parts'")
    if scaling == "base":
        if dim == 2:
            raise ValueError("rotary_frequencies: 'base' needs more than one pair")
        base = base * factor ** (dim / (dim - 2))
    f = torch.tensor([base ** (-2.0 * n / dim) for n in range(dim // 2)], dtype=torch.float64)
    if scaling == "linear":
        f = f / factor
    elif scaling == "parts":
        if original_length is None or original_length <= 0 or not 0 <= low < high:
            raise ValueError("rotary_frequencies: 'parts' needs original_length > 0 and 0 <= low < high")
        turns = original_length * f / (2 * math.pi)
        keep = ((turns - low) / (high - low)).clamp(0, 1)
        f = f * (keep + (1 - keep) / factor)
    return f.to(device) if device is not None else f


@_on_device
def _rotary_run(index, x, positions, frequencies, interleaved, amplitude, inverse):
    b, l, h, d = shape = x.shape
    y = x.new_empty(shape)
    if b and l and h:
        st = None
        if not x.is_contiguous():
            if x.stride(3) != 1 and d > 1:
                x = x.contiguous()
            else:
                st = _lib.int64s(*(0 if n == 1 else s for n, s in zip(shape, x.stride()[:3])))
        flags = ((_lib.SM_ROTARY_INTERLEAVED if interleaved else 0)
                 | (_lib.SM_ROTARY_INVERSE if inverse else 0)
                 | (_lib.SM_ROTARY_POS64 if positions.dtype == torch.int64 else 0))
        ps = positions.stride(0) if b > 1 and positions.dim() == 2 else 0
        rc = _lib.load().sm_rotary(
            x.data_ptr(), positions.data_ptr(), frequencies.data_ptr(), y.data_ptr(), _TOKEN_DTYPES[x.dtype],
            b, l, h, d, 2 * frequencies.shape[0], st, ps, flags, amplitude, _raw_stream(index))
        if rc:
            _lib.check(rc, "sm_rotary")
    return y


def _rotary_checks(x, positions, frequencies, layout):
    """(device index, positions, frequencies) as the kernel takes them, or the refusal: for the turn and
    the turn back."""
    what = "rotary"
    _tensors(what, "x", x, "positions", positions, "frequencies", frequencies)
    shape, pshape = x.shape, positions.shape
    if len(shape) != 4:
        raise RuntimeError(f"{what}: expected (B, L, heads, D) tokens, got {tuple(shape)}")
    _token_dtype(x, what, "x")
    b, l, _, d = shape
    if (positions.dtype not in _POSITIONS or pshape[-1:] != (l,)
            or not (len(pshape) == 1 or (len(pshape) == 2 and pshape[0] == b))):
        raise RuntimeError(f"{what}: positions must be ({l},) or ({b}, {l}) int32 or int64, got "
                           f"{tuple(pshape)} {positions.dtype}")
    if frequencies.dtype != torch.float64 or frequencies.dim() != 1:
        raise RuntimeError(f"{what}: frequencies must be one row of float64, got "
                           f"{tuple(frequencies.shape)} {frequencies.dtype}")
    if not 2 <= 2 * frequencies.shape[0] <= d:
        raise RuntimeError(f"{what}: {frequencies.shape[0]} pairs do not fit heads of {d} values")
    if layout not in ("half", "interleaved"):
        raise ValueError(f"{what}: layout must be 'half' or 'interleaved'")
    if frequencies.requires_grad:
        raise RuntimeError(f"{what}: frequencies have no gradient")
    _no_tangents(what, x, frequencies)
    index = _one_device(x, positions, frequencies)
    if positions.stride(-1) != 1:
        positions = positions.contiguous()
    if not frequencies.is_contiguous():
        frequencies = frequencies.contiguous()
    return index, positions, frequencies


class _Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, positions, frequencies, interleaved, amplitude):
        ctx.save_for_backward(positions, frequencies)
        ctx.how = interleaved, amplitude
        return _rotary_run(x.get_device(), x, positions, frequencies, interleaved, amplitude, False)

    @staticmethod
    @_first_order
    def backward(ctx, dy):
        return (_rotary_run(dy.get_device(), dy, *ctx.saved_tensors, *ctx.how, True), None, None, None, None)


def rotary(x, positions, frequencies, layout="half", amplitude=1.0):
    """Rotary positions of (B,L,heads,D) tokens: the first ``2 * len(frequencies)`` values of every
    head are turned in pairs by ``positions * frequencies`` radians, the others pass through.

    ``positions``: (L,) or (B,L) int32 / int64; ``frequencies``: float64 on the tokens' device, kept by
    the caller (``rotary_frequencies``).  ``layout``: ``"half"`` pairs value n with n + R/2,
    ``"interleaved"`` 2n with 2n + 1.  ``amplitude`` multiplies the turned values.  The angle is formed
    in 64 bits, so far positions are as exact as near ones; one rounding, to the tokens' type.
    Differentiable in x (reverse mode).
    """
    if _traced():
        return _ops().rotary(x, positions, frequencies, layout, float(amplitude))
    index, positions, frequencies = _rotary_checks(x, positions, frequencies, layout)
    interleaved, amplitude = layout == "interleaved", float(amplitude)
    if x.requires_grad and torch.is_grad_enabled():
        return _Rotary.apply(x, positions, frequencies, interleaved, amplitude)
    return _rotary_run(index, x, positions, frequencies, interleaved, amplitude, False)


# ------------------------------------------------------------------------------------- RMS norm
def _rows(t, c):
    """(the tensor as rows of c contiguous values, their stride)."""
    if t.is_contiguous():
        return t, c
    t = t.reshape(-1, c)
    if c > 1 and t.stride(1) != 1:
        t = t.contiguous()
    return t, t.stride(0) if t.shape[0] > 1 else c


def _norm_checks(what, x, weight, residual, eps):
    _tensors(what, "x", x, "weight", weight)
    if residual is not None:
        _tensors(what, "residual", residual)
    shape, dtype = x.shape, x.dtype
    if weight.dim() != 1 or shape[-1:] != weight.shape:
        raise RuntimeError(f"{what}: expected (..., C) rows and (C,) weight, got {tuple(shape)} and "
                           f"{tuple(weight.shape)}")
    if not 1 <= shape[-1] <= 65536:
        raise RuntimeError(f"{what}: rows of 1 to 65536 values, got {shape[-1]}")
    _token_dtype(x, what, "x")
    if weight.dtype not in (dtype, torch.float32):
        raise TypeError(f"{what}: weight must be {dtype} or float32, got {weight.dtype}")
    if residual is not None:
        if residual.dtype not in (dtype, torch.float32):
            raise TypeError(f"{what}: residual must be {dtype} or float32, got {residual.dtype}")
        if residual.shape != shape:
            raise RuntimeError(f"{what}: x/residual shape mismatch {tuple(shape)} vs {tuple(residual.shape)}")
    if not 0.0 <= float(eps) < 3.4e38:
        raise ValueError(f"{what}: eps must be finite and not negative, got {eps}")
    _no_tangents(what, x, weight, residual)
    return _one_device(x, weight) if residual is None else _one_device(x, weight, residual)


@_on_device
def _norm_forward(index, x, weight, residual, eps, e4m3=None):
    """(y, summed or None), or with ``e4m3`` (the group) (q, scales, summed or None)."""
    shape, code = x.shape, _TOKEN_DTYPES[x.dtype]
    c = shape[-1]
    summed = None if residual is None else residual.new_empty(shape)
    if e4m3 is None:
        y, scales = x.new_empty(shape), None
    else:
        y = x.new_empty(shape, dtype=torch.float8_e4m3fn)
        scales = x.new_empty((*shape[:-1], -(-c // e4m3) if e4m3 else 1), dtype=torch.float32)
    n = y.numel() // c
    if n:
        x, xs = _rows(x, c)
        rcode, rs, rp, sp = code, c, None, None
        if residual is not None:
            residual, rs = _rows(residual, c)
            rcode, rp, sp = _TOKEN_DTYPES[residual.dtype], residual.data_ptr(), summed.data_ptr()
        if not weight.is_contiguous():
            weight = weight.contiguous()
        lib = _lib.load()
        if e4m3 is None:
            rc = lib.sm_rms_norm(x.data_ptr(), rp, weight.data_ptr(), y.data_ptr(), sp, code, rcode,
                                 _TOKEN_DTYPES[weight.dtype], n, c, xs, rs, eps, _raw_stream(index))
        else:
            rc = lib.sm_rms_norm_e4m3(
                x.data_ptr(), rp, weight.data_ptr(), y.data_ptr(), scales.data_ptr(), sp, code, rcode,
                _TOKEN_DTYPES[weight.dtype], n, c, xs, rs, e4m3, eps, _raw_stream(index))
        if rc:
            _lib.check(rc, "sm_rms_norm")
    return (y, summed) if e4m3 is None else (y, scales, summed)


@_on_device
def _norm_backward(index, summed, weight, dy, dsummed, dtype, eps):
    """(dx, dresidual in summed's type or None where that is dx, dweight)."""
    c = summed.shape[-1]
    dx = summed.new_empty(summed.shape, dtype=dtype)
    dres = None if summed.dtype == dtype else summed.new_empty(summed.shape)
    dw = weight.new_empty(weight.shape)
    n = summed.numel() // c
    lib = _lib.load()
    nws = lib.sm_rms_norm_backward_workspace_bytes(n, c)
    ws = summed.new_empty(nws, dtype=torch.uint8) if nws else None
    summed, ss = _rows(summed, c)
    dy, ys = _rows(dy, c)
    zs, zp = c, None
    if dsummed is not None:
        dsummed, zs = _rows(dsummed, c)
        zp = dsummed.data_ptr()
    weight = weight.contiguous()
    _lib.check(lib.sm_rms_norm_backward(
        summed.data_ptr(), weight.data_ptr(), dy.data_ptr(), zp, dx.data_ptr(),
        None if dres is None else dres.data_ptr(), dw.data_ptr(), _TOKEN_DTYPES[dtype],
        _TOKEN_DTYPES[summed.dtype], _TOKEN_DTYPES[weight.dtype], n, c, ss, ys, zs, eps,
        ws.data_ptr() if nws else None, nws, _raw_stream(index)), "sm_rms_norm_backward")
    return dx, dres, dw


class _RmsNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, eps):
        ctx.save_for_backward(x, weight)
        ctx.eps = eps
        return _norm_forward(x.get_device(), x, weight, None, eps)[0]

    @staticmethod
    @_first_order
    def backward(ctx, dy):
        x, weight = ctx.saved_tensors
        dx, _, dw = _norm_backward(x.get_device(), x, weight, dy, None, x.dtype, ctx.eps)
        return dx, dw, None


class _AddRmsNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, residual, eps):
        y, summed = _norm_forward(x.get_device(), x, weight, residual, eps)
        ctx.save_for_backward(summed, weight)
        ctx.eps, ctx.dtype = eps, x.dtype
        ctx.set_materialize_grads(False)
        return y, summed

    @staticmethod
    @_first_order
    def backward(ctx, dy, dsummed):
        summed, weight = ctx.saved_tensors
        if dy is None:  # only the stream was used
            if dsummed is None:
                return None, None, None, None
            return dsummed.to(ctx.dtype), torch.zeros_like(weight), dsummed, None
        dx, dres, dw = _norm_backward(summed.get_device(), summed, weight, dy, dsummed, ctx.dtype, ctx.eps)
        return dx, dw, dx if dres is None else dres, None


def rms_norm(x, weight, residual=None, eps=1e-6):
    """Root-mean-square norm of (..., C) rows: ``y = s / sqrt(mean(s^2) + eps) * weight``.

    Without a residual ``s = x`` and y is returned.  With one ``s = x + residual``, rounded to the
    residual's type, and ``(y, s)`` is returned: s is the stream that the next layer adds to, and y is
    the norm of s as it is handed on.  x is fp32, fp16 or bf16, y has its type; weight (C,) and
    residual have it or are fp32 (a 32-bit stream beside 16-bit layers).  C is 1 to 65536; sums are
    fp32.  Differentiable once, in reverse mode, in x, weight and residual (weight's gradient is summed
    in one order).
    """
    if _traced():
        if residual is None:
            return _ops().rms_norm(x, weight, float(eps))
        return _ops().add_rms_norm(x, weight, residual, float(eps))
    index = _norm_checks("rms_norm", x, weight, residual, eps)
    eps = float(eps)
    if residual is None:
        if _grads_wanted(x, weight):
            return _RmsNorm.apply(x, weight, eps)
        return _norm_forward(index, x, weight, None, eps)[0]
    if _grads_wanted(x, weight, residual):
        return _AddRmsNorm.apply(x, weight, residual, eps)
    return _norm_forward(index, x, weight, residual, eps)


def rms_norm_e4m3(x, weight, residual=None, eps=1e-6, group=None):
    """``rms_norm`` with y in 8 bits, for a product that takes them: ``(q, scales)``, or ``(q, scales,
    s)`` with a residual, where ``y ~ q * scales``.

    q is (..., C) float8_e4m3fn: ``s w * 448 / max|s w|``, formed in 64 bits and rounded to 32 and then to 8;
    a scale is max|y| / 448 (rounded to fp32 by itself) over the row (``group=None``; scales (..., 1)) or
    over each 128 values of it (``group=128``; scales (..., ceil(C / 128))), and 1 where y is 0.  Forward only: x and residual that require a gradient are
    refused, and the backward pass of a weight's raises.
    """
    if group not in (None, 128):
        raise ValueError(f"rms_norm_e4m3: group must be None (a row) or 128, got {group}")
    if _traced():
        if residual is None:
            return _ops().rms_norm_e4m3(x, weight, float(eps), group or 0)
        return _ops().add_rms_norm_e4m3(x, weight, residual, float(eps), group or 0)
    index = _norm_checks("rms_norm_e4m3", x, weight, residual, eps)
    if _grads_wanted(x, residual):
        raise NotImplementedError("rms_norm_e4m3 is forward only: call it under torch.no_grad()")
    args = index, x, weight, residual, float(eps), group or 0
    out = _ForwardOnly.apply(lambda: _norm_forward(*args), weight) if _grads_wanted(weight) else _norm_forward(*args)
    return out[:2] if residual is None else out
