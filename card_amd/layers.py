"""Layer operators of guidance networks and conditional heads on the device: dropout with a mask that is never stored
(card_dropout), root-mean-square norm with the residual's addition (card_rms_norm) and products of few rows with 4-bit
weights (card_linear4).

All take fp32, bf16 and fp16 tensors on the GPU, launch on the current stream of the tensor's device, never synchronise and
raise CardError for what the kernels do not cover.  `dropout` and `rms_norm` have a backward pass (of first order);
`rms_norm_e4m3` and `QuantLinear` are for inference and refuse tensors that ask for a gradient.  Tensors that are not
contiguous are copied first, as everywhere in card_amd.
"""
import ctypes as C
import weakref

import torch

from . import _lib
from ._lib import CardError
from .sampler import _dev_f32, _require_cuda

E4M3_MAX = 448.0

_DTYPES = {torch.float32: _lib.DTYPE_F32, torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_F16}


def _dtype(t, name):
    d = _DTYPES.get(t.dtype)
    if d is None:
        raise CardError(f"{name}: dtype {t.dtype} is none of float32, bfloat16, float16")
    return d


def _current_stream(index):
    return torch.cuda.current_stream(index).cuda_stream


# the handle alone, without the Stream object around it: 0.1 us instead of 1.9
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", _current_stream)


def _call(device, fn, what, *args):
    """fn(*args, current stream of `device`) with that device current"""
    index = device.index
    if torch.cuda.current_device() == index:
        status = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(device):
            status = fn(*args, _raw_stream(index))
    if status != _lib.CARD_OK:
        _lib.check(status, what)


def _same(t, like, shape, name):
    if t.shape != shape or t.dtype is not like.dtype or t.device != like.device:
        raise CardError(f"{name}: expected {tuple(shape)} {like.dtype} on {like.device}, got {tuple(t.shape)} {t.dtype} on {t.device}")
    return t if t.is_contiguous() else t.contiguous()


def _wants_grad(*tensors):
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


# ------------------------------------------------------------------------------------------------ dropout
def _dropout_forward(x, residual, state, key):
    dt, rows, cols, n_z, p, seed, elem_offset, draw = key
    y = torch.empty_like(x) if n_z == 1 else x.new_empty(x.shape[:-1] + (n_z, cols))
    _call(x.device, _lib.lib().card_dropout, "card_dropout", x.data_ptr(), residual.data_ptr() if residual is not None else None,
          y.data_ptr(), dt, rows, cols, n_z, p, seed, elem_offset, state.data_ptr() if state is not None else None, draw)
    return y


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, state, key):
        ctx.key, ctx.shape = key, x.shape
        ctx.save_for_backward(state)          # numbers written into it before the backward pass are noticed
        return _dropout_forward(x, residual, state, key)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g):
        dt, rows, cols, n_z, p, seed, elem_offset, draw = ctx.key
        (state,) = ctx.saved_tensors
        dx = None
        if ctx.needs_input_grad[0]:
            gc = g.contiguous()
            dx = torch.empty(ctx.shape, dtype=g.dtype, device=g.device)
            _call(g.device, _lib.lib().card_dropout_backward, "card_dropout_backward", gc.data_ptr(), dx.data_ptr(), dt, rows, cols,
                  n_z, p, seed, elem_offset, state.data_ptr() if state is not None else None, draw)
        return dx, g if ctx.needs_input_grad[1] else None, None, None


def dropout(x, p, *, seed, elem_offset=0, draw=0, n_z=1, residual=None):
    """residual + keep * x / (1 - p): card_dropout.  x is (..., cols); with n_z > 1 every row gets n_z masks and the result
    is (..., n_z, cols), as the sampler expands a row to n_z chains.

    The mask is a function of (seed, elem_offset + index of the output element, draw) alone, like the sampler's normals: the
    same three give the same mask in the backward pass, on every device and under any sharding, and nothing is stored.  Give
    each layer of a step its own `draw` and each step its own seed.  `seed` is an int (modulo 2^64), or an int64 tensor of two
    numbers {seed, element offset} on x's device that the kernels read when they run: a captured graph then draws new masks
    when the program writes new numbers into it.  A dropped element is 0 even where x is infinite or NaN.  The keep
    probability has 32 bits.  `residual` (of the result's shape and type) is added in 32 bits before the only rounding."""
    _require_cuda(x.device)
    dt = _dtype(x, "dropout")
    n_z, draw, elem_offset = int(n_z), int(draw), int(elem_offset)
    if x.dim() < 1:
        raise CardError("dropout: x is a scalar; expected (..., cols)")
    if n_z < 1 or not 0 <= draw < 2 ** 31 or not 0 <= elem_offset < 2 ** 63 or n_z >= 2 ** 31:
        raise CardError(f"dropout: n_z={n_z}, draw={draw} or elem_offset={elem_offset} out of range")
    state = None
    if torch.is_tensor(seed):
        state, seed = seed, 0
        if state.dtype is not torch.int64 or state.numel() != 2 or state.device != x.device or not state.is_contiguous():
            raise CardError(f"dropout: a seed tensor holds two int64 numbers on {x.device}, got {tuple(state.shape)} {state.dtype} on {state.device}")
    cols = int(x.shape[-1])
    if residual is not None:
        residual = _same(residual, x, x.shape if n_z == 1 else x.shape[:-1] + (n_z, cols), "dropout: residual")
    xc = x if x.is_contiguous() else x.contiguous()
    key = (dt, xc.numel() // cols if cols else 0, cols, n_z, float(p), int(seed) & (2 ** 64 - 1), elem_offset, draw)
    if _wants_grad(x, residual):
        return _Dropout.apply(xc, residual, state, key)
    return _dropout_forward(xc, residual, state, key)


# ------------------------------------------------------------------------------------------------ norm
def _norm_forward(x, residual, weight, eps, e4m3):
    cols = int(x.shape[-1])
    rows = x.numel() // cols
    h = torch.empty_like(x) if residual is not None else None
    scale = torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device) if e4m3 else None
    y = torch.empty_like(x, dtype=torch.float8_e4m3fn) if e4m3 else torch.empty_like(x)
    dt = _DTYPES[x.dtype]
    _call(x.device, _lib.lib().card_rms_norm, "card_rms_norm", x.data_ptr(), residual.data_ptr() if h is not None else None,
          weight.data_ptr() if weight is not None else None, dt, _DTYPES[weight.dtype] if weight is not None else dt, rows, cols, eps,
          h.data_ptr() if h is not None else None, y.data_ptr(), _lib.DTYPE_E4M3 if e4m3 else dt, scale.data_ptr() if e4m3 else None)
    return y, scale, h


class _RmsNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, eps):
        y, _, h = _norm_forward(x, residual, weight, eps, False)
        ctx.save_for_backward(x if h is None else h, weight)
        ctx.eps = eps
        ctx.set_materialize_grads(False)
        return y if h is None else (y, h)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g, gh=None):
        h, weight = ctx.saved_tensors
        cols = int(h.shape[-1])
        rows = h.numel() // cols
        dt, wt = _DTYPES[h.dtype], _DTYPES[h.dtype if weight is None else weight.dtype]
        g = g if g is None else g.contiguous()
        gh = gh if gh is None else gh.contiguous()
        dx = torch.empty_like(h)
        dw = ws = None
        nbytes = C.c_uint64()
        if ctx.needs_input_grad[2]:
            dw = torch.empty_like(weight)
            _lib.check(_lib.lib().card_rms_norm_backward_workspace_bytes(dt, rows, cols, C.byref(nbytes)), "card_rms_norm_backward_workspace_bytes")
            ws = torch.empty(nbytes.value, dtype=torch.uint8, device=h.device)
        ptr = lambda t: t.data_ptr() if t is not None else None  # noqa: E731
        _call(h.device, _lib.lib().card_rms_norm_backward, "card_rms_norm_backward", h.data_ptr(), ptr(weight), ptr(g), ptr(gh), dt, wt,
              rows, cols, ctx.eps, dx.data_ptr(), ptr(dw), ptr(ws), nbytes.value)
        need = ctx.needs_input_grad
        return dx if need[0] else None, dx if need[1] else None, dw, None


def _norm_args(x, weight, residual, eps, what):
    _require_cuda(x.device)
    _dtype(x, what)
    if x.dim() < 1 or x.shape[-1] < 1:
        raise CardError(f"{what}: x has shape {tuple(x.shape)}; expected (..., cols) with cols >= 1")
    if weight is not None:
        if weight.dim() != 1 or weight.shape[0] != x.shape[-1] or weight.dtype not in (torch.float32, x.dtype) or weight.device != x.device:
            raise CardError(f"{what}: weight: expected ({x.shape[-1]},) {x.dtype} or float32 on {x.device}, got {tuple(weight.shape)} "
                            f"{weight.dtype} on {weight.device}")
        weight = weight if weight.is_contiguous() else weight.contiguous()
    if residual is not None:
        residual = _same(residual, x, x.shape, f"{what}: residual")
    return (x if x.is_contiguous() else x.contiguous()), weight, residual, float(eps)


def rms_norm(x, weight=None, *, residual=None, eps=1e-6):
    """h / sqrt(mean(h^2) + eps) * weight over the last dimension, with h = x + residual: card_rms_norm.  Returns y, or
    (y, h) where a residual is given: h is the next layer's residual.  x, residual, y and h have one type; weight has it too
    or is float32.  Differentiable in x, residual and weight; the backward pass starts from h as it was stored."""
    args = _norm_args(x, weight, residual, eps, "rms_norm")
    if _wants_grad(x, weight, residual):
        return _RmsNorm.apply(args[0], args[2], args[1], args[3])
    y, _, h = _norm_forward(args[0], args[2], args[1], args[3], False)
    return y if h is None else (y, h)


def rms_norm_e4m3(x, weight=None, *, residual=None, eps=1e-6):
    """rms_norm with its result in 8 bits: (q, scale) or (q, scale, h), with q float8_e4m3fn and scale (...,) float32, so that
    q * scale[..., None] stands for y; scale = max |y| / 448 of each row.  What QuantLinear takes as (x, x_scale)."""
    if _wants_grad(x, weight, residual):
        raise CardError("rms_norm_e4m3 has no backward pass; use rms_norm, or torch.no_grad()")
    x, weight, residual, eps = _norm_args(x, weight, residual, eps, "rms_norm_e4m3")
    y, scale, h = _norm_forward(x, residual, weight, eps, True)
    return (y, scale) if h is None else (y, scale, h)


# ------------------------------------------------------------------------------------------------ 4-bit weights
class QuantLinear:
    """A Linear layer with 4-bit weights, packed on one GPU; immutable after construction (card_linear4).

    w[o, k] = (q[o, k] - zero[o, k // group]) * scale[o, k // group]: q (out, in) uint8 with values 0..15, scale (out,
    ceil(in / group)) float32, zero likewise uint8 (0..15) or None = 8 everywhere, bias (out,) or None; group 32, 64 or 128."""

    def __init__(self, q, scale, zero=None, bias=None, *, group, device=None):
        device = torch.device(device) if device is not None else q.device
        _require_cuda(device)
        if q.dim() != 2 or q.dtype is not torch.uint8:
            raise CardError(f"QuantLinear: q is (out, in) uint8, got {tuple(q.shape)} {q.dtype}")
        out_f, in_f = (int(n) for n in q.shape)
        group = int(group)
        if group not in (32, 64, 128):
            raise CardError(f"QuantLinear: group={group} is none of 32, 64, 128")
        groups = -(-in_f // group)
        if tuple(scale.shape) != (out_f, groups):
            raise CardError(f"QuantLinear: scale is ({out_f}, {groups}), got {tuple(scale.shape)}")
        if zero is not None and (tuple(zero.shape) != (out_f, groups) or zero.dtype is not torch.uint8):
            raise CardError(f"QuantLinear: zero is ({out_f}, {groups}) uint8, got {tuple(zero.shape)} {zero.dtype}")
        if bias is not None and tuple(bias.shape) != (out_f,):
            raise CardError(f"QuantLinear: bias is ({out_f},), got {tuple(bias.shape)}")
        keep = [q.to(device).contiguous(), _dev_f32(scale, device), zero if zero is None else zero.to(device).contiguous(),
                bias if bias is None else _dev_f32(bias, device)]
        d = _lib.Linear4Desc()
        d.struct_bytes, d.in_features, d.out_features, d.group = C.sizeof(_lib.Linear4Desc), in_f, out_f, group
        d.q, d.scale, d.zero, d.bias = (None if t is None else t.data_ptr() for t in keep)
        h = C.c_void_p()
        L = _lib.lib()
        self.device = keep[0].device
        # the pack kernels read `keep` on the current stream; the caching allocator is stream-ordered
        _call(self.device, lambda stream: L.card_linear4_create(C.byref(d), stream, C.byref(h)), "card_linear4_create")
        self.in_features, self.out_features, self.group = in_f, out_f, group
        self._h = h.value
        weakref.finalize(self, L.card_linear4_destroy, h)

    @classmethod
    def from_float(cls, weight, bias=None, *, group=128, device=None):
        """The nearest 4-bit weights of a float weight (out, in): card_linear4_quantize, with zero points."""
        device = torch.device(device) if device is not None else weight.device
        return cls(*quantize_weight(_dev_f32(weight, device), group=group), bias, group=group, device=device)

    def forward(self, x, x_scale=None, *, gamma=None, slope=None, out_dtype=None):
        """act(gamma * (x w^T + bias)): card_linear4_forward.  x (..., in) in fp32, bf16 or fp16, or float8_e4m3fn with
        x_scale (...,) float32, the scale of each row; gamma (out,) float32: a ConditionalLinear's embedding row; slope: a
        LeakyReLU's negative slope (0 = ReLU), None = no activation; out_dtype: x's type by default (bf16 for 8-bit rows).
        Made for one to some tens of rows, right for up to 65535."""
        dev = self.device
        if x.device != dev:
            raise CardError(f"QuantLinear: x is on {x.device}, the weights are on {dev}")
        if x.dim() < 1 or x.shape[-1] != self.in_features:
            raise CardError(f"QuantLinear: x has shape {tuple(x.shape)}; expected (..., {self.in_features})")
        if _wants_grad(x, x_scale, gamma):
            raise CardError("QuantLinear has no backward pass; call it under torch.no_grad() or detach its input")
        if x.dtype is torch.float8_e4m3fn:
            xt = _lib.DTYPE_E4M3
            if x_scale is None or x_scale.shape != x.shape[:-1] or x_scale.dtype is not torch.float32 or x_scale.device != dev:
                raise CardError(f"QuantLinear: 8-bit rows come with x_scale {tuple(x.shape[:-1])} float32 on {dev}")
            x_scale = x_scale if x_scale.is_contiguous() else x_scale.contiguous()
        else:
            xt = _dtype(x, "QuantLinear")
            if x_scale is not None:
                raise CardError("QuantLinear: x_scale goes with float8_e4m3fn rows")
        if out_dtype is None:
            out_dtype = torch.bfloat16 if xt == _lib.DTYPE_E4M3 else x.dtype
        yt = _DTYPES.get(out_dtype)
        if yt is None:
            raise CardError(f"QuantLinear: out_dtype {out_dtype} is none of float32, bfloat16, float16")
        if gamma is not None:
            if tuple(gamma.shape) != (self.out_features,) or gamma.dtype is not torch.float32 or gamma.device != dev:
                raise CardError(f"QuantLinear: gamma is ({self.out_features},) float32 on {dev}, got {tuple(gamma.shape)} {gamma.dtype} on {gamma.device}")
            gamma = gamma if gamma.is_contiguous() else gamma.contiguous()
        x = x if x.is_contiguous() else x.contiguous()
        y = torch.empty(x.shape[:-1] + (self.out_features,), dtype=out_dtype, device=dev)
        _call(dev, _lib.lib().card_linear4_forward, "card_linear4_forward", self._h, x.data_ptr(), xt,
              x_scale.data_ptr() if x_scale is not None else None, x.numel() // self.in_features,
              gamma.data_ptr() if gamma is not None else None, 1.0 if slope is None else float(slope), y.data_ptr(), yt)
        return y

    __call__ = forward


def quantize_weight(weight, *, group=128):
    """(q, scale, zero) of a float weight (out, in) on the GPU, as QuantLinear takes them: card_linear4_quantize.  Per group
    of columns scale = (max - min) / 15 over its values and zero, so that zero is exact."""
    _require_cuda(weight.device)
    if weight.dim() != 2 or weight.numel() == 0:
        raise CardError(f"quantize_weight: weight is (out, in), got {tuple(weight.shape)}")
    if int(group) not in (32, 64, 128):
        raise CardError(f"quantize_weight: group={group} is none of 32, 64, 128")
    w = _dev_f32(weight, weight.device)
    out_f, in_f = (int(n) for n in w.shape)
    groups = -(-in_f // int(group))
    q = torch.empty(out_f, in_f, dtype=torch.uint8, device=w.device)
    scale = torch.empty(out_f, groups, dtype=torch.float32, device=w.device)
    zero = torch.empty(out_f, groups, dtype=torch.uint8, device=w.device)
    _call(w.device, _lib.lib().card_linear4_quantize, "card_linear4_quantize", w.data_ptr(), out_f, in_f, int(group), q.data_ptr(),
          scale.data_ptr(), zero.data_ptr())
    return q, scale, zero
