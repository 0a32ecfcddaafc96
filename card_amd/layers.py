"""Layer operators of guidance networks and conditional heads on the device: dropout with a mask that is never stored
(card_dropout), root-mean-square norm with the residual's addition (card_rms_norm) and products of few rows with 4-bit
weights (card_linear4).

All take fp32, bf16 and fp16 tensors on the GPU, launch on the current stream of the tensor's device, never synchronise and
raise CardError for what the kernels do not cover.  `dropout` and `rms_norm` have a backward pass (of first order);
a captured backward pass needs its forward pass in the same capture and no older graph of the same tensors.  Tensors with a
forward-mode tangent and calls under torch.jit.trace are refused.
`rms_norm_e4m3` and `QuantLinear` are for inference and refuse tensors that ask for a gradient.  Tensors that are not
contiguous are copied first, as everywhere in card_amd.
"""
import ctypes as C
import os

import torch

from . import _lib
from ._lib import CardError
from .sampler import _dev_f32, _ptr, _require_cuda, _stream

_EXT_PATH = os.path.join(os.path.dirname(os.path.abspath(__file__)), "_card_torch.so")
_ext = None


def _load():
    """The torch binding of the operators (csrc/card_torch.cpp), bound to the library that _lib.lib() loads."""
    global _ext
    if _ext is None:
        L = _lib.lib()
        if not os.path.exists(_EXT_PATH):
            raise CardError(f"{_EXT_PATH} is missing: build it with `make -C card_amd/csrc` (or __graft_entry__.build()).")
        from . import _card_torch
        names = ("card_last_error", "card_dropout", "card_dropout_backward", "card_rms_norm", "card_rms_norm_backward",
                 "card_rms_norm_backward_workspace_bytes", "card_linear4_forward", "card_linear4_workspace_bytes")
        _card_torch.init({n: C.cast(getattr(L, n), C.c_void_p).value for n in names}, CardError)
        _ext = _card_torch
    return _ext


def dropout(x, p, *, seed, elem_offset=0, draw=0, n_z=1, residual=None):
    """residual + keep * x / (1 - p): card_dropout.  x is (..., cols); with n_z > 1 every row gets n_z masks and the result
    is (..., n_z, cols), as the sampler expands a row to n_z chains.

    The mask is a function of (seed, elem_offset + index of the output element, draw) alone, like the sampler's normals: the
    same three give the same mask in the backward pass, on every device and under any sharding, and nothing is stored.  Give
    each layer of a step its own `draw` and each step its own seed.  `seed` is an int (modulo 2^64), or an int64 tensor of two
    numbers {seed, element offset} on x's device that the kernels read when they run: a captured graph then draws new masks
    when the program writes new numbers into it.  A dropped element is 0 even where x is infinite or NaN.  The keep
    probability has 32 bits.  `residual` (of the result's shape and type) is added in 32 bits before the only rounding."""
    state = None
    if torch.is_tensor(seed):
        state, seed = seed, 0
    return (_ext or _load()).dropout(x, p, int(seed) & 0xFFFFFFFFFFFFFFFF, state, elem_offset, draw, n_z, residual)


def rms_norm(x, weight=None, *, residual=None, eps=1e-6):
    """h / sqrt(mean(h^2) + eps) * weight over the last dimension, with h = x + residual: card_rms_norm.  Returns y, or
    (y, h) where a residual is given: h is the next layer's residual.  x, residual, y and h have one type; weight has it too
    or is float32.  Differentiable in x, residual and weight; the backward pass starts from h as it was stored."""
    out = (_ext or _load()).rms_norm(x, weight, residual, eps)
    return tuple(out) if residual is not None else out[0]


def rms_norm_e4m3(x, weight=None, *, residual=None, eps=1e-6):
    """rms_norm with its result in 8 bits: (q, scale) or (q, scale, h), with q float8_e4m3fn and scale (...,) float32, so that
    q * scale[..., None] stands for y; scale = max |y| / 448 of each row (2^-140 at least; 0 for a row of zeros).  What QuantLinear takes as (x, x_scale)."""
    return tuple((_ext or _load()).rms_norm_e4m3(x, weight, residual, eps))


class QuantLinear:
    """A Linear layer with 4-bit weights, packed on one GPU (on the current stream); immutable after construction
    (card_linear4).  It holds the weights that a captured graph reads: keep it as long as the graph.  copy.copy shares them;
    deep copies and pickles are refused.

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
        with torch.cuda.device(self.device):
            _lib.check(L.card_linear4_create(C.byref(d), _stream(self.device), C.byref(h)), "card_linear4_create")
        self._index = self.device.index
        self.in_features, self.out_features, self.group = in_f, out_f, group
        self._h = _lib.Handle(h.value, L.card_linear4_destroy)

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
        return (_ext or _load()).linear4(self._h.value, self._index, self.in_features, self.out_features, x, x_scale, gamma,
                                         1.0 if slope is None else slope, out_dtype)

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
    with torch.cuda.device(w.device):
        _lib.check(_lib.lib().card_linear4_quantize(_ptr(w), out_f, in_f, int(group), _ptr(q), _ptr(scale), _ptr(zero), _stream(w.device)),
                   "card_linear4_quantize")
    return q, scale, zero
