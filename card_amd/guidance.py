"""The guidance network f_phi on the device (card_fphi_*): y_0_hat = f_phi(x), evaluated inside the sampling call.

Reference: regression/model.py:55-82 DeterministicFeedForwardNeuralNetwork and the OLS guidance of
Diffusion.compute_guiding_prediction (regression/card_regression.py:111-124).  The reference evaluates f_phi once per
test minibatch (:1021) and then tiles x, y_0_hat and y_T_mean n_z times (:1027-1035); with `Sampler.run(..., fphi=g,
n_z=n)` both happen inside card_sampler_run: one kernel over the un-tiled rows, then the sampling kernels expand rows to
chains themselves.
"""
import ctypes as C
import weakref

import torch

from . import _lib
from ._lib import CardError
from .sampler import _content_hash, _dev_f32, _fingerprint, _ptr, _require_cuda, _stream


class GuidanceNet:
    """A packed f_phi on one GPU.  Immutable after construction.  `dropout`: the rates of the hidden layers' Dropout, which
    `mc_dropout` applies (`forward` is the eval-mode network)."""

    def __init__(self, weights, biases, *, negative_slope=0.01, bn_scale=None, bn_shift=None, dropout=None, device):
        device = torch.device(device)
        _require_cuda(device)
        n = len(weights)
        if not 1 <= n <= _lib.FPHI_MAX_LAYERS:
            raise CardError(f"f_phi with {n} Linear layers; the kernel takes 1..{_lib.FPHI_MAX_LAYERS}")
        d = _lib.FphiDesc()
        d.struct_bytes = C.sizeof(_lib.FphiDesc)
        d.n_layers = n
        d.negative_slope = float(negative_slope)
        keep = []

        def dev(t):
            t = _dev_f32(t, device)
            keep.append(t)
            return t.data_ptr()

        d.dims[0] = int(weights[0].shape[1])
        for l, W in enumerate(weights):
            if W.dim() != 2 or int(W.shape[1]) != d.dims[l]:
                raise CardError(f"f_phi layer {l}: weight {tuple(W.shape)} does not take {d.dims[l]} inputs")
            d.dims[l + 1] = int(W.shape[0])
            d.W[l] = dev(W)
            if biases[l] is not None:
                d.b[l] = dev(biases[l])
            if bn_scale is not None and bn_scale[l] is not None:
                d.bn_scale[l], d.bn_shift[l] = dev(bn_scale[l]), dev(bn_shift[l])
        self.device, self.dim_in, self.dim_out = device, int(d.dims[0]), int(d.dims[n])
        self.dropout = _rates(dropout, n)
        h = C.c_void_p()
        L = _lib.lib()
        with torch.cuda.device(device):
            _lib.check(L.card_fphi_create(C.byref(d), _stream(device), C.byref(h)), "card_fphi_create")
        self._h = _lib.Handle(h.value, L.card_fphi_destroy)

    @classmethod
    def from_module(cls, net, device=None, *, weight_bits=None, group=64):
        """From a DeterministicFeedForwardNeuralNetwork (its `.network` Sequential: Linear, [BatchNorm1d], LeakyReLU,
        Dropout per hidden layer, then Linear -- regression/model.py:70-79) or any Sequential of those layer types.
        weight_bits=4: the weights in 4 bits with a scale per `group` columns (QuantGuidanceNet); the layers may then be of
        any width and may have an nn.RMSNorm ahead of them."""
        d = describe_guidance(net)
        device = device if device is not None else d["weights"][0].device
        if weight_bits == 4:
            return QuantGuidanceNet(d, group=group, device=device)
        if weight_bits is not None:
            raise CardError(f"f_phi: weight_bits={weight_bits}; 4, or None for fp32")
        if any(n is not None for n in d["norms"]):
            raise CardError("f_phi: RMSNorm layers run with weight_bits=4 only")
        sc = [None if bn is None else _bn_fold(bn)[0] for bn in d["batchnorm"]]
        sh = [None if bn is None else _bn_fold(bn)[1] for bn in d["batchnorm"]]
        return cls(d["weights"], d["biases"], negative_slope=d["negative_slope"], bn_scale=sc, bn_shift=sh,
                   dropout=d["dropout"], device=device)

    @classmethod
    def from_ols(cls, beta, device=None):
        """OLS guidance (regression/card_regression.py:76-92, :115-117): beta is (1 + x_dim, y_dim), y = cat(1, x).mm(beta)."""
        device = device if device is not None else beta.device
        return cls([beta[1:].t().contiguous()], [beta[0].contiguous()], device=device)

    def forward(self, x, out=None):
        """(rows, dim_out) = f_phi(x): card_fphi_forward (compute_guiding_prediction, regression/card_regression.py:111-124)."""
        x = _dev_f32(x, self.device)
        if x.dim() != 2 or x.shape[1] != self.dim_in:
            raise CardError(f"f_phi: x must be (rows, {self.dim_in}), got {tuple(x.shape)}")
        rows = int(x.shape[0])
        if out is None:
            out = torch.empty(rows, self.dim_out, device=self.device, dtype=torch.float32)
        with torch.cuda.device(self.device):
            _lib.check(_lib.lib().card_fphi_forward(self._h, _ptr(x), rows, _ptr(out), _stream(self.device)),
                       "card_fphi_forward")
        return out

    __call__ = forward

    def mc_dropout(self, x, n_z, *, seed, chain_offset=0):
        """(rows, n_z, dim_out): the network with its Dropout layers active, n_z masks for every row (Monte-Carlo dropout):
        card_fphi_forward_mc.  Hidden layer l drops what `card_amd.dropout(..., seed=seed, draw=l)` drops of its (rows * n_z,
        width) outputs; chain_offset: the first row's number times n_z where rows are sharded."""
        x, n_z, chain_offset = self._mc_args(x, n_z, chain_offset)
        rows = int(x.shape[0])
        out = torch.empty(rows, n_z, self.dim_out, device=self.device, dtype=torch.float32)
        p = (C.c_double * max(1, len(self.dropout)))(*self.dropout)
        with torch.cuda.device(self.device):
            _lib.check(_lib.lib().card_fphi_forward_mc(self._h, _ptr(x), rows, n_z, p, int(seed) & (2 ** 64 - 1), chain_offset,
                                                       _ptr(out), _stream(self.device)), "card_fphi_forward_mc")
        return out

    def _rows(self, x):
        x = _dev_f32(x, self.device)
        if x.dim() != 2 or x.shape[1] != self.dim_in:
            raise CardError(f"f_phi: x must be (rows, {self.dim_in}), got {tuple(x.shape)}")
        return x

    def _mc_args(self, x, n_z, chain_offset):
        if self.dropout is None:
            raise CardError("f_phi: no Dropout rates, or Dropout layers other than one behind each hidden layer")
        x = self._rows(x)
        if not 1 <= int(n_z) < 2 ** 31 or not 0 <= int(chain_offset) < 2 ** 52:
            raise CardError(f"f_phi: n_z={n_z} or chain_offset={chain_offset} out of range")
        return x, int(n_z), int(chain_offset)


def _rates(dropout, n_layers):
    if dropout is None:
        return None
    p = [float(v) for v in dropout]
    if len(p) != n_layers - 1 or not all(0.0 <= v <= 1.0 for v in p):
        raise CardError(f"f_phi: dropout rates {p} for {n_layers - 1} hidden layers")
    return p


class QuantGuidanceNet(GuidanceNet):
    """f_phi with 4-bit weights: per layer [RMSNorm to e4m3 (card_rms_norm)], the 4-bit product with bias, folded BatchNorm and
    LeakyReLU in its epilogue (card_linear4), and in `mc_dropout` the dropout (card_dropout).  Rows stay fp32 between layers,
    8-bit behind a norm.  Where the sampler takes a GuidanceNet it takes this one; the network then runs ahead of the sampling
    kernels instead of as their first."""

    def __init__(self, description, *, group=64, device):
        from .layers import QuantLinear
        device = torch.device(device)
        _require_cuda(device)
        d = description
        self.dim_in, self.dim_out = d["dims"][0], d["dims"][-1]
        self.dropout, self.slope = _rates(d["dropout"], len(d["weights"])), d["negative_slope"]
        self._h = None
        self.layers = []
        for W, b, bn, norm in zip(d["weights"], d["biases"], d["batchnorm"], d["norms"]):
            W = _dev_f32(W, device)
            b = _dev_f32(b, device) if b is not None else torch.zeros(W.shape[0], device=device)
            if bn is not None:
                sc, sh = (_dev_f32(t, device) for t in _bn_fold(bn))
                W, b = W * sc[:, None], b * sc + sh
            lin = QuantLinear.from_float(W, b, group=group, device=device)
            w = None if norm is None or norm.weight is None else _dev_f32(norm.weight, device)
            self.layers.append((norm is not None, w, 0.0 if norm is None else _eps(norm), lin))
        self.device = self.layers[0][3].device

    def _layer(self, l, h):
        from .layers import rms_norm_e4m3
        norm, w, eps, lin = self.layers[l]
        scale = None
        if norm:
            h, scale = rms_norm_e4m3(h, w, eps=eps)
        return lin.forward(h, scale, slope=self.slope if l < len(self.layers) - 1 else None, out_dtype=torch.float32)

    def forward(self, x, out=None):
        """(rows, dim_out) = f_phi(x)."""
        h = self._rows(x)
        if out is not None and not (tuple(out.shape) == (h.shape[0], self.dim_out) and out.dtype is torch.float32 and out.device == self.device):
            raise CardError(f"f_phi: out must be ({h.shape[0]}, {self.dim_out}) float32 on {self.device}, got {tuple(out.shape)} {out.dtype} on {out.device}")
        with torch.no_grad():
            h = torch.cat([self._part(h[i:i + _lib.LINEAR4_MAX_ROWS]) for i in range(0, h.shape[0], _lib.LINEAR4_MAX_ROWS)]) \
                if h.shape[0] > _lib.LINEAR4_MAX_ROWS else self._part(h)
            return h if out is None else out.copy_(h)

    __call__ = forward

    def _part(self, h):
        for l in range(len(self.layers)):
            h = self._layer(l, h)
        return h

    def mc_dropout(self, x, n_z, *, seed, chain_offset=0):
        """GuidanceNet.mc_dropout with 4-bit weights: the same masks."""
        from .layers import dropout
        x, n_z, chain_offset = self._mc_args(x, n_z, chain_offset)
        most = max(1, _lib.LINEAR4_MAX_ROWS // n_z)
        if n_z > _lib.LINEAR4_MAX_ROWS:
            raise CardError(f"f_phi: n_z={n_z} > {_lib.LINEAR4_MAX_ROWS} with 4-bit weights")
        if (chain_offset + int(x.shape[0]) * n_z) * max(lin.out_features for _, _, _, lin in self.layers) >= 2 ** 63:
            raise CardError(f"f_phi: chain_offset={chain_offset} out of range for layers of this width")
        parts = []
        with torch.no_grad():
            for i in range(0, max(1, x.shape[0]), most):
                h = x[i:i + most]
                rows, chains, first = int(h.shape[0]), 1, chain_offset + i * n_z
                for l in range(len(self.layers)):
                    h = self._layer(l, h)
                    # rows become chains at the first layer that drops something; the layers ahead of it run once per row
                    if l < len(self.dropout) and self.dropout[l] > 0:
                        z, chains = (n_z, n_z) if chains == 1 else (1, chains)
                        h = dropout(h, self.dropout[l], seed=seed, elem_offset=first * h.shape[1], draw=l, n_z=z).reshape(rows * n_z, h.shape[1])
                parts.append(h.reshape(rows, chains, self.dim_out).expand(rows, n_z, self.dim_out))
        return parts[0].contiguous() if len(parts) == 1 else torch.cat(parts)


def _eps(norm):
    return torch.finfo(torch.float32).eps if norm.eps is None else float(norm.eps)


def _bn_fold(m):
    """eval-mode BatchNorm1d as (scale, shift) per feature"""
    s = (m.weight if m.affine else torch.ones_like(m.running_var)) / torch.sqrt(m.running_var + m.eps)
    return s, (m.bias if m.affine else torch.zeros_like(m.running_mean)) - m.running_mean * s


def describe_guidance(net):
    """Recognise f_phi (device-free, like card_amd.sampler.describe): walk the `.network` Sequential of a
    DeterministicFeedForwardNeuralNetwork (regression/model.py:70-79) -- or any Sequential of Linear / BatchNorm1d /
    LeakyReLU / ReLU / Dropout / RMSNorm / Identity -- and return {"dims": [dim_in, hidden..., dim_out], "weights": [Linear.weight
    ...], "biases": [...], "batchnorm": [the BatchNorm1d module that follows layer l, or None], "negative_slope": float,
    "dropout": [the Dropout rate behind hidden layer l] (None: Dropout layers elsewhere), "norms": [the RMSNorm ahead of layer l, or None]}
    with the module's own Parameter objects.  Raises CardError for train-mode BatchNorm / Dropout, foreign layers and orders other
    than Linear, [BatchNorm], activation -- which is what the kernels compute -- with Dropout anywhere."""
    import torch.nn as nn
    net = getattr(net, "module", net) if isinstance(net, (nn.DataParallel, nn.parallel.DistributedDataParallel)) else net
    seq = getattr(net, "network", net)
    Ws, bs, bns, slope = [], [], [], None
    drops, norms, norm, active, simple = [], [], None, False, True
    for m in seq.children():
        if isinstance(m, nn.Linear):
            if Ws and not active:
                raise CardError("f_phi: a Linear layer behind another without an activation between them")
            Ws.append(m.weight)
            bs.append(m.bias)
            bns.append(None)
            drops.append(0.0)
            norms.append(norm)
            if norm is not None and tuple(norm.normalized_shape) != (m.in_features,):
                raise CardError(f"f_phi: RMSNorm over {tuple(norm.normalized_shape)} ahead of a Linear layer of {m.in_features} inputs")
            norm, active = None, False
        elif isinstance(m, nn.BatchNorm1d):
            if m.training or not m.track_running_stats:
                raise CardError("f_phi BatchNorm1d must be in eval mode with running statistics (the reference calls "
                                "cond_pred_model.eval() before testing, regression/card_regression.py:951)")
            if not Ws or bns[-1] is not None or norm is not None or active:
                raise CardError("f_phi: BatchNorm1d must follow a Linear layer, ahead of its activation")
            bns[-1] = m
            simple = simple and drops[-1] == 0
        elif isinstance(m, (nn.LeakyReLU, nn.ReLU)):
            s = m.negative_slope if isinstance(m, nn.LeakyReLU) else 0.0
            if norm is not None:
                raise CardError("f_phi: an activation between RMSNorm and its Linear layer")
            if not Ws or (active and s != 0):          # a second ReLU changes nothing
                raise CardError("f_phi: an activation stands once behind a Linear layer")
            if slope is not None and slope != s:
                raise CardError("f_phi: activations with different slopes")
            slope, active = s, True
        elif isinstance(m, nn.Dropout):
            if m.training and m.p > 0:
                raise CardError("f_phi Dropout must be in eval mode (identity); call .eval() on the guidance model")
            if m.p > 0:
                if not Ws or drops[-1] > 0 or norm is not None:
                    simple = False
                else:
                    drops[-1] = float(m.p)
        elif isinstance(m, nn.RMSNorm):
            if norm is not None or (Ws and not active):
                raise CardError("f_phi: RMSNorm stands once ahead of a Linear layer, behind the activation of the layer before")
            norm = m
        elif isinstance(m, nn.Identity):
            pass
        else:
            raise CardError(f"f_phi: layer type {type(m).__name__} is not part of regression/model.py:70-79")
    if not Ws:
        raise CardError("f_phi: no Linear layer found")
    if norm is not None:
        raise CardError("f_phi: RMSNorm behind the output layer")
    if active:
        raise CardError("f_phi: an activation behind the output layer")
    simple = simple and drops[-1] == 0
    if bns[-1] is not None:
        raise CardError("f_phi: BatchNorm after the output layer is not part of regression/model.py:70-79")
    dims = [int(Ws[0].shape[1])]
    for l, W in enumerate(Ws):
        if W.dim() != 2 or int(W.shape[1]) != dims[-1]:
            raise CardError(f"f_phi layer {l}: weight {tuple(W.shape)} does not take {dims[-1]} inputs")
        dims.append(int(W.shape[0]))
    return {"dims": dims, "weights": Ws, "biases": bs, "batchnorm": bns, "negative_slope": 0.01 if slope is None else float(slope),
            "dropout": drops[:-1] if simple else None, "norms": norms}


_gcache = weakref.WeakKeyDictionary()


def _settings(net):
    """What describe_guidance reads of a network besides its tensors: its modules in their order with the numbers they hold"""
    names = ("training", "p", "negative_slope", "eps", "track_running_stats")
    numbers = lambda m: (v if isinstance(v, (int, float)) else None for v in (getattr(m, n, None) for n in names))  # noqa: E731
    return tuple((type(m), *numbers(m)) for m in net.modules())


def guidance_for(f_phi):
    """The cached GuidanceNet of an `nn.Module` (DeterministicFeedForwardNeuralNetwork), or of an OLS coefficient tensor
    (1 + x_dim, y_dim); a GuidanceNet passes through.  Re-packed when the weights change (identity + content check, like
    sampler_for), or the modules' own numbers: Dropout rates, slopes, eps, train mode."""
    if isinstance(f_phi, GuidanceNet):
        return f_phi
    if torch.is_tensor(f_phi):
        return GuidanceNet.from_ols(f_phi)                 # a (1 + x_dim) x y_dim matrix: packing it is one tiny copy
    fp = (_fingerprint(f_phi), _settings(f_phi))
    hit = _gcache.get(f_phi)
    h = None
    if hit is not None and hit[0] == fp:
        h = _content_hash(f_phi)
        if h == hit[2]:
            return hit[1]
    g = GuidanceNet.from_module(f_phi)
    _gcache[f_phi] = (fp, g, _content_hash(f_phi) if h is None else h)
    return g
