"""Residual feed-forward layers of the wide nets: LayerNorm, ResidualDenseLayer, GatedFfnBlock, and the `block_cfg` by which GeoNet and
RadianceNet take them as their hidden layers.  The reference's nets have plain DenseLayers only
(arcnerf/models/base_modules/geo_rad_model/linear_network_module.py:16-335); without `block_cfg` nothing of this is used.

On CUDA tensors the layers run csrc/norm.hip and csrc/dense.hpp (ops.autograd.layer_norm, linear_act_residual, gated_ffn).  First order: the
normals of a net made of them cannot be differentiated again (forward_with_grad under a loss on the normals raises)."""
import torch
import torch.nn as nn

from ...utils.cfgs_utils import get_value_from_cfgs_field as _opt
from .linear import Linear

_DTYPES = {'float32': torch.float32, 'bfloat16': torch.bfloat16, 'float16': torch.float16}


def _as(t, dtype):
    return t if t is None else t.to(dtype)


def _add_to_stream(x, h, branch):
    """x + branch(residual) in x's type: in the branch's last epilogue where h, x in the type that the branch computes in, holds all of x; else
    outside, so that neither the stream nor its gradient loses bits to a narrower branch"""
    if torch.promote_types(x.dtype, h.dtype) == h.dtype:
        return branch(h).to(x.dtype)
    return (x + branch(None)).to(x.dtype)


class LayerNorm(nn.Module):
    """torch.nn.LayerNorm over the last dimension (same parameters and state_dict keys)"""

    def __init__(self, dim, eps=1e-5):
        super().__init__()
        self.eps = eps
        self.weight, self.bias = nn.Parameter(torch.ones(dim)), nn.Parameter(torch.zeros(dim))

    def forward(self, x):
        from ...ops.autograd import layer_norm
        return layer_norm(x, self.weight, self.bias, self.eps)


class ResidualDenseLayer(Linear):
    """x + act(norm(x) W^T + b): one norm and one product whose epilogue adds the bias, the activation and the residual.  `dtype` is the type the
    layer computes in (its parameters stay float32, and a wider x keeps its type and bits: _add_to_stream)"""

    def __init__(self, dim, act='relu', beta=1.0, norm=True, bias=True, dtype=torch.float32):
        super().__init__(dim, dim, bias=bias)
        self.act, self.beta, self.dtype = act, beta, dtype
        self.norm = LayerNorm(dim) if norm else None

    def forward(self, x):
        from ...ops.autograd import linear_act_residual
        h = x.to(self.dtype)
        n = h if self.norm is None else self.norm(h)
        w, b = _as(self.weight, self.dtype), _as(self.bias, self.dtype)
        return _add_to_stream(x, h, lambda res: linear_act_residual(n, w, b, res, act=self.act, beta=self.beta))


class GatedFfnBlock(nn.Module):
    """x + down(act(gate(n)) * up(n)), n = norm(x): `gate` and `up` as one kernel, the residual in the epilogue of `down`.  `dtype` as
    ResidualDenseLayer has it"""

    def __init__(self, dim, hidden, act='silu', beta=1.0, norm=True, bias=True, dtype=torch.float32):
        super().__init__()
        self.in_features = self.out_features = dim
        self.act, self.beta, self.dtype = act, beta, dtype
        self.norm = LayerNorm(dim) if norm else None
        self.gate, self.up, self.down = nn.Linear(dim, hidden, bias=bias), nn.Linear(dim, hidden, bias=bias), nn.Linear(hidden, dim, bias=bias)

    def forward(self, x):
        from ...ops.autograd import gated_ffn
        d = self.dtype
        h = x.to(d)
        n = h if self.norm is None else self.norm(h)
        w = [_as(layer.weight, d) for layer in (self.gate, self.up, self.down)]
        b = [_as(layer.bias, d) for layer in (self.gate, self.up, self.down)]
        return _add_to_stream(x, h, lambda res: gated_ffn(n, *w, *b, residual=res, act=self.act, beta=self.beta))


def build_block(cfg, dim, bias=True):
    """cfg: type 'gated' (default) | 'dense', hidden (gated; default 2 dim), act ('silu' / 'relu'), beta (softplus), norm (True), dtype ('float32' |
    'bfloat16' | 'float16')"""
    kind, dtype = _opt(cfg, 'type', 'gated'), _opt(cfg, 'dtype', 'float32')
    if dtype not in _DTYPES:
        raise NotImplementedError('No block dtype {} (one of {})'.format(dtype, sorted(_DTYPES)))
    common = dict(beta=_opt(cfg, 'beta', 1.0), norm=_opt(cfg, 'norm', True), bias=bias, dtype=_DTYPES[dtype])
    if kind == 'gated':
        return GatedFfnBlock(dim, _opt(cfg, 'hidden', 2 * dim), act=_opt(cfg, 'act', 'silu'), **common)
    if kind == 'dense':
        return ResidualDenseLayer(dim, act=_opt(cfg, 'act', 'relu'), **common)
    raise NotImplementedError('No block type {}'.format(kind))
