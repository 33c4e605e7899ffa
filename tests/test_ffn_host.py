"""CPU checks of the residual feed-forward layers: the modules' arithmetic and parameters, the nets that take them, and what the C entry points
and the Python front end refuse before anything reaches a device."""
import ctypes as C

import pytest
import torch

from arcnerf_amd import _native as N
from arcnerf_amd.models.base_modules import GatedFfnBlock, LayerNorm, ResidualDenseLayer, build_block, build_geo_model, build_radiance_model
from arcnerf_amd.ops import autograd as A
from arcnerf_amd.ops import functional as F
from arcnerf_amd.utils.cfgs_utils import dict_to_obj

FREQ = {'type': 'FreqEmbedder', 'input_dim': 3, 'n_freqs': 0}      # the coordinates themselves (the encoding kernel runs on the GPU only)


def test_layers_compute_their_formulas():
    torch.manual_seed(0)
    x = torch.randn(7, 12, dtype=torch.float64)
    fn = torch.nn.functional
    n = LayerNorm(12)
    n.weight.data.normal_()
    n.bias.data.normal_()
    want = fn.layer_norm(x.float(), (12,), n.weight, n.bias)
    assert torch.allclose(n(x.float()), want)
    d = ResidualDenseLayer(12, act='softplus', beta=3.0, norm=False, dtype=torch.float64)
    assert torch.allclose(d(x), x + fn.softplus(fn.linear(x, d.weight.double(), d.bias.double()), beta=3.0))
    g = GatedFfnBlock(12, 20, act='gelu', norm=False, dtype=torch.float64)
    w = {k: v.double() for k, v in g.state_dict().items()}
    h = fn.gelu(fn.linear(x, w['gate.weight'], w['gate.bias'])) * fn.linear(x, w['up.weight'], w['up.bias'])
    assert torch.allclose(g(x), x + fn.linear(h, w['down.weight'], w['down.bias']))
    for act, f in (('relu', fn.relu), ('sigmoid', torch.sigmoid), ('silu', fn.silu), (None, lambda v: v)):
        w1 = torch.randn(5, 12, dtype=torch.float64)
        assert torch.allclose(A.linear_act_residual(x, w1, act=act), f(x @ w1.t()))


def test_block_config():
    b = build_block(dict_to_obj({'hidden': 24, 'act': 'silu', 'dtype': 'bfloat16'}), 16)
    assert type(b) is GatedFfnBlock and b.gate.weight.shape == (24, 16) and b.dtype == torch.bfloat16 and b.norm is not None
    assert b.gate.weight.dtype == torch.float32
    b = build_block(dict_to_obj({'type': 'dense', 'norm': False}), 16, bias=False)
    assert type(b) is ResidualDenseLayer and b.norm is None and b.bias is None and b.act == 'relu'
    assert build_block(dict_to_obj({'type': 'gated'}), 16).gate.weight.shape == (32, 16)
    for bad in ({'type': 'other'}, {'dtype': 'float8'}):
        with pytest.raises(NotImplementedError):
            build_block(dict_to_obj(bad), 16)


def test_nets_with_blocks():
    torch.manual_seed(0)
    cfg = {'W': 32, 'D': 4, 'skips': [], 'W_feat': 16, 'encoder': FREQ, 'geometric_init': False, 'block_cfg': {'hidden': 40}}
    geo = build_geo_model(dict_to_obj(cfg))
    assert [type(layer).__name__ for layer in geo.layers] == ['DenseLayer'] + ['GatedFfnBlock'] * 3 + ['Linear']
    x = torch.randn(9, 3)
    sdf, feat = geo(x)
    assert sdf.shape == (9, 1) and feat.shape == (9, 16)
    (sdf.sum() + feat.sum()).backward()
    assert all(p.grad is not None and torch.isfinite(p.grad).all() for p in geo.parameters())
    rad = build_radiance_model(dict_to_obj({'mode': 'vf', 'W': 24, 'D': 3, 'W_feat_in': 16, 'encoder': {'view': FREQ}, 'block_cfg': {'type': 'dense'}}))
    assert [type(layer).__name__ for layer in rad.layers] == ['DenseLayer'] + ['ResidualDenseLayer'] * 2 + ['DenseLayer']
    rgb = rad(x, torch.randn(9, 3), None, feat.detach())
    assert rgb.shape == (9, 3) and ((rgb > 0) & (rgb < 1)).all()
    with pytest.raises(AssertionError):
        build_geo_model(dict_to_obj(dict(cfg, skips=[1])))
    with pytest.raises(AssertionError):
        build_geo_model(dict_to_obj(dict(cfg, weight_norm=True)))
    plain = build_geo_model(dict_to_obj({k: v for k, v in cfg.items() if k != 'block_cfg'}))
    assert [type(layer).__name__ for layer in plain.layers] == ['DenseLayer'] * 4 + ['Linear']


@pytest.fixture(scope='module')
def lib():
    import os
    if not os.path.exists(N.LIB_PATH):
        import __graft_entry__ as ge
        ge.build()
    return N.lib()


def test_entry_points_refuse_before_a_launch(lib):
    p = C.c_void_p(4096)        # never read: every call below is refused, or has no rows
    n = None
    assert lib.arcn_layer_norm_fwd(p, 8, n, n, 3, 0, 1e-5, p, n, 4, 8, n) == -1                  # no such type
    assert lib.arcn_layer_norm_fwd(p, 8, n, n, 0, 1, 1e-5, p, n, 4, 8, n) == -1                  # bf16 parameters of f32 rows
    assert lib.arcn_layer_norm_fwd(p, 7, n, n, 0, 0, 1e-5, p, n, 4, 8, n) == -1                  # rows overlap
    assert lib.arcn_layer_norm_fwd(p, 8, n, n, 0, 0, 1e-5, n, n, 4, 8, n) == -1
    assert lib.arcn_layer_norm_fwd(p, 8, n, n, 0, 0, 1e-5, p, n, 4, 0, n) == -1
    assert lib.arcn_layer_norm_fwd(n, 8, n, n, 0, 0, 1e-5, n, n, 0, 8, n) == 0
    need = lib.arcn_layer_norm_bwd_scratch_floats(4, 8, 0)
    assert need >= 16
    assert lib.arcn_layer_norm_bwd(p, 8, p, 8, n, p, 0, 0, p, p, n, p, need - 1, 4, 8, n) == -1
    assert lib.arcn_layer_norm_bwd(p, 8, p, 8, n, n, 0, 0, p, n, n, n, 0, 4, 8, n) == -1          # no statistics
    assert lib.arcn_layer_norm_bwd(p, 8, p, 8, n, p, 0, 0, p, p, n, p, need, 0, 8, n) == -1       # a weight gradient over no rows
    assert lib.arcn_dense_fwd(p, 8, p, n, n, 0, p, 0, 3, 1.0, 4, 8, 8, n) == -1                   # an activation of the other kernels
    assert lib.arcn_dense_fwd(p, 8, p, n, n, 0, p, 0, 4, 0.0, 4, 8, 8, n) == -1                   # softplus with beta 0
    assert lib.arcn_dense_fwd(p, 8, p, n, p, 7, p, 0, 0, 1.0, 4, 8, 8, n) == -1                   # residual rows overlap
    assert lib.arcn_dense_fwd(p, 8, p, n, n, 0, p, 5, 0, 1.0, 4, 8, 8, n) == -1
    assert lib.arcn_dense_fwd(p, 8, p, n, n, 0, p, 0, 0, 1.0, -1, 8, 8, n) == -1
    assert lib.arcn_dense_fwd(n, 8, n, n, n, 0, n, 2, 8, 1.0, 0, 8, 8, n) == 0
    assert b'dense_fwd' in lib.arcn_last_error()
    assert lib.arcn_dense_dz(p, 8, p, n, n, 8, p, p, 0, 1, 1.0, 4, 8, 8, n) == -1
    assert lib.arcn_dense_dx(p, 7, p, p, p, 0, 4, 7, 8, n) == -1                                  # two halves of an odd width
    assert lib.arcn_dense_dw_scratch_floats(1000, 64, 32, 0) >= 64 * 33
    assert lib.arcn_dense_dw_scratch_floats(1000, 64, 32, 9) == 0
    assert lib.arcn_dense_dw(p, 64, p, 32, p, n, 0, p, 64 * 33 - 1, 1000, 64, 32, n) == -1
    assert lib.arcn_gated_fwd(p, 8, p, n, n, n, p, 0, 7, 1.0, 4, 8, 8, n) == -1
    assert lib.arcn_gated_bwd(p, 8, p, p, n, n, p, 7, p, p, 0, 7, 1.0, 4, 8, 8, 8, n) == -1


def test_front_end_refuses_cpu_tensors_and_mixed_devices():
    x, w = torch.zeros(4, 8), torch.zeros(8, 8)
    for call in (lambda: F.layer_norm_fwd(x), lambda: F.dense_fwd(x, w), lambda: F.gated_fwd(x, w, w), lambda: F.dense_dx(x, w), lambda: F.dense_dw(x, x)):
        with pytest.raises(RuntimeError):
            call()
    with pytest.raises(RuntimeError):
        A.linear_act_residual(x, w, act='tanh')
    assert set(F.DENSE_ACT.values()) == {0, 1, 2, 4, 7, 8}
