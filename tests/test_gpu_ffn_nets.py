"""GeoNet / RadianceNet with residual blocks on the GPU against the same modules in float64 on the CPU, and inside a NeRF model's training step."""
import copy
import os

import pytest
import torch

from conftest import ROOT

pytestmark = pytest.mark.gpu

FREQ = {'type': 'FreqEmbedder', 'input_dim': 3, 'n_freqs': 0}      # the coordinates themselves (the encoding kernel runs on the GPU only)


def nets(block, dtype='float32'):
    from arcnerf_amd.models.base_modules import build_geo_model, build_radiance_model
    from arcnerf_amd.utils.cfgs_utils import dict_to_obj
    torch.manual_seed(0)
    block = dict(block, dtype=dtype)
    geo = build_geo_model(dict_to_obj({'W': 64, 'D': 4, 'skips': [], 'W_feat': 32, 'encoder': FREQ, 'geometric_init': False, 'act_cfg': {'type': 'Softplus', 'beta': 1.0},
                                       'block_cfg': block}))
    rad = build_radiance_model(dict_to_obj({'mode': 'vf', 'W': 64, 'D': 3, 'W_feat_in': 32, 'encoder': {'view': FREQ}, 'act_cfg': {'type': 'Softplus', 'beta': 1.0},
                                            'block_cfg': block}))
    return geo, rad


def in_64(net):
    net = copy.deepcopy(net).double()
    for m in net.modules():
        if isinstance(getattr(m, 'dtype', None), torch.dtype):
            m.dtype = torch.float64
    return net


@pytest.mark.parametrize('block', [{'hidden': 96, 'act': 'silu'}, {'hidden': 80, 'act': 'gelu', 'norm': False}, {'type': 'dense', 'act': 'softplus'}],
                         ids=['gated', 'gated-no-norm', 'dense'])
@pytest.mark.parametrize('dtype,rel', [('float32', 2e-5), ('bfloat16', 0.06), ('float16', 0.0075)])
def test_nets_match_float64(block, dtype, rel):
    """2-norms of outputs and of every gradient.  16 bits: at most 15 roundings of stored tensors lie on a path (five blocks of norm, product and
    sum), each of at most u = 2^-8 / 2^-11: 15 u.  f32: sums of at most 230 terms in a chain of 12 products, 12 * 230 * 2^-24 / 8 for random
    signs"""
    geo, rad = nets(block, dtype)
    geo64, rad64 = in_64(geo), in_64(rad)
    geo, rad = geo.cuda(), rad.cuda()
    g = torch.Generator().manual_seed(1)
    x, d = torch.randn(3000, 3, generator=g), torch.randn(3000, 3, generator=g)
    c1, c2 = torch.randn(3000, 1, generator=g), torch.randn(3000, 3, generator=g)

    def run(geo, rad, *t):
        sdf, feat = geo(t[0])
        rgb = rad(t[0], t[1], None, feat)
        ((sdf * t[2]).sum() + (rgb * t[3]).sum()).backward()
        return {'sdf': sdf, 'feat': feat, 'rgb': rgb, **{'geo.' + k: p.grad for k, p in geo.named_parameters()}, **{'rad.' + k: p.grad for k, p in rad.named_parameters()}}

    got, want = run(geo, rad, x.cuda(), d.cuda(), c1.cuda(), c2.cuda()), run(geo64, rad64, x.double(), d.double(), c1.double(), c2.double())
    for k, v in want.items():
        assert ((got[k].double().cpu() - v).norm() / v.norm()).item() <= rel, k


def test_normals_of_a_block_net_cannot_be_differentiated_again():
    geo, _ = nets({'hidden': 96})
    geo = geo.cuda()
    sdf, feat, grad = geo.forward_with_grad(torch.randn(64, 3, device='cuda'))
    with pytest.raises(RuntimeError):
        grad.square().sum().backward()


@pytest.mark.parametrize('dtype', ['float32', 'bfloat16'])
def test_nerf_model_with_blocks_trains(dtype):
    """a step of the NeRF model whose nets have residual blocks: every parameter gets a finite gradient, twice the same bits"""
    from arcnerf_amd.models import build_model
    from arcnerf_amd.utils.cfgs_utils import load_configs
    over = ['--model.geometry.W', '64', '--model.geometry.D', '3', '--model.geometry.W_feat', '64', '--model.radiance.W', '64',
            '--model.radiance.D', '2', '--model.radiance.W_feat_in', '64', '--model.rays.perturb', 'False', '--model.rays.noise_std', '0.0',
            '--model.geometry.block_cfg.hidden', '96', '--model.geometry.block_cfg.dtype', dtype, '--model.radiance.block_cfg.type', 'dense',
            '--model.radiance.block_cfg.dtype', dtype]
    torch.manual_seed(0)
    cfg = load_configs(os.path.join(ROOT, 'configs', 'nerf.yaml'), over)
    cfg.model.geometry.skips = []
    model = build_model(cfg, None).cuda()
    g = torch.Generator().manual_seed(2)
    rays_d = torch.nn.functional.normalize(torch.randn(128, 3, generator=g), dim=-1)
    feed = {'rays_o': (-4 * rays_d).cuda(), 'rays_d': rays_d.cuda()}
    grads = []
    for _ in range(2):
        model.zero_grad(set_to_none=True)
        out = model({k: v[None] for k, v in feed.items()}, inference_only=False)
        sum(v.square().mean() for k, v in out.items() if k.startswith('rgb')).backward()
        grads.append({k: p.grad.clone() for k, p in model.named_parameters() if p.grad is not None})
    blocks = [k for k in grads[0] if '.gate.' in k or '.up.' in k or '.down.' in k or '.norm.' in k]
    assert len(blocks) >= 16
    for k in blocks:
        assert torch.isfinite(grads[0][k]).all() and grads[0][k].abs().max().item() > 0, k
        assert torch.equal(grads[0][k], grads[1][k]), k
