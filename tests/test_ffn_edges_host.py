"""CPU checks of what the feed-forward layers' native nodes refuse before anything else, and of the modules on them."""
import pytest
import torch

from arcnerf_amd import _native as N


@pytest.fixture(scope='module')
def nodes():
    import os
    if not os.path.exists(N.NODES_PATH):
        import __graft_entry__ as ge
        ge.build()
    return N.torch_nodes()


def node_calls(nodes):
    """name -> (call of its operands, operands): every operand given"""
    x, v, w = torch.randn(4, 8), torch.randn(8), torch.randn(8, 8)
    return {
        'layer_norm': (lambda x, w, b: nodes.layer_norm(x, w, b, 1e-5), [x, v, v]),
        'linear_act_residual': (lambda x, w, b, r: nodes.linear_act_residual(x, w, b, r, 7, 1.0), [x, w, v, x]),
        'gated_ffn': (lambda x, wg, wu, wd, bg, bu, bd, r: nodes.gated_ffn(x, wg, wu, wd, bg, bu, bd, r, 7, 1.0), [x, w, w, w, v, v, v, x]),
    }


@pytest.mark.parametrize('name', ['layer_norm', 'linear_act_residual', 'gated_ffn'])
def test_a_tangent_in_any_operand_is_refused(nodes, name):
    import torch.autograd.forward_ad as fw
    call, ops = node_calls(nodes)[name]
    with fw.dual_level():
        for k in range(len(ops)):
            for grad in (False, True):
                with_dual = [fw.make_dual(t.detach().requires_grad_(grad), torch.ones_like(t)) if i == k else t for i, t in enumerate(ops)]
                with pytest.raises(RuntimeError, match='forward-mode'):
                    call(*with_dual)


@pytest.mark.filterwarnings('ignore::DeprecationWarning')
@pytest.mark.parametrize('name', ['layer_norm', 'linear_act_residual', 'gated_ffn'])
def test_a_trace_is_refused(nodes, name):
    call, ops = node_calls(nodes)[name]
    with pytest.raises(RuntimeError, match='cannot be traced'):
        torch.jit.trace(call, tuple(ops))


# ---- the modules --------------------------------------------------------------------------------------------------------------------------
FREQ = {'type': 'FreqEmbedder', 'input_dim': 3, 'n_freqs': 0}      # the coordinates themselves (the encoding kernel runs on the GPU only)


@pytest.mark.parametrize('block', [{'type': 'dense'}, {'type': 'gated'}], ids=['dense', 'gated'])
def test_blocks_refuse_the_geometric_initialisation(block):
    """which is on by default and makes a sphere of plain layers only"""
    from arcnerf_amd.models.base_modules import build_geo_model
    from arcnerf_amd.utils.cfgs_utils import dict_to_obj
    cfg = {'W': 32, 'D': 4, 'skips': [], 'W_feat': 0, 'encoder': FREQ, 'block_cfg': block}
    for more in ({}, {'geometric_init': True}):
        with pytest.raises(AssertionError, match='geometric'):
            build_geo_model(dict_to_obj(dict(cfg, **more)))
    net = build_geo_model(dict_to_obj(dict(cfg, geometric_init=False)))
    assert len(net.layers) == 5
    # without blocks, and with no layer that would be one, the initialisation is there as ever
    torch.manual_seed(0)
    x = torch.nn.functional.normalize(torch.randn(500, 3), dim=-1) * 2
    for more in ({'block_cfg': None}, {'D': 1}):
        sdf, _ = build_geo_model(dict_to_obj(dict(cfg, W=256, geometric_init=True, **more)))(x)
        assert (sdf - 1).abs().mean().item() < 0.5


STREAMS = [(torch.float32, 'bfloat16'), (torch.float32, 'float16'), (torch.float16, 'bfloat16'), (torch.bfloat16, 'float32'), (torch.float32, 'float32')]


def check_stream(x_type, dtype, kind, device):
    """a block whose branch is zero hands x and its gradient on, bit for bit"""
    from arcnerf_amd.models.base_modules import build_block
    from arcnerf_amd.utils.cfgs_utils import dict_to_obj
    block = build_block(dict_to_obj({'type': kind, 'dtype': dtype, 'act': 'silu'}), 24).to(device)
    last = block.down if kind == 'gated' else block
    torch.nn.init.zeros_(last.weight)
    torch.nn.init.zeros_(last.bias)
    g = torch.Generator().manual_seed(0)
    x = (torch.randn(30, 24, generator=g) * 3 + 0.123).to(x_type).to(device).requires_grad_(True)
    y = block(x)
    assert y.dtype == x_type and torch.equal(y, x)
    dy = torch.randn(30, 24, generator=g).to(x_type).to(device)
    dx, dw = torch.autograd.grad(y, [x, last.weight], dy)
    assert torch.equal(dx, dy)              # (a zero weight hands no gradient to the branch's input)
    assert dw.dtype == torch.float32 and torch.isfinite(dw).all()


@pytest.mark.parametrize('kind', ['gated', 'dense'])
@pytest.mark.parametrize('x_type,dtype', STREAMS)
def test_a_narrow_branch_leaves_a_wide_stream_its_bits(x_type, dtype, kind):
    check_stream(x_type, dtype, kind, 'cpu')


# ---- sizes ------------------------------------------------------------------------------------------------------------------------------
def test_backward_products_take_what_a_gated_forward_takes(nodes):
    """a hidden width of up to 2^24 is two halves of that in the backward (no rows: nothing is launched)"""
    lib, n = N.lib(), None
    for hid in (1 << 23, (1 << 23) + 1, 1 << 24):
        assert lib.arcn_gated_fwd(n, 1, n, n, n, n, n, 0, 7, 1.0, 0, 1, hid, n) == 0
        assert lib.arcn_gated_bwd(n, 1, n, n, n, n, n, 1, n, n, 0, 7, 1.0, 0, 1, hid, 1, n) == 0
        assert lib.arcn_dense_dx(n, 2 * hid, n, n, n, 0, 0, 2 * hid, 1, n) == 0
        assert lib.arcn_dense_dw_scratch_floats(1, 2 * hid, 1, 0) >= 4 * hid
    for big in ((1 << 25) + 1, (1 << 31) - 1):
        assert lib.arcn_dense_dx(n, big, n, n, n, 0, 0, big, 1, n) == -1
        assert lib.arcn_dense_dw_scratch_floats(1, big, 1, 0) == 0
    for bad in (0, -1, -(1 << 31)):
        assert lib.arcn_dense_dx(n, 1, n, n, n, 0, 0, bad, 1, n) == -1
        assert lib.arcn_dense_dw_scratch_floats(1, bad, 1, 0) == 0


@pytest.mark.parametrize('name', ['layer_norm', 'linear_act_residual', 'gated_ffn'])
@pytest.mark.parametrize('how', [dict(tracing_mode='real'), dict(tracing_mode='real', pre_dispatch=True)], ids=['', 'pre-dispatch'])
def test_a_trace_into_a_graph_module_is_refused(nodes, name, how):
    """it would record the allocation of a result and nothing that fills it"""
    from torch.fx.experimental.proxy_tensor import make_fx
    call, ops = node_calls(nodes)[name]
    with pytest.raises(RuntimeError, match='cannot be traced'):
        make_fx(call, **how)(*ops)


def test_column_sums_are_refused_before_a_launch(nodes):
    """of f32, without room or a host number for them, more of them than there can be"""
    import ctypes as C
    lib, p, n = N.lib(), C.c_void_p(4096), None      # (4096 is never read)
    num = C.c_int64(7)
    need = lib.arcn_bias_sums_floats(200, 8)
    assert need >= 4 * 8 and lib.arcn_bias_sums_floats(0, 8) == 0 and lib.arcn_bias_sums_floats(-1, 8) == 0 and lib.arcn_bias_sums_floats(1, 0) == 0
    dz = lambda sums, room, at, dtype: lib.arcn_dense_dz_sums(p, 8, p, n, p, 8, p, n, sums, room, at, dtype, 7, 1.0, 200, 8, 8, n)
    gated = lambda sums, room, at, dtype: lib.arcn_gated_bwd_sums(p, 8, p, p, n, n, p, 8, p, p, sums, room, at, dtype, 7, 1.0, 200, 8, 4, 8, n)
    for call in (dz, gated):
        assert call(p, need, C.byref(num), 0) == -1
        assert call(p, need - 1, C.byref(num), 1) == -1
        assert call(p, need, n, 2) == -1
    assert lib.arcn_dense_dz_sums(n, 8, n, n, n, 8, n, n, p, 0, C.byref(num), 1, 7, 1.0, 0, 8, 8, n) == 0 and num.value == 0      # no rows
    for dtype, rows in ((0, 1), (1, -1), (1, 5)):
        assert lib.arcn_dense_dw_sums(p, 8, p, 8, p, rows, p, p, dtype, p, 1 << 20, 200, 8, 8, n) == -1
