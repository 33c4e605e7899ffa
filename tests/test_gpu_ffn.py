"""Layer norm, the dense layer with activation and residual and the gated feed-forward block (csrc/norm.hip, csrc/dense.hpp) against float64,
forward and backward.  The bounds are elementwise and worst case: with u the unit roundoff of the tensors' type (bf16 2^-8, f16 2^-11, f32
2^-24) and e = 2^-24, a sum of n products is within (n + c) e of the sum of their sizes, a value that is stored is within u of itself,
and both are carried through the formulas below.  (The f32 products' three-way bf16 splits drop less than e of a product: inside c.)"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]
IDS = ['f32', 'bf16', 'f16']
E = 2.0 ** -24
C0 = 24          # roundings beside a sum's own: conversions, the activation's evaluation, the epilogue


def unit(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    """half a step of the type's subnormal numbers: the rounding of a result below its normal range"""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps


def randn(seed, *shape, dtype, scale=1.0, offset=0.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g, dtype=torch.float64) * scale + offset).to(dtype)


def pitched(t, pitch):
    """t on the GPU as a column slice of a wider buffer whose other columns are NaN"""
    if not pitch:
        return t.cuda()
    wide = torch.full((t.shape[0], t.shape[1] + pitch), float('nan'), dtype=t.dtype, device='cuda')
    wide[:, pitch // 2:pitch // 2 + t.shape[1]] = t.cuda()
    return wide[:, pitch // 2:pitch // 2 + t.shape[1]]


def close(got, want, tol, what):
    assert got.dtype in TYPES
    got = got.detach().double().cpu()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    off = (got - want).abs() - (tol + 1e-300)
    assert torch.isfinite(got).all(), what + ' is not finite'
    assert off.max().item() <= 0, '{}: {:.3g} over its bound at {}'.format(what, off.max().item(), int(off.argmax()))


def act64(z, act, beta=1.0):
    """value, slope, and a bound on the slope's own slope"""
    z = z.detach().requires_grad_(True)
    fn = torch.nn.functional
    y = {None: lambda v: v * 1.0, 'relu': fn.relu, 'sigmoid': torch.sigmoid, 'silu': lambda v: v * torch.sigmoid(v),
         'gelu': lambda v: v * 0.5 * torch.erfc(-v / math.sqrt(2)), 'softplus': lambda v: torch.logaddexp(beta * v, torch.zeros_like(v)) / beta}[act](z)
    s, = torch.autograd.grad(y.sum(), z)
    return y.detach(), s.detach(), {None: 0.0, 'relu': 0.0, 'sigmoid': 0.1, 'silu': 0.5, 'gelu': 0.8, 'softplus': beta / 4}[act]


# ---- layer norm -------------------------------------------------------------------------------------------------------------------------
def norm_bounds(x, w, b, dy, eps, dtype, wtype):
    """the float64 results and their bounds"""
    S, C = x.shape
    u, n_e = unit(dtype), (C + C0) * E
    mean = x.mean(1, keepdim=True)
    d = x - mean
    r = 1 / (d.square().mean(1, keepdim=True) + eps).sqrt()
    n = d * r
    y = n * w + b
    mean_err = n_e * x.abs().mean(1, keepdim=True)
    # the sum of squares sees (d + mean_err)^2: its cross term vanishes in exact arithmetic, what is left is inside n_e and mean_err^2
    r_rel = n_e + 0.5 * (mean_err * r).square() + mean_err * r * n_e
    n_err = r * (mean_err + 4 * E * d.abs()) + n.abs() * r_rel
    res = {'y': (y, u * y.abs() + tiny(dtype) + (w.abs() * n_err + 4 * E * (y.abs() + b.abs())) * (1 + u))}
    g = dy * w
    gm, gnm = g.mean(1, keepdim=True), (g * n).mean(1, keepdim=True)
    dx = r * (g - gm - n * gnm)
    ga, gna = g.abs().mean(1, keepdim=True), (g * n).abs().mean(1, keepdim=True)
    size = r * (g.abs() + ga + n.abs() * gna)
    dx_err = size * (2 * n_e + r_rel) + r * (n_err * gna + n.abs() * (g.abs() * n_err).mean(1, keepdim=True))
    res['dx'] = (dx, u * dx.abs() + tiny(dtype) + dx_err * (1 + u))
    dw, db, uw = (dy * n).sum(0), dy.sum(0), unit(wtype)
    res['dw'] = (dw, uw * dw.abs() + tiny(wtype) + 1.01 * ((dy.abs() * n_err).sum(0) + (S + C0) * E * (dy * n).abs().sum(0)))
    res['db'] = (db, uw * db.abs() + tiny(wtype) + 1.01 * (S + C0) * E * dy.abs().sum(0))
    return res


@pytest.mark.parametrize('dtype', TYPES, ids=IDS)
@pytest.mark.parametrize('rows,width,pitch', [(1, 1, 0), (1, 256, 0), (5, 2, 0), (3, 8, 3), (70, 33, 0), (65, 64, 1), (130, 100, 0), (257, 256, 0), (31, 319, 2),
                                              (9, 512, 8), (6, 1000, 0), (33, 2048, 0), (5, 2051, 0), (7, 4096, 1), (3, 8192, 0), (3, 8200, 5)])
def test_layer_norm(dtype, rows, width, pitch):
    from arcnerf_amd.ops import autograd as A
    for wtype in {dtype, torch.float32}:
        x, dy = randn(1, rows, width, dtype=dtype, offset=0.5), randn(2, rows, width, dtype=dtype)
        w, b = randn(3, width, dtype=wtype, scale=0.2, offset=1.0), randn(4, width, dtype=wtype, scale=0.2)
        want = norm_bounds(x.double(), w.double(), b.double(), dy.double(), 1e-5, dtype, wtype)
        xg, wg, bg = pitched(x, pitch).requires_grad_(True), w.cuda().requires_grad_(True), b.cuda().requires_grad_(True)
        y = A.layer_norm(xg, wg, bg, 1e-5)
        close(y, *want['y'], 'y')
        dx, dw, db = torch.autograd.grad(y, [xg, wg, bg], pitched(dy, pitch))
        assert dw.dtype == wtype and db.dtype == wtype
        close(dx, *want['dx'], 'dx')
        close(dw, *want['dw'], 'dw')
        close(db, *want['db'], 'db')


@pytest.mark.parametrize('dtype', TYPES, ids=IDS)
def test_layer_norm_many_rows_and_repeatable(dtype):
    """more rows than the backward's grid holds at once: every workgroup strides; twice the same bits"""
    from arcnerf_amd.ops import autograd as A
    rows, width = 40003, 36
    x, dy = randn(1, rows, width, dtype=dtype, offset=-2.0), randn(2, rows, width, dtype=dtype)
    w, b = randn(3, width, dtype=dtype, offset=1.0), randn(4, width, dtype=dtype)
    want = norm_bounds(x.double(), w.double(), b.double(), dy.double(), 1e-3, dtype, dtype)
    leaves = [t.cuda().requires_grad_(True) for t in (x, w, b)]
    y = A.layer_norm(*leaves, 1e-3)
    got = torch.autograd.grad(y, leaves, dy.cuda(), retain_graph=True)
    again = torch.autograd.grad(y, leaves, dy.cuda())
    close(y, *want['y'], 'y')
    for k, a, c in zip(('dx', 'dw', 'db'), got, again):
        close(a, *want[k], k)
        assert torch.equal(a, c), k


def test_layer_norm_constant_rows_far_from_zero():
    """no variance: the result is the bias; the centred form keeps it so at any offset"""
    from arcnerf_amd.ops import functional as F
    x = torch.full((4, 300), 1000.0, device='cuda')
    b = torch.linspace(-1, 1, 300, device='cuda')
    y, stats = F.layer_norm_fwd(x, None, b, want_stats=True)
    # mean: within (300 + c) e of 1000, which 1 / sqrt(eps) = 316 carries into y
    assert (y - b).abs().max().item() <= 1000 * (300 + C0) * E * 317
    assert torch.isfinite(stats).all()


def test_layer_norm_without_parameters_and_empty():
    from arcnerf_amd.ops import autograd as A
    x = randn(1, 6, 40, dtype=torch.float32).cuda().requires_grad_(True)
    one, zero = torch.ones(40, dtype=torch.float64), torch.zeros(40, dtype=torch.float64)
    dy = randn(2, 6, 40, dtype=torch.float32)
    want = norm_bounds(x.detach().double().cpu(), one, zero, dy.double(), 1e-5, torch.float32, torch.float32)
    y = A.layer_norm(x)
    close(y, *want['y'], 'y')
    close(torch.autograd.grad(y, x, dy.cuda())[0], *want['dx'], 'dx')
    xe, w = torch.zeros(0, 7, 40, device='cuda', requires_grad=True), torch.ones(40, device='cuda', requires_grad=True)
    y = A.layer_norm(xe, w)
    assert y.shape == (0, 7, 40)
    gx, gw = torch.autograd.grad(y.sum(), [xe, w])
    assert gx.shape == xe.shape and gw.abs().max().item() == 0
    b = torch.zeros(40, device='cuda', requires_grad=True)
    gb, = torch.autograd.grad(A.layer_norm(x.detach(), None, b).sum(), b)
    assert torch.equal(gb, torch.full((40,), 6.0, device='cuda'))


# ---- dense layer ------------------------------------------------------------------------------------------------------------------------
def dense_bounds(x, w, b, r, dy, act, beta, dtype):
    S, K = x.shape
    N = w.shape[0]
    u, t = unit(dtype), tiny(dtype)
    z = x @ w.t() + b
    z_err = (K + C0) * E * (x.abs() @ w.abs().t() + b.abs())
    a, s, curve = act64(z, act, beta)
    y = a + r
    res = {'y': (y, u * y.abs() + t + (1.2 * z_err + C0 * E * (a.abs() + z.abs() + 1 / max(beta, 1.0)) * (act is not None) + E * y.abs()) * (1 + u))}
    dz = dy * s
    s_err = (C0 * E + curve * z_err) if act else torch.zeros_like(z)
    u_dz = (u * dz.abs() + t) if act else torch.zeros_like(z)
    dz_err = u_dz + dy.abs() * s_err * (1 + u)
    dx = dz @ w
    res['dx'] = (dx, u * dx.abs() + t + ((dz_err + (N + C0) * E * dz.abs()) @ w.abs()) * 1.01)
    dw = dz.t() @ x
    res['dw'] = (dw, u * dw.abs() + t + ((dz_err + (S + C0) * E * dz.abs()).t() @ x.abs()) * 1.01)
    db = dz.sum(0)
    res['db'] = (db, u * db.abs() + t + (dz_err + (S + C0) * E * dz.abs()).sum(0) * 1.01)
    return res


def dense_inputs(rows, k, n, dtype, seed=10):
    x, w = randn(seed, rows, k, dtype=dtype), randn(seed + 1, n, k, dtype=dtype, scale=k ** -0.5)
    return x, w, randn(seed + 2, n, dtype=dtype, scale=0.3), randn(seed + 3, rows, n, dtype=dtype), randn(seed + 4, rows, n, dtype=dtype)


def check_dense(rows, k, n, dtype, act, beta=1.0, pitch=0, bias=True, residual=True):
    from arcnerf_amd.ops import autograd as A
    x, w, b, r, dy = dense_inputs(rows, k, n, dtype)
    if act == 'relu':
        # keep the pre-activations away from the jump of the slope: multiples of 1/16 with an odd numerator, exact in every type
        x, w = (x * 2).round().clamp(-3, 3) / 2, (w * 4).round().clamp(-2, 2) / 2
        b = torch.full_like(b, 0.125)
    zero = torch.zeros((), dtype=torch.float64)
    want = dense_bounds(x.double(), w.double(), b.double() if bias else zero.expand(n), r.double() if residual else zero.expand(rows, n), dy.double(), act, beta, dtype)
    xg, wg = pitched(x, pitch).requires_grad_(True), w.cuda().requires_grad_(True)
    bg = b.cuda().requires_grad_(True) if bias else None
    rg = pitched(r, pitch).requires_grad_(True) if residual else None
    y = A.linear_act_residual(xg, wg, bg, rg, act=act, beta=beta)
    close(y, *want['y'], 'y')
    with torch.no_grad():
        assert torch.equal(A.linear_act_residual(xg, wg, bg, rg, act=act, beta=beta), y)
    leaves = [t for t in (xg, wg, bg, rg) if t is not None]
    grads = dict(zip([k_ for k_, t in zip(('dx', 'dw', 'db', 'dr'), (xg, wg, bg, rg)) if t is not None], torch.autograd.grad(y, leaves, pitched(dy, pitch))))
    for key in ('dx', 'dw') + (('db',) if bias else ()):
        close(grads[key], *want[key], key)
    if residual:
        assert torch.equal(grads['dr'].cpu(), dy)


@pytest.mark.parametrize('dtype', TYPES, ids=IDS)
@pytest.mark.parametrize('rows,k,n,pitch', [(1, 1, 1, 0), (1, 256, 256, 0), (2, 31, 17, 1), (16, 32, 16, 0), (17, 33, 15, 0), (32, 520, 70, 3), (33, 8, 8, 0), (33, 64, 64, 0), (65, 100, 1030, 0), (999, 40, 48, 1),
                                            (40, 96, 200, 0), (130, 283, 131, 5), (257, 319, 129, 2), (1000, 7, 3, 0)])
def test_dense_sizes(dtype, rows, k, n, pitch):
    check_dense(rows, k, n, dtype, 'silu', pitch=pitch)


@pytest.mark.parametrize('dtype', TYPES, ids=IDS)
def test_dense_large_tiles(dtype):
    """enough tiles for the 128 x 128 kernels of all three products, none of them whole"""
    check_dense(33001, 129, 130, dtype, 'gelu')
    check_dense(16500, 264, 136, dtype, None, pitch=8)


@pytest.mark.parametrize('dtype', TYPES, ids=IDS)
@pytest.mark.parametrize('rows,k,n,act,pitch', [(16384, 8, 8, 'silu', 0), (16401, 128, 128, 'gelu', 0), (20000, 100, 60, 'softplus', 3), (17000, 256, 256, 'silu', 0),
                                                (16999, 250, 13, 'sigmoid', 1), (40007, 33, 256, 'gelu', 0), (16400, 128, 512, 'silu', 0), (70001, 63, 31, None, 0), (33001, 9, 129, 'relu', 5)])
def test_dense_small_layer_many_rows(dtype, rows, k, n, act, pitch):
    """layers whose weight stays on chip (16-bit types), every wave with several groups of rows and a last partial one"""
    check_dense(rows, k, n, dtype, act, pitch=pitch, bias=act != 'silu', residual=act != 'sigmoid')


@pytest.mark.parametrize('dtype', TYPES, ids=IDS)
@pytest.mark.parametrize('act,beta', [(None, 1.0), ('relu', 1.0), ('sigmoid', 1.0), ('softplus', 1.0), ('softplus', 100.0), ('gelu', 1.0)])
def test_dense_activations(dtype, act, beta):
    check_dense(77, 40, 50, dtype, act, beta)
    check_dense(9, 40, 50, dtype, act, beta, bias=False, residual=False)


@pytest.mark.parametrize('rows', [200, 16400])
def test_dense_infinite_input_stays_in_its_row(rows):
    """an infinity in one input row: its pre-activations are infinite and the slopes zero, every other row is as without it"""
    from arcnerf_amd.ops import autograd as A
    x, w, b, _, dy = (t.cuda() for t in dense_inputs(rows, 24, 13, torch.bfloat16))
    bad = x.clone()
    bad[5, 3] = float('inf')
    w[:, 3] = w[:, 3].abs() + 0.25
    got = []
    for t in (x, bad):
        t = t.requires_grad_(True)
        y = A.linear_act_residual(t, w, b, act='sigmoid')
        got.append((y.detach(), torch.autograd.grad(y, t, dy)[0]))
    keep = torch.arange(rows, device='cuda') != 5
    assert torch.equal(got[0][0][keep], got[1][0][keep]) and torch.equal(got[0][1][keep], got[1][1][keep])
    assert (got[1][0][5] == 1).all() and (got[1][1][5] == 0).all()


def test_dense_far_preactivations():
    """the activations at pre-activations where an exponential over- or underflows"""
    from arcnerf_amd.ops import autograd as A
    z = torch.tensor([-3e38, -1e4, -200.0, -90.0, -20.0, -1e-6, 0.0, 1e-6, 20.0, 90.0, 200.0, 1e4, 3e38], device='cuda')
    for rows in (13, 52):
        x = z.repeat(rows // 13)[:, None].clone().requires_grad_(True)
        w = torch.ones(1, 1, device='cuda')
        for act in ('relu', 'sigmoid', 'softplus', 'silu', 'gelu'):
            y = A.linear_act_residual(x, w, act=act)
            g, = torch.autograd.grad(y.sum(), x)
            ref, slope, _ = act64(x.detach().double().cpu(), act)
            assert torch.isfinite(y).all() and torch.isfinite(g).all(), act
            assert ((y.double().cpu() - ref).abs() <= C0 * E * (1 + ref.abs())).all(), act
            assert ((g.double().cpu() - slope)[ref != 0].abs() <= 2 * C0 * E).all(), act


def test_dense_broadcast_transposed_and_shared_inputs():
    """an expanded input, a transposed weight, the input as its own residual: gradients add up as autograd has them"""
    from arcnerf_amd.ops import autograd as A
    row = randn(1, 1, 24, dtype=torch.float32)
    w = randn(2, 24, 24, dtype=torch.float32, scale=0.2)
    rg, wg = row.cuda().requires_grad_(True), w.t().contiguous().cuda().requires_grad_(True)
    x = rg.expand(50, 24)
    y = A.linear_act_residual(x, wg.t(), None, x, act='silu')
    g_row, g_w = torch.autograd.grad(y.sum(), [rg, wg])
    r64, w64 = row.double().requires_grad_(True), w.double().requires_grad_(True)
    x64 = r64.expand(50, 24)
    y64 = torch.nn.functional.silu(x64 @ w64.t()) + x64
    h_row, h_w = torch.autograd.grad(y64.sum(), [r64, w64])
    # 50 equal rows; sums of 50 x 24 products of size <= ~4: (1200 + c) e of their sizes
    assert ((y.double().cpu() - y64).abs() <= 64 * E * (1 + x64.abs() @ w.double().abs().t() + y64.abs())).all()
    tol = (1200 + C0) * E * 50
    assert (g_row.double().cpu() - h_row).abs().max().item() <= tol * (1 + w.double().abs().sum(0).max().item())
    assert (g_w.t().double().cpu() - h_w).abs().max().item() <= tol * (1 + row.double().abs().max().item())


def test_dense_gradients_against_differences():
    """central differences of the float32 layer: step h = 2^-7, error h^2 / 6 times the third derivative (|act'''| <= 2) and the values' rounding / h"""
    from arcnerf_amd.ops import autograd as A
    x, w, b, r, dy = (t.cuda() for t in dense_inputs(5, 6, 7, torch.float32))
    h = 2.0 ** -7
    for act in ('silu', 'gelu', 'softplus', 'sigmoid'):
        leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
        grads = torch.autograd.grad(A.linear_act_residual(*leaves, r, act=act), leaves, dy)
        for at, (t, g) in enumerate(zip((x, w, b), grads)):
            for k in (0, t.numel() // 2, t.numel() - 1):
                val = []
                for sgn in (1, -1):
                    moved = [v.clone() for v in (x, w, b)]
                    moved[at].view(-1)[k] += sgn * h
                    val.append((A.linear_act_residual(*moved, r, act=act).double() * dy.double()).sum().item())
                scale = dy.abs().sum().item() * (1 + x.abs().max().item()) ** 3
                assert abs((val[0] - val[1]) / (2 * h) - g.view(-1)[k].item()) <= scale * (h * h / 3 + 64 * E / h), (act, at, k)


def test_dense_empty_batch_and_leading_dimensions():
    from arcnerf_amd.ops import autograd as A
    w = torch.ones(5, 3, device='cuda', requires_grad=True)
    b = torch.ones(5, device='cuda', requires_grad=True)
    x = torch.zeros(0, 3, device='cuda', requires_grad=True)
    y = A.linear_act_residual(x, w, b, act='relu')
    assert y.shape == (0, 5)
    gx, gw, gb = torch.autograd.grad(y.sum(), [x, w, b])
    assert gx.shape == (0, 3) and gw.abs().max().item() == 0 and gb.abs().max().item() == 0
    x3 = randn(1, 2, 3, 4, 3, dtype=torch.float32).cuda()
    y3 = A.linear_act_residual(x3, w, b, torch.zeros(2, 3, 4, 5, device='cuda'), act='relu')
    assert torch.equal(y3.view(-1, 5), A.linear_act_residual(x3.view(-1, 3), w, b, act='relu'))


def test_dense_rows_past_32_bit_offsets():
    """the last rows of a buffer of more than 2^32 bytes and 2^31 elements"""
    from arcnerf_amd.ops import functional as F
    rows, pitch = 140000, 16384                    # 2.3e9 elements
    wide = torch.empty(rows, pitch, dtype=torch.bfloat16, device='cuda')
    x = wide[:, 16000:16040]
    x.copy_(randn(1, rows, 40, dtype=torch.float32).cuda())
    w = randn(2, 24, 40, dtype=torch.bfloat16).cuda()
    y, packed = F.dense_fwd(x, w, act='silu'), F.dense_fwd(x.contiguous(), w, act='silu')
    assert torch.equal(y, packed)
    n, packed = F.layer_norm_fwd(x), F.layer_norm_fwd(x.contiguous())
    assert torch.equal(n, packed)
    dw, packed = F.dense_dw(y, x)[0], F.dense_dw(y, x.contiguous())[0]
    assert torch.equal(dw, packed)


# ---- gated block ------------------------------------------------------------------------------------------------------------------------
def gated_bounds(x, wg, wu, wd, bg, bu, bd, r, dy, act, beta, dtype):
    (S, K), H, N = x.shape, wg.shape[0], wd.shape[0]
    u, t = unit(dtype), tiny(dtype)
    g, up = x @ wg.t() + bg, x @ wu.t() + bu
    g_err = (K + C0) * E * (x.abs() @ wg.abs().t() + bg.abs())
    u_err = (K + C0) * E * (x.abs() @ wu.abs().t() + bu.abs())
    a, s, curve = act64(g, act, beta)
    a_err = 1.2 * g_err + C0 * E * (a.abs() + g.abs() + 1)
    h = a * up
    h_err = u * h.abs() + t + (a_err * up.abs() + a.abs() * u_err + a_err * u_err + E * h.abs()) * (1 + u)
    y = h @ wd.t() + bd + r
    res = {'y': (y, u * y.abs() + t + ((h_err + (H + C0) * E * h.abs()) @ wd.abs().t() + C0 * E * (bd.abs() + r.abs() + y.abs())) * 1.01)}
    dh = dy @ wd
    dh_err = (N + C0) * E * (dy.abs() @ wd.abs())
    s_err = C0 * E + curve * g_err
    dg, du = dh * up * s, dh * a
    dg_err = u * dg.abs() + t + 1.01 * (dh_err * (up * s).abs() + dh.abs() * (u_err * s.abs() + up.abs() * s_err) + C0 * E * dg.abs())
    du_err = u * du.abs() + t + 1.01 * (dh_err * a.abs() + dh.abs() * a_err + C0 * E * du.abs())
    dx = dg @ wg + du @ wu
    res['dx'] = (dx, u * dx.abs() + t + 1.01 * ((dg_err + (2 * H + C0) * E * dg.abs()) @ wg.abs() + (du_err + (2 * H + C0) * E * du.abs()) @ wu.abs()))
    sum_e = (S + C0) * E
    for k, v, e in (('g', dg, dg_err), ('u', du, du_err)):
        res['dw' + k] = (v.t() @ x, u * (v.t() @ x).abs() + t + 1.01 * (e + sum_e * v.abs()).t() @ x.abs())
        res['db' + k] = (v.sum(0), u * v.sum(0).abs() + t + 1.01 * (e + sum_e * v.abs()).sum(0))
    dwd = dy.t() @ h
    res['dwd'] = (dwd, u * dwd.abs() + t + 1.01 * dy.abs().t() @ (h_err + sum_e * h.abs()))
    res['dbd'] = (dy.sum(0), u * dy.sum(0).abs() + t + 1.01 * sum_e * dy.abs().sum(0))
    return res


def gated_inputs(rows, k, hid, n, dtype):
    p = dict(x=randn(20, rows, k, dtype=dtype), wg=randn(21, hid, k, dtype=dtype, scale=k ** -0.5), wu=randn(22, hid, k, dtype=dtype, scale=k ** -0.5),
             wd=randn(23, n, hid, dtype=dtype, scale=hid ** -0.5), bg=randn(24, hid, dtype=dtype, scale=0.2), bu=randn(25, hid, dtype=dtype, scale=0.2),
             bd=randn(26, n, dtype=dtype, scale=0.2), r=randn(27, rows, n, dtype=dtype))
    return p, randn(28, rows, n, dtype=dtype)


def check_gated(rows, k, hid, n, dtype, act='silu', beta=1.0, pitch=0, bias=True, residual=True):
    from arcnerf_amd.ops import autograd as A
    p, dy = gated_inputs(rows, k, hid, n, dtype)
    z = torch.zeros((), dtype=torch.float64)
    q = {key: v.double() for key, v in p.items()}
    if not bias:
        q.update(bg=z.expand(hid), bu=z.expand(hid), bd=z.expand(n))
    if not residual:
        q['r'] = z.expand(rows, n)
    want = gated_bounds(*(q[key] for key in ('x', 'wg', 'wu', 'wd', 'bg', 'bu', 'bd', 'r')), dy.double(), act, beta, dtype)
    d = {key: (pitched(v, pitch) if key in ('x', 'r') else v.cuda()).requires_grad_(True) for key, v in p.items()
         if (bias or key not in ('bg', 'bu', 'bd')) and (residual or key != 'r')}
    y = A.gated_ffn(d['x'], d['wg'], d['wu'], d['wd'], d.get('bg'), d.get('bu'), d.get('bd'), d.get('r'), act=act, beta=beta)
    close(y, *want['y'], 'y')
    names = list(d)
    grads = dict(zip(names, torch.autograd.grad(y, [d[key] for key in names], pitched(dy, pitch))))
    for key in names:
        if key == 'r':
            assert torch.equal(grads['r'].cpu(), dy)
        else:
            close(grads[key], *want['d' + key], 'd' + key)


@pytest.mark.parametrize('dtype', TYPES, ids=IDS)
@pytest.mark.parametrize('rows,k,hid,n,pitch', [(1, 1, 1, 1, 0), (1, 256, 1024, 256, 0), (8, 64, 96, 64, 0), (17, 33, 31, 29, 1), (32, 40, 65, 40, 0), (33, 32, 32, 32, 0), (100, 20, 1100, 20, 0), (1024, 24, 40, 16, 0),
                                                (61, 131, 347, 131, 3), (300, 48, 130, 24, 0), (129, 72, 64, 200, 8)])
def test_gated_sizes(dtype, rows, k, hid, n, pitch):
    check_gated(rows, k, hid, n, dtype, pitch=pitch)


@pytest.mark.parametrize('dtype', TYPES, ids=IDS)
def test_gated_large_tiles(dtype):
    check_gated(8301, 130, 260, 136, dtype, 'gelu')
    check_gated(33000, 264, 72, 264, dtype, 'silu', bias=False, residual=False)


@pytest.mark.parametrize('dtype', TYPES, ids=IDS)
@pytest.mark.parametrize('act', ['gelu', 'sigmoid', 'softplus', None])
def test_gated_activations(dtype, act):
    check_gated(50, 24, 40, 24, dtype, act, bias=act != 'gelu', residual=act != 'sigmoid')


def test_gated_shared_weight_and_partial_gradients():
    """one weight as gate and up projection; gradients asked of some of the leaves only"""
    from arcnerf_amd.ops import autograd as A
    p, dy = gated_inputs(40, 24, 32, 24, torch.float32)
    w, wd, x, bu = p['wg'].cuda().requires_grad_(True), p['wd'].cuda(), p['x'].cuda(), p['bu'].cuda().requires_grad_(True)
    y = A.gated_ffn(x, w, w, wd, b_up=bu)
    dw, dbu = torch.autograd.grad(y, [w, bu], dy.cuda())
    z = torch.zeros(1, dtype=torch.float64)
    q = {key: v.double() for key, v in p.items()}
    want = gated_bounds(q['x'], q['wg'], q['wg'], q['wd'], z.expand(32), q['bu'], z.expand(24), z.expand(40, 24), dy.double(), 'silu', 1.0, torch.float32)
    close(dw, want['dwg'][0] + want['dwu'][0], want['dwg'][1] + want['dwu'][1] + E * (want['dwg'][0] + want['dwu'][0]).abs(), 'dw')
    close(dbu, *want['dbu'], 'dbu')
    wd2 = p['wd'].cuda().requires_grad_(True)
    dwd, = torch.autograd.grad(A.gated_ffn(x, w.detach(), w.detach(), wd2, b_up=bu.detach()), wd2, dy.cuda())
    close(dwd, *want['dwd'], 'dwd')


# ---- a whole block, streams and graphs ----------------------------------------------------------------------------------------------------
def block(A, x, p):
    n = A.layer_norm(x, p['nw'], p['nb'])
    x = A.gated_ffn(n, p['wg'], p['wu'], p['wd'], residual=x)
    return A.linear_act_residual(x, p['wo'], p['bo'], act='gelu')


def block_params(dtype, k, hid, n):
    return {'nw': randn(30, k, dtype=dtype, scale=0.1, offset=1.0), 'nb': randn(31, k, dtype=dtype, scale=0.1),
            'wg': randn(32, hid, k, dtype=dtype, scale=k ** -0.5), 'wu': randn(33, hid, k, dtype=dtype, scale=k ** -0.5),
            'wd': randn(34, k, hid, dtype=dtype, scale=hid ** -0.5), 'wo': randn(35, n, k, dtype=dtype, scale=k ** -0.5),
            'bo': randn(36, n, dtype=dtype, scale=0.1)}


@pytest.mark.parametrize('dtype,rel', [(torch.float32, 64 * E), (torch.bfloat16, 8 * 2.0 ** -8), (torch.float16, 8 * 2.0 ** -11)], ids=IDS)
def test_block_forward_and_backward(dtype, rel):
    """norm, gated block with residual, dense layer, as a residual net runs them.  In the 2-norm: each of the chain's at most 8 stored tensors in
    front of a result adds one relative rounding (f32: a sum's random-sign roundings, sqrt of the longest, 300, times 3)"""
    from arcnerf_amd.ops import autograd as A
    p = block_params(dtype, 72, 160, 40)
    x, dy = randn(37, 300, 72, dtype=dtype), randn(38, 300, 40, dtype=dtype)
    leaves = {k: v.cuda().requires_grad_(True) for k, v in dict(p, x=x).items()}
    y = block(A, leaves['x'], leaves)
    got = dict(zip(leaves, torch.autograd.grad(y, list(leaves.values()), dy.cuda())), y=y)
    ref = {k: v.double().requires_grad_(True) for k, v in dict(p, x=x).items()}
    fn = torch.nn.functional
    n = fn.layer_norm(ref['x'], (72,), ref['nw'], ref['nb'])
    m = (fn.silu(n @ ref['wg'].t()) * (n @ ref['wu'].t())) @ ref['wd'].t() + ref['x']
    y64 = fn.gelu(m @ ref['wo'].t() + ref['bo'])
    want = dict(zip(ref, torch.autograd.grad(y64, list(ref.values()), dy.double())), y=y64)
    for k, v in want.items():
        assert ((got[k].double().cpu() - v).norm() / v.norm()).item() <= rel, k


@pytest.mark.parametrize('dtype', TYPES, ids=IDS)
def test_block_on_a_side_stream_and_replayed(dtype):
    """a side stream gives the same bits; a captured training pass replays to the eager result, with other work and other inputs in between, also
    beside a second graph of the same calls"""
    from arcnerf_amd.ops import autograd as A
    p = {k: v.cuda().requires_grad_(True) for k, v in block_params(dtype, 72, 160, 40).items()}
    xs = [randn(40 + i, 300, 72, dtype=dtype).cuda() for i in range(3)]
    dy = randn(39, 300, 40, dtype=dtype).cuda()

    def run(x):
        x = x.detach().requires_grad_(True)
        y = block(A, x, p)
        return (y.detach(),) + torch.autograd.grad(y, [x] + list(p.values()), dy)

    want = [run(x) for x in xs]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run(xs[0])
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want[0]))
    del got
    held = [xs[0].clone(), xs[1].clone()]
    graphs, outs = [], []
    for h in held:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(run(h))
        graphs.append(g)
    for trip in range(4):
        for k in (0, 1):
            held[k].copy_(xs[(trip + k) % 3])
        graphs[0].replay()
        graphs[1].replay()
        eager = run(xs[(trip + 2) % 3])
        torch.cuda.synchronize()
        for k in (0, 1):
            for a, b in zip(outs[k], want[(trip + k) % 3]):
                assert torch.equal(a, b), (trip, k)
        assert all(torch.equal(a, b) for a, b in zip(eager, want[(trip + 2) % 3]))


def test_second_differentiation_is_refused():
    from arcnerf_amd.ops import autograd as A
    x = randn(1, 40, 16, dtype=torch.float32).cuda().requires_grad_(True)
    w = randn(2, 16, 16, dtype=torch.float32).cuda()
    for y in (A.layer_norm(x), A.linear_act_residual(x, w, act='silu'), A.gated_ffn(x, w, w, w)):
        g, = torch.autograd.grad(y.square().sum(), x, create_graph=True)
        with pytest.raises(RuntimeError):
            torch.autograd.grad(g.sum(), x)


def test_gpu_refusals():
    from arcnerf_amd.ops import autograd as A
    x, w = torch.zeros(4, 8, device='cuda'), torch.zeros(6, 8, device='cuda')
    bad = [lambda: A.linear_act_residual(x, w.bfloat16()), lambda: A.linear_act_residual(x.double(), w.double()), lambda: A.linear_act_residual(x, torch.zeros(6, 7, device='cuda')),
           lambda: A.linear_act_residual(x, w, torch.zeros(5, device='cuda')), lambda: A.linear_act_residual(x, w, None, torch.zeros(4, 5, device='cuda')),
           lambda: A.linear_act_residual(x, w, None, torch.zeros(1, 6, device='cuda')), lambda: A.linear_act_residual(x, w, act='tanh'),
           lambda: A.linear_act_residual(x, w, act='softplus', beta=0.0), lambda: A.linear_act_residual(x, w.cpu()), lambda: A.linear_act_residual(x, w[:, :0]),
           lambda: A.layer_norm(x, torch.ones(7, device='cuda')), lambda: A.layer_norm(x, torch.ones(8, device='cuda', dtype=torch.float16)),
           lambda: A.layer_norm(x.half(), torch.ones(8, device='cuda'), torch.ones(8, device='cuda').half()), lambda: A.layer_norm(x, torch.ones(8)),
           lambda: A.layer_norm(torch.zeros(3, 0, device='cuda')), lambda: A.gated_ffn(x, w, w[:5], torch.zeros(8, 6, device='cuda')),
           lambda: A.gated_ffn(x, w, w, torch.zeros(8, 7, device='cuda')), lambda: A.gated_ffn(x, w, w, torch.zeros(8, 6, device='cuda'), b_up=torch.zeros(5, device='cuda'))]
    for k, call in enumerate(bad):
        with pytest.raises(RuntimeError):
            call()
            pytest.fail('call {} went through'.format(k))
