"""Calls of layer norm, the dense layer and the gated block at the edges of what they take: second and forward-mode derivatives, traces, tails
of the activations, the 256-wide kernels, sums that are exact, the calls without autograd."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def leaf(seed, *shape, dtype=torch.float32, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dtype).cuda().requires_grad_(True)


# ---- second derivatives -----------------------------------------------------------------------------------------------------------------
def small_calls():
    """name -> (function of the leaves, leaves by name): all three operators with every operand a leaf"""
    from arcnerf_amd.ops import autograd as A
    x, r = leaf(1, 40, 16), leaf(2, 40, 16)
    w, b, w2, wd = leaf(3, 16, 16), leaf(4, 16), leaf(5, 16, 16), leaf(6, 16, 16)
    return {
        'layer_norm': (lambda t: A.layer_norm(t['x'], t['w'], t['b']), dict(x=x, w=leaf(7, 16), b=b)),
        'linear_act_residual': (lambda t: A.linear_act_residual(t['x'], t['w'], t['b'], t['r'], act='silu'), dict(x=x, w=w, b=b, r=r)),
        'linear_act_residual without act': (lambda t: A.linear_act_residual(t['x'], t['w'], t['b'], t['r']), dict(x=x, w=w, b=b, r=r)),
        'gated_ffn': (lambda t: A.gated_ffn(t['x'], t['wg'], t['wu'], t['wd'], t['bg'], t['bu'], t['bd'], t['r']),
                      dict(x=x, wg=w, wu=w2, wd=wd, bg=b, bu=leaf(8, 16), bd=leaf(9, 16), r=r)),
    }


@pytest.mark.parametrize('name', ['layer_norm', 'linear_act_residual', 'linear_act_residual without act', 'gated_ffn'])
def test_a_loss_on_gradients_raises_whatever_else_it_holds(name):
    """a loss with a term in the result and one in its gradient: every way of differentiating it raises, none returns the first term alone"""
    fn, t = small_calls()[name]
    for wrt in t:
        def loss():
            y = fn(t)
            g, = torch.autograd.grad(y.square().sum(), t[wrt], create_graph=True)
            assert g.requires_grad
            return y.sum() + g.square().sum()
        for call in (lambda l: torch.autograd.grad(l, t['x']), lambda l: torch.autograd.grad(l, t['w' if 'w' in t else 'wd']), lambda l: l.backward(inputs=[t['x']]),
                     lambda l: l.backward(), lambda l: torch.autograd.grad(l, t['x'], allow_unused=True)):
            with pytest.raises(RuntimeError, match='differentiated once'):
                call(loss())


def test_a_loss_on_gradients_raises_through_the_incoming_gradient():
    """only the incoming gradient depends on the leaf that is asked for"""
    from arcnerf_amd.ops import autograd as A
    x, w, s = leaf(1, 40, 16), leaf(2, 16, 16), leaf(3, 40, 16)
    y = A.linear_act_residual(x.detach(), w, act='gelu')
    g, = torch.autograd.grad((y * s).sum(), w, create_graph=True)
    with pytest.raises(RuntimeError, match='differentiated once'):
        torch.autograd.grad(s.square().sum() + g.square().sum(), s)


@pytest.mark.parametrize('name', ['layer_norm', 'linear_act_residual', 'gated_ffn'])
def test_gradients_with_a_graph_are_the_gradients(name):
    """create_graph alone changes no value, and other terms of a loss are differentiated as ever"""
    fn, t = small_calls()[name]
    leaves = list(t.values())
    plain = torch.autograd.grad(fn(t).square().sum(), leaves)
    graph = torch.autograd.grad(fn(t).square().sum(), leaves, create_graph=True)
    for k, a, b in zip(t, plain, graph):
        assert torch.equal(a, b), k
    z = leaf(20, 5)
    got, = torch.autograd.grad(z.square().sum() + graph[0].sum(), z)
    assert torch.equal(got, 2 * z.detach())


# ---- forward-mode derivatives -----------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize('name', ['layer_norm', 'linear_act_residual', 'gated_ffn'])
def test_forward_mode_is_refused(name):
    """a tangent in any operand, with and without a graph, and through torch.func: refused, never dropped"""
    import torch.autograd.forward_ad as fw
    fn, t = small_calls()[name]
    with fw.dual_level():
        for k in t:
            for grad in (False, True):
                dual = {j: fw.make_dual(v.detach().requires_grad_(grad), torch.ones_like(v)) if j == k else v.detach() for j, v in t.items()}
                with pytest.raises(RuntimeError, match='forward-mode'):
                    fn(dual)
    x = t['x'].detach()
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda v: fn(dict({j: u.detach() for j, u in t.items()}, x=v)), (x,), (torch.ones_like(x),))


@pytest.mark.filterwarnings('ignore::DeprecationWarning')
@pytest.mark.parametrize('name', ['layer_norm', 'linear_act_residual', 'gated_ffn'])
def test_a_trace_is_refused(name):
    """with and without a graph, also where only a captured parameter meets the traced input"""
    fn, t = small_calls()[name]
    for grad in (False, True):
        with torch.set_grad_enabled(grad), pytest.raises(RuntimeError, match='cannot be traced'):
            torch.jit.trace(lambda x: fn(dict(t, x=x)), (t['x'].detach(),))
    y = fn(t)                                   # (nothing of the failed trace stays)
    assert torch.isfinite(y).all()


# ---- tails of the activations -----------------------------------------------------------------------------------------------------------
E24 = 2.0 ** -24


def values_and_slopes(z, act, rows=None):
    """act and act' at the numbers z, exactly the pre-activations of layers of one input with weight 1: of the dense layer's and the gated block's
    kernels for few rows and for many"""
    from arcnerf_amd.ops import autograd as A
    one = torch.ones(1, 1, dtype=z.dtype, device='cuda')
    for n in (z.numel(), 2000):
        x = z.repeat(-(-n // z.numel()))[:, None].cuda().requires_grad_(True)
        y = A.linear_act_residual(x, one, act=act)
        s, = torch.autograd.grad(y.sum(), x)
        yield 'dense', n, y[:z.numel(), 0].detach().double().cpu(), s[:z.numel(), 0].double().cpu()
        # the up projection is 1 by its bias: h = act(z), dg = act'(z), dx = dg
        y = A.gated_ffn(x, one, torch.zeros_like(one), one, b_up=one[0], act=act)
        s, = torch.autograd.grad(y.sum(), x)
        yield 'gated', n, y[:z.numel(), 0].detach().double().cpu(), s[:z.numel(), 0].double().cpu()


def gelu64(z):
    import math
    cdf = 0.5 * torch.erfc(z * -math.sqrt(0.5))
    phi = torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    return z * cdf, cdf + z * phi


def test_gelu_far_below_zero_f32():
    """Relative to the value, e = 2^-24: the argument of erfc carries 2 e (a constant, a product), which its condition number, at most z^2 + 1,
    carries on; erfcf 16 ulp = 32 e, the products 2 e.  The slope adds z phi: z^2 / 2 e of its exponent and 8 e of constants, products and the exponential,
    and cancels against cdf, at most 0.21 of it from -2 on: 1 / (1 - 0.21) < 1.3."""
    z = -torch.linspace(2, 9, 141)
    y64, s64 = gelu64(z.double())
    zz = z.double() ** 2
    tol_y = (2 * (zz + 1) + 34) * E24
    tol_s = 1.3 * (zz / 2 + 8 + 0.21 * tol_y / E24) * E24 + 2 * E24
    for what, n, y, s in values_and_slopes(z, 'gelu'):
        assert ((y - y64).abs() <= tol_y * y64.abs()).all(), (what, n)
        assert ((s - s64).abs() <= tol_s * s64.abs()).all(), (what, n)


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float16], ids=['bf16', 'f16'])
def test_gelu_far_below_zero_16_bits(dtype):
    """every number of the type in [-9, -2]: half a step of the result's type, and 2e-5 of the evaluation (the fit 1.5e-5, the exponent's rounding
    z^2 / 2 2^-24 and those of the products)"""
    z = -torch.arange(2.0, 9.0, 2.0 ** -9).to(dtype).unique()
    half, least = torch.finfo(dtype).eps / 2, torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2
    y64, s64 = gelu64(z.double())
    for what, n, y, s in values_and_slopes(z, 'gelu'):
        assert ((y - y64).abs() <= (half + 2e-5) * y64.abs() + least).all(), (what, n)
        assert ((s - s64).abs() <= (half + 2e-5) * s64.abs() + least).all(), (what, n)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16, torch.float16], ids=['f32', 'bf16', 'f16'])
def test_sigmoid_slope_far_from_zero(dtype):
    """s (1 - s) relative to its value on both sides of zero, e = 2^-24: the exponent's rounding |z| e (16 bits; f32 puts it back), 16 e of the
    exponential, the reciprocal and the products, and half a step of the result"""
    z = torch.cat([torch.arange(4.0, 30.0, 2.0 ** -4), -torch.arange(4.0, 30.0, 2.0 ** -4)]).to(dtype)
    half, least = torch.finfo(dtype).eps / 2, torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2
    zz = z.double()
    y64, s64 = torch.sigmoid(zz), torch.sigmoid(zz) * torch.sigmoid(-zz)
    for what, n, y, s in values_and_slopes(z, 'sigmoid'):
        assert ((y - y64).abs() <= (half + (zz.abs() + 16) * E24) * y64 + least).all(), (what, n)
        assert ((s - s64).abs() <= (half + 1.01 * (zz.abs() + 16) * E24) * s64 + least).all(), (what, n)


# ---- the modules ------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize('kind', ['gated', 'dense'])
def test_a_narrow_branch_leaves_a_wide_stream_its_bits(kind):
    from test_ffn_edges_host import STREAMS, check_stream
    for x_type, dtype in STREAMS:
        check_stream(x_type, dtype, kind, 'cuda')


# ---- sizes and sums that are exact ------------------------------------------------------------------------------------------------------
def test_gated_widest_hidden_layer():
    """more than 2^23 hidden features, whose two halves are more than 2^24 in the backward; everything in {-1, 0, 1}, so every sum is exact"""
    from arcnerf_amd.ops import autograd as A
    hid = (1 << 23) + 72
    g = torch.Generator(device='cuda').manual_seed(0)
    wg, wu, wd = (torch.randint(-1, 2, (hid,), generator=g, device='cuda').float() for _ in range(3))
    x = torch.ones(1, 1, device='cuda', requires_grad=True)
    leaves = [x] + [w.clone().requires_grad_(True) for w in (wg[:, None], wu[:, None], wd[None])]
    y = A.gated_ffn(*leaves, act=None)
    dx, dwg, dwu, dwd = torch.autograd.grad(y, leaves, torch.ones_like(y))
    assert y.item() == (wg * wu * wd).double().sum().item() and dx.item() == 2 * (wg * wu * wd).double().sum().item()
    assert torch.equal(dwg[:, 0], wd * wu) and torch.equal(dwu[:, 0], wd * wg) and torch.equal(dwd[0], wg * wu)


# ---- the calls without autograd ---------------------------------------------------------------------------------------------------------
TYPES = [torch.float32, torch.bfloat16, torch.float16]
IDS = ['f32', 'bf16', 'f16']


def wide_rows(seed, rows, width, dtype):
    """a column slice of a wider buffer"""
    return leaf(seed, rows, width + 5, dtype=dtype).detach()[:, 3:3 + width]


def same(a, b):
    assert len(a) == len(b)
    for k, (u, v) in enumerate(zip(a, b)):
        assert (u is None) == (v is None) and (u is None or (u.dtype == v.dtype and torch.equal(u, v))), k


@pytest.mark.parametrize('dtype', TYPES, ids=IDS)
@pytest.mark.parametrize('rows,width', [(1, 8), (37, 45), (300, 256), (0, 16)])
def test_layer_norm_calls_are_the_nodes(dtype, rows, width):
    from arcnerf_amd.ops import autograd as A, functional as F
    for wt in (dtype, torch.float32):
        x, dy = wide_rows(1, rows, width, dtype), wide_rows(2, rows, width, dtype)
        w, b = leaf(3, width, dtype=wt), leaf(4, width, dtype=wt)
        xg = x.detach().requires_grad_(True)
        y, stats = F.layer_norm_fwd(x, w.detach(), b.detach(), want_stats=True)
        yn = A.layer_norm(xg, w, b)
        same((y, F.layer_norm_fwd(x, w.detach(), b.detach())), (yn.detach(),) * 2)
        want = torch.autograd.grad(yn, [xg, w, b], dy)
        same(F.layer_norm_bwd(x, dy, w.detach(), stats), want)
        spread = torch.full((rows, 5), float('nan'), device='cuda')
        spread[:, 1:3] = stats                                              # statistics that are not contiguous
        same(F.layer_norm_bwd(x, dy, w.detach(), spread[:, 1:3], want_dx=False), (None,) + want[1:])
        same(F.layer_norm_bwd(x, dy, w.detach(), stats, want_dw=False, want_db=False), (want[0], None, None))
        # no weight: the type of the bias's gradient is the caller's
        bn = leaf(4, width, dtype=wt)
        db, = torch.autograd.grad(A.layer_norm(x, None, bn), bn, dy)
        same(F.layer_norm_bwd(x, dy, None, stats, want_dx=False, want_dw=False, param_dtype=wt), (None, None, db))


@pytest.mark.parametrize('dtype', TYPES, ids=IDS)
@pytest.mark.parametrize('rows,k,n', [(1, 8, 8), (37, 45, 21), (500, 128, 72), (17000, 40, 56), (30000, 40, 56), (0, 16, 8)])
def test_dense_calls_are_the_nodes(dtype, rows, k, n):
    from arcnerf_amd.ops import autograd as A, functional as F
    x, dy, r = wide_rows(1, rows, k, dtype), wide_rows(2, rows, n, dtype), wide_rows(3, rows, n, dtype)
    w, b = leaf(4, n, k, dtype=dtype, scale=0.2), leaf(5, n, dtype=dtype)
    wd, bd = w.detach(), b.detach()
    for act in ('gelu', 'softplus', None):
        xg = x.detach().requires_grad_(True)
        y = A.linear_act_residual(xg, w, b, r, act=act, beta=2.0)
        same((F.dense_fwd(x, wd, bd, r, act, 2.0),), (y.detach(),))
        want = torch.autograd.grad(y, [xg, w, b], dy)
        dz, dx, sums = F.dense_dz(x, wd, bd, dy, act, 2.0, want_dx=True, want_sums=True)
        assert (sums is not None) == (rows > 0 and act is not None and dtype != torch.float32)
        same((dx,) + F.dense_dw(dz, x, True, sums), want)
        same(F.dense_dw(dz, x, sums=sums), (want[1], None))
        same(F.dense_dz(x, wd, bd, dy, act, 2.0, want_dx=True) + F.dense_dw(dz, x), (dz, dx, want[1], None))
        if act is None or rows < 24576:                                     # (else dx comes from the kernel of dz, in another order of sums)
            alone = F.dense_dz(x, wd, bd, dy, act, 2.0)
            same((alone, F.dense_dx(alone, wd)), (dz, dx))
            alone, some = F.dense_dz(x, wd, bd, dy, act, 2.0, want_sums=True)
            same((alone, some), (dz, sums))


@pytest.mark.parametrize('dtype', TYPES, ids=IDS)
@pytest.mark.parametrize('rows,k,hid,n', [(1, 8, 16, 8), (37, 45, 21, 30), (700, 64, 136, 72), (0, 8, 8, 8)])
def test_gated_calls_are_the_nodes(dtype, rows, k, hid, n):
    from arcnerf_amd.ops import autograd as A, functional as F
    x, dy, r = wide_rows(1, rows, k, dtype), wide_rows(2, rows, n, dtype), wide_rows(3, rows, n, dtype)
    p = {'wg': leaf(4, hid, k, dtype=dtype, scale=0.2), 'wu': leaf(5, hid, k, dtype=dtype, scale=0.2), 'wd': leaf(6, n, hid, dtype=dtype, scale=0.2),
         'bg': leaf(7, hid, dtype=dtype), 'bu': leaf(8, hid, dtype=dtype), 'bd': leaf(9, n, dtype=dtype)}
    q = {name: t.detach() for name, t in p.items()}
    xg = x.detach().requires_grad_(True)
    y = A.gated_ffn(xg, p['wg'], p['wu'], p['wd'], p['bg'], p['bu'], p['bd'], r, act='silu')
    h = F.gated_fwd(x, q['wg'], q['wu'], q['bg'], q['bu'])
    same((F.dense_fwd(h, q['wd'], q['bd'], r),), (y.detach(),))
    want = dict(zip(['x'] + list(p), torch.autograd.grad(y, [xg] + list(p.values()), dy)))
    dgu, sums = F.gated_bwd(x, q['wg'], q['wu'], q['bg'], q['bu'], dy, q['wd'], want_sums=True)
    same((F.gated_bwd(x, q['wg'], q['wu'], q['bg'], q['bu'], dy, q['wd']),), (dgu,))
    dw, db = F.dense_dw(dgu, x, True, sums)
    same((F.dense_dx(dgu, q['wg'], q['wu']), dw[:hid], dw[hid:], db[:hid], db[hid:]) + F.dense_dw(dy, h, want_db=True),
         tuple(want[name] for name in ('x', 'wg', 'wu', 'bg', 'bu', 'wd', 'bd')))


def test_calls_without_autograd_refuse():
    from arcnerf_amd.ops import functional as F
    x, w, st = torch.zeros(4, 8, device='cuda'), torch.zeros(6, 8, device='cuda'), torch.zeros(4, 2, device='cuda')
    bad = [lambda: F.layer_norm_bwd(x, x, None, st, param_dtype=torch.float64), lambda: F.layer_norm_bwd(x, x, None, st, param_dtype=torch.bfloat16),
           lambda: F.layer_norm_bwd(x, x, None, st[:3]), lambda: F.layer_norm_bwd(x, x, None, st.half()), lambda: F.layer_norm_bwd(x, x[:3], None, st),
           lambda: F.layer_norm_bwd(x, x, torch.ones(7, device='cuda'), st), lambda: F.dense_dz(x, w, None, x, 'silu'), lambda: F.dense_dz(x, w, None, x[:, :6].half(), 'silu'),
           lambda: F.dense_dw(x, x, True, torch.zeros(1, 7, device='cuda')), lambda: F.dense_dw(x, x, True, torch.zeros(1, 8, device='cuda')),
           lambda: F.dense_dw(x.half(), x.half(), True, torch.zeros(2, 8, device='cuda')), lambda: F.dense_dw(x.half(), x.half(), True, torch.zeros(1, 8, device='cuda').half()),
           lambda: F.dense_dx(x, w), lambda: F.dense_dx(x[:, :7], w[:3], w[:3]), lambda: F.dense_dx(x, w[:4], w[:3]), lambda: F.dense_dw(x, x[:3]),
           lambda: F.gated_fwd(x, w, w[:5]), lambda: F.gated_bwd(x, w, w, None, None, x, torch.zeros(8, 5, device='cuda')),
           lambda: F.gated_bwd(x, w, w, None, None, x[:, :7], torch.zeros(8, 6, device='cuda'))]
    for k, call in enumerate(bad):
        with pytest.raises(RuntimeError):
            call()
            pytest.fail('call {} went through'.format(k))


# ---- exact sums: a row, a tile or a slab that is lost or counted twice changes them, whatever the number of rows --------------------------
def ints(seed, *shape, dtype):
    """-1, 0, 1: products and sums of up to 2^24 of them are exact in float32"""
    g = torch.Generator(device='cuda').manual_seed(seed)
    return torch.randint(-1, 2, shape, generator=g, device='cuda').to(dtype)


def exact(a, b):
    """a product of integers, float64"""
    return a.double() @ b.double()


@pytest.mark.parametrize('dtype', TYPES, ids=IDS)
@pytest.mark.parametrize('rows,k,n', [(1, 1, 1), (255, 24, 40), (1000, 7, 3), (33001, 129, 130), (16400, 128, 72), (24577, 128, 512), (70001, 63, 31), (17000, 256, 256), (20003, 520, 520),
                                      (33100, 520, 520), (66000, 264, 264), (300007, 16, 16)])
def test_dense_sums_are_exact(dtype, rows, k, n):
    """forward, dx, dW and db of the layer without an activation and of one whose activation is the identity (relu above zero: the kernels that compute
    the slope): integers, rounded once.  At most 300007 terms, 2^18.2; a bias of 1024 is above any sum of 520 terms."""
    from arcnerf_amd.ops import autograd as A
    x, w, r, dy = ints(1, rows, k, dtype=dtype), ints(2, n, k, dtype=dtype), ints(3, rows, n, dtype=dtype), ints(4, rows, n, dtype=dtype)
    z, dx, dw, db = exact(x, w.t()), exact(dy, w), exact(dy.t(), x), dy.double().sum(0)
    for act, offset in ((None, 1), ('relu', 1024)):
        b = torch.full((n,), offset, dtype=dtype, device='cuda')
        leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
        y = A.linear_act_residual(*leaves, r, act=act)
        assert torch.equal(y.detach(), (z + offset + r.double()).to(dtype)), (act, 'y')
        for name, got, want in zip(('dx', 'dw', 'db'), torch.autograd.grad(y, leaves, dy), (dx, dw, db)):
            assert torch.equal(got, want.to(dtype)), (act, name)


@pytest.mark.parametrize('dtype', TYPES, ids=IDS)
@pytest.mark.parametrize('rows,k,hid,n', [(1, 1, 1, 1), (300, 24, 40, 16), (8301, 130, 260, 136), (33000, 264, 520, 264), (50001, 256, 264, 256)])
def test_gated_sums_are_exact(dtype, rows, k, hid, n):
    """the block without an activation, all of it integers: h = g u, du = dh g and dg = dh u are rounded to the type (the bias gradients are the sums of
    what they were before), every result once.  Sums of k <= 264 terms are below 2^9, h below 2^18, dh below 2^9 (n <= 264) and the others far
    inside 2^24 (random signs: 2^8.5 sqrt(33000))."""
    from arcnerf_amd.ops import autograd as A
    x, dy, r = ints(1, rows, k, dtype=dtype), ints(2, rows, n, dtype=dtype), ints(3, rows, n, dtype=dtype)
    wg, wu, wd = ints(4, hid, k, dtype=dtype), ints(5, hid, k, dtype=dtype), ints(6, n, hid, dtype=dtype)
    bg, bu, bd = ints(7, hid, dtype=dtype), ints(8, hid, dtype=dtype), ints(9, n, dtype=dtype)
    leaves = [t.clone().requires_grad_(True) for t in (x, wg, wu, wd, bg, bu, bd)]
    y = A.gated_ffn(*leaves, r, act=None)
    got = torch.autograd.grad(y, leaves, dy)
    g, u, dh = exact(x, wg.t()) + bg.double(), exact(x, wu.t()) + bu.double(), exact(dy, wd)
    h, dg, du = ((a * b).to(dtype).double() for a, b in ((g, u), (dh, u), (dh, g)))
    assert torch.equal(y.detach(), (exact(h, wd.t()) + bd.double() + r.double()).to(dtype))
    want = (exact(dg, wg) + exact(du, wu), exact(dg.t(), x), exact(du.t(), x), exact(dy.t(), h), (dh * u).sum(0), (dh * g).sum(0), dy.double().sum(0))
    for name, a, b in zip(('dx', 'dwg', 'dwu', 'dwd', 'dbg', 'dbu', 'dbd'), got, want):
        assert torch.equal(a, b.to(dtype)), name


@pytest.mark.parametrize('dtype', TYPES, ids=IDS)
@pytest.mark.parametrize('rows,k,n', [(3, 8, 16), (1001, 24, 40), (1001, 25, 41), (16500, 64, 136), (25001, 64, 136), (33001, 129, 130), (40003, 256, 256), (70001, 100, 500), (33100, 520, 520)])
def test_bias_gradient_has_no_rounded_terms(dtype, rows, k, n):
    """weights of zero: dz = dy act'(b), the same digits in every row, which a 16-bit dz rounds the same way every time.  The sum is rounded once; its
    terms carry 24 e (e = 2^-24) of the slope and the product, and no chain of its additions is longer than 256."""
    from arcnerf_amd.ops import autograd as A
    b = torch.linspace(-3, 3, n).to(dtype)
    dy = ints(1, rows, n, dtype=dtype).abs() + 1
    w = torch.zeros(n, k, dtype=dtype, device='cuda', requires_grad=True)
    x, bg = ints(2, rows, k, dtype=dtype).requires_grad_(True), b.cuda().requires_grad_(True)
    y = A.linear_act_residual(x, w, bg, act='sigmoid')
    s = torch.sigmoid(b.double()) * torch.sigmoid(-b.double())
    want = s * dy.double().sum(0).cpu()
    tol = torch.finfo(dtype).eps / 2 * want + (256 + 24) * E24 * want
    for leaves in ([x, w, bg], [bg]):
        db = torch.autograd.grad(y, leaves, dy, retain_graph=True)[-1].double().cpu()
        assert ((db - want).abs() <= tol).all(), ((db - want).abs() / tol).max().item()


@pytest.mark.parametrize('dtype', TYPES, ids=IDS)
@pytest.mark.parametrize('rows,width', [(1, 8), (129, 8), (300001, 8), (40003, 64), (40003, 256), (40003, 512), (40003, 1024), (5001, 2048), (3001, 4096), (2501, 8192)])
def test_layer_norm_weight_gradients_are_exact(dtype, rows, width):
    """rows of as many +1 as -1 have mean 0 and, at a width that is a power of two, variance 1: n = x, and with eps = 0 and integers for dy the
    weight's gradient sum dy x and the bias's sum dy are integers, rounded once"""
    from arcnerf_amd.ops import autograd as A
    half = torch.rand(rows, width, generator=torch.Generator(device='cuda').manual_seed(1), device='cuda').argsort(1) < width // 2
    x = torch.where(half, 1.0, -1.0).to(dtype)
    dy = ints(2, rows, width, dtype=dtype)
    w, b = torch.ones(width, dtype=dtype, device='cuda', requires_grad=True), torch.zeros(width, dtype=dtype, device='cuda', requires_grad=True)
    y = A.layer_norm(x, w, b, eps=0.0)
    assert torch.equal(y.detach(), x)
    dw, db = torch.autograd.grad(y, [w, b], dy)
    assert torch.equal(dw, (dy.double() * x.double()).sum(0).to(dtype)) and torch.equal(db, dy.double().sum(0).to(dtype))


# ---- the 256-wide tiles of the 16-bit types ----------------------------------------------------------------------------------------------
@pytest.mark.parametrize('dtype', TYPES[1:], ids=IDS[1:])
@pytest.mark.parametrize('rows,k,n,act', [(66000, 264, 264, 'silu'), (65537, 256, 256, 'gelu'), (33100, 520, 520, 'softplus'), (33100, 328, 776, None)])
def test_dense_256_wide(dtype, rows, k, n, act):
    """more than 256 tiles of 256 x 256 with a reduction of 256 or more: rows, features and reduction that end inside a tile or a step"""
    from test_gpu_ffn import check_dense
    check_dense(rows, k, n, dtype, act)


@pytest.mark.parametrize('dtype', TYPES[1:], ids=IDS[1:])
@pytest.mark.parametrize('rows,k,hid,n,act', [(33000, 264, 520, 264, 'silu'), (32900, 256, 256, 72, 'gelu')])
def test_gated_256_wide(dtype, rows, k, hid, n, act):
    """the same of the gated block, whose backward has tiles of 128 features x 192 rows and a second reduction over n"""
    from test_gpu_ffn import check_gated
    check_gated(rows, k, hid, n, dtype, act)


def test_256_wide_strided_rows():
    """a pitch of whole 16-byte packs keeps the direct loads; one of single elements does not: the same results, bit for bit where the tiles agree, and
    what lies between the rows is not touched"""
    from arcnerf_amd.ops import functional as F
    rows, k, n = 66001, 264, 264
    x, w, dz = ints(1, rows, k, dtype=torch.bfloat16), ints(2, n, k, dtype=torch.bfloat16), ints(3, rows, n, dtype=torch.bfloat16)
    want = (exact(x, w.t()).bfloat16(), exact(dz, w).bfloat16(), exact(dz.t(), x).bfloat16())
    for pitch in (8, 3):
        wx, wz = (torch.full((rows, t.shape[1] + pitch), float('nan'), dtype=torch.bfloat16, device='cuda') for t in (x, dz))
        wx[:, :k], wz[:, :n] = x, dz
        got = (F.dense_fwd(wx[:, :k], w), F.dense_dx(wz[:, :n], w), F.dense_dw(wz[:, :n], wx[:, :k])[0])
        for name, a, b in zip(('y', 'dx', 'dw'), got, want):
            assert torch.equal(a, b), (pitch, name)
        assert torch.isnan(wx[:, k:]).all() and torch.isnan(wz[:, n:]).all()


# ---- relu at pre-activations that are never zero ------------------------------------------------------------------------------------------
@pytest.mark.parametrize('dtype', TYPES, ids=IDS)
@pytest.mark.parametrize('rows,k,hid,n', [(50, 24, 40, 24), (8301, 130, 260, 136)])
def test_relu_off_zero(dtype, rows, k, hid, n):
    """x in halves, weights in quarters: the products are eighths and a bias of 1/16 keeps every sum off zero, exactly in every type"""
    from arcnerf_amd.ops import autograd as A
    from test_gpu_ffn import close, dense_bounds, gated_bounds, gated_inputs
    p, dy = gated_inputs(rows, k, hid, n, dtype)
    p['x'], p['wg'] = (p['x'] * 2).round().clamp(-3, 3) / 2, (p['wg'] * 4 * k ** 0.5).round().clamp(-2, 2) / 4
    p['bg'] = torch.full_like(p['bg'], 0.0625)
    q = {name: t.double() for name, t in p.items()}
    assert (q['x'] @ q['wg'].t() + q['bg']).abs().min().item() >= 0.0625
    d = {name: t.cuda().requires_grad_(True) for name, t in p.items()}
    order = ('x', 'wg', 'wu', 'wd', 'bg', 'bu', 'bd', 'r')
    want = gated_bounds(*(q[name] for name in order), dy.double(), 'relu', 1.0, dtype)
    y = A.gated_ffn(*(d[name] for name in order), act='relu')
    close(y, *want['y'], 'y')
    for name, g in zip(order[:7], torch.autograd.grad(y, [d[name] for name in order[:7]], dy.cuda())):
        close(g, *want['d' + name], 'd' + name)
    r, dh = torch.zeros(rows, hid, dtype=torch.float64), (dy[:, :1] + torch.zeros(rows, hid, dtype=dtype))
    want = dense_bounds(q['x'], q['wg'], q['bg'], r, dh.double(), 'relu', 1.0, dtype)
    y = A.linear_act_residual(d['x'], d['wg'], d['bg'], act='relu')
    close(y, *want['y'], 'dense y')
    for key, g in zip(('dx', 'dw', 'db'), torch.autograd.grad(y, [d['x'], d['wg'], d['bg']], dh.cuda())):
        close(g, *want[key], 'dense ' + key)


# ---- tensors whose numbers are not what memory holds ----------------------------------------------------------------------------------------
def negated(t):
    """-t as a view that is negated on reading, as the imaginary part of a conjugate is"""
    v = torch.complex(torch.zeros_like(t), t).conj().imag
    assert v.is_neg() and torch.equal(v, -t)
    return v


@pytest.mark.parametrize('name', ['layer_norm', 'linear_act_residual', 'linear_act_residual without act', 'gated_ffn'])
def test_negated_views(name):
    """any operand, and the gradient that comes in, as a view with its sign in the tensor and not in memory"""
    fn, t = small_calls()[name]
    dy = leaf(30, 40, 16).detach()
    for k in list(t) + ['dy']:
        results = []
        for sign in (lambda v: -v, negated):
            at = {j: (sign(v.detach()) if j == k else v.detach()).requires_grad_(True) for j, v in t.items()}
            y = fn(at)
            with torch.no_grad():
                assert torch.equal(fn(at), y)
            results.append((y.detach(),) + torch.autograd.grad(y, list(at.values()), sign(dy) if k == 'dy' else dy))
        same(*results)


def test_negated_views_in_the_calls_without_autograd():
    from arcnerf_amd.ops import functional as F
    x, dy, w, b = (leaf(k, *s).detach() for k, s in enumerate([(40, 16), (40, 24), (24, 16), (24,)]))
    nx, nw, nb, ndy = (negated(t) for t in (x, w, b, dy))
    same((F.dense_fwd(nx, nw, nb, ndy, 'silu'), F.layer_norm_fwd(nx), F.dense_dx(ndy, nw)) + F.dense_dw(ndy, nx, True),
         (F.dense_fwd(-x, -w, -b, -dy, 'silu'), F.layer_norm_fwd(-x), F.dense_dx(-dy, -w)) + F.dense_dw(-dy, -x, True))


@pytest.mark.parametrize('name', ['layer_norm', 'linear_act_residual', 'gated_ffn'])
def test_transforms_raise_or_are_right(name):
    """traces into a graph module are refused, and so are batched and functional derivatives (by torch); other modes see the calls that are made"""
    from torch.fx.experimental.proxy_tensor import make_fx
    from torch.utils.flop_counter import FlopCounterMode
    fn, t = small_calls()[name]
    d = {j: v.detach() for j, v in t.items()}
    call = lambda x: fn(dict(d, x=x))
    x = d['x']
    for refused in (lambda: make_fx(call)(x), lambda: make_fx(call, pre_dispatch=True)(x), lambda: make_fx(call, tracing_mode='fake')(x),
                    lambda: torch.func.vmap(call)(torch.stack([x, x])), lambda: torch.func.grad(lambda v: call(v).sum())(x), lambda: torch.func.functionalize(call)(x),
                    lambda: torch.autograd.grad(fn(t), t['x'], torch.ones(2, 40, 16, device='cuda'), is_grads_batched=True)):
        with pytest.raises(RuntimeError):
            refused()
    want = call(x)
    with FlopCounterMode(display=False):
        assert torch.equal(call(x), want)
    assert torch.equal(call(x), want)


# ---- infinities and NaN stay in their rows --------------------------------------------------------------------------------------------------
def rows_apart(fn, x, dy, bad_rows):
    """results of every row but the bad ones are, bit for bit, those without them"""
    out = []
    for values in ((), (float('nan'), float('inf'), -float('inf'))):
        t = x.clone()
        for k, v in enumerate(values):
            t[bad_rows[k], k % x.shape[1]] = v
        t.requires_grad_(True)
        y = fn(t)
        out.append((y.detach(), torch.autograd.grad(y, t, dy)[0]))
    keep = torch.ones(x.shape[0], dtype=torch.bool, device='cuda')
    keep[bad_rows] = False
    for name, a, b in zip(('y', 'dx'), *out):
        assert torch.isfinite(a).all() and torch.equal(a[keep], b[keep]), name
    return out[1]


@pytest.mark.parametrize('dtype', TYPES, ids=IDS)
@pytest.mark.parametrize('width', [3, 20, 64, 100, 256, 319, 512, 1000, 2048, 4096, 8192, 8200])
def test_layer_norm_keeps_rows_apart(dtype, width):
    from arcnerf_amd.ops import autograd as A
    rows = 70
    x, dy, w, b = (leaf(k, *s, dtype=dtype).detach() for k, s in enumerate([(rows, width), (rows, width), (width,), (width,)]))
    y, dx = rows_apart(lambda t: A.layer_norm(t, w, b), x, dy, [5, 17, 69])
    assert all(torch.isnan(t[r]).all() for t in (y, dx) for r in (5, 17, 69))


@pytest.mark.parametrize('dtype', TYPES, ids=IDS)
@pytest.mark.parametrize('rows,k,n', [(20, 24, 13), (300, 45, 21), (16400, 24, 13), (30001, 24, 13), (33001, 129, 130), (66000, 264, 264)])
def test_dense_and_gated_keep_rows_apart(dtype, rows, k, n):
    from arcnerf_amd.ops import autograd as A
    x, dy, r = (leaf(j, rows, s, dtype=dtype).detach() for j, s in enumerate((k, n, n)))
    w, b, wd = leaf(4, n, k, dtype=dtype, scale=k ** -0.5).detach(), leaf(5, n, dtype=dtype).detach(), leaf(6, n, n, dtype=dtype, scale=n ** -0.5).detach()
    bad = [5, 17, rows - 1]
    for act in ('silu', 'gelu', 'softplus', 'relu', 'sigmoid'):
        rows_apart(lambda t: A.linear_act_residual(t, w, b, r, act=act), x, dy, bad)
        rows_apart(lambda t: A.gated_ffn(t, w, w, wd, b, b, b, r, act=act), x, dy, bad)


# ---- more than 2^31 rows --------------------------------------------------------------------------------------------------------------------
def test_more_rows_than_a_launch_has_threads():
    """2^31 + 77 rows of one 16-bit number, more than 2^32 threads along a grid's first dimension where 64 rows have a workgroup of 256: every row
    of the results is there, and a sum over the rows holds the last ones (x is zero but for 9 rows)"""
    from arcnerf_amd.ops import functional as F
    rows = (1 << 31) + 77
    x = torch.empty(rows, 1, dtype=torch.bfloat16, device='cuda')
    for a in range(0, rows, 1 << 28):
        x[a:a + (1 << 28)].random_(1, 100)
    one = torch.ones(1, 1, dtype=torch.bfloat16, device='cuda')
    assert torch.equal(F.dense_fwd(x, one, act='relu'), x)
    assert torch.equal(F.dense_dz(x, one, None, x, 'relu'), x)
    assert torch.equal(F.dense_dx(x, one), x)
    assert torch.equal(F.gated_fwd(x, torch.zeros_like(one), one, b_gate=one[0], act=None), x)
    assert torch.equal(F.gated_bwd(x, torch.zeros_like(one), one, one[0], None, x, one, act=None)[:, 1:], x)      # du = dy
    y = F.layer_norm_fwd(x, None, one[0])
    assert y.min().item() == 1 and y.max().item() == 1
    del y
    at = torch.tensor([0, 1, 77777, 1 << 30, (1 << 31) - 1, 1 << 31, rows - 40, rows - 2, rows - 1], device='cuda')
    few = torch.zeros_like(x)
    few[at] = torch.tensor([1, 2, 4, 8, 16, 32, 64, 128, 256], device='cuda').bfloat16()[:, None]
    ones = torch.ones_like(x)
    dw, db = F.dense_dw(few, ones, want_db=True)
    assert dw.item() == 512 and db.item() == 512       # 511, rounded to 8 bits
    assert F.dense_dw(ones, few)[0].item() == 512


def test_weight_gradient_of_more_elements_than_a_launch_has_threads():
    """65544 x 65536 weights, more than 2^32: the outer product of one row, exact"""
    from arcnerf_amd.ops import functional as F
    n, k = 65544, 65536
    dz, x = ints(1, 1, n, dtype=torch.bfloat16), ints(2, 1, k, dtype=torch.bfloat16)
    dw, db = F.dense_dw(dz, x, want_db=True)
    assert torch.equal(db, dz[0])
    for a in range(0, n, 8192):
        assert torch.equal(dw[a:a + 8192], dz[0, a:a + 8192, None] * x)


# ---- captured passes ------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize('dtype', TYPES, ids=IDS)
def test_training_passes_with_biases_replay(dtype):
    """a gated block and a dense layer with all their biases, whose column sums are a buffer of the pass: replays with other inputs, eager passes of
    the same shapes in between, are the eager results"""
    from arcnerf_amd.ops import autograd as A
    rows, k, hid = 30000, 40, 72
    p = [leaf(j, *s, dtype=dtype, scale=0.2) for j, s in enumerate([(hid, k), (hid, k), (k, hid), (hid,), (hid,), (k,), (k, k), (k,)])]
    xs, dy = [leaf(20 + j, rows, k, dtype=dtype).detach() for j in range(3)], leaf(30, rows, k, dtype=dtype).detach()

    def run(x):
        x = x.detach().requires_grad_(True)
        y = A.linear_act_residual(A.gated_ffn(x, *p[:6], residual=x), p[6], p[7], act='gelu')
        return (y.detach(),) + torch.autograd.grad(y, [x] + p, dy)

    want = [run(x) for x in xs]
    held = xs[0].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(held)
    for trip in range(4):
        held.copy_(xs[trip % 3])
        graph.replay()
        eager = run(xs[(trip + 1) % 3])
        torch.cuda.synchronize()
        same(out, want[trip % 3])
        same(eager, want[(trip + 1) % 3])


@pytest.mark.parametrize('dtype', TYPES[1:], ids=IDS[1:])
@pytest.mark.parametrize('rows,k,n,act,pitch', [(24576, 8, 8, 'silu', 0), (24593, 128, 128, 'gelu', 0), (26000, 100, 60, 'softplus', 3), (24600, 128, 512, 'silu', 0), (27001, 125, 13, 'sigmoid', 1)])
def test_dense_weight_on_chip(dtype, rows, k, n, act, pitch):
    """dz and dx of one kernel: the fewest rows that take it, partial groups of rows, widths and features that end inside a pack"""
    from test_gpu_ffn import check_dense
    check_dense(rows, k, n, dtype, act, pitch=pitch, bias=act != 'silu', residual=act != 'sigmoid')
