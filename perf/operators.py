"""The residual feed-forward layers of wide coordinate nets, as they are measured: layer norm, a dense layer with bias, activation and
residual, and the gated feed-forward block, each forward alone (a served point or a rendered view) and forward + backward (training).

`own` False: the operators in elementary float32 torch operations, rounded once at the end, whatever the inputs' type.  `own` True:
the framework's operators (arcnerf_amd.ops.autograd), called as a model calls them.

The widths are the repository's (256-wide nets with 63 / 283 / 319-wide inputs, chunks of 131072 points, views of 2^20 points) or generic.
"""
import math

import torch

own = False

_TYPES = {'f32': torch.float32, 'bf16': torch.bfloat16, 'f16': torch.float16}
_EPS = 1e-5


def listed():
    return [
        # one point of a served model: the whole call is launches and latency
        dict(name='norm one row bf16', op='norm', dtype='bf16', train=False, rows=1, width=256, pitch=0),
        # a training chunk of the 256-wide nets in the framework's own precision
        dict(name='norm train f32', op='norm', dtype='f32', train=True, rows=131072, width=256, pitch=0),
        # a whole view's points in 16 bits: pure streaming
        dict(name='norm train bf16 large', op='norm', dtype='bf16', train=True, rows=1 << 20, width=256, pitch=0),
        # the skip concatenation's width (63 + 256), rows that start at any 2-byte boundary of a wider buffer
        dict(name='norm train f16 odd', op='norm', dtype='f16', train=True, rows=20011, width=319, pitch=2),
        # one point through one wide layer: the weight is read once, nothing else matters
        dict(name='dense one row bf16', op='dense', dtype='bf16', train=False, rows=1, width=1024, out=1024, act='silu', bias=True,
             residual=True, pitch=0),
        # a hidden layer of the 8 x 256 nets over a training chunk, in f32
        dict(name='dense train f32', op='dense', dtype='f32', train=True, rows=131072, width=256, out=256, act='softplus', bias=True,
             residual=True, pitch=0),
        # the same layer in 16 bits over two chunks
        dict(name='dense train bf16', op='dense', dtype='bf16', train=True, rows=262144, width=256, out=256, act='silu', bias=True,
             residual=True, pitch=0),
        # the radiance net's odd input width, an odd output, odd row count, a column slice of a wider buffer as the input
        dict(name='dense train f16 odd', op='dense', dtype='f16', train=True, rows=10007, width=283, out=131, act='gelu', bias=True,
             residual=True, pitch=5),
        # a handful of points through a served block
        dict(name='ffn eight rows bf16', op='ffn', dtype='bf16', train=False, rows=8, width=256, hidden=1024, act='silu', bias=False,
             residual=True, pitch=0),
        # a training step of one block in f32
        dict(name='ffn train f32', op='ffn', dtype='f32', train=True, rows=32768, width=256, hidden=512, act='silu', bias=True,
             residual=True, pitch=0),
        # the largest: a wide block in 16 bits, bound by the matrix cores
        dict(name='ffn train bf16 large', op='ffn', dtype='bf16', train=True, rows=65536, width=512, hidden=2048, act='silu', bias=False,
             residual=True, pitch=0),
        # nothing divides anything
        dict(name='ffn train f16 odd', op='ffn', dtype='f16', train=True, rows=5003, width=131, hidden=347, act='gelu', bias=True,
             residual=False, pitch=0),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """rows from one to 2^20, widths from 8 to 1024 (norm: to 4096), hidden to 2048, half of the sizes as they fall (odd ones among them) and half
    rounded to 8; scaled down in rows where the case would cost more than the largest listed ones"""
    op = rng.choice(['norm', 'dense', 'ffn'])
    case = dict(op=op, dtype=rng.choice(['f32', 'bf16', 'f16']), train=rng.random() < 0.7)
    even = rng.random() < 0.5

    def size(lo, hi):
        n = _log(rng, lo, hi)
        return max(lo, n // 8 * 8) if even else n
    rows = _log(rng, 1, 1 << 20)
    case['width'] = size(8, 4096 if op == 'norm' else 1024)
    case['pitch'] = 0 if even or rng.random() < 0.5 else rng.randrange(1, 9)
    if op == 'norm':
        case['rows'] = max(1, min(rows, (1 << 28) // case['width']))
        return case
    # the derivative of relu jumps at zero, where the last bit of a sum decides: it is drawn for forward passes only
    acts = ['silu', 'gelu', 'softplus'] if case['train'] else ['silu', 'gelu', 'relu', 'sigmoid']
    case['act'] = rng.choice(acts if op == 'ffn' else acts + ['none'])
    if op == 'dense':
        case['out'] = size(8, 1024)
        per_row = 6 * case['width'] * case['out'] + 400 * (case['width'] + case['out'])
    else:
        case['hidden'] = size(8, 2048)
        per_row = 18 * case['width'] * case['hidden'] + 400 * (case['width'] + case['hidden'])
    most = 1.2e12 if case['dtype'] != 'f32' else 1.2e11
    case['rows'] = max(1, min(rows, int(most / per_row), 1 << 19))
    case['bias'] = rng.random() < 0.5
    case['residual'] = rng.random() < 0.5
    return case


def prepare(case, seed):
    """activations of unit size with an offset per row, weights at the scale of their initialisation, gradients of unit size (a scaled loss):
    all made from the seed on the GPU"""
    dtype, rows, width = _TYPES[case['dtype']], case['rows'], case['width']
    gen = torch.Generator(device='cuda')
    gen.manual_seed(int(seed))

    def normal(*shape, scale=1.0, offset=0.0):
        t = torch.randn(*shape, generator=gen, device='cuda', dtype=torch.float32)
        return t.mul_(scale).add_(offset).to(dtype)

    train = bool(case['train'])
    s = {'case': case}
    wide = normal(rows, width + case['pitch'])
    if case['op'] == 'norm':
        wide += normal(rows, 1)
    s['x'] = wide[:, :width]
    leaves = ['x']
    if case['op'] == 'norm':
        s['weight'], s['bias'] = normal(width, scale=0.1, offset=1.0), normal(width, scale=0.1)
        leaves += ['weight', 'bias']
        out = width
    elif case['op'] == 'dense':
        out = case['out']
        s['weight'] = normal(out, width, scale=width ** -0.5)
        s['bias'] = normal(out, scale=0.1) if case['bias'] else None
        leaves += ['weight', 'bias']
    else:
        hid, out = case['hidden'], width
        s['w_gate'], s['w_up'] = normal(hid, width, scale=width ** -0.5), normal(hid, width, scale=width ** -0.5)
        s['w_down'] = normal(width, hid, scale=hid ** -0.5)
        s['b_gate'] = normal(hid, scale=0.1) if case['bias'] else None
        s['b_up'] = normal(hid, scale=0.1) if case['bias'] else None
        s['b_down'] = normal(width, scale=0.1) if case['bias'] else None
        leaves += ['w_gate', 'w_up', 'w_down', 'b_gate', 'b_up', 'b_down']
    if case['op'] != 'norm':
        s['residual'] = normal(rows, out) if case['residual'] else None
    s['leaves'] = [k for k in leaves if s[k] is not None]
    if train:
        s['dy'] = normal(rows, out)
        for k in s['leaves']:
            s[k] = s[k].detach().requires_grad_(True)
    return s


def run(s):
    case = s['case']
    if own:
        return _run_own(s)
    with torch.no_grad():
        f = {k: v.float() if torch.is_tensor(v) else v for k, v in s.items()}
        out = {'norm': _plain_norm, 'dense': _plain_dense, 'ffn': _plain_ffn}[case['op']](case, f)
        return {k: v.to(_TYPES[case['dtype']]) for k, v in out.items() if v is not None}


def _run_own(s):
    from arcnerf_amd.ops import autograd as A
    case = s['case']
    if not case['train']:
        with torch.no_grad():
            return {'y': _call(A, case, s)}
    y = _call(A, case, s)
    grads = torch.autograd.grad(y, [s[k] for k in s['leaves']], s['dy'])
    return dict(zip(['d_' + k for k in s['leaves']], grads), y=y.detach())


def _call(A, case, s):
    if case['op'] == 'norm':
        return A.layer_norm(s['x'], s['weight'], s['bias'], eps=_EPS)
    if case['op'] == 'dense':
        return A.linear_act_residual(s['x'], s['weight'], s['bias'], s['residual'], act=case['act'])
    return A.gated_ffn(s['x'], s['w_gate'], s['w_up'], s['w_down'], s['b_gate'], s['b_up'], s['b_down'], residual=s['residual'],
                       act=case['act'])


def work(case):
    """each input read once, each output written once; the products a pass cannot do without (two per gradient of a product)"""
    size = 4 if case['dtype'] == 'f32' else 2
    r, w, train = case['rows'], case['width'], case['train']
    if case['op'] == 'norm':
        return {'bytes': size * (r * w * (4 if train else 2) + w * (4 if train else 2)), 'flops': r * w * (20 if train else 8)}
    if case['op'] == 'dense':
        n = case['out']
        rows_io = r * (w + n * (2 if case['residual'] else 1)) + (r * (n + w) if train else 0)
        weights = (w * n + (n if case['bias'] else 0)) * (2 if train else 1)
        return {'bytes': size * (rows_io + weights), 'flops': 2.0 * r * w * n * (3 if train else 1)}
    h = case['hidden']
    rows_io = r * w * (3 if case['residual'] else 2) + (2 * r * w if train else 0)
    weights = (3 * w * h + (2 * h + w if case['bias'] else 0)) * (2 if train else 1)
    return {'bytes': size * (rows_io + weights), 'flops': 6.0 * r * w * h * (3 if train else 1)}


# ---- the plain forms: float32 -------------------------------------------------------------------------------------------------------
def _act(z, name):
    """act(z), act'(z)"""
    if name == 'none':
        return z, torch.ones_like(z)
    if name == 'relu':
        on = (z > 0).float()
        return z * on, on
    if name == 'softplus':
        e = torch.exp(-z.abs())
        return torch.clamp(z, min=0) + torch.log1p(e), torch.where(z >= 0, 1 / (1 + e), e / (1 + e))
    e = torch.exp(-z.abs())
    sig = torch.where(z >= 0, 1 / (1 + e), e / (1 + e))
    if name == 'sigmoid':
        return sig, sig * (1 - sig)
    if name == 'silu':
        return z * sig, sig * (1 + z * (1 - sig))
    if name == 'gelu':
        cdf = 0.5 * torch.erfc(z * -math.sqrt(0.5))
        return z * cdf, cdf + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi))
    raise ValueError(name)


def _plain_norm(case, f):
    x = f['x']
    d = x - x.mean(1, keepdim=True)
    rstd = 1 / torch.sqrt((d * d).mean(1, keepdim=True) + _EPS)
    n = d * rstd
    y = n * f['weight'] + f['bias']
    if not case['train']:
        return {'y': y}
    g = f['dy'] * f['weight']
    dx = rstd * (g - g.mean(1, keepdim=True) - n * (g * n).mean(1, keepdim=True))
    return {'y': y, 'd_x': dx, 'd_weight': (f['dy'] * n).sum(0), 'd_bias': f['dy'].sum(0)}


def _plain_dense(case, f):
    z = f['x'] @ f['weight'].t()
    if f['bias'] is not None:
        z = z + f['bias']
    a, slope = _act(z, case['act'])
    y = a if f['residual'] is None else a + f['residual']
    if not case['train']:
        return {'y': y}
    dz = f['dy'] * slope
    return {'y': y, 'd_x': dz @ f['weight'], 'd_weight': dz.t() @ f['x'], 'd_bias': None if f['bias'] is None else dz.sum(0)}


def _plain_ffn(case, f):
    g, u = f['x'] @ f['w_gate'].t(), f['x'] @ f['w_up'].t()
    if case['bias']:
        g, u = g + f['b_gate'], u + f['b_up']
    a, slope = _act(g, case['act'])
    h = a * u
    y = h @ f['w_down'].t()
    if case['bias']:
        y = y + f['b_down']
    if f['residual'] is not None:
        y = y + f['residual']
    if not case['train']:
        return {'y': y}
    dy = f['dy']
    dh = dy @ f['w_down']
    dg, du = dh * u * slope, dh * a
    out = {'y': y, 'd_x': dg @ f['w_gate'] + du @ f['w_up'], 'd_w_gate': dg.t() @ f['x'], 'd_w_up': du.t() @ f['x'], 'd_w_down': dy.t() @ h}
    if case['bias']:
        out.update(d_b_gate=dg.sum(0), d_b_up=du.sum(0), d_b_down=dy.sum(0))
    return out


# ---- 64 bits, from the definitions: torch's own differentiation of the formulas in double ------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    v = {k: t.detach().double().requires_grad_(bool(case['train']) and k in s['leaves']) for k, t in s.items() if torch.is_tensor(t)}
    F = torch.nn.functional
    act = {'none': lambda z: z, 'relu': F.relu, 'softplus': lambda z: torch.logaddexp(z, torch.zeros_like(z)), 'sigmoid': torch.sigmoid,
           'silu': lambda z: z * torch.sigmoid(z), 'gelu': lambda z: z * (1 + torch.special.erf(z / math.sqrt(2))) / 2}.get(case.get('act'))
    with torch.set_grad_enabled(bool(case['train'])):
        if case['op'] == 'norm':
            var, mean = torch.var_mean(v['x'], dim=1, unbiased=False, keepdim=True)
            y = (v['x'] - mean) / (var + _EPS).sqrt() * v['weight'] + v['bias']
        elif case['op'] == 'dense':
            y = act(F.linear(v['x'], v['weight'], v.get('bias')))
        else:
            h = act(F.linear(v['x'], v['w_gate'], v.get('b_gate'))) * F.linear(v['x'], v['w_up'], v.get('b_up'))
            y = F.linear(h, v['w_down'], v.get('b_down'))
        if v.get('residual') is not None:
            y = y + v['residual']
        if not case['train']:
            return {'y': y}
        grads = torch.autograd.grad(y, [v[k] for k in s['leaves']], v['dy'])
        return dict(zip(['d_' + k for k in s['leaves']], grads), y=y.detach())
