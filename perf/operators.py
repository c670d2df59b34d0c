"""Workloads of the dense-network operators: the linear layer with its epilogue, layer norm, and activations kept in 8 bits.

    linear      y = act(x W' + b) + r, forward alone or with the gradients of x, W, b and r; `save8` keeps the x that the
                weight gradient needs as 8-bit integers with one power of two for every 32 features of a row
    norm        y = (z - mean) / sqrt(var + eps) * g + b with z = x or z = x + r (z is an output then), forward alone or with
                the gradients of x, r, g and b; `save8` as above for the z that the backward pass needs
    pack        an activation into the 8-bit form and back

`own` False: plain torch operations in fp32, each output rounded once. `own` True: `ursabench_amd.fused_linear`,
`ursabench_amd.fused_norm`, `ursabench_amd.act8`. `exact`: the definitions in fp64.
"""
import math

import torch
import torch.nn as nn

own = False

_DTYPES = {'float32': torch.float32, 'bfloat16': torch.bfloat16, 'float16': torch.float16}
_BLOCK = 32                                  # features that share one power of two in the 8-bit form
_MOST_FLOPS = 6 * 8192 * 2048 * 8192         # of the largest listed linear case
_MOST_NUMBERS = 16384 * 4096                 # of the largest listed norm case


def _linear(rows, fin, fout, dtype, act='none', residual=False, train=True, save8=False):
    return dict(kind='linear', rows=rows, fin=fin, fout=fout, dtype=dtype, act=act, residual=residual, train=train, save8=save8)


def _norm(rows, features, dtype, add=False, train=True, save8=False):
    return dict(kind='norm', rows=rows, features=features, dtype=dtype, add=add, train=train, save8=save8)


def _pack(rows, features, dtype):
    return dict(kind='pack', rows=rows, features=features, dtype=dtype)


def listed():
    return [
        # one token through the widening layer of a feed-forward block: the weights are read once, latency counts
        dict(_linear(1, 4096, 4096, 'bfloat16', act='gelu', train=False), name='linear_one_token'),
        # the predictive of one ensemble member over a test batch: no gradients, relu, fp32 like every sampler here
        dict(_linear(2048, 1024, 1024, 'float32', act='relu', train=False), name='linear_member_predictive'),
        # the first layer of models.MLP200MNIST at the samplers' batch of 128, as the samplers train it
        dict(_linear(128, 784, 200, 'float32', act='relu'), name='linear_mnist_step'),
        # a feed-forward block's widening layer in the samplers' own type
        dict(_linear(4096, 1024, 4096, 'float32', act='gelu'), name='linear_train_fp32'),
        # the same layer at the size of a large step in bf16
        dict(_linear(8192, 2048, 8192, 'bfloat16', act='gelu'), name='linear_train_bf16'),
        # odd sizes everywhere, a shortcut added in the epilogue
        dict(_linear(1000, 1111, 777, 'float16', act='silu', residual=True), name='linear_odd_fp16'),
        # the narrowing layer with its shortcut; the wide input is what fills the memory, so it is kept in 8 bits
        dict(_linear(8192, 4096, 1024, 'bfloat16', residual=True, save8=True), name='linear_save8_bf16'),
        # the shortcut's sum and the norm behind it for one token
        dict(_norm(1, 4096, 'bfloat16', add=True, train=False), name='norm_one_token'),
        # an odd width, rows that are not a multiple of anything
        dict(_norm(777, 1111, 'float16'), name='norm_odd_fp16'),
        # sum and norm of a large step, with the weight's gradient over 16,384 rows
        dict(_norm(16384, 4096, 'bfloat16', add=True), name='norm_train_bf16'),
        # the norm of an fp32 step with its input kept in 8 bits
        dict(_norm(8192, 2048, 'float32', save8=True), name='norm_save8_fp32'),
        # a wide activation into its 8-bit form and back
        dict(_pack(8192, 4096, 'bfloat16'), name='pack_bf16'),
    ]


def _spread(rng, low, high):
    """A whole number between low and high, even over its logarithm; one in two a multiple of 64 where that fits."""
    n = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    if rng.random() < 0.5 and n >= 64:
        n -= n % 64
    return max(low, min(high, n))


def draw(rng):
    dtype = rng.choice(['float32', 'bfloat16', 'float16'])
    kind = rng.choice(['linear', 'linear', 'norm', 'norm', 'pack'])
    if kind == 'linear':
        train = rng.random() < 0.6
        save8 = train and rng.random() < 0.4
        # relu among the forward cases only: at large sizes some sums land within a rounding of its gate, which is no
        # difference in y but one of the whole term in a gradient
        act = rng.choice(['none', 'gelu', 'silu'] if train else ['none', 'relu', 'gelu', 'silu'])
        while True:
            rows, fin, fout = _spread(rng, 16 if train else 1, 8192), _spread(rng, 48, 8192), _spread(rng, 10, 8192)
            # fp32 products cost the plain form and its fp64 check the most
            if 2 * rows * fin * fout * (3 if train else 1) <= _MOST_FLOPS // (4 if dtype == 'float32' else 1):
                break
        return _linear(rows, fin, fout, dtype, act=act, residual=rng.random() < 0.5, train=train, save8=save8)
    if kind == 'norm':
        train = rng.random() < 0.7
        while True:
            rows, features = _spread(rng, 1, 16384), _spread(rng, 24, 16384)
            if rows * features <= _MOST_NUMBERS // (2 if dtype == 'float32' else 1):
                break
        return _norm(rows, features, dtype, add=rng.random() < 0.5, train=train, save8=train and rng.random() < 0.4)
    while True:
        rows, features = _spread(rng, 1, 8192), _spread(rng, 24, 8192)
        if rows * features <= _MOST_NUMBERS // 2:
            return _pack(rows, features, dtype)


# ---- inputs ---------------------------------------------------------------------------------
def _stream(g, rows, features, dtype):
    """Values of a residual stream: some features sit off zero, a few are an order of magnitude larger than the rest."""
    x = torch.randn(rows, features, generator=g, device='cuda')
    scale = torch.exp(0.4 * torch.randn(features, generator=g, device='cuda'))
    scale = torch.where(torch.rand(features, generator=g, device='cuda') < 0.01, scale * 10, scale)
    return (x * scale + 0.3 * torch.randn(features, generator=g, device='cuda')).to(dtype)


def prepare(case, seed):
    g = torch.Generator(device='cuda').manual_seed(seed)
    dtype, rows = _DTYPES[case['dtype']], case['rows']
    s = dict(case=case)
    if case['kind'] == 'pack':
        s['x'] = _stream(g, rows, case['features'], dtype)
        return s
    train = case['train']
    if case['kind'] == 'linear':
        fin, fout = case['fin'], case['fout']
        fc = nn.Linear(fin, fout, device='cuda')
        bound = 1 / math.sqrt(fin)
        with torch.no_grad():
            fc.weight.copy_((2 * torch.rand(fout, fin, generator=g, device='cuda') - 1) * bound)
            fc.bias.copy_((2 * torch.rand(fout, generator=g, device='cuda') - 1) * bound)
        s['fc'] = fc.to(dtype).requires_grad_(train)
        s['x'] = torch.randn(rows, fin, generator=g, device='cuda').to(dtype).requires_grad_(train)
        s['r'] = _stream(g, rows, fout, dtype).requires_grad_(train) if case['residual'] else None
        width = fout
    else:
        width = case['features']
        ln = nn.LayerNorm(width, device='cuda')
        with torch.no_grad():
            ln.weight.copy_(1 + 0.2 * torch.randn(width, generator=g, device='cuda'))
            ln.bias.copy_(0.2 * torch.randn(width, generator=g, device='cuda'))
        s['ln'] = ln.to(dtype).requires_grad_(train)
        s['x'] = _stream(g, rows, width, dtype).requires_grad_(train)
        s['r'] = torch.randn(rows, width, generator=g, device='cuda').to(dtype).requires_grad_(train) if case['add'] else None
    if train:
        s['dy'] = (torch.randn(rows, width, generator=g, device='cuda') / math.sqrt(rows)).to(dtype)
        if case['kind'] == 'norm' and case['add']:
            s['dz'] = (torch.randn(rows, width, generator=g, device='cuda') / math.sqrt(rows)).to(dtype)
    return s


# ---- the plain forms ------------------------------------------------------------------------
def _power_of_two(e):
    """2^e in fp32 from its bits (torch.ldexp multiplies by a pow() that is a rounding off: half-way values would move)."""
    return ((e.int() + 127) << 23).view(torch.float32)


def _plain_unpacked(x):
    """The values that the 8-bit form of x stands for, in fp32: blocks of 32 features share the power of two s = 2^(k - 7),
    k the exponent of the block's largest magnitude m 2^k (1/2 <= m < 1); x / s rounded to the nearest whole number (ties to
    the even one), at most 127 in magnitude."""
    rows, n = x.shape
    pad = -n % _BLOCK
    v = torch.nn.functional.pad(x.float(), (0, pad)).view(rows, -1, _BLOCK)
    k = torch.frexp(v.abs().amax(-1, keepdim=True))[1]
    e = (k - 7).clamp(min=-24 if x.dtype == torch.float16 else -126)
    q = torch.round(v * _power_of_two(-e)).clamp(-127, 127)
    return (q * _power_of_two(e)).view(rows, -1)[:, :n]


def _plain_act(z, act):
    """(act(z), act'(z)) in fp32."""
    if act == 'relu':
        return z.clamp(min=0), (z > 0).float()
    if act == 'gelu':
        phi = 0.5 * (1 + torch.erf(z * math.sqrt(0.5)))
        return z * phi, phi + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi))
    if act == 'silu':
        s = 1 / (1 + torch.exp(-z))
        return z * s, s * (1 + z * (1 - s))
    return z, None


def _plain_linear(s):
    case, dtype = s['case'], s['x'].dtype
    x, w, b = s['x'].detach().float(), s['fc'].weight.detach().float(), s['fc'].bias.detach().float()
    a, da = _plain_act(x @ w.t() + b, case['act'])
    y = (a if s['r'] is None else a + s['r'].detach().float()).to(dtype)
    if not case['train']:
        return dict(y=y)
    dz = s['dy'].float() if da is None else s['dy'].float() * da
    kept = _plain_unpacked(s['x'].detach()) if case['save8'] else x
    out = dict(y=y, dx=(dz @ w).to(dtype), dw=(dz.t() @ kept).to(dtype), db=dz.sum(0).to(dtype))
    if s['r'] is not None:
        out['dr'] = s['dy']
    return out


def _plain_norm(s):
    case, dtype, eps = s['case'], s['x'].dtype, s['ln'].eps
    g, b = s['ln'].weight.detach().float(), s['ln'].bias.detach().float()
    z = s['x'].detach()
    out = {}
    if s['r'] is not None:
        z = out['z'] = (z.float() + s['r'].detach().float()).to(dtype)      # the norm sees the sum as it is stored
    v = z.float()
    mean = v.mean(1, keepdim=True)
    rstd = 1 / torch.sqrt(((v - mean) ** 2).mean(1, keepdim=True) + eps)
    out['y'] = ((v - mean) * rstd * g + b).to(dtype)
    if not case['train']:
        return out
    xhat = ((_plain_unpacked(z) if case['save8'] else v) - mean) * rstd
    dy = s['dy'].float()
    t = dy * g
    dx = rstd * (t - t.mean(1, keepdim=True) - xhat * (t * xhat).mean(1, keepdim=True))
    if s['r'] is not None:
        dx = dx + s['dz'].float()
    out.update(dx=dx.to(dtype), dg=(dy * xhat).sum(0).to(dtype), db=dy.sum(0).to(dtype))
    if s['r'] is not None:
        out['dr'] = out['dx']
    return out


# ---- the framework's operators --------------------------------------------------------------
def _own_linear(s):
    from ursabench_amd.fused_linear import linear_act
    case, fc = s['case'], s['fc']
    act = None if case['act'] == 'none' else case['act']
    if not case['train']:
        return dict(y=linear_act(fc, s['x'], act, s['r']))
    y = linear_act(fc, s['x'], act, s['r'], save8=case['save8'])
    leaves = [s['x'], fc.weight, fc.bias] + ([] if s['r'] is None else [s['r']])
    return dict(zip(('y', 'dx', 'dw', 'db', 'dr'), (y.detach(),) + torch.autograd.grad(y, leaves, s['dy'])))


def _own_norm(s):
    from ursabench_amd.fused_norm import add_layer_norm, layer_norm
    case, ln = s['case'], s['ln']
    if s['r'] is None:
        y = layer_norm(ln, s['x'], save8=case['save8'])
        if not case['train']:
            return dict(y=y)
        dx, dg, db = torch.autograd.grad(y, (s['x'], ln.weight, ln.bias), s['dy'])
        return dict(y=y.detach(), dx=dx, dg=dg, db=db)
    z, y = add_layer_norm(ln, (s['x'], s['r']), save8=case['save8'])
    if not case['train']:
        return dict(z=z, y=y)
    dx, dg, db, dr = torch.autograd.grad((z, y), (s['x'], ln.weight, ln.bias, s['r']), (s['dz'], s['dy']))
    return dict(z=z.detach(), y=y.detach(), dx=dx, dg=dg, db=db, dr=dr)


def run(state):
    kind = state['case']['kind']
    if own:
        if kind == 'pack':
            from ursabench_amd import act8
            return act8.unpack(act8.pack(state['x']))
        return _own_linear(state) if kind == 'linear' else _own_norm(state)
    if kind == 'pack':
        return _plain_unpacked(state['x']).to(state['x'].dtype)
    return _plain_linear(state) if kind == 'linear' else _plain_norm(state)


def work(case):
    size = torch.finfo(_DTYPES[case['dtype']]).bits // 8
    rows = case['rows']
    if case['kind'] == 'pack':
        n = rows * case['features']
        kept = n + rows * -(-case['features'] // _BLOCK)
        return dict(bytes=2 * n * size + 2 * kept, flops=4 * n)                       # x in, the kept form out and in, x out
    if case['kind'] == 'linear':
        fin, fout = case['fin'], case['fout']
        xs, ws, ys = rows * fin, fin * fout + fout, rows * fout
        numbers = xs + ws + ys * (2 if case['residual'] else 1)
        flops = 2 * rows * fin * fout
        if case['train']:                                                             # dy in; dx, dW, db out
            numbers += ys + xs + ws
            flops *= 3
        return dict(bytes=numbers * size, flops=flops)
    n, add = rows * case['features'], case['add']
    numbers = n * (4 if add else 2) + 2 * case['features']                            # x (, r) in, y (, z) out
    if case['train']:
        numbers += n * (3 if add else 2) + 2 * case['features']                       # dy (, dz) in, dx out
    return dict(bytes=numbers * size, flops=n * (8 if not case['train'] else 20))


# ---- the definitions in fp64 ----------------------------------------------------------------
def _exact_unpacked(x):
    """As the 8-bit form is defined, from the exponent field of the block's largest magnitude as an fp64 number."""
    rows, n = x.shape
    blocks = -(-n // _BLOCK)
    v = torch.zeros(rows, blocks * _BLOCK, dtype=torch.float64, device=x.device)
    v[:, :n] = x.double()
    v = v.reshape(rows * blocks, _BLOCK)
    top = v.abs().max(dim=1).values
    field = (top.view(torch.int64) >> 52) & 0x7ff                       # top = 1.f * 2^(field - 1023)
    power = torch.where(field == 0, torch.full_like(field, -126), field - 1023 - 6)
    power = torch.maximum(power, torch.full_like(power, -24 if x.dtype == torch.float16 else -126))
    step = ((power + 1023) << 52).view(torch.float64)[:, None]            # 2^power, exactly
    whole = torch.round(v / step)
    whole = torch.minimum(torch.maximum(whole, torch.full_like(whole, -127)), torch.full_like(whole, 127))
    return (whole * step).reshape(rows, blocks * _BLOCK)[:, :n]


def exact(case, seed):
    s = prepare(case, seed)
    x = s['x'].detach()
    if case['kind'] == 'pack':
        return _exact_unpacked(x)
    if case['kind'] == 'linear':
        w, b = s['fc'].weight.detach().double(), s['fc'].bias.detach().double()
        z = torch.addmm(b, x.double(), w.t())
        act = case['act']
        if act == 'gelu':
            a = 0.5 * z * torch.erfc(-z / math.sqrt(2))
            slope = 0.5 * torch.erfc(-z / math.sqrt(2)) + z * torch.exp(-z.square() / 2) / math.sqrt(2 * math.pi)
        elif act == 'silu':
            a, slope = z * torch.sigmoid(z), torch.sigmoid(z) + z * torch.sigmoid(z) * torch.sigmoid(-z)
        elif act == 'relu':
            a, slope = torch.where(z > 0, z, torch.zeros_like(z)), (z > 0).double()
        else:
            a, slope = z, torch.ones_like(z)
        out = dict(y=a if s['r'] is None else a + s['r'].detach().double())
        if case['train']:
            dz = s['dy'].double() * slope
            out['dx'] = torch.mm(dz, w)
            out['dw'] = torch.mm(dz.t(), _exact_unpacked(x) if case['save8'] else x.double())
            out['db'] = dz.sum(dim=0)
            if s['r'] is not None:
                out['dr'] = s['dy'].double()
        return out
    g, b, n = s['ln'].weight.detach().double(), s['ln'].bias.detach().double(), case['features']
    out = {}
    if s['r'] is not None:
        x = (x.double() + s['r'].detach().double()).to(x.dtype)
        out['z'] = x.double()
    v = x.double()
    centred = v - v.sum(1, keepdim=True) / n
    rstd = (centred.square().sum(1, keepdim=True) / n + s['ln'].eps).rsqrt()
    out['y'] = centred * rstd * g + b
    if case['train']:
        dy = s['dy'].double()
        xhat = (centred if not case['save8'] else centred + (_exact_unpacked(x) - v)) * rstd
        inner = dy * g
        dx = rstd * (inner - inner.sum(1, keepdim=True) / n - xhat * ((inner * xhat).sum(1, keepdim=True) / n))
        out['dx'] = dx if s['r'] is None else dx + s['dz'].double()
        out['dg'] = (dy * xhat).sum(dim=0)
        out['db'] = dy.sum(dim=0)
        if s['r'] is not None:
            out['dr'] = out['dx']
    return out
