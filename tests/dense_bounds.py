"""fp64 definitions of K15 - K17 and, beside each, how far a right launch may be from it - derived from its roundings, element by
element. u = eps / 2 of the element type is one rounding to it, f = 2^-24 one fp32 rounding."""
import math

import torch

F = 2.0 ** -24
TYPES = {'float32': torch.float32, 'bfloat16': torch.bfloat16, 'float16': torch.float16}


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def last_rounding(value, dtype):
    """One rounding of `value` to dtype: half a step, or half the smallest subnormal number."""
    return half_step(dtype) * value.abs() + torch.finfo(dtype).smallest_normal * half_step(dtype)


def act(z, name):
    """(act, act', bound on |act'|, bound on |act''|): gelu' <= 1.13, silu' <= 1.1; |gelu''| <= 0.8, |silu''| <= 0.5."""
    if name == 'relu':
        return z.clamp(min=0), (z > 0).double(), 1.0, 0.0
    if name == 'gelu':
        phi = 0.5 * torch.erfc(-z / math.sqrt(2))
        return z * phi, phi + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi), 1.13, 0.8
    if name == 'silu':
        s = torch.sigmoid(z)
        return z * s, s * (1 + z * (1 - s)), 1.1, 0.5
    return z, torch.ones_like(z), 1.0, 0.0


def product_error(sum_abs, k, dtype):
    """An fp32 sum of k products whose magnitudes add up to sum_abs, in any order: k roundings of at most the running sum. fp32
    operands are six partial products each (6 k roundings), and what the split leaves out - two products of at most 2^-7 and 2^-16
    of the operands, one of 2^-16 twice - is below 2^-21.9 of each product."""
    if dtype == torch.float32:
        return sum_abs * ((6 * k + 8) * F + 2.0 ** -21.9)
    return sum_abs * ((k + 8) * F)


def linear(x, w, b, r, name, dy=None, kept=None):
    """(values, bounds): dicts y (, dx, dw, db). All operands are tensors of the type under test (or None); `kept`: what stands
    for x in dw (fp64)."""
    t = x.dtype
    X, W = x.double(), w.double()
    z = X @ W.t()
    zs = X.abs() @ W.abs().t()
    if b is not None:
        z, zs = z + b.double(), zs + b.double().abs()
    ez = product_error(zs, X.shape[1] + 1, t)
    a, da, l1, l2 = act(z, name)
    y = a if r is None else a + r.double()
    # the activation: its distribution function to 2^-22 of the smaller tail, a few roundings of its factors; the residual's sum: one
    ey = l1 * ez + (0 if name is None else 12 * F * (z.abs() + 1)) + F * (a.abs() + y.abs())
    values, bounds = dict(y=y), dict(y=ey + last_rounding(y, t))
    if dy is None:
        return values, bounds
    DY = dy.double()
    dz = DY * da
    if name is None:
        edz32 = torch.zeros_like(dz)
        edz = edz32
    else:
        # act' at the z that was kept: rounded to the type, and off by its sum's error; relu's gate is taken as given where the
        # tests keep z away from 0
        edz32 = DY.abs() * (l2 * (ez + last_rounding(z, t)) + 16 * F)
        edz = edz32 + last_rounding(dz.abs() + edz32, t)
    M, N = dz.shape
    KX = X if kept is None else kept
    for key, left, right, eleft, n in (('dx', dz, W, edz, N), ('dw', dz.t(), KX, edz.t(), M)):
        v = left @ right
        s = (left.abs() + eleft) @ right.abs()
        values[key] = v
        bounds[key] = eleft @ right.abs() + product_error(s, n, t) + last_rounding(v, t)
    values['db'] = dz.sum(0)
    bounds['db'] = edz32.sum(0) + (M + 4) * F * (dz.abs() + edz32).sum(0) + last_rounding(dz.sum(0), t)
    return values, bounds


def unpacked(x):
    """The 8-bit form's values in fp64."""
    rows, n = x.shape
    blocks = -(-n // 32)
    v = torch.zeros(rows, blocks * 32, dtype=torch.float64, device=x.device)
    v[:, :n] = x.double()
    v = v.view(rows, blocks, 32)
    top = v.abs().amax(-1, keepdim=True)
    finite = torch.isfinite(v).all(-1, keepdim=True)
    k = torch.frexp(torch.where(finite, top, torch.zeros_like(top)))[1]
    e = (k - 7).clamp(min=-24 if x.dtype == torch.float16 else -126).double()
    e = torch.where(top > 0, e, torch.full_like(e, -24 if x.dtype == torch.float16 else -126))
    q = torch.round(v / 2 ** e).clamp(-127, 127)
    return torch.where(finite, q * 2 ** e, torch.full_like(v, math.nan)).view(rows, -1)[:, :n]


def norm(z, g, b, eps, dy=None, dz=None, kept=None):
    """(values, bounds): y (, dx, dg, db) for z as it is stored. A sum over D numbers runs in at most 64 roundings a number here (32
    in a register walk, the rest of a tree) up to D = 16,384; longer rows add D / 8192 each."""
    t, pt = z.dtype, z.dtype if g is None else g.dtype
    Z = z.double()
    D = Z.shape[1]
    n = 64 + 2 * D / 8192
    mean = Z.mean(1, keepdim=True)
    var = ((Z - mean) ** 2).mean(1, keepdim=True)
    rstd = 1 / torch.sqrt(var + eps)
    xhat = (Z - mean) * rstd
    off = Z.abs().mean(1, keepdim=True) * rstd                        # an error of the mean, in units of the result
    G = torch.ones(D, dtype=torch.float64) if g is None else g.double()
    B = torch.zeros(D, dtype=torch.float64) if b is None else b.double()
    exh = n * F * (xhat.abs() * (1 + off) + off)                      # of xhat: the mean's, the variance's, a few products
    y = xhat * G + B
    values = dict(y=y)
    bounds = dict(y=exh * G.abs() + 4 * F * (xhat.abs() * G.abs() + B.abs()) + last_rounding(y, t))
    if dy is None:
        return values, bounds
    if kept is not None:
        xhat = (kept - mean) * rstd
        exh = n * F * (xhat.abs() * (1 + off) + off) + 2 * F * kept.abs() * rstd
    DY = dy.double()
    T = DY * G
    m1, m2 = T.mean(1, keepdim=True), (T * xhat).mean(1, keepdim=True)
    em1 = n * F * T.abs().mean(1, keepdim=True)
    em2 = (T.abs() * exh).mean(1, keepdim=True) + n * F * (T * xhat).abs().mean(1, keepdim=True)
    dx = rstd * (T - m1 - xhat * m2)
    edx = rstd * (em1 + xhat.abs() * em2 + exh * m2.abs() + 6 * F * (T.abs() + m1.abs() + (xhat * m2).abs())) + n * F * (1 + off) * dx.abs()
    if dz is not None:
        dx = dx + dz.double()
        edx = edx + F * dx.abs()
    M = Z.shape[0]
    dg, db = (DY * xhat).sum(0), DY.sum(0)
    values.update(dx=dx, dg=dg, db=db)
    bounds.update(dx=edx + last_rounding(dx, t), dg=(DY.abs() * exh).sum(0) + (M + 16) * F * (DY * xhat).abs().sum(0) + last_rounding(dg, pt),
                  db=(M + 16) * F * DY.abs().sum(0) + last_rounding(db, pt))
    return values, bounds


def check(got, values, bounds, where=''):
    """Every element of got[key] within its bound of values[key]. What lies over the type's largest number by half a step (65,520 in
    fp16) rounds to that infinity: it has to where the whole bound lies there, and may where a part does."""
    for key, t in got.items():
        v, e = values[key], bounds[key]
        g = t.detach().double().to(v.device)
        assert g.shape == v.shape, (where, key, g.shape, v.shape)
        top = torch.finfo(t.dtype).max * (1 + half_step(t.dtype) / 2)
        must, may = v.abs() - e > top, (v.abs() + e > top) & (g == v.sign() * math.inf)
        assert torch.equal(g[must], v[must].sign() * math.inf), (where, key)
        off = (g - v).abs().masked_fill(must | may, 0)
        assert torch.isfinite(off).all(), (where, key)
        worst = float((off / e.clamp(min=1e-300)).max()) if off.numel() else 0.0
        assert worst <= 1, f'{where} {key}: {worst:.3g} times the bound, largest difference {float(off.max()):.3g}'
