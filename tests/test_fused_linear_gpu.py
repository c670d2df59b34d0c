"""K15: act(x W' + b) + r and its gradients against the definition in fp64, at the sizes, types and forms where a launch can go wrong.
Every tolerance is a bound on the launch's roundings (dense_bounds)."""
import pytest
import torch
import torch.nn as nn

import dense_bounds as B

pytestmark = pytest.mark.gpu
DEV = 'cuda'


def _case(M, K, N, dtype, seed=0, bias=True, residual=False, away=None):
    """Operands; `away`: scale of a bias that keeps |z| off relu's gate (alternating in sign over the features)."""
    g = torch.Generator().manual_seed(seed + 1000 * M + 10 * K + N)
    t = B.TYPES[dtype]
    x, w = torch.randn(M, K, generator=g).to(t), (torch.randn(N, K, generator=g) / max(K, 1) ** 0.5).to(t)
    b = torch.randn(N, generator=g)
    if away:
        b = away * (1 - 2 * (torch.arange(N) % 2)).float()
    r = torch.randn(M, N, generator=g).to(t) if residual else None
    dy = (torch.randn(M, N, generator=g) / max(M, 1) ** 0.5).to(t)
    return x, w, b.to(t) if bias else None, r, dy


def _run(x, w, b, r, act, dy=None, save8=False):
    from ursabench_amd.fused_linear import linear_act
    fc = nn.Linear(w.shape[1], w.shape[0], bias=b is not None, device=DEV, dtype=w.dtype)
    with torch.no_grad():
        fc.weight.copy_(w)
        if b is not None:
            fc.bias.copy_(b)
    fc.requires_grad_(dy is not None)
    X = x.detach().to(DEV).requires_grad_(dy is not None)
    R = None if r is None else r.detach().to(DEV).requires_grad_(dy is not None)
    y = linear_act(fc, X, act, R, save8=save8)
    if dy is None:
        return dict(y=y)
    leaves = dict(dx=X, dw=fc.weight)
    if b is not None:
        leaves['db'] = fc.bias
    if R is not None:
        leaves['dr'] = R
    got = dict(zip(leaves, torch.autograd.grad(y, list(leaves.values()), dy.to(DEV))))
    if R is not None:
        assert torch.equal(got.pop('dr').to(dy.device), dy)
    return dict(y=y, **got)


SIZES = [(1, 1, 1), (1, 8, 16), (2, 31, 3), (3, 5, 7), (16, 64, 64), (17, 33, 65), (64, 128, 128), (65, 130, 131), (100, 784, 200),
         (128, 200, 10), (130, 64, 129), (257, 96, 300), (5, 4100, 40), (33, 2048, 72), (400, 24, 16), (1000, 32, 8)]


@pytest.mark.parametrize('dtype', list(B.TYPES))
@pytest.mark.parametrize('M,K,N', SIZES)
def test_forward_and_gradients_at_odd_and_even_sizes(M, K, N, dtype):
    x, w, b, r, dy = _case(M, K, N, dtype, residual=True)
    B.check(_run(x, w, b, r, 'gelu', dy), *B.linear(x, w, b, r, 'gelu', dy), where=(M, K, N, dtype))


@pytest.mark.parametrize('dtype', list(B.TYPES))
@pytest.mark.parametrize('M,K,N', [(600, 520, 1100), (520, 1048, 520), (1100, 264, 1032), (300, 4096, 300), (2100, 130, 150), (777, 555, 333)])
def test_larger_tiles_and_cut_contractions(M, K, N, dtype):
    x, w, b, r, dy = _case(M, K, N, dtype, residual=True)
    B.check(_run(x, w, b, r, 'silu', dy), *B.linear(x, w, b, r, 'silu', dy), where=(M, K, N, dtype))


@pytest.mark.parametrize('save8', [False, True])
@pytest.mark.parametrize('dtype', list(B.TYPES))
@pytest.mark.parametrize('M,K,N', [(3592, 3600, 3608), (2056, 2056, 2056), (4104, 72, 4104), (200, 4104, 4104), (4104, 4104, 72), (3600, 3601, 3600)])
def test_whole_tiles_and_their_edges(M, K, N, dtype, save8):
    """Sizes that give every product of the step its largest tiles (and its second largest, and one it cannot use them for), none
    a multiple of a tile or of a step over the contraction; fp64 on the device."""
    x, w, b, r, dy = (None if t is None else t.to(DEV) for t in _case(M, K, N, dtype, residual=True))
    B.check(_run(x, w, b, r, 'silu', dy, save8=save8), *B.linear(x, w, b, r, 'silu', dy, kept=B.unpacked(x) if save8 else None), where=(M, K, N, dtype))


@pytest.mark.parametrize('dtype', list(B.TYPES))
@pytest.mark.parametrize('residual', [False, True])
@pytest.mark.parametrize('bias', [False, True])
@pytest.mark.parametrize('act', [None, 'gelu', 'silu'])
def test_every_epilogue(act, bias, residual, dtype):
    x, w, b, r, dy = _case(70, 72, 90, dtype, bias=bias, residual=residual)
    B.check(_run(x, w, b, r, act, dy), *B.linear(x, w, b, r, act, dy), where=(act, bias, residual, dtype))


@pytest.mark.parametrize('dtype', list(B.TYPES))
def test_relu_with_its_gate_away_from_zero(dtype):
    x, w, b, r, dy = _case(70, 72, 90, dtype, residual=True, away=8.0)
    assert float((x.double() @ w.double().t() + b.double()).abs().min()) > 1
    B.check(_run(x, w, b, r, 'relu', dy), *B.linear(x, w, b, r, 'relu', dy))


@pytest.mark.parametrize('dtype', list(B.TYPES))
@pytest.mark.parametrize('M', [1, 2, 5, 8, 16, 17, 31, 48, 64])
@pytest.mark.parametrize('K,N', [(256, 512), (1000, 333), (4096, 96), (72, 1030), (8200, 40), (5003, 200), (2051, 2100)])
def test_few_rows(M, K, N, dtype):
    x, w, b, r, _ = _case(M, K, N, dtype, residual=True)
    B.check(_run(x, w, b, r, 'gelu'), *B.linear(x, w, b, r, 'gelu'), where=(M, K, N, dtype))


@pytest.mark.parametrize('dtype', list(B.TYPES))
@pytest.mark.parametrize('M,K,N', [(1, 32, 16), (40, 64, 48), (130, 100, 72), (300, 1111, 200), (1000, 256, 136), (600, 1056, 1100)])
def test_input_kept_in_8_bits(M, K, N, dtype):
    x, w, b, r, dy = _case(M, K, N, dtype)
    x[:, 3] *= 40                                                    # a feature that sets its blocks' scale
    got = _run(x, w, b, r, 'gelu', dy, save8=True)
    B.check(got, *B.linear(x, w, b, r, 'gelu', dy, kept=B.unpacked(x)), where=(M, K, N, dtype))


def test_gradients_against_differences():
    """Central differences of sum(c y) along a random direction, fp32: the launches' forward error over the step, and the third
    derivative's h^2 term (gelu''' <= 2; every |dz| of the step <= h |direction z|)."""
    M, K, N, h = 20, 48, 40, 2.0 ** -5
    x, w, b, r, c = _case(M, K, N, 'float32', residual=True)
    g = torch.Generator().manual_seed(5)
    vx, vw, vb, vr = (torch.randn(t.shape, generator=g) * s for t, s in ((x, 0.1), (w, 0.02), (b, 0.1), (r, 0.1)))
    got = _run(x, w, b, r, 'gelu', c)
    slope = sum(float((got[k].double().cpu() * v.double()).sum()) for k, v in (('dx', vx), ('dw', vw), ('db', vb))) + float((c.double() * vr.double()).sum())
    side, err = [], 0.0
    for s in (h, -h):
        args = (x + s * vx, w + s * vw, b + s * vb, r + s * vr)
        side.append(float((_run(*args, 'gelu')['y'].double().cpu() * c.double()).sum()))
        moved = B.linear(*args, 'gelu')[1]['y']
        err += float((moved * c.double().abs()).sum())
        # the moved operands are rounded to fp32 themselves: 2^-24 of each, through the sums
        err += B.F * float(((args[0].abs().double() @ args[1].abs().double().t() * 2 + args[2].abs() + args[3].abs()) * 1.13 * c.abs()).sum())
    dz1 = vx.double() @ w.double().t() + x.double() @ vw.double().t() + vb.double()
    dz2 = 2 * (vx.double() @ vw.double().t())
    third = (2 * dz1.abs() ** 3 + 3 * 0.8 * (dz1 * dz2).abs() + 4 * h * dz2.abs() ** 2) * c.abs().double()
    values, bounds = B.linear(x, w, b, r, 'gelu', c)
    own = sum(float((bounds[k] * v.double().abs()).sum()) for k, v in (('dx', vx), ('dw', vw), ('db', vb)))
    assert abs((side[0] - side[1]) / (2 * h) - slope) <= err / (2 * h) + h * h / 6 * 1.5 * float(third.sum()) + own


def test_leading_dimensions_strides_and_offsets():
    from ursabench_amd.fused_linear import linear_act
    torch.manual_seed(0)
    for t in B.TYPES.values():
        fc = nn.Linear(40, 24, device=DEV, dtype=t)
        base = torch.randn(3, 7, 81, device=DEV).to(t)
        x = base[:, :, 1:41]                                         # rows 81 apart, one element off alignment
        r = torch.randn(24, device=DEV).to(t).expand(3, 7, 24)       # one vector for every row
        want = linear_act(fc, x.contiguous().view(21, 40), 'silu', r.contiguous().view(21, 24)).view(3, 7, 24)
        assert torch.equal(linear_act(fc, x, 'silu', r), want)
        assert torch.equal(linear_act(fc, base.transpose(0, 1)[:, :, 1:41], 'silu', r.transpose(0, 1)), want.transpose(0, 1))
        one = torch.randn(41, device=DEV).to(t)[1:]
        assert torch.equal(linear_act(fc, one), linear_act(fc, one.clone()[None])[0])
        # a contiguous view whose storage starts at an odd element, as weights in a flat arena do
        flat = torch.zeros(1 + fc.weight.numel(), device=DEV, dtype=t)
        flat[1:].copy_(fc.weight.detach().view(-1))
        other = nn.Linear(40, 24, device=DEV, dtype=t)
        other.weight.data, other.bias.data = flat[1:].view(24, 40), fc.bias.data
        assert torch.equal(linear_act(other, x, 'silu', r), want)
        xb = x.detach().requires_grad_()
        rb = r.detach().requires_grad_()
        gx, gr, gw = torch.autograd.grad(linear_act(fc, xb, 'silu', rb), (xb, rb, fc.weight), torch.ones(1, device=DEV, dtype=t).expand(3, 7, 24))
        assert gx.shape == xb.shape and gr.shape == rb.shape and torch.equal(gr, torch.ones_like(gr))
        other.weight.requires_grad_()
        assert torch.equal(torch.autograd.grad(linear_act(other, x, 'silu', r).sum(), other.weight)[0], gw)


def test_broadcast_residual_gets_the_summed_gradient():
    from ursabench_amd.fused_linear import linear_act
    fc = nn.Linear(16, 24, device=DEV)
    v = torch.randn(24, device=DEV, requires_grad=True)
    y = linear_act(fc, torch.randn(9, 16, device=DEV), None, v.expand(9, 24))
    assert torch.equal(torch.autograd.grad(y.sum(), v)[0], torch.full((24,), 9.0, device=DEV))


@pytest.mark.parametrize('frozen', ['x', 'w', 'b', 'xw', 'wb', 'xb', 'xwb'])
def test_only_the_gradients_that_are_wanted(frozen):
    from ursabench_amd.fused_linear import linear_act
    x, w, b, r, dy = _case(33, 40, 50, 'float32', residual=True)
    full = _run(x, w, b, r, 'gelu', dy)
    fc = nn.Linear(40, 50, device=DEV)
    with torch.no_grad():
        fc.weight.copy_(w), fc.bias.copy_(b)
    fc.weight.requires_grad_('w' not in frozen), fc.bias.requires_grad_('b' not in frozen)
    X, R = x.to(DEV).requires_grad_('x' not in frozen), r.to(DEV).requires_grad_()
    leaves = {k: t for k, t in (('dx', X), ('dw', fc.weight), ('db', fc.bias)) if t.requires_grad}
    got = torch.autograd.grad(linear_act(fc, X, 'gelu', R), [*leaves.values(), R], dy.to(DEV))
    assert torch.equal(got[-1].cpu(), dy)
    for k, t in zip(leaves, got):
        assert torch.equal(t, full[k]), k


def test_differentiable_once_and_no_changes_in_place():
    """create_graph gives the same gradients, differentiating them raises; so does a backward pass over an operand that changed."""
    from ursabench_amd.fused_linear import linear_act
    from ursabench_amd.fused_norm import add_layer_norm, layer_norm
    fc, ln = nn.Linear(40, 40, device=DEV), nn.LayerNorm(40, device=DEV)
    x = torch.randn(3, 9, 40, device=DEV, requires_grad=True)
    for f in (lambda: linear_act(fc, x, 'gelu', x), lambda: layer_norm(ln, x), lambda: sum(add_layer_norm(ln, (x, 2 * x)))):
        want = torch.autograd.grad(f().square().sum(), x)[0]
        g = torch.autograd.grad(f().square().sum(), x, create_graph=True)[0]
        assert torch.equal(g, want)
        with pytest.raises(RuntimeError, match='double backward'):
            g.sum().backward()
    y = linear_act(fc, x, 'gelu')
    with torch.no_grad():
        fc.weight.mul_(2)
    with pytest.raises(RuntimeError, match='modified by an inplace'):
        y.sum().backward()
    z, y = add_layer_norm(ln, (x, 2 * x))
    z.mul_(2)
    with pytest.raises(RuntimeError, match='modified by an inplace'):
        y.sum().backward()


def test_nothing_is_kept_behind_a_dropped_graph():
    from ursabench_amd.fused_linear import linear_act
    from ursabench_amd.fused_norm import add_layer_norm
    fc, ln = nn.Linear(512, 512, device=DEV), nn.LayerNorm(512, device=DEV)
    x = torch.randn(4, 256, 512, device=DEV, requires_grad=True)
    held = []
    for _ in range(4):
        for save8 in (False, True):
            z, y = add_layer_norm(ln, (x, x), save8=save8)
            linear_act(fc, y, 'gelu', z, save8=save8).sum().backward()
            del z, y
        torch.cuda.synchronize()
        held.append(torch.cuda.memory_allocated())
    assert held[-1] == held[0], held


def test_empty_batches():
    from ursabench_amd.fused_linear import linear_act
    for t in B.TYPES.values():
        for save8 in (False, True):
            fc = nn.Linear(40, 24, device=DEV, dtype=t)
            x = torch.empty(0, 40, device=DEV, dtype=t, requires_grad=True)
            y = linear_act(fc, x, 'gelu', save8=save8)
            assert y.shape == (0, 24)
            dx, dw, db = torch.autograd.grad(y, (x, fc.weight, fc.bias), torch.empty(0, 24, device=DEV, dtype=t))
            assert dx.shape == (0, 40) and not dw.any() and not db.any() and dw.shape == (24, 40)


def test_no_features_and_no_rows_at_the_kernels():
    """An empty contraction is a sum of nothing: zeros, in every direction."""
    from ursabench_amd import _native
    k = _native.default_kernels()
    z = lambda *s: torch.empty(s, device=DEV, dtype=torch.bfloat16)      # noqa: E731
    dx, dw, db = k.linear_backward(z(300, 0), z(300, 40), z(0, 40))
    assert dx.shape == (300, 40) and not dx.any() and dw.shape == (0, 40) and db.shape == (0,)
    b = torch.randn(24, device=DEV).bfloat16()
    for M in (5, 300):
        assert torch.equal(k.linear_act(z(M, 0), z(24, 0), b)[0], b.expand(M, 24))
    dx, dg, db = k.layer_norm_backward(z(0, 40), torch.empty(2, 0, device=DEV), x=z(0, 40), need_dgamma=True, need_dbeta=True)
    assert dx.shape == (0, 40) and dg.shape == db.shape == (40,) and not dg.any() and not db.any()


@pytest.mark.parametrize('dtype', list(B.TYPES))
def test_infinities_and_nans_stay_in_their_rows(dtype):
    """Other rows keep their bits; the row itself is not finite."""
    from ursabench_amd.fused_linear import linear_act
    x, w, b, r, dy = _case(70, 72, 90, dtype)
    t = B.TYPES[dtype]
    fc = nn.Linear(72, 90, device=DEV, dtype=t)
    clean = linear_act(fc, x.to(DEV), 'gelu')
    for bad in (float('inf'), float('-inf'), float('nan')):
        z = x.clone()
        z[5, 7] = bad
        y = linear_act(fc, z.to(DEV))
        assert not torch.isfinite(y[5]).any()
        y = linear_act(fc, z.to(DEV), 'gelu')
        keep = [i for i in range(70) if i != 5]
        assert torch.equal(y[keep], clean[keep])
        X = z.to(DEV).requires_grad_()
        dw = torch.autograd.grad(linear_act(fc, X, save8=True), fc.weight, dy.to(DEV))[0]
        assert torch.isnan(dw[:, :32]).all() and torch.isfinite(dw[:, 32:]).all()     # the block of 32 features, no other


@pytest.mark.parametrize('dtype', list(B.TYPES))
@pytest.mark.parametrize('M,K,N', [(100, 99, 71), (300, 200, 136), (90, 33, 40), (1000, 1111, 777)])
def test_nans_in_one_column_stay_in_it(M, K, N, dtype):
    """The column next to a row's end in memory is the next row's first: what is NaN there reaches the gradients of that column
    (or what is contracted with it) and nothing else."""
    from ursabench_amd import _native
    k, t = _native.default_kernels(), B.TYPES[dtype]
    x, w, dy = (torch.randn(*s, device=DEV).to(t) for s in ((M, K), (N, K), (M, N)))
    bad = lambda v: torch.cat([torch.full_like(v[:, :1], float('nan')), v[:, 1:]], 1).contiguous()      # noqa: E731
    _, dw, _ = k.linear_backward(dy, bad(x), w)
    assert dw[:, 0].isnan().all() and dw[:, 1:].isfinite().all()
    dx, _, _ = k.linear_backward(dy, x, bad(w))
    assert dx[:, 0].isnan().all() and dx[:, 1:].isfinite().all()
    dx, dw, db = k.linear_backward(bad(dy), x, w)
    assert dx.isnan().all() and dw[0].isnan().all() and dw[1:].isfinite().all() and db[0].isnan() and db[1:].isfinite().all()
    q, e = k.act8_pack(bad(x))
    _, dw, _ = k.linear_backward(dy, None, w, q=q, e=e, in_features=K)
    assert dw[:, :32].isnan().all() and dw[:, 32:].isfinite().all()                   # a block of 32 with a NaN in it is NaN
    x[-1] = float('nan')
    y = k.linear_act(x, w)[0]
    assert y[-1].isnan().all() and y[:-1].isfinite().all()


@pytest.mark.parametrize('act', ['gelu', 'silu', 'relu'])
def test_sums_beyond_the_type_have_their_slope(act):
    """z = -96,000 is -inf in fp16 where it is kept: y = 0 and the gradient 0, not NaN; z = 96,000: y = inf, the gradient's factor 1;
    a NaN in z stays one."""
    from ursabench_amd import _native
    from ursabench_amd.fused_linear import linear_act
    fc = nn.Linear(8, 2, bias=False, device=DEV, dtype=torch.float16)
    with torch.no_grad():
        fc.weight.copy_(torch.tensor([[-6000.0] * 8, [6000.0] * 8]))
    x = torch.full((3, 8), 2.0, device=DEV, dtype=torch.float16, requires_grad=True)
    y = linear_act(fc, x, act)
    assert torch.equal(y[:, 0], torch.zeros_like(y[:, 0])) and torch.isinf(y[:, 1]).all()
    dy = torch.tensor([[1.0, 2.0 ** -10]] * 3, device=DEV, dtype=torch.float16)
    dx, dw = torch.autograd.grad(y, (x, fc.weight), dy)
    assert torch.equal(dx, torch.full_like(dx, 6000 / 1024)) and torch.equal(dw, torch.tensor([[0.0] * 8, [6 / 1024] * 8], device=DEV, dtype=torch.float16))
    z = torch.full((3, 2), float('nan'), device=DEV)
    db = _native.default_kernels().linear_backward(torch.ones(3, 2, device=DEV), in_features=8, z=z, activation=act, need_dx=False, need_dw=False)[2]
    assert torch.isnan(db).all() or act == 'relu'


@pytest.mark.parametrize('M', [40, 100])
def test_large_and_small_magnitudes_fp32(M):
    """The three-way split holds over fp32's exponents: products of 2^100 and 2^-100, of the largest numbers, and of numbers
    whose low parts are subnormal."""
    from ursabench_amd import _native
    k = _native.default_kernels()
    g = torch.Generator().manual_seed(3)
    x, w = torch.randn(M, 64, generator=g), torch.randn(48, 64, generator=g)
    for sx, sw in ((2.0 ** 100, 2.0 ** -100), (2.0 ** -100, 2.0 ** 100), (2.0 ** 120, 2.0 ** -60), (2.0 ** -60, 2.0 ** -40)):
        a, c = x * sx, w * sw
        got = k.linear_act(a.to(DEV), c.to(DEV))[0].double().cpu()
        want, bound = B.linear(a, c, None, None, None)
        # below 2^-117 the low parts of an operand are subnormal bf16 numbers, kept to 2^-133: 2^-134 of each times the other
        low = 2.0 ** -134 * (a.abs().double().sum(1)[:, None] + c.abs().double().sum(1)[None, :])
        assert ((got - want['y']).abs() <= bound['y'] + low).all(), (sx, sw)
    top = torch.full((M, 32), torch.finfo(torch.float32).max)
    got = k.linear_act(top.to(DEV), torch.full((16, 32), 2.0 ** -10, device=DEV))[0].double().cpu()
    want = float(top[0, 0]) * 2.0 ** -10 * 32
    assert ((got - want).abs() <= 1e-6 * want).all()


def test_offsets_past_32_bits():
    """More than 2^32 bytes of y, z and dy (and 2^31 elements): the last rows and features, and the column sums over all rows."""
    from ursabench_amd import _native
    k = _native.default_kernels()
    M, K, N = 70000, 8, 32768
    g = torch.Generator(device=DEV).manual_seed(0)
    x = torch.randn(M, K, generator=g, device=DEV).bfloat16()
    w = torch.randn(N, K, generator=g, device=DEV).bfloat16()
    y, z = k.linear_act(x, w, activation='silu', save_z=True)
    assert y.numel() > 2 ** 31
    tail = slice(M - 300, M)
    B.check(dict(y=y[tail]), *B.linear(x[tail], w, None, None, 'silu'))
    del z
    dx, dw, db = k.linear_backward(y, x, w)
    yt = y[tail].double()
    want = yt @ w.double()
    bound = B.product_error(yt.abs() @ w.double().abs(), N, torch.bfloat16) + B.last_rounding(want, torch.bfloat16)
    assert ((dx[tail].double() - want).abs() <= bound).all()
    cols = slice(N - 64, N)
    yc = y[:, cols].double()
    want, s = yc.t() @ x.double(), yc.abs().t() @ x.double().abs()
    assert ((dw[cols].double() - want).abs() <= B.product_error(s, M, torch.bfloat16) + B.last_rounding(want, torch.bfloat16)).all()
    assert ((db[cols].double() - yc.sum(0)).abs() <= (M + 16) * B.F * yc.abs().sum(0) + B.last_rounding(yc.sum(0), torch.bfloat16)).all()


def test_the_same_call_gives_the_same_bits():
    for M, K, N, dtype in ((300, 4096, 300, 'bfloat16'), (300, 1000, 200, 'float32')):
        x, w, b, r, dy = _case(M, K, N, dtype, residual=True)
        one = _run(x, w, b, r, 'gelu', dy)
        for _ in range(3):
            for key, t in _run(x, w, b, r, 'gelu', dy).items():
                assert torch.equal(t, one[key]), key


def test_side_streams_at_once():
    """Two streams run the same layer on their own inputs; each waits for what it uses."""
    from ursabench_amd.fused_linear import linear_act
    fc = nn.Linear(512, 700, device=DEV).requires_grad_(False)
    xs = [torch.randn(300, 512, device=DEV) for _ in range(4)]
    want = [linear_act(fc, x, 'gelu') for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [None] * 4
    for i, x in enumerate(xs):
        s = streams[i % 2]
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got[i] = linear_act(fc, x, 'gelu')
    for s in streams:
        torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_training_steps_on_side_streams_at_once():
    """Forward and backward of one layer's copies on two streams: their scratch is their own."""
    from ursabench_amd.fused_linear import linear_act
    fcs = [nn.Linear(2048, 640, device=DEV) for _ in range(4)]
    xs = [torch.randn(300, 2048, device=DEV, requires_grad=True) for _ in range(4)]
    dy = torch.randn(300, 640, device=DEV)

    def step(fc, x, save8):
        return torch.autograd.grad(linear_act(fc, x, 'gelu', save8=save8), (x, fc.weight, fc.bias), dy)
    want = [step(fc, x, i > 1) for i, (fc, x) in enumerate(zip(fcs, xs))]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for i, (fc, x) in enumerate(zip(fcs, xs)):
        with torch.cuda.stream(streams[i % 2]):
            got.append(step(fc, x, i > 1))
    for s in streams:
        torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for g, w in zip(got, want) for a, b in zip(g, w))


@pytest.mark.parametrize('save8', [False, True])
def test_one_tensor_in_both_places_and_one_layer_twice(save8):
    """The input as its own residual: its gradient is the layer's and dy; a layer called twice: both calls' gradients."""
    from ursabench_amd.fused_linear import linear_act
    fc = nn.Linear(136, 136, device=DEV)
    x, dy = torch.randn(100, 136, device=DEV, requires_grad=True), torch.randn(100, 136, device=DEV)
    y = linear_act(fc, x, 'silu', x, save8=save8)
    got = torch.autograd.grad(y, (x, fc.weight, fc.bias), dy, retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(got, torch.autograd.grad(y, (x, fc.weight, fc.bias), dy)))
    r = x.detach().clone().requires_grad_()
    yr = linear_act(fc, x, 'silu', r, save8=save8)
    dx, dw, db, dr = torch.autograd.grad(yr, (x, fc.weight, fc.bias, r), dy)
    assert torch.equal(y, yr) and torch.equal(dr, dy) and torch.equal(got[0], dx + dy) and torch.equal(got[1], dw) and torch.equal(got[2], db)
    h = linear_act(fc, x, 'silu', save8=save8)
    both = torch.autograd.grad(linear_act(fc, h, save8=save8), (x, fc.weight), dy)
    h2 = h.detach().requires_grad_()
    dh, dw2 = torch.autograd.grad(linear_act(fc, h2, save8=save8), (h2, fc.weight), dy)
    dx1, dw1 = torch.autograd.grad(linear_act(fc, x, 'silu', save8=save8), (x, fc.weight), dh)
    assert torch.equal(both[0], dx1) and torch.equal(both[1], dw1 + dw2)


@pytest.mark.parametrize('dtype', list(B.TYPES))
def test_captured_step_replays_like_the_eager_one(dtype):
    """Forward and backward of a layer (cut contractions among them) in a graph: several replays on new inputs with eager work and
    synchronisations between, every one equal to the eager call."""
    from ursabench_amd import _capture
    from ursabench_amd.fused_linear import linear_act
    t = B.TYPES[dtype]
    torch.manual_seed(1)
    fc = nn.Linear(1000, 200, device=DEV, dtype=t)
    x = torch.zeros(96, 1000, device=DEV, dtype=t, requires_grad=True)
    dy = torch.zeros(96, 200, device=DEV, dtype=t)

    def step(a, c, save8):
        return torch.autograd.grad(linear_act(fc, a, 'gelu', save8=save8), (a, fc.weight, fc.bias), c)

    for save8 in (False, True):
        side = _capture.side_streams(torch.device(DEV, 0), 1)[0]
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(x, dy, save8)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with _capture.capture(graph):
            out = step(x, dy, save8)
        for k in range(4):
            a, c = torch.randn(96, 1000, device=DEV).to(t), torch.randn(96, 200, device=DEV).to(t)
            with torch.no_grad():
                x.copy_(a), dy.copy_(c)
            graph.replay()
            torch.cuda.synchronize()
            got = [o.clone() for o in out]
            want = step(a.requires_grad_(), c, save8)
            torch.cuda.synchronize()
            for p, q in zip(got, want):
                assert torch.equal(p, q), (save8, k)


def test_what_takes_the_stock_path():
    """Autocast, mixed types, fp64, hooks, subclasses and the switch: fc(x) and the stock activation, same bits."""
    import torch.nn.functional as F
    from ursabench_amd import fused_linear
    from ursabench_amd.fused_linear import linear_act
    fc = nn.Linear(40, 24, device=DEV)
    x = torch.randn(9, 40, device=DEV)
    with torch.autocast('cuda', dtype=torch.bfloat16):
        y = linear_act(fc, x, 'relu')
        assert y.dtype == torch.bfloat16 and torch.equal(y, F.relu(fc(x)))
    d = nn.Linear(40, 24, device=DEV, dtype=torch.float64)
    assert torch.equal(linear_act(d, x.double(), 'silu'), F.silu(d(x.double())))
    with pytest.raises(RuntimeError):
        linear_act(fc, x.to(torch.bfloat16))
    seen = []
    hook = fc.register_forward_hook(lambda *a: seen.append(1))
    linear_act(fc, x)
    hook.remove()
    assert seen

    class Doubled(nn.Linear):
        def forward(self, x):
            return 2 * super().forward(x)

    two = Doubled(40, 24, device=DEV)
    assert torch.equal(linear_act(two, x, 'relu'), F.relu(two(x)))
    old = fused_linear.enabled(False)
    try:
        assert torch.equal(linear_act(fc, x, 'gelu'), F.gelu(fc(x)))
    finally:
        fused_linear.enabled(old)


def test_saved_memory():
    """What a layer keeps for its backward pass: x in 8 bits is 33 / 128 of its fp32 size."""
    from ursabench_amd.fused_linear import linear_act
    fc = nn.Linear(4096, 16, device=DEV)
    held = []
    for save8 in (False, True):
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        y = linear_act(fc, torch.randn(2048, 4096, device=DEV, requires_grad=True).mul(2), save8=save8)
        held.append(torch.cuda.memory_allocated() - before)
        del y
    full = 2048 * 4096 * 4
    assert held[0] - held[1] == full - full // 4 - full // 128


def test_models_take_it_when_asked():
    """models.MLP / LeNet5 with in_models(True): logits and gradients of the stock networks to fp32 rounding (the gates' inputs of
    this seed are not within it of zero: the same units are open)."""
    from ursabench_amd import fused_linear, models
    assert fused_linear.in_models() is False
    for make, shape in ((lambda: models.MLP(200, 784, 10), (64, 1, 28, 28)), (lambda: models.LeNet5(10), (32, 1, 28, 28))):
        torch.manual_seed(0)
        net = make().to(DEV)
        x, y = torch.randn(shape, device=DEV), torch.randint(0, 10, shape[:1], device=DEV)

        def step():
            logits = net(x)
            return logits.detach(), torch.autograd.grad(torch.nn.functional.cross_entropy(logits, y), list(net.parameters()))

        want, gw = step()
        calls = []
        real, fused_linear.linear_act = fused_linear.linear_act, lambda *a, **k: calls.append(1) or real(*a, **k)
        old = fused_linear.in_models(True)
        try:
            got, gg = step()
        finally:
            fused_linear.in_models(old)
            fused_linear.linear_act = real
        assert len(calls) == 3
        # fp32 sums of at most 800 terms through three layers, two orders of summation: 800 x 2^-24 x 3 of the scale
        assert float((got - want).abs().max()) <= 1.5e-4 * float(want.abs().max())
        for a, b in zip(gg, gw):
            assert float((a - b).abs().max()) <= 3e-4 * float(b.abs().max())


def test_sampler_runs_on_it():
    """An SGHMC chain (captured steps) on the MLP with the launches in: the graph path runs and its members are finite and differ."""
    from ursabench_amd import fused_linear, inference, models
    from ursabench_amd.data import synthetic
    torch.manual_seed(0)
    train = synthetic(512, (1, 28, 28), 10, seed=0, device=torch.device(DEV, 0), batch_size=128)
    old = fused_linear.in_models(True)
    try:
        s = inference.SGHMC({'lr': 0.01, 'prior_std': 0.5, 'num_samples': 2, 'alpha': 0.5, 'burn_in_epochs': 0},
                            models.MLP(200, 784, 10).to(DEV), train, device=torch.device(DEV, 0))
        members = s.sample()
        assert s.engine.stats['graph_replays'] > 0
    finally:
        fused_linear.in_models(old)
    a, b = (torch.cat([p.detach().view(-1) for p in m.parameters()]) for m in members)
    assert torch.isfinite(a).all() and torch.isfinite(b).all() and not torch.equal(a, b)
