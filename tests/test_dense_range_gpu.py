"""The dense blocks (K15, K16) at the ends of their types' range and precision, against the definition in fp64."""
import math

import pytest
import torch
import torch.nn as nn

import dense_bounds as B

pytestmark = pytest.mark.gpu
DEV = 'cuda'
INF, NAN = math.inf, math.nan


def _unpacked(x):
    """The 8-bit form's values, by the host: its powers of two are exact (the device's fp64 pow is off by a rounding for some, which
    breaks ties the other way)."""
    return B.unpacked(x.cpu()).to(DEV)


# ---- fp32 sums past the range -------------------------------------------------------------------
# Every form of the fp32 product: (M, K, N) whose forward is 64 x 64 tiles, 64 x 64 with the contraction cut, 128 x 128 (rows that the
# large form does not take), the large form, the large form with the contraction cut; and, for comparison, up to 64 rows.
FORMS = [(100, 40, 72), (100, 2040, 72), (2100, 33, 2052), (4104, 72, 2056), (1032, 4104, 1040), (40, 72, 72)]


def _signed(M, K, N):
    """x with a tenth of its rows near 2^100, w near 2^100 with one sign a feature: a sum of the large rows is above 2^200 in
    magnitude, of that sign - and so are, past the range each, the products with the operands' low parts, which have either sign. The
    others are inside the range."""
    g = torch.Generator(device=DEV).manual_seed(M + K + N)
    x, w = 1 + torch.rand(M, K, generator=g, device=DEV), 1 + torch.rand(N, K, generator=g, device=DEV)
    big = torch.arange(M, device=DEV) % 10 == 3
    x[big] *= 2.0 ** 100
    w *= 2.0 ** 100 * (1 - 2 * (torch.arange(N, device=DEV) % 2).float())[:, None]
    return x, w, big


def _agrees(got, want, k):
    """Infinities and NaNs of `want` (fp32's: |sum| >= 2^128) exactly, the rest to an fp32 sum's rounding; all terms of a sum have one sign."""
    want = torch.where(want.abs() >= 2.0 ** 128, want.sign() * INF, want)
    got = got.double()
    assert torch.equal(got.isnan(), want.isnan())
    assert torch.equal(got[want.isinf()], want[want.isinf()])
    fine = want.isfinite()
    assert ((got - want)[fine].abs() <= B.product_error(want[fine].abs(), k, torch.float32)).all()


@pytest.mark.parametrize('M,K,N', FORMS)
def test_fp32_sums_past_the_range_are_infinite(M, K, N):
    """Finite operands whose sum fp32 cannot hold: the infinity of its sign in every form and direction, whatever the low parts' signs;
    relu of -inf is 0. The other rows keep their values."""
    from ursabench_amd import _native
    k = _native.default_kernels()
    x, w, big = _signed(M, K, N)
    want = x.double() @ w.double().t()
    assert (want[big].abs() > 2.0 ** 128).all()
    _agrees(k.linear_act(x, w)[0], want, K)
    _agrees(k.linear_act(x, w, activation='relu')[0], want.clamp(min=0), K)
    # dx = dy w: dy takes x's place, [M, N'] with N' = K, w as it is stored for the other direction
    wt = w.t().contiguous()
    _agrees(k.linear_backward(x, None, wt, need_dw=False, need_db=False)[0], want, K)
    # dw = dy' x
    xt = x.t().contiguous()
    _agrees(k.linear_backward(xt, wt, need_dx=False, need_db=False)[1], want, K)


@pytest.mark.parametrize('M,K,N', [(70, 100, 72), (4104, 72, 2056), (1032, 4104, 1040)])
def test_fp32_sums_past_the_range_with_the_input_in_8_bits(M, K, N):
    from ursabench_amd import _native
    k = _native.default_kernels()
    x, w, _ = _signed(M, K, N)
    q, e = k.act8_pack(w.t().contiguous())                                  # dw [M, N] = x (as dy' [K, M]) times the kept [K, N]
    kept = _unpacked(w.t())
    got = k.linear_backward(x.t().contiguous(), None, None, q=q, e=e, in_features=N, need_dx=False, need_db=False)[1]
    _agrees(got, x.double() @ kept, K)


@pytest.mark.parametrize('M,K,N', FORMS)
def test_fp32_infinities_and_nans_enter_sums_as_they_do_in_fp32(M, K, N):
    from ursabench_amd import _native
    k = _native.default_kernels()
    g = torch.Generator(device=DEV).manual_seed(K)
    x, w = 1 + torch.rand(M, K, generator=g, device=DEV), 1 + torch.rand(N, K, generator=g, device=DEV)
    w *= (1 - 2 * (torch.arange(N, device=DEV) % 2).float())[:, None]
    x[5, K - 1], x[7, 3], x[8, 0], x[M - 1, K // 2] = INF, -INF, NAN, INF
    w[2, K - 1], w[4, 3], w[N - 1, 1] = 0, INF, NAN
    want = x.double() @ w.double().t()
    assert want[5, 2].isnan() and want[5, 3] == -INF and want[7, 4] == -INF and want[8].isnan().all() and want[0, 4] == INF
    for act, f in ((None, lambda z: z), ('relu', torch.relu)):
        _agrees(k.linear_act(x, w, activation=act)[0], f(want), K)
    wt = w.t().contiguous()
    _agrees(k.linear_backward(x, None, wt, need_dw=False, need_db=False)[0], want, K)
    _agrees(k.linear_backward(x.t().contiguous(), wt, need_dx=False, need_db=False)[1], want, K)


def test_fp32_the_largest_numbers_and_a_row_among_many():
    """The largest number times one, sums that end exactly at it, and a row's answer beside 3 rows and beside 300."""
    from ursabench_amd import _native
    k = _native.default_kernels()
    top = torch.finfo(torch.float32).max
    x, w, big = _signed(300, 72, 72)
    few = k.linear_act(x[:4].contiguous(), w)[0]
    many = k.linear_act(x, w)[0]
    assert torch.equal(few.isfinite(), many[:4].isfinite()) and torch.equal(few[3], many[3]) and few[3].isinf().all()
    x, w = torch.zeros(300, 72, device=DEV), torch.zeros(72, 72, device=DEV)
    x[:, 5], w[:, 5] = top, 1
    x[:, 9], w[1::2, 9] = 1, top                                            # 2 top: past the range
    y = k.linear_act(x, w)[0]
    assert (y[:, 0::2] == top).all() and (y[:, 1::2] == INF).all()


@pytest.mark.parametrize('M,K,N', FORMS)
def test_fp32_operands_near_the_smallest(M, K, N):
    """From 2^-110 up the three parts of an operand hold all of it; below, its low part ends at the smallest bf16 number, 2^-133: half of
    that is lost of each operand, times the other. Subnormal operands among them."""
    from ursabench_amd import _native
    k = _native.default_kernels()
    g = torch.Generator(device=DEV).manual_seed(N)
    for scale in (-110, -113, -118, -126, -131):
        x = (1 + torch.rand(M, K, generator=g, device=DEV)) * 2.0 ** scale
        w = (1 + torch.rand(N, K, generator=g, device=DEV)) * 2.0 ** 100
        want = x.double() @ w.double().t()
        bound = B.product_error(want, K, torch.float32) + (0 if scale >= -110 else 2.0 ** -134 * w.double().abs().sum(1))
        for got in (k.linear_act(x, w)[0], k.linear_backward(x, None, w.t().contiguous(), need_dw=False, need_db=False)[0],
                    k.linear_backward(x.t().contiguous(), w.t().contiguous(), need_dx=False, need_db=False)[1]):
            assert ((got.double() - want).abs() <= bound).all(), scale


# ---- rows far from zero -------------------------------------------------------------------------
def _norm_bound(z, eps, g, b, stored_mean):
    """(y, bound on y or on what follows from xhat) of a row-wise norm whose mean is corrected by the mean of what it leaves. n roundings a
    sum as in dense_bounds.norm. First mean: off by d1 <= (n + 1) F max|z|. v = z - mean: F |v|. The mean of v: off by (n + 1) F mean|v|,
    with mean|v| <= deviation + d1. The variance around it: (n + 4) F (var + d1^2). `stored_mean`: the backward pass has the mean
    rounded once more, to fp32: F |mean|."""
    Z = z.double()
    n = 64 + 2 * Z.shape[1] / 8192
    mean = Z.mean(1, keepdim=True)
    var = ((Z - mean) ** 2).mean(1, keepdim=True)
    rstd = 1 / torch.sqrt(var + eps)
    d1 = (n + 1) * B.F * Z.abs().amax(1, keepdim=True)
    centre = (n + 2) * B.F * (var.sqrt() + d1) + 2 * B.F * ((Z - mean).abs() + d1) + (B.F * mean.abs() if stored_mean else 0)
    xhat = (Z - mean) * rstd
    relative = (n + 4) * B.F * (var + d1 ** 2) / (var + eps) + 4 * B.F
    if stored_mean:
        relative = relative + (B.F * mean.abs() * rstd) ** 2
    return xhat, rstd, centre * rstd + relative * (xhat.abs() + centre * rstd)


@pytest.mark.parametrize('dtype', list(B.TYPES))
@pytest.mark.parametrize('D', [7, 24, 100, 777, 1000, 1111, 2500, 5000, 10000, 16000, 20000])
def test_constant_rows_are_zero(D, dtype):
    """The mean of D equal numbers is that number, whether or not 1 / D is one: y is the bias and the gradients of the scale are 0."""
    from ursabench_amd.fused_norm import add_layer_norm, layer_norm
    t = B.TYPES[dtype]
    ln = nn.LayerNorm(D, device=DEV)
    with torch.no_grad():
        ln.bias.fill_(0.5)
    ln = ln.to(t)
    # whole and dyadic numbers whose sums fp32 holds exactly; the others round on the way
    x = torch.tensor([1000.0, 2.5, -3.0, 0.0, 0.1, 1234.567, -33333.0, 1e-3], device=DEV).to(t)[:, None].expand(8, D).contiguous()
    if dtype != 'float32':
        x[6] = -1000
    xhat, _, bound = _norm_bound(x, 1e-5, None, None, False)
    assert float(xhat.abs().max()) <= 1e-6
    y = layer_norm(ln, x)
    assert ((y.double() - 0.5).abs() <= bound + xhat.abs() + B.half_step(t) * 0.5).all() and (y[:4] == 0.5).all()
    z, y = add_layer_norm(ln, (x, torch.zeros_like(x)))
    assert torch.equal(z, x) and (y[:4] == 0.5).all()
    X = x[:4].clone().requires_grad_()
    dx, dg = torch.autograd.grad(layer_norm(ln, X), (X, ln.weight), torch.ones(4, D, device=DEV, dtype=t))
    assert not dg.any() and not dx.any()                    # xhat is 0, and a constant gradient has no component that moves y


@pytest.mark.parametrize('D', [7, 100, 1000, 1111, 5000, 10000, 20000])
def test_fp32_rows_far_from_zero(D):
    """Deviation 1e-5 of the mean, eps 1e-12 of its square and more."""
    from ursabench_amd import _native
    k = _native.default_kernels()
    g = torch.Generator(device=DEV).manual_seed(D)
    for mean, deviation in ((1000.0, 0.03), (-77.7, 1e-3), (1.0, 1e-4), (3e4, 3.0)):
        x = mean + deviation * torch.randn(9, D, generator=g, device=DEV)
        gamma, dy = 1 + 0.3 * torch.randn(D, generator=g, device=DEV), torch.randn(9, D, generator=g, device=DEV)
        eps = 1e-5
        xhat, rstd, bound = _norm_bound(x, eps, None, None, False)
        _, y, stats, _, _ = k.layer_norm(x, eps=eps, stats=True)
        assert ((y.double() - xhat).abs() <= bound + B.last_rounding(xhat, torch.float32)).all(), (mean, deviation)
        true = x.double().mean(1)
        n = 64 + 2 * D / 8192
        off = (n + 3) * B.F * ((x.double() - true[:, None]).abs().mean(1) + (n + 1) * B.F * x.double().abs().amax(1))
        assert ((stats[0].double() - true).abs() <= off + B.F * true.abs()).all()      # one rounding of the mean, and the correction's own
        _, _, e = _norm_bound(x, eps, None, None, True)
        dx, dg, db = k.layer_norm_backward(dy, stats, gamma, x=x, need_dgamma=True, need_dbeta=True)
        DY = dy.double()
        want = (DY * xhat).sum(0)
        assert ((dg.double() - want).abs() <= (DY.abs() * e).sum(0) + 25 * B.F * (DY * xhat).abs().sum(0) + B.last_rounding(want, torch.float32)).all()


@pytest.mark.parametrize('D', [7, 49, 1000, 1111, 4099, 10000, 20000])
def test_a_constant_gradient_moves_nothing(D):
    """t = dy gamma equal along a row that is constant itself: dx = rstd (t - mean t) = 0, the mean of D equal numbers being that number."""
    from ursabench_amd import _native
    k = _native.default_kernels()
    x = torch.full((9, D), 2.5, device=DEV)
    dy = torch.tensor([1.0, 3.0, 77.0, -1000.0, 801.0, 0.375, 1023.0, 5.0, 11.0], device=DEV)[:, None].expand(9, D).contiguous()   # sums are exact
    _, _, stats, _, _ = k.layer_norm(x, eps=1e-5, stats=True)
    assert torch.equal(stats[0], x[:, 0])
    dx, dg, _ = k.layer_norm_backward(dy, stats, x=x, need_dgamma=True)
    assert not dx.any() and not dg.any()


@pytest.mark.parametrize('D', [64, 777, 5000, 20000])
def test_fp32_rows_whose_variance_is_past_the_range(D):
    """Squares above 2^128: the variance is infinite and 1 / sqrt of it 0, so y is the bias - not a NaN of two infinities."""
    from ursabench_amd import _native
    k = _native.default_kernels()
    g = torch.Generator(device=DEV).manual_seed(D)
    x = torch.randn(4, D, generator=g, device=DEV) * torch.tensor([1e20, 1e28, 1e33, 1.0], device=DEV)[:, None]
    beta = torch.full((D,), 0.5, device=DEV)
    _, y, stats, _, _ = k.layer_norm(x, torch.ones(D, device=DEV), beta, eps=1e-5, stats=True)
    assert (y[:3] == 0.5).all() and not stats[1, :3].any() and y[3].isfinite().all() and stats[1, 3] > 0.5


# ---- rows of a million features -----------------------------------------------------------------
@pytest.mark.parametrize('dtype,M,D', [('float32', 3, 16385), ('bfloat16', 4, 20000), ('bfloat16', 40, 70001), ('float32', 9, 2 ** 20 + 5), ('float16', 40, 2 ** 20 + 5),
                                       ('bfloat16', 6, 4500001), ('float32', 2, 4500000)])
def test_column_sums_of_long_rows(dtype, M, D):
    """One slice of the rows (no scratch), few and many: dgamma and dbeta, together and each alone, from x and from its 8-bit form."""
    from ursabench_amd import _native
    k, t = _native.default_kernels(), B.TYPES[dtype]
    g = torch.Generator(device=DEV).manual_seed(D)
    x, dy = (torch.randn(M, D, generator=g, device=DEV).to(t) for _ in range(2))
    for pt in {t, torch.float32}:
        gamma = torch.ones(D, device=DEV, dtype=pt)
        _, _, stats, q, e = k.layer_norm(x, gamma, eps=1e-5, stats=True, save8=True)
        for kept, source in ((None, dict(x=x)), (_unpacked(x), dict(q=q, e=e))):
            Z, DY = x.double(), dy.double()
            mean, var = Z.mean(1, keepdim=True), Z.var(1, unbiased=False, keepdim=True)
            xhat = ((Z if kept is None else kept) - mean) / torch.sqrt(var + 1e-5)
            n = 64 + 2 * D / 8192
            exh = n * B.F * (xhat.abs() * 2 + 2)                                 # |mean| and the deviation's roundings are below one each
            want = dict(dg=(DY * xhat).sum(0), db=DY.sum(0))
            bound = dict(dg=(DY.abs() * exh).sum(0) + (M + 16) * B.F * (DY * xhat).abs().sum(0) + B.last_rounding(want['dg'], pt),
                         db=(M + 16) * B.F * DY.abs().sum(0) + B.last_rounding(want['db'], pt))
            _, dg, db = k.layer_norm_backward(dy, stats, gamma, need_dx=False, need_dgamma=True, need_dbeta=True, **source)
            B.check(dict(dg=dg, db=db), want, bound, where=(dtype, M, D, pt))
            assert torch.equal(k.layer_norm_backward(dy, stats, gamma, need_dx=False, need_dgamma=True, **source)[1], dg)
            assert torch.equal(k.layer_norm_backward(dy, stats, gamma, need_dx=False, need_dbeta=True, **source)[2], db)


# ---- the roundings of a 16-bit layer's gradients ------------------------------------------------
@pytest.mark.parametrize('dtype,act', [('bfloat16', 'gelu'), ('bfloat16', 'silu'), ('float16', 'gelu'), ('float16', 'silu')])
@pytest.mark.parametrize('M,K,N', [(300, 200, 333), (2048, 1024, 2048)])
def test_gradients_carry_the_rounding_of_z_of_dz_and_their_own(M, K, N, dtype, act):
    """Against the formula with z and dz rounded to the type, dx and dW are off by one rounding - the root of the mean square of the
    result's own, and no third one. An fp32 sum that ends beside a tie of z or dz may round to the other side: a sum's error is 2^-20 of
    its scale at most, which moves 2^-12 of the elements (bf16; fp16: 2^-9) by a step, 1 / sqrt(12) of which is a rounding's root mean
    square: sqrt(1 + 12 x 2^-9) of it together, and two operands so: 5 % in all."""
    from ursabench_amd import _native
    k, t = _native.default_kernels(), B.TYPES[dtype]
    g = torch.Generator(device=DEV).manual_seed(M)
    x, dy = torch.randn(M, K, generator=g, device=DEV).to(t), (torch.randn(M, N, generator=g, device=DEV) / M ** 0.5).to(t)
    w, b = ((2 * torch.rand(*s, generator=g, device=DEV) - 1) / K ** 0.5 for s in ((N, K), (N,)))
    w, b = w.to(t), b.to(t)
    once = lambda v: v.to(t).double()                                            # noqa: E731
    z = once(x.double() @ w.double().t() + b.double())
    _, kept = k.linear_act(x, w, b, activation=act, save_z=True)
    exact = dy.double() * B.act(z, act)[1]
    dz = once(exact)
    got = k.linear_backward(dy, x, w, kept, activation=act)
    for v, want in zip(got, (dz @ w.double(), dz.t() @ x.double(), exact.sum(0))):
        assert float((v.double() - want).norm()) <= 1.05 * float((once(want) - want).norm())
