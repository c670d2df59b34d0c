"""K15 - K17 on the host: argument checks of the C entries (before any launch), refusals, and the stock path of host tensors."""
import ctypes

import pytest
import torch
import torch.nn as nn
import torch.nn.functional as F

F32, BF16, F16 = 0, 1, 2


@pytest.fixture(scope='module')
def lib():
    from ursabench_amd import _native
    return _native.load_library()


@pytest.fixture(scope='module')
def p():
    """A 16-byte aligned host address that no refused call reads."""
    p.buf = (ctypes.c_float * 64)()
    a = ctypes.addressof(p.buf)
    return a + -a % 16


def test_linear_entries_refuse_bad_arguments(lib, p):
    fwd, bwd, ws, bws = lib.ursa_linear_act, lib.ursa_linear_bwd, lib.ursa_linear_ws_bytes, lib.ursa_linear_bwd_ws_bytes
    assert fwd(p, p, None, None, p, None, None, 4, 4, 4, 3, 0, None) == -4            # no such type
    assert fwd(p, p, None, None, p, None, None, 4, 4, 4, F32, 4, None) == -4          # no such activation
    assert fwd(p, p, None, None, p, None, None, -1, 4, 4, F32, 0, None) == -2
    assert fwd(p, p, None, None, p, None, None, 1 << 31, 4, 4, F32, 0, None) == -2
    assert fwd(p, p, None, None, p, None, None, 1 << 20, 1 << 20, 4, F32, 0, None) == -2    # more workgroups than a launch has
    assert fwd(p, p, None, None, p, None, None, 4, 1 << 28, 4, F32, 0, None) == -2
    assert fwd(p, p, None, None, p, None, None, 4, 4, 1 << 28, F32, 0, None) == -2
    assert fwd(None, p, None, None, p, None, None, 4, 4, 4, F32, 0, None) == -1
    assert fwd(p, None, None, None, p, None, None, 4, 4, 4, F32, 0, None) == -1
    assert fwd(p, p, None, None, None, None, None, 4, 4, 4, F32, 0, None) == -1
    assert fwd(p + 2, p, None, None, p, None, None, 4, 4, 4, F32, 0, None) == -3
    assert fwd(p, p, p + 1, None, p, None, None, 4, 4, 4, BF16, 0, None) == -3
    assert fwd(None, None, None, None, None, None, None, 0, 4, 4, F32, 0, None) == 0  # no rows: nothing to do
    assert ws(65, 64, 1 << 16, F32) > 0 and ws(4, 64, 1 << 16, F32) > 0 and ws(4, 64, 1 << 10, F32) == 0
    assert fwd(p, p, None, None, p, None, None, 65, 64, 1 << 16, F32, 0, None) == -1  # a cut contraction without its scratch
    ok = dict(dy=p, x=p, q=None, e=None, w=p, z=p, dx=p, dw=p, db=p, ws=p, M=4, N=4, K=4, t=F16, act=2)
    back = lambda **k: bwd(*{**ok, **k}.values(), None)                               # noqa: E731
    assert back(t=3) == -4 and back(act=4) == -4 and back(M=-1) == -2 and back(N=1 << 31) == -2 and back(K=1 << 31) == -2
    assert back(M=1 << 20, K=1 << 20) == -2 and back(M=1 << 20, K=1 << 28) == -2 and back(N=1 << 20, K=1 << 20) == -2   # too many tiles of dx, of dw
    assert back(dy=None) == -1 and back(w=None) == -1 and back(ws=None) == -1
    assert back(z=None) == -1                                                         # an activation without z
    assert back(x=None) == -1 and back(q=p, e=p) == -1 and back(x=None, q=p) == -1    # neither x nor its 8-bit form; both; q without e
    assert back(dx=p + 1) == -3 and back(x=None, q=p + 4, e=p) == -3 and back(ws=p + 4) == -3
    assert back(dx=None, dw=None, db=None) == 0 and back(N=0) == 0                    # nothing to do
    assert bws(4, 4, 4, F16, 0, 1, 1, 0) == 0 and bws(4, 4, 4, F16, 2, 1, 1, 0) == 256 and bws(4, 4, 4, F16, 2, 0, 0, 1) == 16
    assert ws(0, 4, 4, F32) == 0 and ws(4, 4, 4, 9) == 0 and bws(-1, 4, 4, F32, 0, 1, 1, 1) == 0


def test_norm_and_pack_entries_refuse_bad_arguments(lib, p):
    fwd, bwd = lib.ursa_layer_norm_fwd, lib.ursa_layer_norm_bwd
    ok = dict(x=p, a=None, z=None, y=p, g=None, b=None, m=None, r=None, q=None, e=None, M=2, D=4, eps=1e-5, t=F32, pt=F32)
    call = lambda **k: fwd(*{**ok, **k}.values(), None)                               # noqa: E731
    assert call(t=3) == -4 and call(t=F32, pt=BF16) == -4 and call(t=BF16, pt=F16) == -4
    assert call(M=-1) == -2 and call(M=1 << 31) == -2 and call(D=1 << 28) == -2
    assert call(eps=-1.0) == -5 and call(eps=float('nan')) == -5
    assert call(x=None) == -1 and call(y=None) == -1 and call(a=p) == -1 and call(z=p) == -1 and call(m=p) == -1 and call(q=p) == -1
    assert call(x=p + 2) == -3 and call(g=p + 2) == -3 and call(q=p + 8, e=p) == -3
    assert call(x=None, M=0) == 0
    ok = dict(x=p, q=None, e=None, dy=p, dz=None, g=None, m=p, r=p, dx=p, dg=None, db=None, ws=None, M=2, D=4, t=F32, pt=F32)
    back = lambda **k: bwd(*{**ok, **k}.values(), None)                               # noqa: E731
    assert back(x=None) == -1 and back(q=p, e=p) == -1 and back(x=None, q=p) == -1 and back(dy=None) == -1 and back(m=None) == -1
    assert back(dg=p) == -1                                                           # a weight gradient without its scratch
    assert back(t=7) == -4 and back(D=-1) == -2 and back(dz=p + 1) == -3
    pack, unpack = lib.ursa_act8_pack, lib.ursa_act8_unpack
    assert pack(None, p, p, 2, 4, F32, None) == -1 and pack(p, p, p, 2, 4, 5, None) == -4 and pack(p, p, p, -2, 4, F32, None) == -2
    assert pack(p, p + 1, p, 2, 4, F32, None) == -3 and pack(None, None, None, 0, 4, F32, None) == 0
    assert unpack(p, None, p, 2, 4, F32, None) == -1 and unpack(p, p, p + 1, 2, 4, BF16, None) == -3


def test_wrappers_refuse_before_they_launch():
    from ursabench_amd import _native, act8
    k = _native.default_kernels()
    x, w = torch.zeros(4, 8), torch.zeros(6, 8)
    with pytest.raises(RuntimeError, match='no CPU path'):
        k.linear_act(x, w)
    with pytest.raises(RuntimeError, match='no CPU path'):
        k.layer_norm(x, eps=1e-5)
    with pytest.raises(RuntimeError, match='no CPU path'):
        act8.pack(x)
    with pytest.raises(ValueError, match='should be'):
        k.linear_act(x, torch.zeros(6, 9))
    with pytest.raises(ValueError, match='activation'):
        k.linear_act(x, w, activation='tanh')
    with pytest.raises(TypeError, match='float32, bfloat16 or float16'):
        k.linear_act(x.double(), w.double())
    with pytest.raises(ValueError, match='8-bit form'):
        k.linear_backward(x, x, w, q=x, e=x)


def test_calls_that_are_refused():
    from ursabench_amd.fused_linear import linear_act
    from ursabench_amd.fused_norm import add_layer_norm, layer_norm
    fc, ln, x = nn.Linear(8, 6), nn.LayerNorm(8), torch.randn(4, 8)
    with pytest.raises(ValueError, match='activation'):
        linear_act(fc, x, 'tanh')
    with pytest.raises(ValueError, match='residual'):
        linear_act(fc, x, None, torch.zeros(6))                      # a broadcast residual: expand it
    with pytest.raises(TypeError, match='nn.Linear'):
        linear_act(nn.Bilinear(8, 8, 6), x)
    with pytest.raises(TypeError, match='nn.LayerNorm'):
        layer_norm(nn.BatchNorm1d(8), x)
    with pytest.raises(TypeError, match='nn.LayerNorm'):
        add_layer_norm(nn.BatchNorm1d(8), (x, x))


def test_host_tensors_take_the_stock_ops():
    from ursabench_amd.fused_linear import linear_act
    from ursabench_amd.fused_norm import add_layer_norm, layer_norm
    torch.manual_seed(0)
    fc, ln, x, r = nn.Linear(8, 6), nn.LayerNorm(8), torch.randn(2, 4, 8), torch.randn(2, 4, 6)
    for name, f in ((None, lambda z: z), ('relu', F.relu), ('gelu', F.gelu), ('silu', F.silu)):
        for save8 in (False, True):
            assert torch.equal(linear_act(fc, x, name, save8=save8), f(fc(x)))
            assert torch.equal(linear_act(fc, x, name, r, save8=save8), f(fc(x)) + r)
    assert torch.equal(layer_norm(ln, x, save8=True), ln(x))
    z, y = add_layer_norm(ln, (x, 2 * x))
    assert torch.equal(z, x + 2 * x) and torch.equal(y, ln(z))


def test_models_keep_their_stock_layers_by_default():
    from ursabench_amd import fused_linear, models
    assert fused_linear.in_models() is False
    torch.manual_seed(0)
    net, x = models.MLP(20, 12, 3), torch.randn(5, 12)
    want = net.fc3(F.relu(net.fc2(F.relu(net.fc1(x)))))
    assert torch.equal(net(x), want)
    old = fused_linear.in_models(True)
    try:
        assert torch.equal(net(x), want)                              # host tensors: the same ops
    finally:
        fused_linear.in_models(old)
