"""Which calls the dense blocks (K15, K16) leave to the stock ops: modules whose call is more than their forward, and tensors that are
more than memory."""
import pytest
import torch
import torch.nn as nn
import torch.nn.functional as F

pytestmark = pytest.mark.gpu
DEV = 'cuda'


def _parts(dtype=torch.float32):
    from ursabench_amd.fused_linear import linear_act
    from ursabench_amd.fused_norm import add_layer_norm, layer_norm
    torch.manual_seed(0)
    fc, ln = nn.Linear(40, 24, device=DEV, dtype=dtype), nn.LayerNorm(40, device=DEV, dtype=dtype)
    with torch.no_grad():
        ln.weight.normal_(), ln.bias.normal_()
    x = torch.randn(9, 40, device=DEV).to(dtype)
    # name -> (module, f(x), the stock ops it stands for)
    return x, {'linear': (fc, lambda v, s=False: linear_act(fc, v, 'gelu', save8=s), lambda v: F.gelu(fc(v))),
               'norm': (ln, lambda v, s=False: layer_norm(ln, v, save8=s), lambda v: ln(v)),
               'add': (ln, lambda v, s=False: torch.cat(add_layer_norm(ln, (v, 2 * v), save8=s)), lambda v: (lambda z: torch.cat((z, ln(z))))(v + 2 * v))}


PARTS = ['linear', 'norm', 'add']


# ---- modules whose call is more than their forward ----------------------------------------------
@pytest.mark.parametrize('part', PARTS)
def test_global_module_hooks_are_called(part):
    from torch.nn.modules import module as m
    x, parts = _parts()
    mod, f, _ = parts[part]
    seen = []
    handles = [m.register_module_forward_pre_hook(lambda n, i: seen.append('pre') if n is mod else None),
               m.register_module_forward_hook(lambda n, i, o: seen.append('post') if n is mod else None),
               m.register_module_full_backward_pre_hook(lambda n, g: seen.append('bpre') if n is mod else None),
               m.register_module_full_backward_hook(lambda n, gi, go: seen.append('bpost') if n is mod else None)]
    try:
        f(x.clone().requires_grad_()).sum().backward()
    finally:
        for h in handles:
            h.remove()
    assert sorted(seen) == ['bpost', 'bpre', 'post', 'pre']


@pytest.mark.parametrize('part', PARTS)
def test_a_forward_set_on_the_instance_is_called(part):
    x, parts = _parts()
    mod, f, stock = parts[part]
    mod.forward = lambda v: 3 * type(mod).forward(mod, v)
    assert torch.equal(f(x), stock(x))
    del mod.forward
    assert not torch.equal(f(x), 3 * stock(x))


# ---- tensors that are more than memory ----------------------------------------------------------
@pytest.mark.parametrize('save8', [False, True])
@pytest.mark.parametrize('part', PARTS)
def test_function_transforms(part, save8):
    """torch.func: vmap, grad, jacrev, jvp, nested, and of constants inside a transform - the stock ops' results."""
    from torch.func import grad, hessian, jacrev, jvp, vjp, vmap
    x, parts = _parts()
    _, g, stock = parts[part]
    f = lambda v: g(v, save8)                                                                             # noqa: E731
    rows = x[:, None]
    assert torch.equal(vmap(f)(rows), vmap(stock)(rows))
    assert torch.equal(vmap(f, in_dims=1, out_dims=1)(x[:, :, None].transpose(1, 2)), vmap(stock, in_dims=1, out_dims=1)(x[:, :, None].transpose(1, 2)))
    for t in (grad, hessian):
        assert torch.equal(t(lambda v: f(v).sum())(x[:2]), t(lambda v: stock(v).sum())(x[:2]))
    assert torch.equal(jacrev(f)(x[:2]), jacrev(stock)(x[:2]))
    assert torch.equal(vjp(f, x)[1](stock(x))[0], vjp(stock, x)[1](stock(x))[0])
    for a, b in zip(jvp(f, (x,), (x.flip(0),)), jvp(stock, (x,), (x.flip(0),))):
        assert torch.equal(a, b)
    assert torch.equal(vmap(lambda v: v.sum() + f(x).sum())(x), vmap(lambda v: v.sum() + stock(x).sum())(x))


def test_an_ensemble_by_vmap_over_its_weights():
    from torch.func import functional_call, stack_module_state, vmap
    from ursabench_amd.fused_linear import linear_act
    from ursabench_amd.fused_norm import layer_norm

    class Net(nn.Module):
        def __init__(self):
            super().__init__()
            self.ln, self.fc = nn.LayerNorm(40), nn.Linear(40, 24)

        def forward(self, x, own):
            return linear_act(self.fc, layer_norm(self.ln, x), 'relu') if own else F.relu(self.fc(self.ln(x)))

    torch.manual_seed(0)
    nets = [Net().to(DEV) for _ in range(3)]
    params, _ = stack_module_state(nets)
    x = torch.randn(9, 40, device=DEV)
    got, want = (vmap(lambda p, own=own: functional_call(nets[0], p, (x, own)))(params) for own in (True, False))
    assert torch.equal(got, want)
    one = functional_call(nets[0], {k: v[1] for k, v in params.items()}, (x, True))      # without a transform: the launches
    assert torch.equal(one, nets[1](x, True))


@pytest.mark.parametrize('part', PARTS)
def test_forward_mode_tangents(part):
    import torch.autograd.forward_ad as fw
    x, parts = _parts()
    mod, f, stock = parts[part]
    for frozen in (True, False):
        mod.requires_grad_(not frozen)
        with fw.dual_level():
            a, b = (fw.unpack_dual(g(fw.make_dual(x, x.flip(0)))) for g in (f, stock))
            assert torch.equal(a.primal, b.primal) and torch.equal(a.tangent, b.tangent)
            assert fw.unpack_dual(f(x)).tangent is None


@pytest.mark.parametrize('part', PARTS)
def test_traced_and_faked_calls(part):
    """torch.jit.trace, make_fx and fake tensors see the stock ops."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.fx.experimental.proxy_tensor import make_fx
    x, parts = _parts()
    mod, f, stock = parts[part]
    mod.requires_grad_(False)
    other = x.flip(0) + 1
    traced = torch.jit.trace(lambda v: f(v), x, check_trace=False)
    assert torch.equal(traced(other), stock(other))
    assert torch.equal(make_fx(lambda v: f(v))(x)(other), stock(other))
    with FakeTensorMode(allow_non_fake_inputs=True) as mode:
        y = f(mode.from_tensor(x))
    assert y.shape == stock(x).shape and y.dtype == x.dtype and isinstance(y, torch._subclasses.FakeTensor)


@pytest.mark.parametrize('part', PARTS)
def test_a_dispatch_mode_sees_the_ops(part):
    from torch.utils.flop_counter import FlopCounterMode
    x, parts = _parts()
    _, f, stock = parts[part]
    with FlopCounterMode(display=False) as a:
        f(x)
    with FlopCounterMode(display=False) as b:
        stock(x)
    assert a.get_total_flops() == b.get_total_flops()


def test_a_tensor_subclass_decides_for_itself():
    from ursabench_amd.fused_linear import linear_act

    class Logged(torch.Tensor):
        seen = []

        @classmethod
        def __torch_function__(cls, func, types, args=(), kwargs=None):
            cls.seen.append(getattr(func, '__name__', str(func)))
            return super().__torch_function__(func, types, args, kwargs)

    x, parts = _parts()
    y = linear_act(parts['linear'][0], x.as_subclass(Logged), 'gelu')
    assert isinstance(y, Logged) and 'linear' in Logged.seen and torch.equal(y.as_subclass(torch.Tensor), parts['linear'][2](x))


@pytest.mark.parametrize('part', PARTS)
def test_batched_and_dual_gradients_are_refused(part):
    """Of a plain call's graph: the launches of the backward pass cannot take a wrapped gradient."""
    import torch.autograd.forward_ad as fw
    x, parts = _parts()
    _, f, _ = parts[part]
    x.requires_grad_()
    y = f(x)
    with pytest.raises(RuntimeError, match='batched'):
        torch.autograd.grad(y, x, torch.ones(3, *y.shape, device=DEV), is_grads_batched=True, retain_graph=True)
    with fw.dual_level(), pytest.raises(RuntimeError, match='dual'):
        torch.autograd.grad(y, x, fw.make_dual(torch.ones_like(y), torch.ones_like(y)), retain_graph=True)
    with fw.dual_level():
        a = torch.autograd.grad(y, x, torch.ones_like(y), retain_graph=True)[0]
    assert torch.equal(a, torch.autograd.grad(y, x, torch.ones_like(y))[0])


def test_8_bit_copies_of_such_tensors_are_refused():
    from torch.func import vmap
    from ursabench_amd import act8
    x, _ = _parts()
    with pytest.raises(ValueError, match='plain tensor'):
        vmap(lambda v: act8.unpack(act8.pack(v)))(x)
    with pytest.raises(ValueError, match='plain tensor'):
        torch.jit.trace(lambda v: act8.unpack(act8.pack(v)), x, check_trace=False)


def test_the_launches_are_back_afterwards():
    """What the tests above leave behind: a plain call takes the launches (their own bits, not the stock ops')."""
    from ursabench_amd import _native
    x, parts = _parts()
    calls, nodes = [], _native.nodes()
    fc, f, _ = parts['linear']
    y = nodes.linear_act(x, fc.weight, fc.bias, None, _native.ACTIVATIONS['gelu'], False)
    assert y is not None and torch.equal(f(x), y)
