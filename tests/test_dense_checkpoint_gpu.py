"""The dense blocks (K15, K16) under activation checkpointing, compiled callers and two threads: the plain call's bits."""
import threading

import pytest
import torch
import torch.nn as nn

pytestmark = pytest.mark.gpu
DEV = 'cuda'


def _block():
    from ursabench_amd.fused_linear import linear_act
    from ursabench_amd.fused_norm import add_layer_norm
    torch.manual_seed(0)
    ln, up, down = nn.LayerNorm(40, device=DEV), nn.Linear(40, 100, device=DEV), nn.Linear(100, 40, device=DEV)

    def f(x, save8=False):
        z, h = add_layer_norm(ln, (x, 2 * x), save8=save8)
        return linear_act(down, linear_act(up, h, 'gelu', save8=save8), None, z, save8=save8)

    return f, [*ln.parameters(), *up.parameters(), *down.parameters()], torch.randn(33, 40, device=DEV, requires_grad=True), torch.randn(33, 40, device=DEV)


@pytest.mark.parametrize('reentrant', [False, True])
@pytest.mark.parametrize('save8', [False, True])
def test_checkpointed_blocks(save8, reentrant):
    from torch.utils.checkpoint import checkpoint
    f, params, x, dy = _block()

    def grads(call):
        for t in (x, *params):
            t.grad = None
        h = call(call(x))
        h.backward(dy)
        return [h.detach()] + [t.grad for t in (x, *params)]

    want = grads(lambda v: f(v, save8))
    got = grads(lambda v: checkpoint(f, v, save8, use_reentrant=reentrant))
    assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_compiled_callers():
    f, params, x, dy = _block()
    g = torch.compile(f, backend='eager')
    want, got = (torch.autograd.grad(h(x), [x, *params], dy) for h in (f, g))
    assert torch.equal(f(x), g(x)) and all(torch.equal(a, b) for a, b in zip(want, got))


def test_two_threads_on_their_own_streams():
    f, params, x, dy = _block()
    want = torch.autograd.grad(f(x), [x, *params], dy)
    torch.cuda.synchronize()
    bad = []

    def work():
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            for _ in range(20):
                v = x.detach().requires_grad_()
                got = torch.autograd.grad(f(v), [v, *params], dy)
                s.synchronize()
                if not all(torch.equal(a, b) for a, b in zip(want, got)):
                    bad.append(1)

    threads = [threading.Thread(target=work) for _ in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad
