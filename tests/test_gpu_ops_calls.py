"""Calls of the learning operators that their own sizes, masks and types do not reach: two captures, lazily negated tensors, saved-tensor hooks, ratios next to the
clipping border, rollouts one after the other."""
import math
import pickle

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_gpu_ops import DT, U, advantages64, check_loss, gen, linear_inputs, loss_inputs, mg, within


@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_policy_loss_backward_in_a_graph_of_its_own(dt):
    """the loss in one graph, its backward pass in another that is replayed several times behind one replay of the first: every replay gives the gradient of the
    factor that it finds, whatever the one before left and the caller did to it"""
    x, a, old, adv, ref, mask = loss_inputs(37, 700, DT[dt], 4)
    x = x.detach().clone().requires_grad_(True)
    scale = torch.ones((), device="cuda")
    make = lambda: mg().policy_loss(x, a, old, adv, mask=mask, ref_log_prob=ref, kl_coef=0.1, entropy_coef=0.01)[0]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        torch.autograd.grad(make(), [x], scale)
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    forward, backward = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(forward):
        loss = make()
    with torch.cuda.graph(backward, pool=forward.pool()):
        d, = torch.autograd.grad(loss, [x], scale, retain_graph=True)
    want = {f: torch.autograd.grad(make(), [x], torch.full((), f, device="cuda"))[0] for f in (1.0, 2.0)}
    for i in range(2):
        forward.replay()
        for f, spoil in ((1.0, False), (2.0, False), (1.0, False), (1.0, True), (2.0, True), (1.0, False)):
            scale.fill_(f)
            if spoil:
                d.fill_(7.0)
            backward.replay()
            torch.cuda.synchronize()
            assert torch.equal(d, want[f]), (i, f, spoil)


def test_a_tangent_of_the_incoming_gradient_is_refused():
    """(forward over reverse: the gradient's own tangent would be lost)"""
    import torch.autograd.forward_ad as fw
    x, a, old, adv, ref, mask = loss_inputs(40, 7, torch.float32, 3)
    x = x.contiguous().requires_grad_(True)
    w = torch.randn((5, 7), generator=gen(1), device="cuda", requires_grad=True)
    for y in (mg().linear(x, w, activation="tanh"), mg().policy_loss(x, a, old, adv)[0]):
        with fw.dual_level():
            g = fw.make_dual(torch.ones_like(y), torch.ones_like(y))
            with pytest.raises((RuntimeError, ValueError), match="forward-mode"):
                torch.autograd.grad(y, [x], g, retain_graph=True)
        torch.autograd.grad(y, [x], torch.ones_like(y))


def test_a_fake_tensor_beside_real_ones_is_refused():
    """(its address is 0: an optional argument would be taken for one that was not given)"""
    from torch._subclasses.fake_tensor import FakeTensorMode
    x, w, b, r, dy = linear_inputs(50, 24, 40, torch.float32, False, True, True, False, 5)
    l, a, old, adv, ref, mask = loss_inputs(40, 7, torch.float32, 3)
    with FakeTensorMode():
        fake = lambda t: torch.empty(t.shape, dtype=t.dtype, device="cuda")
        fb, fr, fref, fmask, fu = fake(b), fake(r), fake(ref), fake(mask), fake(ref)
    for call in (lambda: mg().linear(x, w, fb), lambda: mg().linear(x, w, residual=fr), lambda: mg().policy_loss(l, a, old, adv, mask=fmask),
                 lambda: mg().policy_loss(l, a, old, adv, ref_log_prob=fref), lambda: mg().sample_actions(l, fu)):
        with pytest.raises(ValueError, match="has no memory"):
            call()
