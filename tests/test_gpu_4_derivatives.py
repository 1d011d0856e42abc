"""GPU: the operators on q and k where a call is traced or a forward-mode level is open."""
import pytest
import torch
from torch.autograd import forward_ad

from vision_longformer_amd import rotary

pytestmark = pytest.mark.gpu


def qk(N, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    q, k, gq, gk = (torch.randn(2, N, h, 32, generator=g, device="cuda").to(torch.bfloat16) for h in (4, 2, 4, 2))
    return q, k, gq, gk


def turn(nx, ny):
    return dict(positions=rotary.grid_positions(nx, ny, device="cuda"), inv_freq=rotary.rotary_frequencies((8, 8), device="cuda"), sections=(8, 8))


@pytest.mark.parametrize("norm", [True, False])
def test_a_traced_call_gives_the_eager_results(norm):
    """on other values than those that it was traced with, and with gradients through it"""
    fn = rotary.vil_qk_norm_rope if norm else rotary.vil_rope
    q, k, gq, gk = qk(30)
    kw = turn(5, 6)
    traced = torch.jit.trace(lambda q, k: fn(q, k, **kw), (q, k), check_trace=False)
    q, k = (v.requires_grad_() for v in qk(30, 1)[:2])
    want, got = fn(q, k, **kw), traced(q, k)
    for a, b in zip((*want, *torch.autograd.grad(want, (q, k), (gq, gk))), (*got, *torch.autograd.grad(got, (q, k), (gq, gk)))):
        assert torch.equal(a, b)


@pytest.mark.parametrize("norm", [True, False])
def test_inside_a_forward_mode_level(norm):
    fn = rotary.vil_qk_norm_rope if norm else rotary.vil_rope
    q, k, _, _ = qk(30)
    kw = turn(5, 6)
    want = fn(q, k, **kw)
    with forward_ad.dual_level():
        for a, b in zip(fn(q, k, **kw), want):
            assert torch.equal(a, b)
        with pytest.raises(NotImplementedError):
            fn(forward_ad.make_dual(q, torch.ones_like(q)), k, **kw)
