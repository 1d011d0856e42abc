"""GPU: the operators on q and k where a call is traced or a forward-mode level is open."""
import pytest
import torch
from torch.autograd import forward_ad

from vision_longformer_amd import act8, ops, rotary

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


@pytest.mark.parametrize("op", ["gelu", "mlp", "window", "dense"])
def test_other_traced_nodes_give_the_eager_results(op):
    """on other values, with gradients through them: 8-bit GELU and MLP block, the attention node with a window and without"""
    g = torch.Generator(device="cuda").manual_seed(0)
    n = lambda *s: torch.randn(*s, generator=g, device="cuda").to(torch.bfloat16)
    if op in ("gelu", "mlp"):
        shape = (1100, 96)
        ws = [n(384, 96) / 10, n(384), n(96, 384) / 20, n(96)]
        fn = act8.vil_gelu_act8 if op == "gelu" else lambda x: act8.vil_mlp_act8(x, *ws)
    else:
        shape = (2, 197, 384)
        kw = rotary.GridTurn(64).of(14, 14, 1, torch.device("cuda"))
        fn = lambda x: ops.vil_rotary_attention_qkv(x, None, None, None, nx=14, ny=14, nglo=1, num_heads=2, w=7 if op == "window" else None, norm=True, **kw)
    traced = torch.jit.trace(fn, (n(*shape),), check_trace=False)
    x = n(*shape).requires_grad_()
    want, got = fn(x), traced(x)
    dy = n(*want.shape)
    assert torch.equal(got, want) and torch.equal(torch.autograd.grad(got, x, dy)[0], torch.autograd.grad(want, x, dy)[0])


@pytest.mark.parametrize("fn", [lambda x: act8.vil_act8_unpack(act8.vil_act8_pack(x)), lambda x: act8.vil_gelu_act8_fwd(x)[0]])
def test_calls_without_a_node_are_not_traced(fn):
    with pytest.raises(RuntimeError, match="no launch"):
        torch.jit.trace(fn, (torch.randn(4, 64, device="cuda"),), check_trace=False)
