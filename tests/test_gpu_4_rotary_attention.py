"""GPU: vil_rotary_attention_qkv (q and k normalised and rotated in front of the attention, one node) at the calls that
test_gpu_4_block.py does not make."""
import pytest
import torch

from vision_longformer_amd import ops, rotary

pytestmark = pytest.mark.gpu
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def rnd(*shape, seed=0, t=torch.float32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda").to(t)


def args(w, t, nx=14, ny=14, B=2, H=2, M=64, nglo=1):
    """a packed projection, biases, norm weights and the grid's rotation; w None: dense"""
    side = (4 * w - 1,) * 2 if w is not None else (2 * nx - 1, 2 * ny - 1)
    return dict(qkv=rnd(B, nglo + nx * ny, 3 * H * M, t=t), bias_table=rnd(side[0] * side[1], H, seed=4), g2l_bias=rnd(2, H, nglo, seed=5),
                g2g_bias=rnd(H, nglo, nglo, seed=6), q_weight=1 + 0.2 * rnd(M, seed=1), k_weight=1 + 0.2 * rnd(M, seed=2), nx=nx, ny=ny,
                w=w, nglo=nglo, num_heads=H, norm=True, **rotary.GridTurn(M).of(nx, ny, nglo, torch.device("cuda")))


LEAVES = ("qkv", "bias_table", "g2l_bias", "g2g_bias", "q_weight", "k_weight")


@pytest.mark.parametrize("w", [7, None])
def test_create_graph_gives_the_same_gradients_and_a_second_derivative_raises(w):
    a = args(w, torch.bfloat16)
    leaves = [a[n].requires_grad_() for n in LEAVES]
    dout = rnd(2, 197, 128, seed=3, t=torch.bfloat16)
    out = ops.vil_rotary_attention_qkv(**a)
    first = torch.autograd.grad(out, leaves, dout, retain_graph=True)
    again = torch.autograd.grad(out, leaves, dout, create_graph=True)
    for x, y, v in zip(first, again, leaves):
        # (bias gradients may add their 392 terms at most in another order: each way is within 392 u of the terms' magnitudes,
        # 392 of them, against a largest sum of sqrt(392) or more of them: 2 x 392 x 2^-24 x sqrt(392) < 2^-10)
        assert torch.equal(x, y) or float((x - y).abs().max()) <= 2.0 ** -10 * float(x.abs().max())
        with pytest.raises(RuntimeError):
            (y.float().square().sum() + v.float().square().sum()).backward(retain_graph=True)
