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


@pytest.mark.parametrize("how", ["wider_rows", "odd_wider_rows", "tokens_first", "one_image"])
@pytest.mark.parametrize("w,t,M", [(7, "bf16", 64), (7, "fp32", 32), (None, "fp32", 64), (None, "bf16", 48), (None, "bf16", 64)])
def test_a_projection_in_other_rows_takes_the_same_kernels(how, w, t, M):
    """a slice of wider rows, or one whose tokens come first, on the matrix-core kernels (which take one stride for k and v) as the packed
    projection itself: where the rotation's kernel is the same too, the same numbers in the same order, so equal outputs and gradients of
    qkv and the norm's weights"""
    H, N, t = 2, 197, TYPES[t]
    a = args(w, t, M=M, H=H, B=1 if how == "one_image" else 2)
    qkv, C3 = a["qkv"], 3 * H * M
    if how == "tokens_first":
        x = qkv.transpose(0, 1).contiguous().transpose(0, 1)
    else:
        wide = torch.zeros(qkv.shape[0], N, C3 + (5 if how == "odd_wider_rows" else 64), device="cuda", dtype=t)
        wide[..., :C3] = qkv
        x = wide[..., :C3]
    assert x.stride(1) != C3 or how == "one_image"
    dout = rnd(qkv.shape[0], N, H * M, seed=3, t=t)
    backend = None if M == 64 and w is None and t == torch.bfloat16 else "mfma"        # (None: the dense family)
    got = []
    for v in (qkv, x):
        leaves = [v.requires_grad_(), *(a[n].requires_grad_() for n in LEAVES[1:])]
        out = ops.vil_rotary_attention_qkv(**{**a, "qkv": v}, backend=backend)
        got.append((out.detach(), torch.autograd.grad(out, leaves, dout)))
    (want, wg), (out, g) = got
    if how == "odd_wider_rows":
        # rows that 16-byte loads do not fit take the element-wise rotation, which adds a row's squares in another order: rotated values may
        # round to the neighbouring number.  Either side is within the attention's bounds of the formulas (gpu_common: fp32 out 2e-5 +
        # 1e-4, gradients 1e-4 + 1e-3; 16 bits 2e-2 + 5e-2, 6 % of the rms + 5 %), so the two are within twice those of each other.
        low = t != torch.float32
        for x, y, grad in ((out, want, False), *((g[i], wg[i], True) for i in range(6))):
            x, y = x.double(), y.double()
            s = float(y.square().mean().sqrt()) if grad else 1.0
            lim = (0.06 * s if grad else 2e-2) + 5e-2 * y.abs() if low else (1e-4 * max(s, 1) if grad else 2e-5) + (1e-3 if grad else 1e-4) * y.abs()
            assert bool(((x - y).abs() <= 2 * lim).all())
        return
    assert torch.equal(out, want)
    for i in (0, 4, 5):
        assert torch.equal(g[i], wg[i]), LEAVES[i]
    for i in (1, 2, 3):                                          # (sums that may come in another order: as above)
        assert float((g[i] - wg[i]).abs().max()) <= 2.0 ** -10 * float(wg[i].abs().max()), LEAVES[i]


def test_rows_beside_a_sliced_projection_are_left_alone():
    a = args(7, torch.bfloat16)
    wide = rnd(2, 197, 400, seed=7, t=torch.bfloat16)
    keep = wide.clone()
    qkv = wide[..., 8:392].detach().requires_grad_()
    out = ops.vil_rotary_attention_qkv(**{**a, "qkv": qkv}, backend="mfma")
    g, = torch.autograd.grad(out, qkv, torch.ones_like(out))
    assert torch.equal(wide, keep) and g.shape == qkv.shape and bool(torch.isfinite(g).all())


@pytest.mark.parametrize("t", ["bf16", "fp32"])
@pytest.mark.parametrize("nx,ny,nglo,M", [(6, 9, 1, 32), (9, 6, 0, 48), (3, 14, 2, 64), (1, 7, 1, 32), (11, 10, 0, 64)])
def test_dense_attention_on_a_grid_that_is_not_square(nx, ny, nglo, M, t):
    """w None: all tokens attend to all, in the dense family (16 bits, 64 channels) and as one chunk of side max(nx, ny).  Bounds of the
    attention kernels' own tests, as in test_gpu_4_block.py."""
    from test_gpu_4_block import attention64
    H, t = 2, TYPES[t]
    a = args(None, t, nx=nx, ny=ny, nglo=nglo, H=H, M=M)
    for n in ("bias_table", "g2l_bias", "g2g_bias"):
        a[n] = None
    turn = {k: a[k] for k in ("positions", "inv_freq", "sections")}
    leaves = [a[n].requires_grad_() for n in ("qkv", "q_weight", "k_weight")]
    dout = rnd(2, nglo + nx * ny, H * M, seed=3, t=t)
    out = ops.vil_rotary_attention_qkv(**a)
    got = torch.autograd.grad(out, leaves, dout)
    d = [v.detach().double().cpu().requires_grad_() for v in leaves]
    ref = attention64(d[0], H, d[1], d[2], turn, M ** -0.5)
    want = torch.autograd.grad(ref, d, dout.double().cpu())
    low = t != torch.float32
    err = (out.detach().double().cpu() - ref.detach()).abs()
    assert bool((err <= (2e-2 + 5e-2 * ref.abs() if low else 2e-5 + 1e-4 * ref.abs())).all()), float(err.max())
    for x, y in zip(got, want):
        err, s = (x.double().cpu() - y).abs(), float(y.square().mean().sqrt())
        assert bool((err <= (0.06 * s + 5e-2 * y.abs() if low else 1e-4 * max(s, 1) + 1e-3 * y.abs())).all()), float(err.max() / s)
