"""GPU: the operators where the framework uses them -- q and k normalised and rotated in front of the attention kernels as one
node, the layers and the model with qk_norm / rotary / act8, and a run of all of them together against 64 bits."""
import math

import pytest
import torch

from vision_longformer_amd import engine, ops, rotary
from vision_longformer_amd.longformer2d import Long2DSCSelfAttention
from vision_longformer_amd.msvit import Attention, Mlp, MsViT

pytestmark = pytest.mark.gpu
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def rnd(*shape, seed=0, t=torch.float32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda").to(t)


def turned(x, cos, sin):
    R = cos.shape[-1]
    return torch.cat([x[..., :R] * cos - x[..., R:] * sin, x[..., R:] * cos + x[..., :R] * sin], -1)


def attention64(qkv, H, wq, wk, turn, scale):
    """plain fp64 attention over all tokens of qkv (B, N, 3C) with the norm (weights given) and the rotation (turn given)"""
    B, N, C3 = qkv.shape
    q, k, v = (t.unflatten(-1, (H, C3 // 3 // H)) for t in qkv.split(C3 // 3, -1))
    if wq is not None:
        q, k = (x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * w for x, w in ((q, wq), (k, wk)))
    if turn is not None:
        axis = [a for a, n in enumerate(turn["sections"]) for _ in range(n)]
        ang = (turn["positions"].double().cpu()[:, axis] * turn["inv_freq"].cpu())[None, :, None]
        q, k = turned(q, torch.cos(ang), torch.sin(ang)), turned(k, torch.cos(ang), torch.sin(ang))
    p = torch.softmax(torch.einsum("bihm,bjhm->bhij", q, k) * scale, -1)
    return torch.einsum("bhij,bjhm->bihm", p, v).flatten(2)


@pytest.mark.parametrize("t", list(TYPES))
@pytest.mark.parametrize("norm,rot", [(True, True), (False, True), (True, False)])
@pytest.mark.parametrize("w,H,M,n", [(7, 3, 32, 7), (7, 2, 64, 7), (None, 3, 64, 10), (None, 2, 32, 6), (7, 1, 48, 6)])
def test_attention_of_normalised_and_rotated_heads(w, H, M, n, norm, rot, t):
    """A grid of one chunk: attention over all tokens.  Bounds of the attention kernels' own tests (gpu_common): fp32 out 2e-5 + 1e-4,
    gradients 1e-4 + 1e-3 of their scale; 16-bit out 2e-2 + 5e-2, gradients 6 % of their rms + 5 %.  The rotated q and k are
    rounded once more, half a step (2^-9 of |q||k| sqrt-summed: under 2e-2 of these scores), inside them."""
    t, B, C = TYPES[t], 2, H * M
    qkv = rnd(B, 1 + n * n, 3 * C, t=t).requires_grad_()
    wq, wk = ((1 + 0.2 * rnd(M, seed=s)).requires_grad_() for s in (1, 2))
    turn = rotary.GridTurn(M).of(n, n, 1, qkv.device) if rot else None
    dout = rnd(B, 1 + n * n, C, seed=3, t=t)
    out = ops.vil_rotary_attention_qkv(qkv, None, None, None, nx=n, ny=n, nglo=1, num_heads=H, w=w, norm=norm,
                                       q_weight=wq if norm else None, k_weight=wk if norm else None, **(turn or {}))
    leaves = [qkv] + ([wq, wk] if norm else [])
    got = torch.autograd.grad(out, leaves, dout)
    ref_leaves = [v.detach().double().cpu().requires_grad_() for v in leaves]
    ref = attention64(ref_leaves[0], H, *(ref_leaves[1:] if norm else (None, None)), turn, M ** -0.5)
    want = torch.autograd.grad(ref, ref_leaves, dout.double().cpu())
    low = t != torch.float32
    err = (out.detach().double().cpu() - ref.detach()).abs()
    assert bool((err <= (2e-2 + 5e-2 * ref.abs() if low else 2e-5 + 1e-4 * ref.abs())).all()), float(err.max())
    for a, b in zip(got, want):
        err, s = (a.double().cpu() - b).abs(), float(b.square().mean().sqrt())
        assert bool((err <= (0.06 * s + 5e-2 * b.abs() if low else 1e-4 * max(s, 1) + 1e-3 * b.abs())).all()), float(err.max() / s)


@pytest.mark.parametrize("mode,exact,nx,ny,w", [(0, 0, 15, 14, 7), (0, 1, 9, 16, 4), (3, 0, 14, 14, 7), (-1, 0, 14, 21, 7), (0, -1, 10, 9, 4)])
def test_one_node_equals_its_parts(mode, exact, nx, ny, w):
    """vil_rotary_attention_qkv against vil_qk_norm_rope, a concatenation and vil_full_attention_qkv: the same kernels on the same
    numbers"""
    H, M, B, t = 2, 32, 2, torch.bfloat16
    C, N = H * M, 1 + nx * ny
    qkv = rnd(B, N, 3 * C, t=t).requires_grad_()
    table, g2l, g2g = rnd((4 * w - 1) ** 2, H, seed=4).requires_grad_(), rnd(2, H, 1, seed=5).requires_grad_(), rnd(H, 1, 1, seed=6).requires_grad_()
    wq, wk = ((1 + 0.2 * rnd(M, seed=s)).requires_grad_() for s in (1, 2))
    turn = rotary.GridTurn(M).of(nx, ny, 1, qkv.device)
    kw = dict(nx=nx, ny=ny, w=w, nglo=1, num_heads=H, mode=mode, exact=exact)
    dout = rnd(B, N, C, seed=3, t=t)
    leaves = (qkv, table, g2l, g2g, wq, wk)
    out = ops.vil_rotary_attention_qkv(qkv, table, g2l, g2g, q_weight=wq, k_weight=wk, norm=True, **turn, **kw)
    got = torch.autograd.grad(out, leaves, dout)
    q, k, v = (x.unflatten(-1, (H, M)) for x in qkv.split(C, -1))
    q, k = rotary.vil_qk_norm_rope(q, k, wq, wk, **turn)
    parts = ops.vil_full_attention_qkv(torch.cat([q, k, v], 2).flatten(2), table, g2l, g2g, **kw)
    assert torch.equal(out, parts)
    for a, b in zip(got, torch.autograd.grad(parts, leaves, dout)):
        assert torch.equal(a, b)


def test_dense_family_takes_it_and_refusals():
    H, M, nx, ny = 2, 64, 12, 10
    C, N = H * M, 1 + nx * ny
    qkv = rnd(2, N, 3 * C, t=torch.bfloat16)
    turn = rotary.GridTurn(M).of(nx, ny, 1, qkv.device)
    table = rnd((2 * nx - 1) * (2 * ny - 1), H)
    kw = dict(nx=nx, ny=ny, nglo=1, num_heads=H)
    out = ops.vil_rotary_attention_qkv(qkv, table, None, None, backend="dense", **turn, **kw)
    q, k, v = (x.unflatten(-1, (H, M)) for x in qkv.split(C, -1))
    q, k = rotary.vil_rope(q, k, **turn)
    assert torch.equal(out, ops.vil_dense_attention(torch.cat([q, k, v], 2).flatten(2), table, None, None, **kw))
    f = ops.vil_rotary_attention_qkv
    for bad in (dict(), dict(norm=True, nx=11), dict(q_weight=rnd(M), **turn), dict(norm=True, num_heads=5), dict(norm=True, w=7, nglo=0, nx=11, ny=11),
                dict(norm=True, w=7, exact=1, mode=2), dict(norm=True, nglo=5, nx=29, ny=4)):
        with pytest.raises(ValueError):
            f(qkv, None, None, None, **{**kw, **bad})
    with pytest.raises(RuntimeError):
        f(qkv.float(), None, None, None, backend="dense", norm=True, **kw)
    with pytest.raises(RuntimeError):
        f(qkv.cpu(), None, None, None, norm=True, **kw)


def test_layers_with_norm_and_rotation():
    """both attention layers under autocast: every parameter has a finite gradient; the rotation and the norm's weights matter"""
    for layer in (Long2DSCSelfAttention(96, num_heads=3, qkv_bias=True, w=7, sharew=True, nglo=1, rpe=True, qk_norm=True, rotary=True),
                  Attention(128, num_heads=2, qkv_bias=True, rpe=True, wx=14, wy=14, nglo=1, qk_norm=True, rotary=True)):
        layer = layer.cuda().train()
        x = rnd(2, 197, layer.proj.in_features).requires_grad_()
        with torch.autocast("cuda", dtype=torch.bfloat16):
            y = layer(x, 14, 14)
        y.float().square().mean().backward()
        for n, p in layer.named_parameters():
            assert p.grad is not None and p.grad.dtype == p.dtype and bool(torch.isfinite(p.grad).all()) and bool((p.grad != 0).any()), n
        with torch.no_grad(), torch.autocast("cuda", dtype=torch.bfloat16):
            again = layer(x, 14, 14)
            assert torch.equal(again, y)
            layer.q_norm.weight.mul_(2)
            assert not torch.equal(layer(x, 14, 14), y)
            layer.turn, keep = None, layer.turn
            assert not torch.equal(layer(x, 14, 14), again)
            layer.turn = keep
    with pytest.raises(ValueError):
        Long2DSCSelfAttention(96, num_heads=3, w=7, sharew=False, nglo=1, qk_norm=True)
    with pytest.raises(ValueError):
        Long2DSCSelfAttention(96, num_heads=3, w=7, sharew=True, nglo=0, rotary=True)
    dropping = Long2DSCSelfAttention(96, num_heads=3, w=7, sharew=True, nglo=1, rotary=True, attn_drop=0.1).cuda().train()
    with pytest.raises(RuntimeError):
        dropping(rnd(1, 197, 96), 14, 14)
    with pytest.raises(RuntimeError):
        Attention(128, num_heads=2, wx=14, wy=14, rotary=True)(torch.zeros(1, 197, 128), 14, 14)


def test_mlp_keeps_a_third_of_the_memory():
    """what a forward pass of the MLP block leaves allocated: x and h in 8 bits (5 C of 33 / 32 bytes a token) against x, h and
    gelu(h) in 16 bits (9 C of 2 bytes), measured with the output in both (2 C more).  Requested bytes: the allocator hands out a
    free block of up to 1 MiB more than asked for, by what was freed before, and counts that as allocated"""
    asked = lambda: torch.cuda.memory_stats()["requested_bytes.all.current"]
    T, C = 4096, 96
    held = {}
    for on in (False, True):
        mlp = Mlp(C, 4 * C, act8=on).cuda().to(torch.bfloat16)
        y = mlp(rnd(T, C, t=torch.bfloat16).requires_grad_())         # (workspaces, tuning)
        y.backward(torch.ones_like(y))
        del y
        torch.cuda.synchronize()
        x = rnd(T, C, t=torch.bfloat16).requires_grad_()
        before = asked()
        y = mlp(x)
        held[on] = asked() - before - y.numel() * 2
        del y
    assert held[True] <= 1.05 * T * 5 * C * 33 / 32 and held[False] >= T * 8 * C * 2


ARCH = "l1,h1,d32,n1,s1,g1,p4,f4,a0_l2,h2,d64,n2,s1,g1,p2,f4,a0_l3,h2,d128,n1,s0,g1,p2,f7,a0"


def test_model_with_everything_trains_as_its_parts_say():
    """One loss and its gradients of a small model with norms, rotation and 8-bit MLP blocks, under bf16 autocast, against the same
    model without act8: the forward differs by the rounding of gelu's place alone, the gradients by the 8-bit values' (2^e of 63.5 to
    127 a block: 0.5 / 63.5 of a block's largest at the most, 0.3 % of it rms) through a handful of blocks: 5 % of each
    gradient's norm holds both with a margin of 4, bf16's own 2^-9 sums included."""
    x = rnd(8, 3, 64, 64)
    grads, outs = [], []
    for on in (False, True):
        torch.manual_seed(0)
        m = MsViT(ARCH, img_size=64, num_classes=10, drop_path_rate=0.0, norm_embed=True, sharew=True, qk_norm=True, rotary=True, act8=on).cuda().train()
        with torch.autocast("cuda", dtype=torch.bfloat16):
            y = m(x)
        y.float().square().mean().backward()
        outs.append(y.detach().float())
        grads.append({n: p.grad.double() for n, p in m.named_parameters()})
    assert float((outs[0] - outs[1]).norm() / outs[0].norm()) < 0.02
    for n, a in grads[0].items():
        assert float((a - grads[1][n]).norm()) <= 0.05 * float(a.norm()) + 1e-7, (n, float((a - grads[1][n]).norm() / a.norm()))


def test_training_step_captured_and_replayed():
    """the captured step of a model with everything walks the eager step's trajectory (as the engine's own test, without the three)"""
    g = torch.Generator().manual_seed(5)
    xs = [torch.randn(8, 3, 64, 64, generator=g).cuda() for _ in range(4)]
    ts = [torch.softmax(torch.randn(8, 10, generator=g), -1).cuda() for _ in range(4)]

    def run(graphed):
        torch.manual_seed(0)
        m = MsViT(ARCH, img_size=64, num_classes=10, drop_path_rate=0.0, norm_embed=True, sharew=True, qk_norm=True, rotary=True, act8=True).cuda().train()
        opt = engine.MasterWeightAdamW(m, lr=1e-3, capturable=graphed)
        losses = []
        if graphed:
            sd, msd = {k: v.clone() for k, v in m.state_dict().items()}, [v.clone() for v in opt.master]
            step = engine.GraphedTrainStep(m, opt, xs[0], ts[0], warmup=2)
            with torch.no_grad():
                for k, v in m.state_dict().items():
                    v.copy_(sd[k])
                for v, w in zip(opt.master, msd):
                    v.copy_(w)
            opt.reset_state()
            for x, t in zip(xs, ts):
                losses.append(float(step(x, t)))
                torch.cuda.synchronize()
                xs[0].sum().item()                         # eager work between the replays
        else:
            for x, t in zip(xs, ts):
                losses.append(float(engine.train_step(m, opt, x, t)))
        return losses, torch.cat([p.detach().float().reshape(-1) for p in m.parameters()])

    (le, pe), (lg, pg) = run(False), run(True)
    # (the engine test's bounds: the two runs tune their products apart, and Adam's first steps move every weight by lr)
    assert max(abs(a - b) for a, b in zip(le, lg)) < 2e-2 and float((pe - pg).abs().max()) < 5e-3


def test_block_against_64_bits():
    """attention layer and MLP block in a row, as a model runs them (bf16 in, rounded once a step), against fp64 of the same formulas:
    out within 2e-2 + 5e-2 (the attention's bound), every gradient within 10 % of its norm: bf16 rounds some 20 tensors on the way,
    2^-9 each, and the 8-bit values add 0.3 % of each block's largest (1 % of a gradient's norm); 10 % is five times their sum."""
    B, n, H, M = 2, 7, 3, 32
    C, N = H * M, 1 + n * n
    torch.manual_seed(1)
    att = Long2DSCSelfAttention(C, num_heads=H, qkv_bias=True, w=7, sharew=True, nglo=1, rpe=False, qk_norm=True, rotary=True).cuda().to(torch.bfloat16)
    mlp = Mlp(C, 4 * C, act8=True).cuda().to(torch.bfloat16)
    with torch.no_grad():
        for p in [*att.parameters(), *mlp.parameters()]:
            if p.dim() == 2:
                p.normal_(0, p.shape[1] ** -0.5)
    x = rnd(B, N, C, t=torch.bfloat16).requires_grad_()
    dy = rnd(B, N, C, seed=2, t=torch.bfloat16)
    y = mlp(att(x, n, n))
    names = ["query.weight", "kv.weight", "proj.weight", "q_norm.weight", "k_norm.weight"]
    ap, mp = dict(att.named_parameters()), dict(mlp.named_parameters())
    leaves = [x] + [ap[k] for k in names] + [mp["fc1.weight"], mp["fc2.weight"]]
    got = torch.autograd.grad(y, leaves, dy)
    d = [v.detach().double().cpu().requires_grad_() for v in leaves]
    X, Q, KV, P, WQ, WK, F1, F2 = d
    b = lambda t: t.detach().double().cpu()
    qkv = torch.cat([X @ Q.t() + b(att.query.bias), X @ KV.t() + b(att.kv.bias)], -1)
    turn = rotary.GridTurn(M).of(n, n, 1, x.device)
    o = attention64(qkv, H, WQ, WK, turn, M ** -0.5) @ P.t() + b(att.proj.bias)
    ref = torch.nn.functional.gelu(o @ F1.t() + b(mlp.fc1.bias)) @ F2.t() + b(mlp.fc2.bias)
    want = torch.autograd.grad(ref, d, dy.double().cpu())
    err = (y.detach().double().cpu() - ref.detach()).abs()
    assert bool((err <= 2e-2 + 5e-2 * ref.abs()).all()), float(err.max())
    for i, (a, w) in enumerate(zip(got, want)):
        assert float((a.double().cpu() - w).norm()) <= 0.1 * float(w.norm()), (i, float((a.double().cpu() - w).norm() / w.norm()))


def test_layer_resumes_after_inference_and_copies():
    """an evaluation under inference_mode first, then training; a deepcopy trains too"""
    import copy
    layer = Attention(128, num_heads=2, rpe=False, wx=8, wy=8, nglo=1, rotary=True, qk_norm=True).cuda().to(torch.bfloat16)
    x = rnd(1, 65, 128, t=torch.bfloat16)
    with torch.inference_mode():
        y = layer(x, 8, 8)
    for m in (layer, copy.deepcopy(layer)):
        z = m(x, 8, 8)
        assert torch.equal(z, y)
        z.float().sum().backward()
        assert m.q_norm.weight.grad is not None and math.isfinite(float(m.q_norm.weight.grad.float().abs().sum()))
