"""Soak tests of the kernels behind rotary positions, the q / k norm and the 8-bit activations, as test_gpu_2_stress.py's: 3000 launches of
each on fixed inputs, every output compared bit for bit with the first launch's on the device, beside a stream of large copies."""
import pytest
import torch

from test_gpu_2_stress import LAUNCHES, _soak
from vision_longformer_amd import _lib, act8, rotary

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    return torch.device("cuda:0")


def rnd(*shape, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda").to(torch.bfloat16)


@pytest.mark.parametrize("T,K,N", [(6400, 384, 1536), (12007, 96, 384), (9001, 192, 768)])
def test_soak_products_with_the_packed_form(dev, T, K, N):
    """fc1 with GELU and packing, then fc2's input gradient with the GELU's backward on what it packed (LDS-DMA rings, stores in inline
    assembly); the first launch against the separate passes"""
    L = _lib.lib()
    x, w1, b, dy, w2 = rnd(T, K), rnd(N, K, seed=1) * 0.1, rnd(N, seed=2), rnd(T, K, seed=3), rnd(K, N, seed=4) * 0.1
    a, again, dh = (torch.empty(T, N, dtype=torch.bfloat16, device=dev) for _ in range(3))
    codes, scales = torch.empty(T, N, dtype=torch.int8, device=dev), torch.empty(T, N // 32, dtype=torch.uint8, device=dev)

    def launch():
        _lib.launch(0, L.vil_gemm_gelu_act8_bf16, x.data_ptr(), w1.data_ptr(), b.data_ptr(), a.data_ptr(), codes.data_ptr(), scales.data_ptr(), T, K, N, K, N)
        _lib.launch(0, L.vil_gemm_dgelu_act8_bf16, dy.data_ptr(), w2.data_ptr(), codes.data_ptr(), scales.data_ptr(), dh.data_ptr(), again.data_ptr(), T, K, N, K, N)

    assert _soak(dev, launch, lambda: [a, codes, scales, dh, again]) == 0
    packed = act8.Act8(codes, scales, (T, N), torch.bfloat16)
    _, want = act8.vil_gelu_act8_bwd(packed, torch.ones_like(dh))
    assert torch.equal(again, want)


@pytest.mark.parametrize("rows,cols", [(4000, 384), (3001, 100)])
def test_soak_packing_and_gelu(dev, rows, cols):
    x, g = rnd(rows, cols), rnd(rows, cols, seed=1)
    out = []

    def launch():
        a, p = act8.vil_gelu_act8_fwd(x)
        out[:] = [a, p.scales.flatten()[:p.scales.numel() // 2 * 2], p.codes.flatten(), *act8.vil_gelu_act8_bwd(p, g), act8.vil_act8_unpack(p)]

    assert _soak(dev, launch, lambda: out) == 0


@pytest.mark.parametrize("B,N,H,M,sections", [(16, 785, 3, 64, (16, 16)), (8, 785, 3, 32, (8, 8)), (3, 183, 1, 48, (9, 8))])
def test_soak_rotation_and_norm(dev, B, N, H, M, sections):
    q, k, gq, gk = (rnd(B, N, H, M, seed=s) for s in range(4))
    w = torch.ones(M, device=dev)
    leaves = [t.requires_grad_() for t in (q, k, w)]
    kw = dict(positions=torch.arange(2 * N, device=dev, dtype=torch.int32).view(N, 2) % 97, inv_freq=rotary.rotary_frequencies(sections, device=dev),
              sections=sections)
    out = []

    def launch():
        y = rotary.vil_qk_norm_rope(q, k, w, w, **kw)
        out[:] = [*(v.detach() for v in y), *torch.autograd.grad(y, leaves, (gq, gk))]

    assert _soak(dev, launch, lambda: out, launches=LAUNCHES // 3) == 0
