"""GPU: activations in 8 bits (csrc/vil_act8.hip): the packed form against its definition bit for bit, the GELU around it against
64 bits, the MLP block built from it against the same arithmetic.

Tolerances, from the arithmetic.  Packing is exact but for the rounding to the code, which both sides do alike: codes, scales and
unpacked values are equal.  GELU, 16-bit: half a step of the type plus 2^-17 relative of cdf (the polynomial's 5.2e-6) and 2^-22 for
the evaluation; fp32: half a step plus 2^-20 relative of the tail Phi(-|x|) (4e-7 with the evaluation), 2^-22 of the rest, and
x^2 2^-24 relative for the exponential's argument."""
import math

import pytest
import torch

from vision_longformer_amd import _lib, act8

pytestmark = pytest.mark.gpu
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def half_step(t, ref):
    f = torch.finfo(t)
    return torch.clamp(ref.abs() * (f.eps / 2), min=f.tiny * f.eps / 2)


def packed_by_definition(x):
    """(codes, scales, values) of x (T, D), block by block on the CPU in 64 bits"""
    t, x = x.dtype, x.detach().cpu().double()
    T, D = x.shape
    nb = -(-D // 32)
    codes, scales, values = torch.zeros(T, D, dtype=torch.int8), torch.zeros(T, nb, dtype=torch.uint8), torch.zeros(T, D, dtype=torch.float64)
    top = 10 if t == torch.float16 else 122
    for i in range(nb):
        v = x[:, 32 * i:32 * i + 32]
        m = v.abs().amax(1)
        bad = ~torch.isfinite(v).all(1)
        _, e = torch.frexp(torch.where(bad, torch.ones_like(m), m) / 127)         # m / 127 = f 2^e, f in [1/2, 1)
        e = torch.where(torch.ldexp(torch.tensor(127.0, dtype=torch.float64), e - 1) >= m, e - 1, e).clamp(min=-126)
        e = torch.where(m == 0, torch.full_like(e, -126), e)
        c = torch.round(v / torch.exp2(e.double())[:, None])
        c = torch.where((e == top)[:, None], c.clamp(-63, 63), c)
        c[bad] = 0
        codes[:, 32 * i:32 * i + 32] = c.to(torch.int8)
        scales[:, i] = torch.where(bad, torch.full_like(e, 255), e + 127).to(torch.uint8)
        w = c * torch.exp2(e.double())[:, None]
        w[bad] = float("nan")
        values[:, 32 * i:32 * i + 32] = w
    return codes, scales, values


def data(T, D, t, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    spread = torch.exp(torch.randn(D, generator=g, device="cuda"))
    return (torch.randn(T, D, generator=g, device="cuda") * spread).to(t)


SHAPES = [(1, 1), (1, 31), (1, 32), (2, 33), (5, 7), (3, 64), (7, 100), (64, 96), (37, 111), (19, 384), (300, 40), (130, 1000), (2, 2050)]


@pytest.mark.parametrize("t", list(TYPES))
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "%dx%d" % s)
def test_pack_and_unpack(shape, t):
    x = data(*shape, TYPES[t])
    p = act8.vil_act8_pack(x)
    codes, scales, values = packed_by_definition(x)
    assert torch.equal(p.scales.cpu(), scales) and torch.equal(p.codes.cpu(), codes)
    for out in TYPES.values():
        assert torch.equal(act8.vil_act8_unpack(p, out).cpu(), values.to(out))
    assert act8.vil_act8_unpack(p).dtype == x.dtype


@pytest.mark.parametrize("t", list(TYPES))
def test_pack_at_the_edges_of_the_type(t):
    """zeros, signed zeros, the smallest and the largest numbers, ties, values just over 127 steps, one non-finite value"""
    t = TYPES[t]
    f = torch.finfo(t)
    x = torch.zeros(12, 64, dtype=t, device="cuda")
    x[1, 0], x[1, 40] = f.max, f.min
    x[2, :3] = torch.tensor([f.max, f.max / 2, -f.max], dtype=t)
    x[3, 5], x[3, 50] = f.tiny, -f.tiny * f.eps                       # smallest normal, smallest subnormal
    x[4, :8] = torch.tensor([127, 0.5, 1.5, 2.5, -0.5, -1.5, 63.5, 126.5], dtype=t)
    x[5, :8] = torch.tensor([127.5, 1, 3, 5, -1, -3, 63, 127], dtype=t)       # steps of 2: odd numbers are ties
    x[6, :4] = torch.tensor([128, -128, 0.99, 1.01], dtype=t)
    x[7, 3], x[7, 33] = float("nan"), 1.0
    x[8, 31], x[8, 32] = float("inf"), 2.0
    x[9, 63] = float("-inf")
    x[10] = torch.linspace(-3, 3, 64).to(t)
    x[11, 0] = -0.0
    codes, scales, values = packed_by_definition(x)
    p = act8.vil_act8_pack(x)
    assert torch.equal(p.scales.cpu(), scales) and torch.equal(p.codes.cpu(), codes)
    y = act8.vil_act8_unpack(p)
    assert torch.equal(y.cpu().nan_to_num(7.0), values.to(t).nan_to_num(7.0)) and torch.equal(y.isnan().cpu(), values.isnan())
    rows = torch.tensor([i for i in range(12) if i not in (7, 8, 9)])
    assert bool(torch.isfinite(y[rows]).all())
    assert bool(y[7, :32].isnan().all()) and y[7, 33] == 1 and bool(y[8, :32].isnan().all()) and y[8, 32] == 2
    # the GELU around it: finite rows stay finite, marked blocks reach the gradient
    a, h8 = act8.vil_gelu_act8_fwd(x)
    assert torch.equal(h8.codes, p.codes) and torch.equal(h8.scales, p.scales)
    assert bool(torch.isfinite(a[rows]).all()) and a[8, 31] == float("inf") and bool(a[7, 3].isnan())
    dh, again = act8.vil_gelu_act8_bwd(h8, torch.ones_like(x))
    assert bool(torch.isfinite(dh[rows]).all()) and bool(dh[7, :32].isnan().all()) and bool(torch.isfinite(dh[7, 32:]).all())
    assert bool(torch.isfinite(again[rows]).all())


def gelu64(x):
    """gelu, gelu' and the tail Phi(-|x|) in fp64"""
    tail = 0.5 * torch.special.erfc(x.abs() * math.sqrt(0.5))
    cdf = torch.where(x < 0, tail, 1 - tail)
    pdf = torch.exp(-x * x / 2) / math.sqrt(2 * math.pi)
    return x * cdf, cdf + x * pdf, tail, cdf, pdf


def gelu_tolerance(x, t):
    """what fp32 adds to cdf and pdf before the result is rounded"""
    _, _, tail, cdf, pdf = gelu64(x)
    fit = 2.0 ** -20 if t == torch.float32 else 2.0 ** -17
    arg = x * x * 2.0 ** -24
    return tail * (fit + arg) + 2.0 ** -22 * cdf, pdf * (arg + 2.0 ** -22)


def check(name, got, ref, tol, t):
    lim = half_step(t, ref) * (1 + 2.0 ** -10) + tol
    err = (got.double() - ref).abs()
    assert got.shape == ref.shape and got.dtype == t and bool((err <= lim).all()), f"{name}: {float((err / lim).max()):.3f} of the bound"


@pytest.mark.parametrize("t", list(TYPES))
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "%dx%d" % s)
def test_gelu_both_ways(shape, t):
    t = TYPES[t]
    h, da = data(*shape, t) * 2, data(*shape, t, 1)
    a, h8 = act8.vil_gelu_act8_fwd(h)
    p = act8.vil_act8_pack(h)
    assert torch.equal(h8.codes, p.codes) and torch.equal(h8.scales, p.scales)
    x = h.double()
    check("a", a, gelu64(x)[0], x.abs() * gelu_tolerance(x, t)[0], t)
    v = act8.vil_act8_unpack(p, torch.float32).double()
    act, slope, _, _, _ = gelu64(v)
    c, d = gelu_tolerance(v, t)
    dh, again = act8.vil_gelu_act8_bwd(h8, da)
    check("dh", dh, da.double() * slope, da.double().abs() * (c + v.abs() * d + 2.0 ** -22 * (slope.abs() + v.abs() * gelu64(v)[4])), t)
    check("again", again, act, v.abs() * c, t)
    alone, none = act8.vil_gelu_act8_bwd(h8, da, want_act=False)
    assert none is None and torch.equal(alone, dh)
    leaf = h.detach().requires_grad_()
    y = act8.vil_gelu_act8(leaf)
    assert torch.equal(y, a) and torch.equal(torch.autograd.grad(y, leaf, da)[0], dh)


def test_gelu_over_the_whole_line():
    """every 16-bit number: no infinity, no NaN from a finite one, the sign and the limits right"""
    for t in (torch.bfloat16, torch.float16):
        x = torch.arange(-2 ** 15, 2 ** 15, device="cuda", dtype=torch.int32).to(torch.int16).view(t)
        x = x[torch.isfinite(x)].view(-1, 1)                         # (a block to itself: packed to within 1 / 127)
        a, h8 = act8.vil_gelu_act8_fwd(x)
        xd = x.double()
        check("a", a, gelu64(xd)[0], xd.abs() * gelu_tolerance(xd, t)[0], t)
        v = act8.vil_act8_unpack(h8, torch.float32).double()
        # half a step of a value alone in its block, |x| > 63.5 steps; at the top exponent the last code is 63: under one step
        # of |x| >= 63 steps
        top = h8.scales == (137 if t == torch.float16 else 249)
        assert bool(((v - xd).abs() <= xd.abs() / torch.where(top, 63.0, 127.0) + 2.0 ** -126).all())
        dh, _ = act8.vil_gelu_act8_bwd(h8, torch.ones_like(x))
        assert bool(torch.isfinite(dh).all()) and float(dh.max()) < 1.2 and float(dh.min()) > -0.2


def test_gradient_against_differences():
    """the gradient is the GELU's slope at the packed value: against central differences of the fp32 forward at that value (h = 2^-7:
    h^2 / 6 times a third derivative under 1 is 1e-5, rounding 2^-23 |a| 2^7 is 6e-5 for |a| < 4)"""
    h = torch.linspace(-4, 4, 512, device="cuda").view(16, 32)
    v = act8.vil_act8_unpack(act8.vil_act8_pack(h))
    up, down = (act8.vil_gelu_act8_fwd(v + s * 2.0 ** -7)[0] for s in (1, -1))
    leaf = h.detach().requires_grad_()
    d, = torch.autograd.grad(act8.vil_gelu_act8(leaf).sum(), leaf)
    assert float((d - (up - down) * 2.0 ** 6).abs().max()) < 1e-4


@pytest.mark.parametrize("how", ["row_stride", "odd_offset", "transposed", "three_axes", "expanded", "odd_row_stride"])
def test_strides_and_alignment(how):
    t = torch.bfloat16
    n = lambda *s: data(math.prod(s[:-1]), s[-1], t).view(*s)
    x = {"row_stride": lambda: n(40, 200)[:, 40:136], "odd_offset": lambda: n(1, 40 * 96 + 1)[0, 1:].view(40, 96),
         "transposed": lambda: n(96, 40).t(), "three_axes": lambda: n(5, 9, 96)[:, 1:], "expanded": lambda: n(1, 96).expand(40, 96),
         "odd_row_stride": lambda: n(40, 101)[:, 3:99]}[how]()
    g = data(*x.reshape(-1, 96).shape, t, 5).view(x.shape)
    g = g.transpose(0, 1).contiguous().transpose(0, 1)
    xc, gc = x.contiguous(), g.contiguous()
    p, q = act8.vil_act8_pack(x), act8.vil_act8_pack(xc)
    assert torch.equal(p.codes, q.codes) and torch.equal(p.scales, q.scales) and p.shape == x.shape
    a, h8 = act8.vil_gelu_act8_fwd(x)
    b, k8 = act8.vil_gelu_act8_fwd(xc)
    assert torch.equal(a, b) and torch.equal(h8.codes, k8.codes)
    for u, v in zip(act8.vil_gelu_act8_bwd(h8, g), act8.vil_gelu_act8_bwd(k8, gc)):
        assert torch.equal(u, v) and u.shape == x.shape


@pytest.mark.parametrize("shape", [(0, 64), (4, 0), (0, 0), (2, 0, 64)])
def test_empty(shape):
    x = torch.zeros(*shape, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    assert act8.vil_act8_unpack(act8.vil_act8_pack(x)).shape == x.shape
    y = act8.vil_gelu_act8(x)
    assert torch.autograd.grad(y, x, torch.ones_like(y))[0].shape == x.shape


def mlp_args(T, C, D, t, bias=True, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=g, device="cuda")
    return [v.to(t).requires_grad_() if v is not None else None for v in
            (n(3, T, C), n(D, C) / C ** 0.5, n(D) * 0.1 if bias else None, n(C, D) / D ** 0.5, n(C) * 0.1 if bias else None)]


@pytest.mark.parametrize("t,T,C,D,bias", [("bf16", 700, 96, 384, True), ("bf16", 50, 48, 192, True), ("bf16", 400, 384, 1536, True),
                                          ("fp16", 65, 96, 384, True), ("fp32", 65, 40, 100, True), ("bf16", 65, 64, 256, False)])
def test_mlp_forward_is_the_plain_one_and_gradients_are_those_at_the_packed_values(t, T, C, D, bias):
    """The forward equals the uncompressed block's arithmetic to the products' rounding; the gradients equal fp64 gradients taken
    at the packed x and h.  Rounded on the way: da, dh and a (half a step each), the products (half a step, fp32 sums): 4 half steps
    of the type, relative to each gradient's scale, and the GEMM's sum of D, C or 3T terms in fp32: 2^-24 sqrt of that, x 8.  Entries
    scatter with the rounding of their terms: 4 half steps x 6 sigma / sqrt of nothing: bound 12 half steps of the rms."""
    t = TYPES[t]
    x, w1, b1, w2, b2 = args = mlp_args(T, C, D, t, bias)
    dy = data(3 * T, C, t, 7).view(3, T, C)
    y = act8.vil_mlp_act8(*args)
    leaves = [v for v in args if v is not None]
    grads = torch.autograd.grad(y, leaves, dy)
    d = lambda v: v.detach().double().cpu() if v is not None else None
    X, W1, B1, W2, B2, DY = (d(v) for v in (x, w1, b1, w2, b2, dy))
    h = torch.nn.functional.linear(X, W1, B1)
    want = torch.nn.functional.linear(gelu64(h)[0], W2, B2)
    eps = torch.finfo(t).eps / 2

    def near(name, got, ref, steps=12):
        got = d(got)
        e, s = (got - ref).square().mean().sqrt(), ref.square().mean().sqrt()
        assert float(e) <= steps * max(eps, 2.0 ** -22) * float(s), (name, float(e / s))

    near("y", y, want)
    # the values that the backward sees: the packed x exactly; h as the device's product rounds it, packed
    x8 = d(act8.vil_act8_unpack(act8.vil_act8_pack(x))).view(-1, C)
    hdev = act8._linear(x.detach().reshape(-1, C), w1.detach(), b1.detach() if bias else None)
    h8 = d(act8.vil_act8_unpack(act8.vil_act8_pack(hdev), torch.float32))
    act, slope, _, _, _ = gelu64(h8)
    g = DY.reshape(-1, C)
    dh = (g @ W2) * slope
    ref = [(dh @ W1).view(3, T, C), dh.t() @ x8, dh.sum(0), g.t() @ act, g.sum(0)]
    if not bias:
        ref = [ref[0], ref[1], ref[3]]
    for i, (a, b) in enumerate(zip(grads, ref)):
        near("grad %d" % i, a, b)


def test_mlp_frozen_parameters_autocast_and_refusals():
    x, w1, b1, w2, b2 = mlp_args(40, 64, 256, torch.float32)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        y = act8.vil_mlp_act8(x, w1, b1, w2, b2)
    assert y.dtype == torch.bfloat16
    grads = torch.autograd.grad(y, (x, w1, b1, w2, b2), torch.ones_like(y))
    assert all(g.dtype == torch.float32 and bool(torch.isfinite(g).all()) for g in grads)
    x, w1, b1, w2, b2 = mlp_args(40, 64, 256, torch.bfloat16)
    for on in range(5):
        args = [v.detach().requires_grad_(i == on) for i, v in enumerate((x, w1, b1, w2, b2))]
        y = act8.vil_mlp_act8(*args)
        full = act8.vil_mlp_act8(*[v.detach().requires_grad_() for v in args])
        assert torch.equal(y, full)
        alone, = torch.autograd.grad(y, args[on], torch.ones_like(y))
        assert alone.shape == args[on].shape and bool(torch.isfinite(alone).all())
    with pytest.raises(ValueError):
        act8.vil_mlp_act8(x, w1, b1, w2[:, :-8], b2)
    with pytest.raises(TypeError):
        act8.vil_mlp_act8(x, w1.float(), b1, w2, b2)


def test_captured_and_replayed_and_other_stream():
    h, da = data(197, 384, torch.bfloat16), data(197, 384, torch.bfloat16, 1)

    def step(v):
        leaf = v[0].detach().requires_grad_()
        y = act8.vil_gelu_act8(leaf)
        return [y.detach(), *torch.autograd.grad(y, leaf, v[1]), act8.vil_act8_unpack(act8.vil_act8_pack(v[0]))]

    first = step((h, da))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = step((h, da))
    s.synchronize()
    for a, b in zip(first, other):
        assert torch.equal(a, b)
    torch.cuda.current_stream().wait_stream(s)
    held = (h.clone(), da.clone())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(held)
    for turn in range(4):
        held[0].copy_(data(197, 384, torch.bfloat16, 20 + turn))
        held[1].copy_(data(197, 384, torch.bfloat16, 30 + turn))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, step(held)):
            assert torch.equal(a, b)


def test_row_stride_past_32_bits_of_offset():
    buf = torch.zeros(40000, 60000, device="cuda", dtype=torch.bfloat16)
    x = data(40000, 96, torch.bfloat16)
    buf[:, 8:104] = x
    p, q = act8.vil_act8_pack(buf[:, 8:104]), act8.vil_act8_pack(x)
    assert torch.equal(p.codes, q.codes) and torch.equal(p.scales, q.scales)


@pytest.mark.parametrize("shape", [(0, 64), (2, 0, 64)])
def test_mlp_of_an_empty_batch(shape):
    _, w1, b1, w2, b2 = mlp_args(4, 64, 256, torch.bfloat16)
    x = torch.zeros(*shape, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    y = act8.vil_mlp_act8(x, w1, b1, w2, b2)
    assert y.shape == (*shape[:-1], 64)
    for g, v in zip(torch.autograd.grad(y, (x, w1, b1, w2, b2), torch.ones_like(y)), (x, w1, b1, w2, b2)):
        assert g.shape == v.shape and bool((g == 0).all())


def test_mlp_of_a_vector_and_of_a_broadcast_gradient():
    x, w1, b1, w2, b2 = mlp_args(40, 64, 256, torch.bfloat16)
    y = act8.vil_mlp_act8(x, w1, b1, w2, b2)
    one = torch.autograd.grad(y, (x, w1, b1, w2, b2), torch.ones_like(y))
    y = act8.vil_mlp_act8(x, w1, b1, w2, b2)
    for a, b in zip(one, torch.autograd.grad(y, (x, w1, b1, w2, b2), torch.ones((), device="cuda", dtype=y.dtype).expand_as(y))):
        # (a broadcast gradient takes the products of another kernel: 12 half steps of the rms, as above)
        assert float((a - b).float().norm()) <= 12 * 2.0 ** -8 * float(a.float().norm())
    v = x[0, 0].detach().requires_grad_()
    y = act8.vil_mlp_act8(v, w1, b1, w2, b2)
    assert y.shape == (64,) and torch.autograd.grad(y, v, torch.ones_like(y))[0].shape == v.shape


def test_non_finite_gradients_stay_visible():
    """fp16 training: an infinite or NaN incoming gradient, or an overflowed pre-activation, is not finite afterwards either"""
    h = data(4, 64, torch.float16)
    da = torch.ones_like(h)
    da[1, 3], da[2, 5] = float("inf"), float("nan")
    h[3, 7] = float("inf")
    _, h8 = act8.vil_gelu_act8_fwd(h)
    dh, again = act8.vil_gelu_act8_bwd(h8, da)
    bad = ~torch.isfinite(dh)
    assert bool(bad[1, 3]) and bool(bad[2, 5]) and bool(bad[3, :32].all()) and int(bad.sum()) == 34 and bool(again[3, :32].isnan().all())


def test_rows_behind_and_channels_beside_are_left_alone():
    buf = torch.zeros(6, 200, device="cuda", dtype=torch.bfloat16)
    buf[:4, 16:113] = data(4, 97, torch.bfloat16)
    keep = buf.clone()
    x = buf[:4, 16:113]
    a, h8 = act8.vil_gelu_act8_fwd(x)
    p = act8.vil_act8_pack(x)
    assert torch.equal(buf, keep) and torch.equal(p.codes, act8.vil_act8_pack(x.contiguous()).codes) and torch.equal(h8.codes, p.codes)


@pytest.mark.parametrize("T", [1, 127, 1100, 2177])
@pytest.mark.parametrize("K,N", [(384, 1536), (96, 384), (192, 768), (416, 128)])
@pytest.mark.parametrize("entry", ["fwd", "bwd"])
def test_products_with_the_packed_form_in_their_epilogue(entry, K, N, T):
    """fc1 with GELU and packing, fc2's input gradient with the GELU's backward.  The operands are small multiples of a power of two,
    so that a sum of the products is exact in 32 bits (below 2^24 units) in any order: codes and scales are those of the product
    rounded to bf16, a and dh are off by the GELU's tolerances alone.  One row has a NaN, one an infinity."""
    L, t = _lib.lib(), torch.bfloat16
    gen = torch.Generator(device="cuda").manual_seed(T + K)
    whole = lambda m, *size: torch.randint(-m, m + 1, size, generator=gen, device="cuda").float()
    x, w, b = whole(8, T, K).to(t), (whole(8, N, K) / 512).to(t), (whole(200, N) / 512).to(t)
    if T > 100:
        x[3, 5], x[T - 1, 7] = float("nan"), float("inf")
    codes = torch.full((T + 1, N), 77, device="cuda", dtype=torch.int8)
    scales = torch.full((T + 1, N // 32), 77, device="cuda", dtype=torch.uint8)
    a = torch.full((T + 1, N + 8), 7.0, device="cuda", dtype=t)                        # a row stride of its own, a row behind the last
    if entry == "fwd":
        _lib.launch(0, L.vil_gemm_gelu_act8_bf16, x.data_ptr(), w.data_ptr(), b.data_ptr(), a.data_ptr(), codes.data_ptr(), scales.data_ptr(), T, K, N, K, N + 8)
        h = (x.cpu().double() @ w.cpu().double().t() + b.cpu().double()).to(t)
        want = act8.vil_act8_pack(h.cuda())
        assert torch.equal(scales[:T], want.scales) and torch.equal(codes[:T], want.codes)
        assert bool((scales[T] == 77).all()) and bool((codes[T] == 77).all())
        hd = h.cuda().double()
        fine = torch.isfinite(hd).all(1)
        assert int(fine.sum()) >= T - 2
        hf = hd[fine]
        check("a", a[:T, :N][fine], gelu64(hf)[0], hf.abs() * gelu_tolerance(hf, t)[0], t)
    else:
        w = w.t().contiguous()
        h8 = act8.vil_act8_pack(2 * data(T, N, t, 4))
        dh = torch.full((T + 1, N + 8), 7.0, device="cuda", dtype=t)
        _lib.launch(0, L.vil_gemm_dgelu_act8_bf16, x.data_ptr(), w.data_ptr(), h8.codes.data_ptr(), h8.scales.data_ptr(), dh.data_ptr(),
                    a.data_ptr(), T, K, N, K, N + 8)
        v = act8.vil_act8_unpack(h8, torch.float32).double()
        act, slope, _, _, pdf = gelu64(v)
        g = (x.cpu().double() @ w.cpu().double()).cuda()
        fine = torch.isfinite(g).all(1)
        assert int(fine.sum()) >= T - 2
        c, d = gelu_tolerance(v, t)
        check("a", a[:T, :N], act, v.abs() * c, t)
        check("dh", dh[:T, :N][fine], (g * slope)[fine], (g.abs() * (c + v.abs() * d + 2.0 ** -22 * (slope.abs() + v.abs() * pdf)))[fine], t)
        if T > 100:
            assert bool(dh[3, :N].isnan().all()) and not bool(torch.isfinite(dh[T - 1, :N]).any())
        assert bool((dh[T] == 7).all()) and bool((dh[:, N:] == 7).all())
    if T > 100 and entry == "fwd":
        assert bool(a[3, :N].isnan().all()) and bool((scales[[3, T - 1]] == 255).all())
    assert bool((a[T] == 7).all()) and bool((a[:, N:] == 7).all())


@pytest.mark.parametrize("C", [96, 384])
def test_mlp_of_the_fused_products_equals_that_of_the_separate_ones(C, monkeypatch):
    """vil_mlp_act8 at a size whose products take the fused epilogues against the same block without them: y, and each gradient, to
    12 half steps of the rms (as above: h and da are rounded in other places)"""
    args = mlp_args(1000, C, 4 * C, torch.bfloat16, seed=3)
    dy = data(3000, C, torch.bfloat16, 7).view(3, 1000, C)
    out = []
    for least in (1024, 1 << 40):
        monkeypatch.setattr(act8, "_FUSE_MIN_T", least)
        y = act8.vil_mlp_act8(*args)
        out.append([y.detach(), *torch.autograd.grad(y, args, dy)])
    for i, (a, b) in enumerate(zip(*out)):
        a, b = a.double(), b.double()
        assert float((a - b).norm()) <= 12 * 2.0 ** -8 * float(b.norm()), (i, float((a - b).norm() / b.norm()))


def test_mlp_of_many_tokens_with_a_broadcast_gradient_an_expanded_or_a_strided_input():
    """sizes that take the products with epilogues: rows that overlap are copied first, so the gradients are those of the copies"""
    x, w1, b1, w2, b2 = mlp_args(1000, 96, 384, torch.bfloat16)
    def grads(x, dy):
        y = act8.vil_mlp_act8(x, w1, b1, w2, b2)
        return [y.detach(), *torch.autograd.grad(y, (x, w1, b1, w2, b2), dy)]

    row = data(1, 96, torch.bfloat16, 5)[0]
    for dy in (row.expand(3, 1000, 96), row[0].expand(3, 1000, 96)):
        for a, b in zip(grads(x, dy), grads(x, dy.contiguous())):
            assert torch.equal(a, b)
    dy = data(3000, 96, torch.bfloat16, 6).view(3, 1000, 96)
    wide = torch.zeros(3, 1000, 104, device="cuda", dtype=torch.bfloat16)
    wide[..., :96] = x.detach()
    off = torch.zeros(3 * 1000 * 96 + 1, device="cuda", dtype=torch.bfloat16)
    off[1:] = x.detach().view(-1)
    want = grads(x, dy)
    for a, b in zip(want, grads(wide[..., :96].requires_grad_(), dy)):
        assert torch.equal(a, b)
    for a, b in zip(want, grads(off[1:].view(3, 1000, 96).requires_grad_(), dy)):         # unaligned: the separate products
        assert float((a - b).float().norm()) <= 12 * 2.0 ** -8 * float(a.float().norm())
    same = x.detach()[:, :1].expand(3, 1000, 96).requires_grad_()
    for a, b in zip(grads(same, dy), grads(same.detach().contiguous().requires_grad_(), dy)):
        assert torch.equal(a, b)


def test_mlp_refuses_parameters_that_do_not_fit():
    x, w1, b1, w2, b2 = mlp_args(1000, 96, 384, torch.bfloat16)
    for args in ((x, w1, b1[:-1], w2, b2), (x, w1, b1[None], w2, b2), (x, w1, b1, w2, b2[:1]), (x, w1, b1, w2, b1)):
        with pytest.raises(ValueError):
            act8.vil_mlp_act8(*args)
    for i in range(1, 5):
        args = [x, w1, b1, w2, b2]
        args[i] = args[i].detach().cpu()
        with pytest.raises(RuntimeError):
            act8.vil_mlp_act8(*args)


def test_mlp_of_many_tokens_captured_and_replayed():
    x, w1, b1, w2, b2 = mlp_args(1000, 96, 384, torch.bfloat16)
    dy = data(3000, 96, torch.bfloat16, 6).view(3, 1000, 96)

    def step(v):
        leaves = [t.detach().requires_grad_() for t in (v, w1, b1, w2, b2)]
        y = act8.vil_mlp_act8(*leaves)
        return [y.detach(), *torch.autograd.grad(y, leaves, dy)]

    v = x.detach().clone()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step(v)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(v)
    for seed in range(3):
        v.copy_(data(3000, 96, torch.bfloat16, seed).view(3, 1000, 96))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        for a, b in zip(got, step(v)):
            # (a product may be split another way in a capture: half a step of the rms)
            assert float((a - b).float().norm()) <= 2.0 ** -8 * float(b.float().norm())


@pytest.mark.parametrize("K", [96, 160])
def test_a_row_that_is_not_finite_stays_in_its_row_of_the_input_gradient(K):
    """K % 64 = 32: the second half of the last block is no row's (the product with h in 16 bits, which shares the loader)"""
    from vision_longformer_amd import linear
    T, N, t = 1100, 384, torch.bfloat16
    dy, w, h = data(T, K, t), data(K, N, t, 1), data(T, N, t, 2)
    want = linear._dgrad_dgelu(dy, w, h)
    bad = dy.clone()
    bad[700, 3], bad[T - 1, 0] = float("nan"), float("inf")
    got = linear._dgrad_dgelu(bad, w, h)
    keep = torch.ones(T, dtype=torch.bool, device="cuda")
    keep[700] = keep[T - 1] = False
    assert torch.equal(got[keep], want[keep]) and bool(got[700].isnan().all()) and bool(torch.isfinite(want).all())
