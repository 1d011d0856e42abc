"""GPU: rotary positions with several axes and the per-head norms of q and k (csrc/vil_qkrope.hip) against the formulas in
64 bits, and against differences.

Tolerances, from the arithmetic.  u = 2^-24 (half a step of fp32).  A stored value is off by half a step of its type plus what
fp32 adds before: the angle's remainder is rounded once (u) and sine and cosine are series of two more roundings, a rotation
rounds three times, so a rotated pair is off by at most 8 u (|a| + |b|).  The norm adds a sum of M squares (<= M u, in
practice a tree), a division, a root and two products: (M + 8) u more, relative.  The backward's dx sums M products once more.
dw adds one product of each row: rounded to (64 + rows / 64) u of the sum of their magnitudes (64 rows or more are added side by
side, 64 covers the tree)."""
import ctypes

import pytest
import torch

from vision_longformer_amd import _lib, rotary

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def half_step(t, ref):
    f = torch.finfo(t)
    return torch.clamp(ref.abs() * (f.eps / 2), min=f.tiny * f.eps / 2)


def rotate(x, cos, sin, layout):
    """fp64: the rotated pairs, and |a| + |b| of each channel's pair"""
    R = cos.shape[-1]
    y, mag = x.clone(), x.abs()
    a, b = (slice(0, R), slice(R, 2 * R)) if layout == "half" else (slice(0, 2 * R, 2), slice(1, 2 * R, 2))
    y[..., a], y[..., b] = x[..., a] * cos - x[..., b] * sin, x[..., b] * cos + x[..., a] * sin
    mag[..., a] = mag[..., b] = x[..., a].abs() + x[..., b].abs()
    return y, mag


def reference(x, w, g, cos, sin, layout, norm, eps):
    """fp64 (y, dx, dw) with the fp32 share of each tolerance"""
    M = x.shape[-1]
    r = 1 / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) if norm else torch.ones_like(x[..., :1])
    w = w if w is not None else torch.ones(M, dtype=torch.float64, device=x.device)
    y, ymag = rotate(x * r * w, cos, sin, layout)
    gi, gmag = rotate(g, cos, -sin, layout)
    k = M + 16 if norm else 8
    out = {"y": (y, k * U * ymag)}
    if not norm:
        return out | {"dx": (gi, k * U * gmag)}
    xh = x * r
    m = (gi * w * xh).mean(-1, keepdim=True)
    mmag = (gmag * (w * xh).abs()).mean(-1, keepdim=True)
    dx = r * (gi * w - xh * m)
    dw = (gi * xh).sum((0, 1, 2))
    rows = x.shape[0] * x.shape[1] * x.shape[2]
    return out | {"dx": (dx, 3 * k * U * r * (gmag * w.abs() + xh.abs() * mmag)),
                  "dw": (dw, (64 + rows / 64 + 2 * k) * U * (gmag * xh.abs()).sum((0, 1, 2)))}


def angles(positions, inv_freq, sections):
    axis = [a for a, n in enumerate(sections) for _ in range(n)]
    t = (positions.double()[..., axis] * inv_freq.double())
    t = (t if t.dim() == 3 else t[None])[:, :, None, :]
    return torch.cos(t), torch.sin(t)


def check(name, got, ref, tol, t):
    lim = half_step(t, ref) * (1 + 2.0 ** -10) + tol
    err = (got.double() - ref).abs()
    assert got.shape == ref.shape and got.dtype == t
    assert bool((err <= lim).all()), f"{name}: {float((err / lim).max()):.3f} of the bound"


def make(B, N, Hq, Hk, M, t, packed, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=g, device="cuda")
    if packed:
        qkv = (n(B, N, (Hq + 2 * Hk) * M) + 0.2).to(t)
        q, k = qkv[..., :Hq * M].unflatten(-1, (Hq, M)), qkv[..., Hq * M:(Hq + Hk) * M].unflatten(-1, (Hk, M))
    else:
        q, k = n(B, N, Hq, M).to(t), n(B, N, Hk, M).to(t)
    return q, k, n(B, N, Hq, M).to(t), n(B, N, Hk, M).to(t), 1 + 0.3 * n(M), 1 + 0.3 * n(M)


def positions_of(kind, B, N, A, seed=1):
    g = torch.Generator(device="cuda").manual_seed(seed)
    if kind == "grid":
        return torch.randint(0, 100, (N, A), generator=g, device="cuda", dtype=torch.int32)
    if kind == "far":
        return torch.randint(-2 ** 27, 2 ** 27, (B, N, A), generator=g, device="cuda", dtype=torch.int32)
    if kind == "int64":
        return torch.randint(0, 2 ** 27, (B, N, A), generator=g, device="cuda", dtype=torch.int64)
    return torch.rand(B, N, A, generator=g, device="cuda") * 57 - 3


CASES = [
    # B, N, Hq, Hk, M, sections, layout, packed, positions
    (2, 65, 3, 3, 32, (8, 8), "half", True, "grid"), (2, 65, 3, 3, 32, (8, 8), "interleaved", True, "grid"),
    (3, 50, 6, 6, 64, (16, 16), "half", True, "grid"), (2, 33, 12, 3, 64, (10, 11, 11), "interleaved", True, "far"),
    (2, 33, 12, 3, 64, (8, 12, 12), "half", True, "far"), (1, 17, 1, 1, 48, (12, 12), "half", True, "scaled"),
    (2, 17, 1, 1, 48, (8, 8), "half", False, "scaled"), (2, 17, 2, 1, 48, (5, 4), "interleaved", False, "scaled"),
    (1, 1, 6, 6, 64, (32,), "half", True, "int64"), (8, 1, 6, 2, 64, (8, 12, 12), "half", True, "int64"),
    (2, 9, 2, 2, 8, (2, 2), "half", True, "grid"), (2, 9, 2, 2, 16, (8,), "half", True, "grid"),
    (2, 9, 2, 2, 16, (3, 2), "half", True, "grid"), (2, 9, 5, 1, 24, (4, 4, 4), "half", True, "grid"),
    (2, 9, 1, 1, 24, (6, 6), "interleaved", True, "grid"), (1, 7, 3, 3, 2, (1,), "half", False, "grid"),
    (1, 7, 3, 3, 10, (2, 1, 1), "interleaved", False, "grid"), (2, 5, 4, 4, 128, (22, 21, 21), "half", True, "grid"),
    (2, 5, 4, 2, 128, (16, 8, 8), "half", True, "far"), (1, 6, 2, 2, 256, (64, 64), "half", True, "grid"),
    (1, 6, 2, 2, 200, (50, 3), "interleaved", True, "grid"), (1, 3, 40, 8, 96, (24, 24), "half", True, "grid"),
    (1, 2500, 1, 1, 32, (8, 8), "half", True, "grid"), (1, 300, 3, 3, 80, (20, 20), "half", True, "scaled"),
    (700, 1, 2, 2, 32, (16,), "half", True, "grid"), (2, 4, 200, 7, 16, (4, 4), "half", True, "grid"),
]


@pytest.mark.parametrize("t", list(TYPES))
@pytest.mark.parametrize("norm", [False, True], ids=["rope", "norm"])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "B%dN%dH%d-%dM%d_%s_%s%s_%s" % (*c[:5], "-".join(map(str, c[5])), c[6][0], "p" if c[7] else "", c[8]))
def test_against_the_formulas(case, norm, t):
    B, N, Hq, Hk, M, sections, layout, packed, kind = case
    t = TYPES[t]
    q, k, gq, gk, wq, wk = make(B, N, Hq, Hk, M, t, packed)
    pos = positions_of(kind, B, N, len(sections))
    f = rotary.rotary_frequencies(sections, device="cuda")
    q, k, wq, wk = (v.detach().requires_grad_() for v in (q, k, wq, wk))
    kw = dict(positions=pos, inv_freq=f, sections=sections, layout=layout)
    if norm:
        yq, yk = rotary.vil_qk_norm_rope(q, k, wq, wk, eps=1e-5, **kw)
    else:
        yq, yk = rotary.vil_rope(q, k, **kw)
    leaves = [q, k] + ([wq, wk] if norm else [])
    grads = torch.autograd.grad((yq, yk), leaves, (gq, gk))
    cos, sin = angles(pos, f, sections)
    for i, (x, w, g, y) in enumerate(((q, wq, gq, yq), (k, wk, gk, yk))):
        ref = reference(x.detach().double(), w.detach().double() if norm else None, g.double(), cos, sin, layout, norm, 1e-5)
        check("y%d" % i, y.detach(), *ref["y"], t)
        check("dx%d" % i, grads[i], *ref["dx"], t)
        if norm:
            check("dw%d" % i, grads[2 + i], *ref["dw"], torch.float32)


def test_norm_without_rotation_and_without_weights():
    q, k, gq, gk, _, _ = make(2, 19, 3, 2, 64, torch.bfloat16, True)
    q, k = q.detach().requires_grad_(), k.detach().requires_grad_()
    yq, yk = rotary.vil_qk_norm_rope(q, k)
    dq, dk = torch.autograd.grad((yq, yk), (q, k), (gq, gk))
    one, zero = torch.ones(1, 1, 1, 0, device="cuda", dtype=torch.float64), torch.zeros(1, 1, 1, 0, device="cuda", dtype=torch.float64)
    for x, g, y, d in ((q, gq, yq, dq), (k, gk, yk, dk)):
        ref = reference(x.detach().double(), None, g.double(), one, zero, "half", True, 1e-6)
        check("y", y.detach(), *ref["y"], torch.bfloat16)
        check("dx", d, *ref["dx"], torch.bfloat16)


@pytest.mark.parametrize("norm", [False, True])
def test_q_alone_equals_q_of_both(norm):
    q, k, gq, gk, wq, wk = make(2, 31, 3, 3, 32, torch.float16, True)
    pos, f = positions_of("grid", 2, 31, 2), rotary.rotary_frequencies((8, 8), device="cuda")
    kw = dict(positions=pos, inv_freq=f, sections=(8, 8))
    fn = (lambda a, b: rotary.vil_qk_norm_rope(a, b, wq, wk if b is not None else None, **kw)) if norm else \
        (lambda a, b: rotary.vil_rope(a, b, **kw))
    q = q.detach().requires_grad_()
    y = fn(q, None)
    both = fn(q, k)
    assert torch.equal(y, both[0])
    assert torch.equal(torch.autograd.grad(y, q, gq)[0], torch.autograd.grad(both, q, (gq, gk))[0])


@pytest.mark.parametrize("wt", [torch.bfloat16, torch.float16])
def test_16_bit_weights_and_frozen_weights(wt):
    q, k, gq, gk, wq, wk = make(2, 40, 3, 3, 64, torch.bfloat16, True)
    pos, f = positions_of("grid", 2, 40, 2), rotary.rotary_frequencies((16, 16), device="cuda")
    wq, wk = wq.to(wt).requires_grad_(), wk.to(wt)
    kw = dict(positions=pos, inv_freq=f, sections=(16, 16))
    yq, yk = rotary.vil_qk_norm_rope(q, k, wq, wk, **kw)
    dw, = torch.autograd.grad((yq, yk), wq, (gq, gk))
    cos, sin = angles(pos, f, (16, 16))
    ref = reference(q.double(), wq.detach().double(), gq.double(), cos, sin, "half", True, 1e-6)
    check("y", yq.detach(), *ref["y"], torch.bfloat16)
    check("dw", dw, *ref["dw"], wt)


@pytest.mark.parametrize("how", ["heads_first", "odd_offset", "every_second_channel", "odd_row", "expanded_batch"])
def test_strides_and_alignment(how):
    B, N, H, M, t = 2, 21, 3, 32, torch.bfloat16
    g = torch.Generator(device="cuda").manual_seed(3)
    n = lambda *s: torch.randn(*s, generator=g, device="cuda").to(t)
    if how == "heads_first":
        q, k = n(B, H, N, M).transpose(1, 2), n(B, H, N, M).transpose(1, 2)
    elif how == "odd_offset":
        q, k = (n(B * N * H * M + 1)[1:].view(B, N, H, M) for _ in range(2))
    elif how == "every_second_channel":
        q, k = (n(B, N, H, 2 * M)[..., ::2] for _ in range(2))
    elif how == "odd_row":
        q, k = (n(B, N, H * M + 3)[..., :H * M].unflatten(-1, (H, M)) for _ in range(2))
    else:
        q, k = (n(1, N, H, M).expand(B, N, H, M) for _ in range(2))
    pos = positions_of("far", B, 2 * N, 2)[:, ::2]                # (rows of the positions a stride apart)
    f = rotary.rotary_frequencies((8, 8), device="cuda")
    kw = dict(positions=pos, inv_freq=f, sections=(8, 8))
    wq = 1 + 0.2 * torch.randn(M, generator=g, device="cuda")
    qc, kc = q.contiguous().requires_grad_(), k.contiguous().requires_grad_()
    want = rotary.vil_qk_norm_rope(qc, kc, wq, wq, **{**kw, "positions": pos.contiguous()})
    q, k = q.detach().requires_grad_(), k.detach().requires_grad_()
    got = rotary.vil_qk_norm_rope(q, k, wq, wq, **kw)

    def same(a, b):
        # A layout that the 16-byte loads do not fit adds a row's M squares and products in another order: r and the mean differ by
        # up to 2 (M + 8) u relative, so a value moves by that share of its pair's and its row's scale (at most 4 (|a| + |b|) of
        # these inputs' largest) and may round to the neighbouring number: one step of the type, eps |b|, or its smallest one.
        if how in ("heads_first", "expanded_batch"):
            return torch.equal(a, b)
        a, b = a.double(), b.double()
        f = torch.finfo(t)
        return bool(((a - b).abs() <= f.eps * b.abs() * (1 + f.eps) + f.tiny * f.eps + 2 * (M + 8) * U * 4 * b.abs().amax()).all())

    for a, b in zip(got, want):
        assert same(a, b) and a.is_contiguous()
    # a gradient that is a slice, and one that is a single broadcast number
    gq = n(B, N, H, 2 * M)[..., M:]
    gk = torch.ones((), device="cuda", dtype=t).expand(B, N, H, M)
    for a, b in zip(torch.autograd.grad(got, (q, k), (gq, gk)), torch.autograd.grad(want, (qc, kc), (gq.contiguous(), gk.contiguous()))):
        assert same(a, b)


@pytest.mark.parametrize("shape", [(0, 5), (3, 0)])
def test_empty_batches(shape):
    q = torch.zeros(*shape, 2, 32, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    w = torch.ones(32, device="cuda", requires_grad=True)
    pos = torch.zeros(shape[1], 2, device="cuda", dtype=torch.int32)
    f = rotary.rotary_frequencies((8, 8), device="cuda")
    yq, yk = rotary.vil_qk_norm_rope(q, q, w, w, positions=pos, inv_freq=f, sections=(8, 8))
    assert yq.shape == yk.shape == (*shape, 2, 32)
    dq, dw = torch.autograd.grad((yq, yk), (q, w), (torch.ones_like(yq), torch.ones_like(yk)))
    assert dq.shape == q.shape and bool((dw == 0).all())


def test_origin_is_left_alone_and_far_positions_keep_their_angle():
    """Position 0 (the global tokens) returns the input bit for bit; a whole number of turns far out does too, to the angle's
    rounding: base 1 and positions that are multiples of 2 pi are not integers, so the check is against fp64 at 2^40."""
    q = torch.randn(1, 4, 2, 64, device="cuda")
    f = rotary.rotary_frequencies((16, 16), device="cuda")
    pos = torch.zeros(4, 2, device="cuda", dtype=torch.int64)
    kw = dict(inv_freq=f, sections=(16, 16))
    assert torch.equal(rotary.vil_rope(q, positions=pos, **kw), q)
    pos[1:, 0] = torch.tensor([2 ** 40, 2 ** 40 + 1, -2 ** 40], device="cuda")
    y = rotary.vil_rope(q, positions=pos, **kw)
    cos, sin = angles(pos, f, (16, 16))
    # (2^40 radians in fp64 are known to 2^40 * 2^-53 * 2 = 2.4e-4: that much of the pair on either side)
    ref, mag = rotate(q.double(), cos, sin, "half")
    assert bool(((y.double() - ref).abs() <= 5e-4 * mag).all())


def test_a_bad_row_stays_in_its_row():
    q, k, gq, gk, wq, wk = make(2, 40, 3, 3, 32, torch.bfloat16, True)
    pos, f = positions_of("grid", 2, 40, 2), rotary.rotary_frequencies((8, 8), device="cuda")
    kw = dict(positions=pos, inv_freq=f, sections=(8, 8))
    clean = rotary.vil_qk_norm_rope(q, k, wq, wk, **kw)
    q2, k2 = q.clone(), k.clone()
    q2[1, 7, 2, 5], k2[0, 3, 0, 31] = float("nan"), float("inf")
    q3, k3 = q2.requires_grad_(), k2.requires_grad_()
    bad = rotary.vil_qk_norm_rope(q3, k3, wq, wk, **kw)
    dq, dk = torch.autograd.grad(bad, (q3, k3), (gq, gk))
    for a, b, at in ((bad[0], clean[0], (1, 7, 2)), (bad[1], clean[1], (0, 3, 0))):
        mask = torch.ones(a.shape[:3], dtype=torch.bool, device="cuda")
        mask[at] = False
        assert torch.equal(a[mask], b[mask]) and bool(a[at].isnan().any())
    assert int(dq.isnan().any(-1).sum()) == 1 and int(dk.isnan().any(-1).sum()) == 1
    # a masked (all-zero) row: the norm of nothing is nothing, and its gradient is finite
    z = torch.zeros(1, 3, 2, 32, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    y = rotary.vil_qk_norm_rope(z, None, wq, positions=pos[:3], inv_freq=f, sections=(8, 8))
    d, = torch.autograd.grad(y, z, torch.ones_like(y))
    assert bool((y == 0).all()) and bool(torch.isfinite(d).all())


def test_gradients_against_differences():
    """fp32 operator, fp64 sums of its outputs: central differences at step h are off by the third derivative's h^2 / 6 and by
    the outputs' rounding, 2 u |y| |g| summed / 2h.  h = 2^-6 keeps the first under 1e-4 relative of values of order one and
    the second under sum * 2^-18."""
    q, k, gq, gk, wq, wk = make(1, 3, 2, 1, 16, torch.float32, False)
    pos, f = positions_of("scaled", 1, 3, 2), rotary.rotary_frequencies((4, 3), device="cuda")
    leaves = [v.detach().requires_grad_() for v in (q, k, wq, wk)]
    kw = dict(positions=pos, inv_freq=f, sections=(4, 3))

    def value(vs):
        with torch.no_grad():
            yq, yk = rotary.vil_qk_norm_rope(*vs, eps=0.1, **kw)
            return float((yq.double() * gq.double()).sum() + (yk.double() * gk.double()).sum())

    grads = torch.autograd.grad(rotary.vil_qk_norm_rope(*leaves, eps=0.1, **kw), leaves, (gq, gk))
    h, total = 2.0 ** -6, float(gq.abs().sum() + gk.abs().sum()) * 3
    for i, (v, d) in enumerate(zip(leaves, grads)):
        for at in range(0, v.numel(), 5):
            vs = [x.detach().clone() for x in leaves]
            vs[i].view(-1)[at] += h
            up = value(vs)
            vs[i].view(-1)[at] -= 2 * h
            slope = (up - value(vs)) / (2 * h)
            assert abs(slope - float(d.reshape(-1)[at])) <= total * 2.0 ** -18 + 2e-3 * max(1.0, abs(slope)), (i, at)


def test_other_stream_and_repeatability():
    q, k, gq, gk, wq, wk = make(4, 197, 6, 6, 64, torch.bfloat16, True)
    pos, f = positions_of("grid", 4, 197, 2), rotary.rotary_frequencies((16, 16), device="cuda")
    kw = dict(positions=pos, inv_freq=f, sections=(16, 16))

    def step():
        leaves = [v.detach().requires_grad_() for v in (q, k, wq, wk)]
        y = rotary.vil_qk_norm_rope(*leaves, **kw)
        return [*(v.detach() for v in y), *torch.autograd.grad(y, leaves, (gq, gk))]

    first = step()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = [v.clone() for v in step()]
    s.synchronize()
    for a, b, c in zip(first, other, step()):
        assert torch.equal(a, b) and torch.equal(a, c)


def test_captured_and_replayed():
    """forward and backward in a graph, replayed on new inputs with eager work and synchronizations in between; two graphs
    replayed in turn share nothing"""
    pos, f = positions_of("grid", 2, 50, 2), rotary.rotary_frequencies((8, 8), device="cuda")
    kw = dict(positions=pos, inv_freq=f, sections=(8, 8))

    def step(v):
        q, k, wq, wk = (x.detach().requires_grad_() for x in (v[0], v[1], v[4], v[5]))
        y = rotary.vil_qk_norm_rope(q, k, wq, wk, **kw)
        return [*(x.detach() for x in y), *torch.autograd.grad(y, (q, k, wq, wk), (v[2], v[3]))]

    graphs = []
    for seed in (0, 1):
        held = list(make(2, 50, 3, 3, 32, torch.bfloat16, True, seed))
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            step(held)
        torch.cuda.current_stream().wait_stream(s)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(held)
        graphs.append((held, graph, out))
    for turn in range(4):
        for held, graph, _ in graphs:
            for a, b in zip(held, make(2, 50, 3, 3, 32, torch.bfloat16, True, 10 + turn)):
                a.copy_(b)
            graph.replay()
        torch.cuda.synchronize()
        for held, graph, out in graphs:
            for a, b in zip(out, step(held)):
                assert torch.equal(a, b)


def test_long_token_axis_past_32_bits_of_offset():
    """one image whose rows span more than 2^31 elements: the last token's row is right"""
    N, M = 40000, 64
    buf = torch.zeros(N, 60000, device="cuda", dtype=torch.bfloat16)        # 4.8 GB, element offsets past 2^31
    x = torch.randn(N, 1, M, device="cuda").to(torch.bfloat16)
    buf[:, :M] = x[:, 0]
    q = buf[:, :M].view(1, N, 1, M)
    pos = torch.arange(N, device="cuda", dtype=torch.int32)[:, None]
    kw = dict(positions=pos, inv_freq=rotary.rotary_frequencies((32,), device="cuda"), sections=(32,))
    assert (N - 1) * 60000 > 2 ** 31
    assert torch.equal(rotary.vil_rope(q, **kw), rotary.vil_rope(x[None], **kw))


def test_the_c_entry_reports_the_launch_contract():
    d = _lib.VilRopeDesc()
    assert _lib.lib().vil_qk_rope_fwd(ctypes.byref(d), *([None] * 9)) < 0


def both_ways(q, k, wq, wk, gq, gk, **kw):
    leaves = [v.detach().requires_grad_() for v in (q, k, wq, wk)]
    y = rotary.vil_qk_norm_rope(*leaves, eps=1e-5, **kw)
    return [v.detach() for v in y], torch.autograd.grad(y, leaves, (gq, gk))


def against_formulas(q, k, wq, wk, gq, gk, pos, f, sections, layout="half"):
    (yq, yk), (dq, dk, dwq, dwk) = both_ways(q, k, wq, wk, gq, gk, positions=pos, inv_freq=f, sections=sections, layout=layout)
    cos, sin = angles(pos, f, sections)
    for x, w, g, y, d, dw in ((q, wq, gq, yq, dq, dwq), (k, wk, gk, yk, dk, dwk)):
        ref = reference(x.detach().double(), w.double(), g.double(), cos, sin, layout, True, 1e-5)
        check("y", y, *ref["y"], x.dtype)
        check("dx", d, *ref["dx"], x.dtype)
        check("dw", dw, *ref["dw"], w.dtype)


@pytest.mark.parametrize("B,N", [(1500, 3), (70000, 1), (3, 700)])
@pytest.mark.parametrize("kind", ["grid", "stream"])
@pytest.mark.parametrize("layout", ["tokens", "heads"])
def test_many_images_and_many_tiles(B, N, kind, layout):
    """more images than the grid's second axis or the backward's workgroups hold, in a layout whose images are one run of tokens and
    in one where they are not; positions shared and each image's own"""
    H, M, t = 2, 16, torch.bfloat16
    q, k, gq, gk, wq, wk = make(B, N, H, H, M, t, False)
    if layout == "heads":
        q, k, gq, gk = (v.transpose(1, 2).contiguous().transpose(1, 2) for v in (q, k, gq, gk))
    pos = positions_of("grid" if kind == "grid" else "far", B, N, 2)
    against_formulas(q, k, wq, wk, gq, gk, pos, rotary.rotary_frequencies((4, 4), device="cuda"), (4, 4))


@pytest.mark.parametrize("how", ["8_byte_offset", "heads_shared_by_stride_0", "16_mb_rows", "one_position_for_all"])
def test_more_layouts(how):
    B, N, H, M, t = 2, 9, 4, 64, torch.float16
    q, k, gq, gk, wq, wk = make(B, N, H, H, M, t, False)
    pos = positions_of("scaled", B, N, 2)
    if how == "8_byte_offset":
        flat = torch.zeros(2, B * N * H * M + 4, device="cuda", dtype=t)
        flat[:, 4:] = torch.stack([q, k]).view(2, -1)
        q, k = flat[0, 4:].view(B, N, H, M), flat[1, 4:].view(B, N, H, M)
    elif how == "heads_shared_by_stride_0":
        q, k = q[:, :, :1].expand(B, N, H, M), k[:, :, :1].expand(B, N, H, M)
    elif how == "16_mb_rows":
        buf = torch.zeros(N, 2 ** 23, device="cuda", dtype=t)
        B, q, k, gq, gk, pos = 1, q[:1], k[:1], gq[:1], gk[:1], pos[:1]
        buf[:, :2 * H * M] = torch.cat([q, k], 2).view(N, -1)
        q, k = buf[:, :H * M].view(1, N, H, M), buf[:, H * M:2 * H * M].view(1, N, H, M)
    else:
        pos = pos[:1, :1].expand(B, N, 2)
    against_formulas(q, k, wq, wk, gq, gk, pos, rotary.rotary_frequencies((16, 16), device="cuda"), (16, 16))


def test_gradient_of_a_broadcast_input():
    """one head of k serving four by expand(): its gradient is the sum of theirs, each rounded once: 4 half steps and the sum's"""
    q, k, gq, gk, wq, wk = make(2, 9, 4, 4, 32, torch.bfloat16, False)
    pos, f = positions_of("grid", 2, 9, 2), rotary.rotary_frequencies((8, 8), device="cuda")
    kw = dict(positions=pos, inv_freq=f, sections=(8, 8))
    one = k[:, :, :1].detach().requires_grad_()
    y = rotary.vil_qk_norm_rope(one.expand(2, 9, 4, 32), None, wk, **kw)
    got, = torch.autograd.grad(y, one, gk)
    four = k[:, :, :1].expand(2, 9, 4, 32).detach().requires_grad_()
    parts, = torch.autograd.grad(rotary.vil_qk_norm_rope(four, None, wk, **kw), four, gk)
    ref = parts.double().sum(2, keepdim=True)
    assert bool(((got.double() - ref).abs() <= 2.0 ** -8 * parts.double().abs().sum(2, keepdim=True) + 1e-30).all())


def test_second_derivatives_are_refused_and_create_graph_is_not():
    q, k, gq, gk, wq, wk = make(1, 5, 2, 2, 32, torch.float32, False)
    pos, f = positions_of("grid", 1, 5, 2), rotary.rotary_frequencies((8, 8), device="cuda")
    q = q.requires_grad_()
    y = rotary.vil_qk_norm_rope(q, None, wq, positions=pos, inv_freq=f, sections=(8, 8))
    first, = torch.autograd.grad(y, q, gq, retain_graph=True)
    again, = torch.autograd.grad(y, q, gq, create_graph=True)
    assert torch.equal(first, again)
    with pytest.raises(RuntimeError):
        again.sum().backward()


def test_two_streams_at_once():
    """calls on two streams in flight together, each with its own weights' gradients: nothing is shared between them"""
    pos, f = positions_of("grid", 16, 785, 2), rotary.rotary_frequencies((16, 16), device="cuda")
    kw = dict(positions=pos, inv_freq=f, sections=(16, 16))
    sets = [make(16, 785, 3, 3, 64, torch.bfloat16, True, seed) for seed in (0, 1)]

    def step(v):
        y, g = both_ways(v[0], v[1], v[4], v[5], v[2], v[3], **kw)
        return [*y, *g]

    want = [step(v) for v in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(step(sets[i]))
    torch.cuda.synchronize()
    for i in (0, 1):
        for turn in got[i]:
            for a, b in zip(turn, want[i]):
                assert torch.equal(a, b)


def test_same_tensor_twice_and_rows_behind_the_last():
    """q and k one tensor: both gradients arrive; a slice's neighbours in memory are left as they were"""
    buf = torch.randn(2, 12, 3, 32, device="cuda")
    keep = buf.clone()
    x = buf[:, :9].detach().requires_grad_()
    pos, f = positions_of("grid", 2, 9, 2), rotary.rotary_frequencies((8, 8), device="cuda")
    kw = dict(positions=pos, inv_freq=f, sections=(8, 8))
    a, b = rotary.vil_rope(x, x, **kw)
    assert torch.equal(a, b)
    one, = torch.autograd.grad(a, x, torch.ones_like(a), retain_graph=True)
    two, = torch.autograd.grad((a, b), x, (torch.ones_like(a), torch.ones_like(b)))
    assert torch.equal(two, 2 * one) and torch.equal(buf, keep)


@pytest.mark.parametrize("t", ["fp32", "bf16"])
@pytest.mark.parametrize("M,sections", [(10, (2,)), (48, (2,)), (48, (8, 8)), (64, (16, 16))])
@pytest.mark.parametrize("scale", [-46, 46, 57])
def test_norm_of_very_small_and_very_large_rows(scale, M, sections, t):
    """rows of 10^-14 (eps = 0), 10^14 and 10^17: their squares fit fp32, and so does everything that the norm and its gradient
    need in the order that the kernels take it"""
    t = TYPES[t]
    q, k, gq, gk, wq, wk = make(2, 33, 3, 3, M, t, False)
    q, k = (v * 2.0 ** scale for v in (q, k))
    pos, f = positions_of("grid", 2, 33, len(sections)), rotary.rotary_frequencies(sections, device="cuda")
    q, k, wq, wk = (v.detach().requires_grad_() for v in (q, k, wq, wk))
    y = rotary.vil_qk_norm_rope(q, k, wq, wk, positions=pos, inv_freq=f, sections=sections, eps=0.0)
    grads = torch.autograd.grad(y, (q, k, wq, wk), (gq, gk))
    cos, sin = angles(pos, f, sections)
    for i, (x, w, g) in enumerate(((q, wq, gq), (k, wk, gk))):
        ref = reference(x.detach().double(), w.detach().double(), g.double(), cos, sin, "half", True, 0.0)
        check("y%d" % i, y[i].detach(), *ref["y"], t)
        check("dx%d" % i, grads[i], *ref["dx"], t)
        check("dw%d" % i, grads[2 + i], *ref["dw"], torch.float32)
