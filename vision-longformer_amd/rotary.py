"""Rotary positions with several axes (rows and columns of a token grid; time, rows and columns of a clip) on the queries
and keys of an attention layer, alone or behind the root-mean-square norm of every head, as one HIP kernel each way
(libvilattn.so: vil_qk_rope_fwd / vil_qk_rope_bwd, csrc/vil_qkrope.hip).

The reference's layers carry positions as learned bias tables (src/models/layers/longformer2d.py:67-100); these operators
serve models trained with rotated queries and keys instead, and grids that no table was trained for.  They sit between the
projection and vil_full_attention / vil_dense_attention: q and k may be slices of the packed projection's output, read in
place.  There is no eager fallback: CPU tensors or a missing library raise."""
import ctypes

import torch

from . import _lib

_DT = {torch.float32: _lib.DTYPE_F32, torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_F16}
_POS = {torch.float32: _lib.POS_F32, torch.int32: _lib.POS_I32, torch.int64: _lib.POS_I64}
_FREQ = {torch.float32: _lib.DTYPE_F32, torch.float64: _lib.DTYPE_F64}
_LAYOUTS = {"half": _lib.ROPE_HALF, "interleaved": _lib.ROPE_INTERLEAVED}
_NO_STRIDES = (0, 0, 0)


def rotary_frequencies(sections, base=10000.0, device=None):
    """(sum(sections),) float64: axis a with n pairs turns its pair j by base^(-j / n) radians per unit of position.
    base: one number, or one per axis."""
    bases = tuple(base) if isinstance(base, (tuple, list)) else (base,) * len(sections)
    if len(bases) != len(sections):
        raise ValueError(f"rotary_frequencies: {len(bases)} bases for {len(sections)} axes")
    return torch.cat([torch.as_tensor(b, dtype=torch.float64) ** (-torch.arange(n, dtype=torch.float64) / max(n, 1))
                      for n, b in zip(sections, bases)]).to(device)


def grid_positions(*sides, nglo=0, device=None):
    """(nglo + prod(sides), len(sides)) int32 positions of a token grid in row-major order, as the layers lay it out: the nglo
    global tokens come first, at the origin (no rotation)."""
    axes = torch.meshgrid(*[torch.arange(int(s), dtype=torch.int32) for s in sides], indexing="ij")
    pos = torch.stack([a.reshape(-1) for a in axes], dim=-1)
    return torch.cat([torch.zeros(int(nglo), len(sides), dtype=torch.int32), pos]).to(device)


def _p(t):
    return ctypes.c_void_p(t.data_ptr()) if t is not None else None


def _rows(t):
    """t (B, N, H, M) with contiguous channels"""
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _check(q, k, wq, wk, positions, inv_freq, sections, layout, name):
    """Everything a call can get wrong, before anything touches the device; returns (sections, layout code)."""
    if q.dim() != 4 or (k is not None and k.dim() != 4):
        raise ValueError(f"{name}: q and k are (images, tokens, heads, channels)")
    B, N, _, M = q.shape
    if q.dtype not in _DT:
        raise TypeError(f"{name} supports float32 / bfloat16 / float16; got {q.dtype}")
    if k is not None:
        if k.dtype != q.dtype:
            raise TypeError(f"{name}: q is {q.dtype}, k is {k.dtype}")
        if k.shape[0] != B or k.shape[1] != N or k.shape[3] != M:
            raise ValueError(f"{name}: q is {tuple(q.shape)}, k is {tuple(k.shape)}: images, tokens and channels have to agree")
    if M < 2 or M % 2 or M > 256:
        raise ValueError(f"{name}: a head of {M} channels (even, 2 to 256)")
    if q.shape[2] < 1 or (k is not None and k.shape[2] < 1):
        raise ValueError(f"{name}: no heads")
    if B * N >= 2 ** 31:
        raise ValueError(f"{name}: {B} x {N} tokens (fewer than 2^31)")
    for w, n in ((wq, "q_weight"), (wk, "k_weight")):
        if w is not None and (w.shape != (M,) or w.dtype not in _DT):
            raise ValueError(f"{name}: {n} has to be ({M},) in float32 / bfloat16 / float16; got {tuple(w.shape)} {w.dtype}")
    if wq is not None and wk is not None and wq.dtype != wk.dtype:
        raise TypeError(f"{name}: q_weight is {wq.dtype}, k_weight is {wk.dtype}")
    if wk is not None and k is None:
        raise ValueError(f"{name}: k_weight without k")
    if (positions is None) != (inv_freq is None) or (positions is None) != (sections is None):
        raise ValueError(f"{name}: positions, inv_freq and sections come together")
    tensors = [q, k, wq, wk, positions, inv_freq]
    if positions is not None:
        sections = tuple(int(n) for n in sections)
        if not 1 <= len(sections) <= 4 or min(sections) < 0 or sum(sections) < 1 or 2 * sum(sections) > M:
            raise ValueError(f"{name}: sections {sections} of a head of {M} channels (1 to 4 axes, 1 to {M // 2} pairs in all)")
        if inv_freq.shape != (sum(sections),) or inv_freq.dtype not in _FREQ:
            raise ValueError(f"{name}: inv_freq has to be ({sum(sections)},) in float64 or float32; got {tuple(inv_freq.shape)} {inv_freq.dtype}")
        A = len(sections)
        if tuple(positions.shape) not in ((N, A), (B, N, A)) or positions.dtype not in _POS:
            raise ValueError(f"{name}: positions have to be ({N}, {A}) or ({B}, {N}, {A}) in int32, int64 or float32; got "
                             f"{tuple(positions.shape)} {positions.dtype}")
        if positions.requires_grad or inv_freq.requires_grad:
            raise ValueError(f"{name} has no gradient for positions and inv_freq")
    if layout not in _LAYOUTS:
        raise ValueError(f"{name}: layout {layout!r} (\"half\" or \"interleaved\")")
    for t in tensors:
        if t is not None and not t.is_cuda:
            raise RuntimeError(f"{name} needs device tensors: the product path is the HIP kernels (libvilattn.so); there is no "
                               "CPU fallback")
        if t is not None and t.device != q.device:
            raise RuntimeError(f"{name}: tensors on {q.device} and {t.device}")
    return sections


def _desc(q, k, wq, wk, positions, inv_freq, cfg, yq=None, yk=None, gq=None, gk=None, dq=None, dk=None):
    """cfg: (sections, layout, norm, eps)"""
    sections, layout, norm, eps = cfg
    B, N, Hq, M = q.shape
    w = wq if wq is not None else wk
    st = []
    for t in (q, k, yq, yk, gq, gk, dq, dk):
        st += t.stride()[:3] if t is not None else _NO_STRIDES
    A, R, pos = 0, 0, (0, 0)
    sec = (0, 0, 0, 0)
    if positions is not None:
        A, R = len(sections), sum(sections)
        sec = sections + (0,) * (4 - A)
        pos = (positions.stride(0) if positions.dim() == 3 else 0, positions.stride(-2))
    return _lib.VilRopeDesc(B, N, Hq, k.shape[2] if k is not None else 0, M, R, A, sec, _LAYOUTS[layout], _DT[q.dtype],
                            _POS[positions.dtype] if A else 0, _FREQ[inv_freq.dtype] if A else 0, int(norm),
                            _DT[w.dtype] if w is not None else 0, eps, *st, *pos)


def _launch(device, fn, desc, *tensors):
    stream = ctypes.c_void_p(torch.cuda.current_stream(device).cuda_stream)
    with torch.cuda.device(device):
        _lib.check(fn(ctypes.byref(desc), *[_p(t) for t in tensors], stream))


def _fwd(q, k, wq, wk, positions, inv_freq, cfg, yq, yk):
    d = _desc(q, k, wq, wk, positions, inv_freq, cfg, yq=yq, yk=yk)
    _launch(q.device, _lib.lib().vil_qk_rope_fwd, d, q, k, wq, wk, positions, inv_freq, yq, yk)


def _bwd(q, k, wq, wk, positions, inv_freq, cfg, gq, gk, dq, dk, dwq, dwk):
    d = _desc(q, k, wq, wk, positions, inv_freq, cfg, gq=gq, gk=gk, dq=dq, dk=dk)
    L = _lib.lib()
    ws = None
    if dwq is not None or dwk is not None:
        # (the call's own: two streams, or two captured graphs, never share it)
        ws = torch.empty(L.vil_qk_rope_workspace_bytes(ctypes.byref(d)) // 4, dtype=torch.float32, device=q.device)
    _launch(q.device, L.vil_qk_rope_bwd, d, gq, gk, q if cfg[2] else None, k if cfg[2] else None, wq, wk, positions, inv_freq,
            dq, dk, dwq, dwk, ws)


class _QKRope(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, wq, wk, positions, inv_freq, cfg):
        q, k = _rows(q), _rows(k) if k is not None else None
        yq = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        yk = torch.empty(k.shape, dtype=k.dtype, device=k.device) if k is not None else None
        _fwd(q, k, wq, wk, positions, inv_freq, cfg, yq, yk)
        # without the norm the gradient is the rotation back: the inputs are kept for their shapes only
        ctx.save_for_backward(*((q, k) if cfg[2] else (None, None)), wq, wk, positions, inv_freq)
        ctx.cfg, ctx.shapes = cfg, (q.shape, k.shape if k is not None else None)
        return yq, yk

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, gq, gk):
        q, k, wq, wk, positions, inv_freq = ctx.saved_tensors
        qs, ks = ctx.shapes
        gq, gk = _rows(gq), _rows(gk) if ks is not None else None
        dq = torch.empty(qs, dtype=gq.dtype, device=gq.device)
        dk = torch.empty(ks, dtype=gk.dtype, device=gk.device) if ks is not None else None
        dwq = torch.empty_like(wq) if wq is not None and ctx.needs_input_grad[2] else None
        dwk = torch.empty_like(wk) if wk is not None and ctx.needs_input_grad[3] else None
        _bwd(q if q is not None else gq, k if k is not None else gk, wq, wk, positions, inv_freq, ctx.cfg, gq, gk, dq, dk, dwq, dwk)
        return dq, dk, dwq, dwk, None, None, None


def _positions(positions):
    return positions if positions is None or positions.stride(-1) == 1 or positions.shape[-1] == 1 else positions.contiguous()


def _apply(name, q, k, wq, wk, positions, inv_freq, sections, layout, norm, eps):
    sections = _check(q, k, wq, wk, positions, inv_freq, sections, layout, name)
    cfg = (sections, layout, norm, float(eps))
    wq, wk = (w.contiguous() if w is not None else None for w in (wq, wk))
    if inv_freq is not None:
        inv_freq = inv_freq.contiguous()
    yq, yk = _QKRope.apply(q, k, wq, wk, _positions(positions), inv_freq, cfg)
    return yq if k is None else (yq, yk)


def vil_rope(q, k=None, *, positions, inv_freq, sections, layout="half"):
    """Rotates q (B, N, Hq, M) and, where it is given, k (B, N, Hk, M); returns the rotated tensors, contiguous.

    positions: (N, axes), or (B, N, axes) where every image has its own, int32 / int64 / float32 (fractions serve grids
               measured in the units of another resolution); no gradient
    inv_freq:  (R,) radians per unit of position (rotary_frequencies), float64 or float32
    sections:  pairs of each axis, in order; R = sum(sections) <= M / 2, the channels from 2R on pass through
    layout:    "half": pair p is channels (p, R + p); "interleaved": (2p, 2p + 1)
    fp32 / bf16 / fp16; any strides with contiguous channels (others are copied); computed in fp32 with fp64 angles."""
    return _apply("vil_rope", q, k, None, None, positions, inv_freq, sections, layout, False, 0.0)


def vil_qk_norm_rope(q, k=None, q_weight=None, k_weight=None, *, positions=None, inv_freq=None, sections=None, layout="half",
                     eps=1e-6):
    """x w / sqrt(mean(x^2) + eps) of every head row of q and k, then vil_rope's rotation, in one pass each way.

    q_weight, k_weight: (M,) or None (ones), shared by the heads; their gradients are summed over images, tokens and heads in a
    fixed order.  Without positions (and inv_freq, sections): the norm alone.  Other arguments as vil_rope's."""
    if not eps >= 0:
        raise ValueError(f"vil_qk_norm_rope: eps {eps}")
    return _apply("vil_qk_norm_rope", q, k, q_weight, k_weight, positions, inv_freq, sections, layout, True, eps)
