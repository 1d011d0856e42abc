"""Rotary positions with several axes (rows and columns of a token grid; time, rows and columns of a clip) on the queries
and keys of an attention layer, alone or behind the root-mean-square norm of every head, as one HIP kernel each way
(libvilattn.so: vil_qk_rope_fwd / vil_qk_rope_bwd, csrc/vil_qkrope.hip).

The reference's layers carry positions as learned bias tables (src/models/layers/longformer2d.py:67-100); these operators
serve models trained with rotated queries and keys instead, and grids that no table was trained for.  They sit between the
projection and vil_full_attention / vil_dense_attention: q and k may be slices of the packed projection's output, read in
place.  There is no eager fallback: CPU tensors or a missing library raise."""
import ctypes

import torch
from torch.autograd import forward_ad

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


def _ptr(t):
    return t.data_ptr() if t is not None else None


def _rows(t):
    """t (B, N, H, M) with contiguous channels"""
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _check(q, k, wq, wk, positions, inv_freq, sections, layout, name):
    """Everything a call can get wrong, before anything touches the device."""
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
    if positions is not None:
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
    for t in (q, k, wq, wk, positions, inv_freq):
        if t is not None and not t.is_cuda:
            raise RuntimeError(f"{name} needs device tensors: the product path is the HIP kernels (libvilattn.so); there is no "
                               "CPU fallback")
        if t is not None and t.device != q.device:
            raise RuntimeError(f"{name}: tensors on {q.device} and {t.device}")


def _dense(shape):
    """strides (image, token, head) of a contiguous tensor"""
    return (shape[1] * shape[2] * shape[3], shape[2] * shape[3], shape[3])


class _Plan:
    """What a call's layout decides (shapes, strides, types, options: nothing of any tensor's values or place): the checks have
    passed, and the descriptors of the forward pass and of a backward pass with contiguous gradients are filled in.  A
    training step makes the same few calls over and over; checking and filling take as long as the launch."""
    __slots__ = ("base", "qs", "ks", "norm", "fwd", "bwd", "ws")

    def __init__(self, q, k, wq, wk, positions, inv_freq, sections, layout, norm, eps):
        B, N, Hq, M = self.qs = tuple(q.shape)
        self.ks, self.norm = tuple(k.shape) if k is not None else None, norm
        w = wq if wq is not None else wk
        A, R, sec, self_pos = 0, 0, (0, 0, 0, 0), (0, 0)
        if positions is not None:
            A, R = len(sections), sum(sections)
            sec = sections + (0,) * (4 - A)
            self_pos = (positions.stride(0) if positions.dim() == 3 else 0, positions.stride(-2))
        head = (B, N, Hq, k.shape[2] if k is not None else 0, M, R, A, sec, _LAYOUTS[layout], _DT[q.dtype],
                _POS[positions.dtype] if A else 0, _FREQ[inv_freq.dtype] if A else 0, int(norm),
                _DT[w.dtype] if w is not None else 0, eps)
        x = q.stride()[:3] + (k.stride()[:3] if k is not None else _NO_STRIDES)
        self.base = head, x, self_pos
        dense = _dense(self.qs) + (_dense(self.ks) if k is not None else _NO_STRIDES)
        self.fwd = _lib.VilRopeDesc(*head, *x, *dense, *_NO_STRIDES * 4, *self_pos)
        self.bwd = self._bwd(dense, dense)
        self.ws = _lib.lib().vil_qk_rope_workspace_bytes(ctypes.byref(self.fwd)) // 4

    def _bwd(self, g, d):
        head, x, pos = self.base
        return _lib.VilRopeDesc(*head, *x, *_NO_STRIDES * 2, *g, *d, *pos)

    def fwd_desc(self, yq, yk):
        """of outputs with other strides"""
        head, x, pos = self.base
        y = yq.stride()[:3] + (yk.stride()[:3] if yk is not None else _NO_STRIDES)
        return _lib.VilRopeDesc(*head, *x, *y, *_NO_STRIDES * 4, *pos)

    def bwd_desc(self, gq, gk, dq=None, dk=None):
        """of gradients (and outputs dq, dk; contiguous where they are None) with other strides"""
        g = gq.stride()[:3] + (gk.stride()[:3] if gk is not None else _NO_STRIDES)
        d = ((dq.stride()[:3] if dq is not None else _dense(self.qs)) +
             ((dk.stride()[:3] if dk is not None else _dense(self.ks)) if self.ks else _NO_STRIDES))
        return self._bwd(g, d)


_PLANS = {}


def _plan(name, q, k, wq, wk, positions, inv_freq, sections, layout, norm, eps):
    index = q.get_device()
    key = (q.shape, q.stride(), q.dtype, index, sections, layout, norm, eps,
           (k.shape, k.stride(), k.dtype, k.get_device()) if k is not None else None,
           (wq.shape, wq.dtype, wq.get_device()) if wq is not None else None,
           (wk.shape, wk.dtype, wk.get_device()) if wk is not None else None,
           (positions.shape, positions.stride(), positions.dtype, positions.get_device(), positions.requires_grad) if positions is not None else None,
           (inv_freq.shape, inv_freq.dtype, inv_freq.get_device(), inv_freq.requires_grad) if inv_freq is not None else None)
    plan = _PLANS.get(key)
    if plan is None:
        _check(q, k, wq, wk, positions, inv_freq, sections, layout, name)
        plan = _Plan(q, k, wq, wk, positions, inv_freq, sections, layout, norm, eps)
        if len(_PLANS) >= 1024:                  # (a program with ever new shapes: start over)
            _PLANS.clear()
        _PLANS[key] = plan
    return plan


def _fwd(plan, q, k, wq, wk, positions, inv_freq, into=None):
    """(yq, yk), contiguous, or `into` two tensors with other strides"""
    if into is None:
        yq = q.new_empty(plan.qs)
        yk = k.new_empty(plan.ks) if k is not None else None
        desc = plan.fwd
    else:
        yq, yk = into
        desc = plan.fwd_desc(yq, yk)
    _lib.launch(q.get_device(), _lib.lib().vil_qk_rope_fwd, desc, q.data_ptr(), _ptr(k), _ptr(wq), _ptr(wk), _ptr(positions),
                _ptr(inv_freq), yq.data_ptr(), _ptr(yk))
    return yq, yk


def _bwd(plan, desc, gq, gk, q, k, wq, wk, positions, inv_freq, dq, dk, need_wq, need_wk):
    """(dwq, dwk); dq and dk are written"""
    dwq = wq.new_empty(wq.shape) if need_wq else None
    dwk = wk.new_empty(wk.shape) if need_wk else None
    # (the call's own workspace: two streams, or two captured graphs, never share it)
    ws = gq.new_empty(plan.ws, dtype=torch.float32) if need_wq or need_wk else None
    _lib.launch(gq.get_device(), _lib.lib().vil_qk_rope_bwd, desc, gq.data_ptr(), _ptr(gk), _ptr(q), _ptr(k), _ptr(wq), _ptr(wk),
                _ptr(positions), _ptr(inv_freq), dq.data_ptr(), _ptr(dk), _ptr(dwq), _ptr(dwk), _ptr(ws))
    return dwq, dwk


class _QKRope(torch.autograd.Function):
    @staticmethod
    @_lib.untraced
    def forward(ctx, q, k, wq, wk, positions, inv_freq, plan):
        """plan: a _Plan of tensors that _inputs has seen, or _inputs' name and options"""
        if not isinstance(plan, _Plan):
            plan, q, k, wq, wk, positions, inv_freq = _inputs(plan[0], q, k, wq, wk, positions, inv_freq, *plan[1:])
        ctx.plan = plan
        # without the norm the gradient is the rotation back: the inputs need not be kept
        ctx.save_for_backward(*((q, k) if plan.norm else (None, None)), wq, wk, positions, inv_freq)
        return _fwd(plan, q, k, wq, wk, positions, inv_freq)

    @staticmethod
    def backward(ctx, gq, gk):
        if not torch.is_grad_enabled():
            return _QKRope.first(ctx, gq, gk)
        # under create_graph: the same values, and an error where a second derivative is asked of them.  The rotation alone is linear: its
        # gradient depends on the incoming one only, the norm's on q and k too.
        return (_QKRope.of_norm if ctx.plan.norm else _QKRope.of_rotation)(ctx, gq, gk)

    @staticmethod
    def first(ctx, gq, gk):
        q, k, wq, wk, positions, inv_freq = ctx.saved_tensors
        plan, need = ctx.plan, ctx.needs_input_grad
        desc = plan.bwd
        if not gq.is_contiguous() or (gk is not None and not gk.is_contiguous()):
            gq, gk = _rows(gq), _rows(gk) if gk is not None else None
            desc = plan.bwd_desc(gq, gk)
        dq = gq.new_empty(plan.qs)
        dk = gk.new_empty(plan.ks) if gk is not None else None
        dwq, dwk = _bwd(plan, desc, gq, gk, q, k, wq, wk, positions, inv_freq, dq, dk, need[2], need[3])
        return dq, dk, dwq, dwk, None, None, None

    of_rotation = staticmethod(torch.autograd.function.once_differentiable(lambda ctx, gq, gk: _QKRope.first(ctx, gq, gk)))
    of_norm = staticmethod(_lib.first_derivative_only(lambda ctx, gq, gk: _QKRope.first(ctx, gq, gk)))


def _inputs(name, q, k, wq, wk, positions, inv_freq, sections, layout, norm, eps):
    """the call's plan and its tensors in the layouts that the kernels take"""
    if q.dim() == 4:
        q = _rows(q)
    if k is not None and k.dim() == 4:
        k = _rows(k)
    if positions is not None:
        if positions.dim() >= 2 and positions.stride(-1) != 1 and positions.shape[-1] != 1:
            positions = positions.contiguous()
        if inv_freq is not None and not inv_freq.is_contiguous():
            inv_freq = inv_freq.contiguous()
    if wq is not None and not wq.is_contiguous():
        wq = wq.contiguous()
    if wk is not None and not wk.is_contiguous():
        wk = wk.contiguous()
    sections = tuple(map(int, sections)) if sections is not None else None
    return _plan(name, q, k, wq, wk, positions, inv_freq, sections, layout, norm, eps), q, k, wq, wk, positions, inv_freq


def _apply(name, q, k, wq, wk, positions, inv_freq, sections, layout, norm, eps):
    if forward_ad._current_level >= 0 or _lib._trace() is not None:
        # a tangent, which only the node refuses; a trace, which records the node and not the launch, and whose sizes are no
        # numbers outside it
        yq, yk = _QKRope.apply(q, k, wq, wk, positions, inv_freq, (name, sections, layout, norm, eps))
        return yq if k is None else (yq, yk)
    plan, *args = _inputs(name, q, k, wq, wk, positions, inv_freq, sections, layout, norm, eps)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in args[:4]):
        yq, yk = _QKRope.apply(*args, plan)
    else:
        yq, yk = _fwd(plan, *args)
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
    return _apply("vil_qk_norm_rope", q, k, q_weight, k_weight, positions, inv_freq, sections, layout, True, float(eps))


class HeadNorm(torch.nn.Module):
    """The (M,) weight of a root-mean-square norm that every head of q, or of k, shares (a parameter `weight`, which
    MsViT.no_weight_decay's rule leaves undecayed); the norm itself runs in the attention's node."""

    def __init__(self, head_dim):
        super().__init__()
        self.weight = torch.nn.Parameter(torch.ones(head_dim))


class QKOptions:
    """Of layers with q_norm, k_norm and turn: one that was pickled before it had them has none."""

    def __setstate__(self, state):
        super().__setstate__(state)
        for name in ("q_norm", "k_norm", "turn"):
            if not hasattr(self, name):
                setattr(self, name, None)


class GridTurn:
    """The rotation of a layer on an nx x ny token grid behind nglo global tokens: half of a head's pairs turn with the row,
    half with the column (the rows take the odd one).  `of(nx, ny, nglo, device)` gives vil_rotary_attention_qkv's positions,
    inv_freq, sections and layout; each grid's tensors are made once (before a stream capture: the layer's first run)."""

    def __init__(self, head_dim, base=10000.0, layout="half"):
        if head_dim % 4:
            raise ValueError(f"GridTurn: a head of {head_dim} channels (a multiple of 4: two axes)")
        if layout not in _LAYOUTS:
            raise ValueError(f"GridTurn: layout {layout!r}")
        pairs = head_dim // 2
        self.sections, self.base, self.layout = (pairs - pairs // 2, pairs // 2), base, layout
        self._made = {}

    def __getstate__(self):
        # a copy or a pickle makes its own: loaded onto another device, these would be there under this one's name
        return {**self.__dict__, "_made": {}}

    def of(self, nx, ny, nglo, device):
        key = (int(nx), int(ny), int(nglo), device)
        made = self._made.get(key)
        if made is None:
            with torch.inference_mode(False):            # (an evaluation may come first, and training save them)
                made = self._made[key] = dict(positions=grid_positions(nx, ny, nglo=nglo, device=device), sections=self.sections,
                                              inv_freq=rotary_frequencies(self.sections, self.base, device), layout=self.layout)
        return made
