"""Activations held in 8 bits between the forward and the backward pass (libvilattn.so: vil_act8_* / vil_gelu_act8_*,
csrc/vil_act8.hip; vil_gemm_*_act8_bf16, csrc/vil_gemm_fused.hip): a general pack / unpack, the exact GELU whose backward
pass reads its pre-activation from the packed form, and the MLP block built from them, whose products carry both in their
epilogues where that is faster.

The reference's Mlp (src/models/msvit.py:17-34) keeps its input, fc1's output h and gelu(h) for the backward pass: 9 C values
of 16 bits a token.  vil_mlp_act8 keeps the input and h in 8 bits (5 C of 1 1/32 bytes) and recomputes gelu from the packed h
for fc2's weight gradient: 29 % of the bytes.  The forward result is the uncompressed one; gradients see the rounding.
There is no eager fallback: CPU tensors or a missing library raise."""
import torch
import torch.nn.functional as F

from . import _lib
from .linear import _fwd_gemm, _bwd_gemm, _wgrad, _colsum

_DT = {torch.float32: _lib.DTYPE_F32, torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_F16}
BLOCK = 32
_MAX_BLOCKS = (2 ** 24 - 1) * 128          # what one launch holds (csrc/vil_act8.hip)


class Act8:
    """A packed activation: codes int8 (rows, cols), scales uint8 (rows, ceil(cols / 32)), the shape and type it had.
    32 neighbouring channels of a row share the power of two 2^(scale - 127), the smallest with max |x| <= 127 * 2^e; a
    value is code * 2^e, code = round(x / 2^e) to even.  Scale 255: the block held an infinity or NaN and stands for NaN."""
    __slots__ = ("codes", "scales", "shape", "dtype")

    def __init__(self, codes, scales, shape, dtype):
        self.codes, self.scales, self.shape, self.dtype = codes, scales, torch.Size(shape), dtype

    @property
    def device(self):
        return self.codes.device

    def nbytes(self):
        return self.codes.numel() + self.scales.numel()


def _check(x, name):
    if x.dtype not in _DT:
        raise TypeError(f"{name} supports float32 / bfloat16 / float16; got {x.dtype}")
    if x.dim() < 1:
        raise ValueError(f"{name}: a tensor with at least one axis")
    n, cols = x.numel(), x.shape[-1]
    if cols >= 2 ** 31 or (n > _MAX_BLOCKS and n // cols * -(-cols // BLOCK) > _MAX_BLOCKS):
        raise ValueError(f"{name}: {tuple(x.shape)} is too large (2^31 blocks of {BLOCK} channels, filled or not)")
    if not x.is_cuda:
        raise RuntimeError(f"{name} needs device tensors: the product path is the HIP kernels (libvilattn.so); there is no CPU "
                           "fallback")


def _check_packed(p, name):
    c, e = p.codes, p.scales
    if (c.dtype != torch.int8 or e.dtype != torch.uint8 or c.dim() != 2 or tuple(e.shape) != (c.shape[0], -(-c.shape[1] // BLOCK))
            or not p.shape or c.shape[1] != p.shape[-1] or c.numel() != p.shape.numel() or not c.is_contiguous() or not e.is_contiguous()):
        raise ValueError(f"{name}: codes {tuple(c.shape)} {c.dtype} and scales {tuple(e.shape)} {e.dtype} of {tuple(p.shape)}")
    if not c.is_cuda or e.device != c.device:
        raise RuntimeError(f"{name} needs device tensors: the product path is the HIP kernels (libvilattn.so); there is no CPU "
                           "fallback")


def _rows(x):
    """x as (rows, cols) with contiguous columns and rows a fixed stride apart (a view where the layout allows it)"""
    cols = x.shape[-1]
    if x.dim() != 2:
        x = x.reshape(x.numel() // cols if cols else 0, cols)
    return x if x.is_contiguous() or ((x.stride(1) == 1 or cols == 1) and x.stride(0) >= cols) else x.contiguous()


def _empty(x2):
    rows, cols = x2.shape
    return x2.new_empty((rows, cols), dtype=torch.int8), x2.new_empty((rows, -(-cols // BLOCK)), dtype=torch.uint8)


def vil_act8_pack(x):
    """x (..., C), fp32 / bf16 / fp16, in 8 bits: an Act8.  No gradient (the packed form is what a backward pass keeps)."""
    _check(x, "vil_act8_pack")
    x2 = _rows(x)
    rows, cols = x2.shape
    codes, scales = _empty(x2)
    _lib.launch(x.get_device(), _lib.lib().vil_act8_pack, x2.data_ptr(), _DT[x.dtype], rows, cols, x2.stride(0), codes.data_ptr(),
                scales.data_ptr())
    return Act8(codes, scales, x.shape, x.dtype)


def vil_act8_unpack(packed, dtype=None):
    """The values that `packed` stands for, in the type it was packed from or in `dtype` (rounded once)."""
    dtype = packed.dtype if dtype is None else dtype
    if dtype not in _DT:
        raise TypeError(f"vil_act8_unpack supports float32 / bfloat16 / float16; got {dtype}")
    _check_packed(packed, "vil_act8_unpack")
    codes = packed.codes
    rows, cols = codes.shape
    y = codes.new_empty(packed.shape, dtype=dtype)
    _lib.launch(codes.get_device(), _lib.lib().vil_act8_unpack, codes.data_ptr(), packed.scales.data_ptr(), rows, cols, y.data_ptr(),
                _DT[dtype])
    return y


def vil_gelu_act8_fwd(h):
    """(gelu(h), h packed): the exact GELU and the packed pre-activation in one pass.  No gradient; see vil_gelu_act8."""
    _check(h, "vil_gelu_act8_fwd")
    h2 = _rows(h)
    rows, cols = h2.shape
    codes, scales = _empty(h2)
    a = h2.new_empty(h.shape)
    _lib.launch(h.get_device(), _lib.lib().vil_gelu_act8_fwd, h2.data_ptr(), _DT[h.dtype], rows, cols, h2.stride(0), a.data_ptr(),
                codes.data_ptr(), scales.data_ptr())
    return a, Act8(codes, scales, h.shape, h.dtype)


def vil_gelu_act8_bwd(packed, da, want_act=True):
    """(dh, a): da * gelu'(v) and, with want_act, gelu(v) (else None), v the values the packed pre-activation stands for."""
    _check(da, "vil_gelu_act8_bwd")
    if da.shape != packed.shape or da.dtype != packed.dtype:
        raise ValueError(f"vil_gelu_act8_bwd: da is {tuple(da.shape)} {da.dtype}, h was {tuple(packed.shape)} {packed.dtype}")
    _check_packed(packed, "vil_gelu_act8_bwd")
    if da.device != packed.device:
        raise RuntimeError(f"vil_gelu_act8_bwd: tensors on {da.device} and {packed.device}")
    g2 = _rows(da)
    rows, cols = g2.shape
    dh = g2.new_empty(da.shape)
    a = g2.new_empty(da.shape) if want_act else None
    _lib.launch(da.get_device(), _lib.lib().vil_gelu_act8_bwd, packed.codes.data_ptr(), packed.scales.data_ptr(), g2.data_ptr(),
                _DT[da.dtype], rows, cols, g2.stride(0), dh.data_ptr(), a.data_ptr() if want_act else None)
    return dh, a


class _GeluAct8Fn(torch.autograd.Function):
    @staticmethod
    @_lib.untraced
    def forward(ctx, h):
        a, packed = vil_gelu_act8_fwd(h)
        ctx.save_for_backward(packed.codes, packed.scales)
        ctx.was = (packed.shape, packed.dtype)
        return a

    @staticmethod
    @_lib.first_derivative_only
    def backward(ctx, da):
        dh, _ = vil_gelu_act8_bwd(Act8(*ctx.saved_tensors, *ctx.was), da, want_act=False)
        return dh


def vil_gelu_act8(h):
    """gelu(h) (exact form) that keeps h in 8 bits for its gradient."""
    _check(h, "vil_gelu_act8")
    return _GeluAct8Fn.apply(h)


def _linear(x2, w, b):
    y = _fwd_gemm(x2, w, b)
    return y if y is not None else F.linear(x2, w, b)


# fc1 with the GELU and the packing in its epilogue, and fc2's input gradient with the GELU's backward on the packed form in its
# epilogue (csrc/vil_gemm_fused.hip), against the library's product and vil_act8.hip's pass over its output; N = 4 K, device us, fused / separate:
#   T x K     100352 x 96   100352 x 192   25088 x 384   25088 x 768   25088 x 1024   2048 x 192    1024 x 384    512 x 192
#   forward      51 / 55       104 / 149       67 / 72      182 / 192      320 / 269    8.5 / 9.6    9.9 / 11.1    8.0 / 8.2
#   backward     55 / 74       138 / 186       76 / 90      236 / 232      382 / 328    9.8 / 11.5   12.4 / 13.1   9.2 / 8.7
# A longer K makes the product the larger part, and the library's is the faster one; few tokens are few tiles.
_FUSE_MIN_T = 1024
_FUSE_FWD_MAX_K, _FUSE_BWD_MAX_K = 768, 384


def _aligned(*ts):
    return all(t is None or (t.dtype == torch.bfloat16 and t.stride(-1) == 1 and t.data_ptr() % 16 == 0
                             and (t.dim() == 1 or (t.stride(0) % 8 == 0 and t.stride(0) >= t.shape[1]))) for t in ts)


def _fused(fn, T, K, N, rs, ts, outs):
    try:
        _lib.launch(outs[0].get_device(), fn, *[t.data_ptr() if t is not None else None for t in ts], *[t.data_ptr() for t in outs], T, K, N, rs, N)
    except _lib.VilAttnError as e:
        if e.code != _lib.VIL_E_BACKEND:
            raise
        return False
    return True


def _fused_fwd(x2, w, b):
    """(gelu(h), h packed) of h = x2 @ w.T + b in one launch that never stores h; None where the separate ones are taken"""
    T, K = x2.shape
    N = w.shape[0]
    if T < _FUSE_MIN_T or K > _FUSE_FWD_MAX_K or K % 32 or N % 128 or not (_aligned(x2, w, b) and w.is_contiguous()):
        return None
    a = x2.new_empty((T, N))
    codes, scales = _empty(a)
    if not _fused(_lib.lib().vil_gemm_gelu_act8_bf16, T, K, N, x2.stride(0), (x2, w, b), (a, codes, scales)):
        return None
    return a, Act8(codes, scales, a.shape, a.dtype)


def _fused_bwd(dy2, w, packed):
    """((dy2 @ w) * gelu'(v), gelu(v)), v the packed values, in one launch; None where the separate ones are taken"""
    T, K = dy2.shape
    N = w.shape[1]
    if T < _FUSE_MIN_T or K > _FUSE_BWD_MAX_K or K % 32 or N % 128 or not (_aligned(dy2, w) and w.is_contiguous()):
        return None
    dh, a = dy2.new_empty((T, N)), dy2.new_empty((T, N))
    if not _fused(_lib.lib().vil_gemm_dgelu_act8_bf16, T, K, N, dy2.stride(0), (dy2, w, packed.codes, packed.scales), (dh, a)):
        return None
    return dh, a


def _weight_grad(dy2, x2, w, want_b):
    fused = _wgrad(dy2, x2, want_b)
    if fused is not None:
        return fused[0].to(w.dtype), fused[1]
    return (dy2.t() @ x2).to(w.dtype), _colsum(dy2) if want_b else None


class _MlpAct8Fn(torch.autograd.Function):
    @staticmethod
    @torch.amp.custom_fwd(device_type="cuda")
    @_lib.untraced
    def forward(ctx, x, w1, b1, w2, b2):
        x2 = _rows(x)
        fused = _fused_fwd(x2, w1, b1)
        a, h8 = fused if fused is not None else vil_gelu_act8_fwd(_linear(x2, w1, b1))
        y = _linear(a, w2, b2)
        x8 = vil_act8_pack(x2) if ctx.needs_input_grad[1] else None      # (x serves fc1's weight gradient alone)
        ctx.save_for_backward(*((x8.codes, x8.scales) if x8 is not None else (None, None)), h8.codes, h8.scales, w1, w2)
        ctx.was = (x.shape, x2.shape, h8.shape, x.dtype, h8.dtype, b1 is not None, b2 is not None)
        return y.view(*x.shape[:-1], w2.shape[0])

    @staticmethod
    @torch.amp.custom_bwd(device_type="cuda")
    @_lib.first_derivative_only
    def backward(ctx, dy):
        xc, xs, hc, hs, w1, w2 = ctx.saved_tensors
        shape, xshape, hshape, xt, ht, has_b1, has_b2 = ctx.was
        need = ctx.needs_input_grad
        dy2 = _rows(dy)                                                 # (a broadcast gradient's rows overlap: copied)
        h8 = Act8(hc, hs, hshape, ht)
        fused = _fused_bwd(dy2, w2, h8)
        if fused is not None:
            dh, a = fused
        else:
            da = _bwd_gemm(dy2, w2)
            dh, a = vil_gelu_act8_bwd(h8, da if da is not None else dy2 @ w2, want_act=need[3])
        dx = dw1 = db1 = dw2 = db2 = None
        if need[3]:
            dw2, db2 = _weight_grad(dy2, a, w2, has_b2 and need[4])
        elif has_b2 and need[4]:
            db2 = _colsum(dy2)
        if need[1]:
            dw1, db1 = _weight_grad(dh, vil_act8_unpack(Act8(xc, xs, xshape, xt)), w1, has_b1 and need[2])
        elif has_b1 and need[2]:
            db1 = _colsum(dh)
        if need[0]:
            dx = _bwd_gemm(dh, w1)
            dx = (dx if dx is not None else dh @ w1).view(shape)
        return dx, dw1, db1, dw2, db2


def vil_mlp_act8(x, w1, b1, w2, b2):
    """F.linear(F.gelu(F.linear(x, w1, b1)), w2, b2) (exact GELU) that keeps x and the pre-activation in 8 bits for the
    backward pass; same autocast semantics as vil_linear.  w1 (D, C), w2 (C', D); biases may be None."""
    if torch.is_autocast_enabled("cuda"):
        dt = torch.get_autocast_dtype("cuda")
        x, w1, w2 = x.to(dt), w1.to(dt), w2.to(dt)
        b1, b2 = (b.to(dt) if b is not None else None for b in (b1, b2))
    _check(x, "vil_mlp_act8")
    if w1.dim() != 2 or w2.dim() != 2 or w1.shape[1] != x.shape[-1] or w2.shape[1] != w1.shape[0]:
        raise ValueError(f"vil_mlp_act8: x {tuple(x.shape)}, w1 {tuple(w1.shape)}, w2 {tuple(w2.shape)}")
    if not (w1.dtype == w2.dtype == x.dtype) or any(b is not None and b.dtype != x.dtype for b in (b1, b2)):
        raise TypeError(f"vil_mlp_act8: x is {x.dtype}, the parameters are {w1.dtype}, {w2.dtype}")
    if any(b is not None and b.shape != w.shape[:1] for b, w in ((b1, w1), (b2, w2))):
        raise ValueError(f"vil_mlp_act8: biases {[tuple(b.shape) for b in (b1, b2) if b is not None]} of weights {tuple(w1.shape)}, {tuple(w2.shape)}")
    if any(p is not None and p.device != x.device for p in (w1, b1, w2, b2)):
        raise RuntimeError(f"vil_mlp_act8: x is on {x.device}, a parameter is not")
    with torch.autocast("cuda", enabled=False):
        return _MlpAct8Fn.apply(x, w1, b1, w2, b2)
