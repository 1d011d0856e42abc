"""CPU: rotary positions / per-head norms and 8-bit activations -- argument checks of the Python and the C entry points, the
descriptor's layout, the helpers.  Nothing is launched."""
import ctypes

import pytest
import torch

from vision_longformer_amd import _lib, act8, rotary

F32, BF16, F16, F64 = _lib.DTYPE_F32, _lib.DTYPE_BF16, _lib.DTYPE_F16, _lib.DTYPE_F64
A16 = ctypes.c_void_p(4096)          # an aligned address that no refused call reads


def _desc(**kw):
    d = _lib.VilRopeDesc()
    base = dict(B=2, N=5, Hq=3, Hk=3, M=32, R=16, axes=2, layout=_lib.ROPE_HALF, dtype=BF16, pos_dtype=_lib.POS_I32,
                freq_dtype=F64, norm=1, w_dtype=F32, eps=1e-6)
    sections = kw.pop("sections", (8, 8))
    for k, v in {**base, **kw}.items():
        setattr(d, k, v)
    for i, n in enumerate(sections):
        d.sections[i] = n
    return d


def _fwd(d, q=A16, k=A16, pos=A16, freq=A16, yq=A16, yk=A16):
    return _lib.lib().vil_qk_rope_fwd(ctypes.byref(d) if d is not None else None, q, k, A16, A16, pos, freq, yq, yk, None)


def _bwd(d, q=A16, gq=A16, dq=A16, wq=A16, dwq=A16, ws=A16):
    return _lib.lib().vil_qk_rope_bwd(ctypes.byref(d), gq, A16, q, A16, wq, A16, A16, A16, dq, A16, dwq, A16, ws, None)


def test_rope_descriptor_layout():
    # 7 + 4 + 6 int32, one float, 8 x 3 + 2 int64
    assert ctypes.sizeof(_lib.VilRopeDesc) == 18 * 4 + 26 * 8


@pytest.mark.parametrize("code,kw", [
    (-2, dict(B=-1)), (-2, dict(Hq=0)), (-2, dict(Hk=-1)), (-2, dict(B=1 << 16, N=1 << 15)),
    (-3, dict(M=31)), (-3, dict(M=0)), (-3, dict(M=258)),
    (-2, dict(R=17, sections=(9, 8))), (-2, dict(R=16, sections=(8, 7))), (-2, dict(axes=5)), (-2, dict(axes=0)),
    (-2, dict(sections=(-8, 24))), (-5, dict(layout=2)), (-7, dict(dtype=F64)), (-7, dict(pos_dtype=3)),
    (-7, dict(freq_dtype=BF16)), (-7, dict(w_dtype=F64)), (-2, dict(norm=0, R=0, axes=0, sections=(0, 0)))])
def test_rope_c_entry_refuses(code, kw):
    assert _fwd(_desc(**kw)) == code
    assert _bwd(_desc(**kw)) == code
    assert _lib.lib().vil_qk_rope_workspace_bytes(ctypes.byref(_desc(**kw))) == 0


def test_rope_c_entry_null_pointers_and_empty_batches():
    assert _fwd(None) == -1
    for kw in (dict(q=None), dict(k=None), dict(pos=None), dict(freq=None), dict(yq=None), dict(yk=None)):
        assert _fwd(_desc(), **kw) == -1, kw
    for kw in (dict(q=None), dict(gq=None), dict(dq=None), dict(wq=None)):
        assert _bwd(_desc(), **kw) == -1, kw
    assert _bwd(_desc(), ws=None) == -9
    assert _bwd(_desc(norm=0)) == -1                            # dw without a norm
    for kw in (dict(B=0), dict(N=0)):                           # nothing to do: no pointer is looked at
        assert _fwd(_desc(**kw), q=None, k=None, yq=None, yk=None) == 0
    assert _lib.lib().vil_qk_rope_workspace_bytes(ctypes.byref(_desc())) % (2 * 32 * 4) == 0
    assert _lib.lib().vil_qk_rope_workspace_bytes(ctypes.byref(_desc(norm=0))) == 0


def test_act8_c_entry_refuses():
    L = _lib.lib()
    assert L.vil_act8_pack(None, BF16, 4, 64, 64, A16, A16, None) == -1
    assert L.vil_act8_pack(A16, BF16, 4, 64, 64, A16, None, None) == -1
    assert L.vil_act8_pack(A16, F64, 4, 64, 64, A16, A16, None) == -7
    assert L.vil_act8_pack(A16, BF16, -1, 64, 64, A16, A16, None) == -2
    assert L.vil_act8_pack(A16, BF16, 4, 64, 63, A16, A16, None) == -2          # rows overlap
    assert L.vil_act8_pack(A16, BF16, 1 << 36, 64, 64, A16, A16, None) == -2
    assert L.vil_act8_pack(None, BF16, 0, 64, 64, None, None, None) == 0
    assert L.vil_act8_pack(None, BF16, 4, 0, 0, None, None, None) == 0
    assert L.vil_act8_unpack(A16, A16, 4, 64, None, F16, None) == -1
    assert L.vil_act8_unpack(A16, A16, 4, 64, A16, 7, None) == -7
    assert L.vil_gelu_act8_fwd(A16, BF16, 4, 64, 64, None, A16, A16, None) == -1
    assert L.vil_gelu_act8_fwd(A16, BF16, 4, 64, 32, A16, A16, A16, None) == -2
    assert L.vil_gelu_act8_bwd(A16, A16, None, BF16, 4, 64, 64, A16, None, None) == -1
    assert L.vil_gelu_act8_bwd(A16, A16, A16, BF16, 4, 64, 8, A16, None, None) == -2


def test_act8_product_entries_refuse():
    L = _lib.lib()
    odd = ctypes.c_void_p(4100)
    f = L.vil_gemm_gelu_act8_bf16
    assert f(None, A16, None, A16, A16, A16, 2048, 96, 384, 96, 384, None) == -1
    assert f(A16, A16, None, A16, A16, None, 2048, 96, 384, 96, 384, None) == -1
    assert f(A16, A16, None, A16, A16, A16, 0, 96, 384, 96, 384, None) == -2
    assert f(A16, A16, None, A16, A16, A16, 2048, 96, 384, 88, 384, None) == -2          # rows overlap
    assert f(A16, A16, None, A16, A16, A16, 2048, 96, 384, 96, 376, None) == -2
    assert f(A16, A16, None, A16, odd, A16, 2048, 96, 384, 96, 384, None) == -8
    assert f(A16, A16, odd, A16, A16, A16, 2048, 96, 384, 96, 384, None) == -8
    assert f(A16, A16, None, A16, A16, A16, 2048, 100, 384, 104, 384, None) == -10
    assert f(A16, A16, None, A16, A16, A16, 2048, 96, 400, 96, 400, None) == -10
    g = L.vil_gemm_dgelu_act8_bf16
    assert g(A16, A16, None, A16, A16, A16, 2048, 96, 384, 96, 384, None) == -1
    assert g(A16, A16, A16, A16, A16, A16, 2048, 96, 400, 96, 400, None) == -10
    assert g(A16, A16, A16, ctypes.c_void_p(4097), A16, A16, 2048, 96, 384, 96, 384, None) == -8
    assert g(A16, A16, A16, A16, A16, A16, 2048, 96, 384, 96, 376, None) == -2
    assert g(A16, A16, A16, A16, A16, A16, 1 << 26, 96, 384, 96, 384, None) == -10           # 32-bit offsets


def test_a_packed_form_of_another_row_length_is_refused():
    """(2, 96) in codes of (4, 48) has as many values, but six scales instead of eight"""
    codes, scales = torch.zeros(2, 96, dtype=torch.int8), torch.zeros(2, 3, dtype=torch.uint8)
    for shape in ((4, 48), (192,), ()):
        with pytest.raises(ValueError):
            act8.vil_act8_unpack(act8.Act8(codes, scales, shape, torch.float32))
    with pytest.raises(RuntimeError):
        act8.vil_act8_unpack(act8.Act8(codes, scales, (2, 96), torch.float32))


def _args(**kw):
    a = dict(q=torch.zeros(2, 6, 3, 32), k=torch.zeros(2, 6, 3, 32), positions=torch.zeros(6, 2, dtype=torch.int32),
             inv_freq=torch.ones(16, dtype=torch.float64), sections=(8, 8))
    a.update(kw)
    return a


Z = torch.zeros


@pytest.mark.parametrize("err,kw", [
    (ValueError, dict(q=Z(6, 3, 32))), (TypeError, dict(q=Z(2, 6, 3, 32).double(), k=None)), (TypeError, dict(k=Z(2, 6, 3, 32).half())),
    (ValueError, dict(k=Z(2, 5, 3, 32))), (ValueError, dict(q=Z(2, 6, 3, 33), k=None)), (ValueError, dict(q=Z(2, 6, 3, 512), k=None)),
    (ValueError, dict(q=Z(2, 6, 0, 32), k=None)), (ValueError, dict(positions=None)), (ValueError, dict(sections=(9, 8))),
    (ValueError, dict(sections=(8, 7))), (ValueError, dict(sections=(24, -8))), (ValueError, dict(sections=(4, 3, 3, 3, 3))),
    (ValueError, dict(inv_freq=Z(16).half())), (ValueError, dict(positions=Z(5, 2))), (ValueError, dict(positions=Z(3, 6, 2))),
    (ValueError, dict(positions=Z(6, 2).half())), (ValueError, dict(positions=Z(6, 2, requires_grad=True))),
    (ValueError, dict(layout="pairs")), (RuntimeError, dict())])
def test_vil_rope_refuses(err, kw):
    with pytest.raises(err):
        rotary.vil_rope(**_args(**kw))


@pytest.mark.parametrize("err,kw", [
    (ValueError, dict(q_weight=Z(31))), (ValueError, dict(q_weight=Z(32).double())), (ValueError, dict(k=None, k_weight=Z(32))),
    (TypeError, dict(q_weight=Z(32), k_weight=Z(32).half())), (ValueError, dict(eps=-1.0)), (ValueError, dict(eps=float("nan"))),
    (RuntimeError, dict(positions=None, inv_freq=None, sections=None))])
def test_vil_qk_norm_rope_refuses(err, kw):
    with pytest.raises(err):
        rotary.vil_qk_norm_rope(**_args(**kw))


def test_act8_refuses():
    x = torch.zeros(4, 64)
    for fn in (act8.vil_act8_pack, act8.vil_gelu_act8_fwd, act8.vil_gelu_act8):
        with pytest.raises(RuntimeError):
            fn(x)
        with pytest.raises(TypeError):
            fn(x.double())
        with pytest.raises(ValueError):
            fn(torch.zeros(()))
    p = act8.Act8(torch.zeros(4, 64, dtype=torch.int8), torch.ones(4, 2, dtype=torch.uint8), (4, 64), torch.float32)
    assert p.nbytes() == 4 * 66 and p.device.type == "cpu"
    with pytest.raises(TypeError):
        act8.vil_act8_unpack(p, torch.float64)
    with pytest.raises(RuntimeError):
        act8.vil_act8_unpack(p)
    with pytest.raises(RuntimeError):
        act8.vil_gelu_act8_bwd(p, x)
    for codes, scales in ((p.codes.float(), p.scales), (p.codes[:, ::2], p.scales), (p.codes, p.scales[:, :1]), (p.codes[:3], p.scales[:3])):
        with pytest.raises(ValueError):
            act8.vil_act8_unpack(act8.Act8(codes, scales, (4, 64), torch.float32))
    with pytest.raises(RuntimeError):
        act8.vil_mlp_act8(x, torch.zeros(8, 64), None, torch.zeros(64, 8), None)


def test_positions_and_frequencies():
    pos = rotary.grid_positions(2, 3, nglo=1)
    assert pos.dtype == torch.int32 and pos.tolist() == [[0, 0], [0, 0], [0, 1], [0, 2], [1, 0], [1, 1], [1, 2]]
    assert rotary.grid_positions(2, 2, 2).shape == (8, 3)
    f = rotary.rotary_frequencies((2, 4), base=(100.0, 16.0))
    assert f.dtype == torch.float64 and torch.allclose(f, torch.tensor([1, 0.1, 1, 0.5, 0.25, 0.125], dtype=torch.float64))
    with pytest.raises(ValueError):
        rotary.rotary_frequencies((2, 4), base=(100.0,))
