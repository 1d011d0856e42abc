"""CPU: the largest tensors of the 8-bit form.  A launch holds under 2^32 work items; a block of 32 channels takes four lanes, two
blocks' worth to a work item, however few of its channels a narrow row fills."""
import ctypes

import pytest
import torch

from vision_longformer_amd import _lib, act8

A16 = ctypes.c_void_p(4096)          # an aligned address that no refused call reads
MOST = (2 ** 24 - 1) * 128           # blocks


@pytest.mark.parametrize("rows,cols", [(MOST + 1, 1), (2 ** 31, 1), (MOST + 1, 32), (MOST // 2 + 1, 33), (2 ** 26, 1024), (32, 2 ** 31 - 1),
                                       (2 ** 36, 1), (2 ** 62, 2), (2 ** 62, 2 ** 31 - 1)])
def test_the_c_entries_refuse_more(rows, cols):
    L, t = _lib.lib(), _lib.DTYPE_BF16
    assert L.vil_act8_pack(A16, t, rows, cols, cols, A16, A16, None) == -2
    assert L.vil_act8_unpack(A16, A16, rows, cols, A16, t, None) == -2
    assert L.vil_gelu_act8_fwd(A16, t, rows, cols, cols, A16, A16, A16, None) == -2
    assert L.vil_gelu_act8_bwd(A16, A16, A16, t, rows, cols, cols, A16, None, None) == -2


@pytest.mark.parametrize("rows,cols,fits", [(MOST, 1, True), (MOST + 1, 1, False), (MOST, 32, True), (MOST + 1, 32, False), (MOST // 2, 33, True),
                                            (MOST // 2 + 1, 33, False), (2 ** 26, 1024, False), (1, 2 ** 31, False), (32, 2 ** 31 - 1, False), (5, 0, True)])
def test_the_python_calls_refuse_more(rows, cols, fits):
    """(tensors without memory: one that fits is refused for its device)"""
    x = torch.empty(rows, cols, dtype=torch.bfloat16, device="meta")
    for fn in (act8.vil_act8_pack, act8.vil_gelu_act8_fwd, act8.vil_gelu_act8):
        with pytest.raises(RuntimeError if fits else ValueError, match="device tensors" if fits else "too large"):
            fn(x)
