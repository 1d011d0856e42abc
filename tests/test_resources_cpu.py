"""CPU: hipcc's resource report of the last build for the products with an epilogue of their own (csrc/vil_gemm_fused.hip)."""
import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.parametrize("kernel,waves", [("k_dgrad_dgelu", 4), ("k_fwd_gelu", 3)])
def test_products_with_an_epilogue_hold_no_scratch(kernel, waves):
    """a reload between a tile's stores waits for all of them; the launch bounds' residency (two workgroups of five waves to a CU need
    four waves a SIMD of k_dgrad_dgelu: 128 registers)"""
    sys.path.insert(0, ROOT)
    import __graft_entry__ as g
    if not os.path.exists(os.path.join(g.OBJ_DIR, "vil_gemm_fused.resources.txt")):
        g.build()
    res = {k: v for k, v in g.kernel_resources().items() if kernel in k}
    assert len(res) == 3, sorted(res)                            # plain, GELU, GELU in its 8-bit form
    for k, v in res.items():
        assert v["scratch"] == 0 and v["occupancy"] >= waves, (k, v)


def test_build_takes_the_arguments_that_it_took():
    """build(), build(True) and build(force=...) are calls that callers have; nothing is compiled here"""
    import inspect
    sys.path.insert(0, ROOT)
    import __graft_entry__ as g
    for args, kw in (((), {}), ((True,), {}), ((), dict(force=True)), ((), dict(force=False))):
        inspect.signature(g.build).bind(*args, **kw)
