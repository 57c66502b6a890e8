"""CPU tests of the expert feed-forward entry points: struct layout and null handles."""
import ctypes

import pytest


@pytest.fixture(scope="module")
def fl():
    import build
    build.build()
    import fletcher
    return fletcher


def test_block_norm_struct_layout(fl):
    # FletcherBlockNorm: 2 int32, 3 float, 1 int32, 1 int64, 6 pointers
    assert ctypes.sizeof(fl.CBlockNorm) == 24 + 8 + 48
    assert fl.CBlockNorm.gate_rows.offset == 24 and fl.CBlockNorm.pre_beta.offset == 72


def test_null_handles_are_refused(fl):
    L = fl.lib()
    h = ctypes.c_void_p()
    assert L.Cuda_Routing_Create(None, 1, 2, 1, ctypes.byref(h)) == 1 and not h.value
    assert L.Cuda_Routing_Free(None) == 0
    assert L.Cuda_Routing_TopK(None, None, 0, 0, 0, 1.0) == 1
    assert L.Cuda_Routing_Assign(None, None, None, 0) == 1
    assert L.Cuda_Routing_Read(None, None, None, None, None) == 1
    assert L.Cuda_Routing_DevicePointers(None, None, None, None, None) == 1
    assert L.Cuda_Linear_Grouped(None, None, 0, 1, None, 1, None, None, 0) == 1
    assert L.Cuda_Combine_Grouped(None, None, 1, None, None, None) == 1
    assert L.Cuda_BlockNorm(None, None, 1, 1, None, None, None) == 1
    assert not L.Cuda_WrapTensor(None, None, 1, 1, 0)


def test_block_norm_keeps_its_tensors(fl):
    class T:
        rows, buf = 3, 1234
    n = fl.BlockNorm(pre=fl.NORM_RMS, gate=T(), residual=T())
    assert n.c.gate_rows == 3 and n.c.gate == 1234 and n.c.post_gamma is None
    with pytest.raises(fl.FletcherError):
        n._ref(4)
