"""What a call of the dense operators leaves for the next one: errors, workspaces."""
import numpy as np
import pytest

from silentotithrandousha_amd import MOE_F32, DeviceBuffer, GatedFfn, MoeError, _ffi
from silentotithrandousha_amd._ffi import check, lib
from tests import dense_ref as ref
from tests.test_gpu_dense import context, dev

pytestmark = pytest.mark.gpu


def test_a_call_out_of_memory_leaves_the_next_one_alone():
    """A workspace of terabytes is refused by the allocation, before anything is enqueued; the next call, and one after a
    refused allocation, report nothing of it."""
    T = inter = 2**20
    H = 2880
    d = context(H)
    try:
        x, y = DeviceBuffer(T * H * 4), DeviceBuffer(T * H * 4)
        block = GatedFfn(inter, (wgu := DeviceBuffer(2 * inter * H * 2)).ptr, None, (wd := DeviceBuffer(inter * H * 2)).ptr, None)
        row, packed = dev(np.ones((1, 32), np.float32)), DeviceBuffer(64)
        codes, scales, _ = ref.act8(np.ones((1, 32)))
        for refused in (lambda: d.ffn_forward_device(block, x, MOE_F32, T, y), lambda: DeviceBuffer(2**46)):
            check(lib().moe_memset_device(packed.ptr, 0, 64))
            with pytest.raises(MoeError) as e:
                refused()
            assert e.value.code == _ffi.MOE_ERR_OOM
            d.act8_pack_device(row, MOE_F32, 1, 32, packed)
            d.synchronize()
            assert np.array_equal(packed.download(np.uint8, (33,)), np.append(codes, scales))
        assert wgu.ptr and wd.ptr
    finally:
        d.close()
