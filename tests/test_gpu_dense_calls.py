"""What a call of the dense operators leaves for the next one: errors, workspaces."""
import ctypes

import numpy as np
import pytest

from silentotithrandousha_amd import MOE_BF16, MOE_F32, DeviceBuffer, GatedFfn, MoeError, _ffi
from silentotithrandousha_amd._ffi import LIB_PATH, check, lib
from tests import dense_ref as ref
from tests.test_gpu_dense import BlockOnDevice, Out, block_case, context, dev, loss_case, run_loss

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


def test_checkpoints_of_2_to_35_values():
    """More values than a launch has threads for: 2^20 rows of 32768 bf16 values packed and read back in place of the rows;
    rows at the start, around 2^34 values and at the end are those of a small call."""
    T, cols = 2**20, 32768
    d = context(32)
    try:
        x, packed = DeviceBuffer(T * cols * 2), DeviceBuffer(d.act8_bytes(T, cols))
        for i in range(32):
            check(lib().moe_synth_fill_device(x.ptr + (i << 31), 1 << 30, 1, i, 1.0, 0.0, None))
        check(lib().moe_synchronize(d.ctx))

        def rows(t, n, back):
            """(codes and scales of n rows from t, or what x holds there)"""
            out = np.empty((n, cols), np.uint16)
            check(lib().moe_memcpy_d2h(out.ctypes.data, x.ptr + t * cols * 2, out.nbytes))
            if back:
                return out
            codes, scales = np.empty((n, cols), np.uint8), np.empty((n, cols // 32), np.uint8)
            check(lib().moe_memcpy_d2h(codes.ctypes.data, packed.ptr + t * cols, codes.nbytes))
            check(lib().moe_memcpy_d2h(scales.ctypes.data, packed.ptr + T * cols + t * (cols // 32), scales.nbytes))
            return codes, scales, ref.act8(ref.from_bf16(out).astype(np.float64))

        places = (0, T // 2 - 1, T // 2 + 1, T - 2)
        d.act8_pack_device(x, MOE_BF16, T, cols, packed)
        d.synchronize()
        values = {}
        for t in places:
            codes, scales, want = rows(t, 2, False)
            assert np.array_equal(codes, want[0]) and np.array_equal(scales, want[1])
            values[t] = want[2]
        d.act8_unpack_device(packed, T, cols, x, MOE_BF16)
        d.synchronize()
        for t in places:
            assert np.array_equal(ref.from_bf16(rows(t, 2, True)).astype(np.float64), values[t])
    finally:
        d.close()


def test_a_wide_head():
    """2^25 rows of the head and 700 tokens: pieces of tokens, and a grid that one launch of them all would be too large for."""
    T, H, V = 700, 32, 2**25
    rng = np.random.default_rng(1)
    d = context(H)
    try:
        w = DeviceBuffer(V * H * 2)
        check(lib().moe_memset_device(w.ptr, 0, V * H * 2))  # every logit 0 but those of the last rows
        tail, tv = ref.rows(rng, (300, H), MOE_BF16, 2 / np.sqrt(H))
        check(lib().moe_memcpy_h2d(w.ptr + (V - 300) * H * 2, tail.ctypes.data, tail.nbytes))
        check(lib().moe_init_lm_head_bf16_device(d.ctx, w.ptr, V, None))
        x, xv = ref.rows(rng, (T, H), MOE_BF16)
        targets = rng.integers(V - 300, V, T).astype(np.int32)
        xd, td, loss, lse = run_loss(d, x, MOE_BF16, targets, V)
        logits = xv @ tv.T
        want = np.log(np.exp(logits).sum(1) + (V - 300))
        # 128 terms of a part, then up to 512 parts a thread and 10 joins, a rounding of 2^-24 each: 2^-14.6 of the sum
        tol = 2.0 ** -14 + 2.0 ** -20 * np.abs(want)
        ref.assert_close(lse.get(), want, tol, "lse")
        ref.assert_close(loss.get(), want - logits[np.arange(T), targets - (V - 300)], 2 * tol, "loss")
    finally:
        d.close()


def test_an_error_of_the_caller_is_not_the_calls():
    """An allocation of the caller's own fails, and the caller has not asked for the error: the calls behind it succeed, and
    leave it to the caller."""
    hip = ctypes.CDLL(LIB_PATH)  # (the library's HIP runtime)
    for name in ("hipMalloc", "hipGetLastError"):
        getattr(hip, name).restype = ctypes.c_int
    T, H, V, I = 20, 64, 100, 40  # noqa: E741
    x, xv, w, wv, targets, dloss = loss_case(MOE_F32, T, H, V)
    c = block_case(MOE_F32, T, H, I)
    d = context(H, w)
    try:
        xd, td, loss, lse = run_loss(d, x, MOE_F32, targets, V)
        b, gd, dx, dw = BlockOnDevice(c), dev(dloss), Out((T, H), MOE_F32), Out((V, H), MOE_F32)
        packed = DeviceBuffer(d.act8_bytes(T, H))
        hip.hipGetLastError()
        assert hip.hipMalloc(ctypes.byref(ctypes.c_void_p()), ctypes.c_size_t(2**46)) == 2  # out of memory
        d.lm_head_loss_device(xd, MOE_F32, td, T, V, loss, lse)
        d.lm_head_loss_backward_device(xd, MOE_F32, td, lse, gd, T, V, dx, dw)
        b.forward(d, MOE_F32, x8=packed)
        b.backward(d, MOE_F32)
        d.act8_pack_device(xd, MOE_F32, T, H, packed)
        d.act8_unpack_device(packed, T, H, dx, MOE_F32)
        assert hip.hipGetLastError() == 2
        d.synchronize()
        want = ref.Loss(xv, wv, targets, dloss.astype(np.float64), MOE_F32)
        ref.assert_close(loss.get(), want.loss, want.loss_tol, "loss")
        ref.assert_close(dw.get(), want.dw, want.dw_tol, "dw")
    finally:
        d.close()
