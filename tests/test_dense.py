"""CPU checks of the dense operators: refusals that need no device, and the 64-bit results that the GPU
tests compare with (differences against the gradients' formulas, the 8-bit form against the number format)."""
import ctypes

import numpy as np
import pytest

from silentotithrandousha_amd import MOE_BF16, MOE_F32, _ffi
from tests import dense_ref as ref


def test_null_context_and_sizes():
    L = _ffi.lib()
    b, g = _ffi.GatedFfn(8), _ffi.GatedFfnGrads()
    calls = [lambda: L.moe_lm_head_loss_device(None, None, 0, None, 1, 1, None, None, None),
             lambda: L.moe_lm_head_loss_backward_device(None, None, 0, None, None, None, 1, 1, None, None, None),
             lambda: L.moe_ffn_forward_device(None, ctypes.byref(b), None, 0, 1, None, None, None),
             lambda: L.moe_ffn_backward_device(None, ctypes.byref(b), None, 0, None, 0, 1, ctypes.byref(g), None),
             lambda: L.moe_act8_pack_device(None, None, 0, 1, 32, None, None),
             lambda: L.moe_act8_unpack_device(None, None, 1, 32, None, 0, None)]
    for call in calls:
        assert call() == _ffi.MOE_ERR_INVALID
        assert b"null context" in L.moe_last_error()
    assert L.moe_act8_bytes(3, 64) == 3 * 64 + 3 * 2
    assert L.moe_act8_bytes(3, 33) == 0 and L.moe_act8_bytes(0, 32) == 0


def test_bf16_helpers():
    x = np.array([1.0, 1.00390625, 1.01171875, -3.1, 0.0, 65504.0], np.float32)
    b = ref.from_bf16(ref.to_bf16(x))
    assert np.array_equal(b[:3], np.array([1.0, 1.0, 1.015625], np.float32))  # ties to even
    assert (np.abs(b - x) <= np.abs(x) * 2.0 ** -8).all()


@pytest.mark.parametrize("V", [1, 7])
def test_loss_reference(V):
    rng = np.random.default_rng(V)
    x, w = rng.standard_normal((4, 6)), rng.standard_normal((V, 6))
    targets, dloss = np.array([0, V - 1, -1, 0]), rng.standard_normal(4)
    at = ref.Loss(x, w, targets, dloss, MOE_F32)
    for name, v in (("dx", x), ("dw", w)):
        d, h = rng.standard_normal(v.shape), 1e-5

        def total(s):
            args = (x + s * d, w) if name == "dx" else (x, w + s * d)
            return float(ref.Loss(*args, targets, dloss, MOE_F32).loss @ dloss)

        numeric = (total(h) - total(-h)) / (2 * h)
        # third derivatives below 100 here, and 16 digits
        assert abs(numeric - (getattr(at, name) * d).sum()) < 100 * h * h + 1e-9


def test_block_reference():
    rng = np.random.default_rng(3)
    T, H, I = 3, 5, 4  # noqa: E741
    p = dict(x=rng.standard_normal((T, H)) * 2, wgu=rng.standard_normal((2 * I, H)) * 2, bgu=rng.standard_normal(2 * I),
             wd=rng.standard_normal((H, I)), bd=rng.standard_normal(H))
    dy = rng.standard_normal((T, H))
    at = ref.Block(**p, dy=dy, dtype=MOE_F32)
    gu = p["x"] @ p["wgu"].T + p["bgu"]
    assert (gu[:, 0::2] > 7).any() and (np.abs(gu[:, 1::2]) > 7).any()  # the clamps are reached
    for name, grad in (("x", "dx"), ("wgu", "dwgu"), ("bgu", "dbgu"), ("wd", "dwd"), ("bd", "dbd")):
        d, h = rng.standard_normal(p[name].shape), 1e-6

        def total(s):
            return float((ref.Block(**dict(p, **{name: p[name] + s * d}), dy=None, dtype=MOE_F32).y * dy).sum())

        numeric = (total(h) - total(-h)) / (2 * h)
        assert abs(numeric - (getattr(at, grad) * d).sum()) < 1e-6, name


@pytest.mark.parametrize("dtype", [MOE_F32, MOE_BF16])
def test_act8_reference(dtype):
    """Every e4m3 value under every scale is its own code; nothing saturates; half a step at most."""
    pos = [m / 8 * 2.0 ** -6 for m in range(8)] + [(1 + m / 8) * 2.0 ** (k - 7) for k in range(1, 16) for m in range(8)]
    vals = np.array(pos[:127])
    for e in (-100, -1, 0, 5, 100):
        x = np.zeros((1, 160))
        x[0, :127], x[0, 127:159:32] = vals, 0
        x[0, [31, 63, 95, 127, 159]] = 448.0  # the same scale for every block
        codes, scales, values = ref.act8(x * 2.0 ** e)
        assert (scales == e + 127).all() and np.array_equal(values, x * 2.0 ** e)
        keep = np.setdiff1d(np.arange(127), [31, 63, 95])
        assert np.array_equal(codes[0, keep], keep)
    rng = np.random.default_rng(4)
    x = ref.rows(rng, (50, 320), dtype)[1]
    codes, scales, values = ref.act8(x)
    top = np.abs(x).reshape(50, -1, 32).max(-1)
    s = 2.0 ** (scales.astype(int) - 127.0)
    assert (top <= 448 * s).all() and (top > 224 * s).all()
    assert (np.abs(values - x) <= np.maximum(2.0 ** -4 * np.abs(x), (2.0 ** -10 * s).repeat(32, 1))).all()
