"""The dense operators (include/moe_dense.h) against 64-bit results with derived tolerances
(tests/dense_ref.py): the loss over the LM head and its gradient, the gated block and its backward pass,
8-bit checkpoints; their refusals, graphs, streams and workspaces; and a run of them together."""
import ctypes
import gc

import numpy as np
import pytest

from silentotithrandousha_amd import (MOE_BF16, MOE_F32, MOE_MXFP8, DeviceBuffer, GatedFfn, GatedFfnGrads,
                                      GpuMoeDispatcher, MoeError)
from silentotithrandousha_amd import synthetic as syn
from silentotithrandousha_amd._ffi import check, lib
from tests import dense_ref as ref

pytestmark = pytest.mark.gpu

TYPES = [MOE_F32, MOE_BF16]
GUARD = 64  # bytes behind each output that must stay as they were


class Out:
    """An output of `shape`, filled with 0xA5 and followed by guard bytes."""

    def __init__(self, shape, dtype):
        self.shape, self.dtype = shape, dtype
        self.n = int(np.prod(shape)) * (4 if dtype == MOE_F32 else 2)
        self.buf = DeviceBuffer.from_array(np.full(self.n + GUARD, 0xA5, np.uint8))
        self.ptr = self.buf.ptr

    def get(self):
        tail = self.buf.download(np.uint8, (self.n + GUARD,))[self.n:]
        assert (tail == 0xA5).all(), "written behind the output"
        return ref.load(self.buf, self.dtype, self.shape)


def dev(a):
    return DeviceBuffer.from_array(a)


def context(H, w=None, inter=32):
    d = GpuMoeDispatcher(H, inter, ref.CLAMP)
    if w is not None:
        d.init_lm_head_bf16(w, w.shape[0])
    return d


# ------------------------------------------------------------------ loss


def loss_case(dtype, T, H, V, seed=0, scale=2.0):
    rng = np.random.default_rng([seed, T, H, V, dtype])
    x, xv = ref.rows(rng, (T, H), dtype)
    w, wv = ref.rows(rng, (V, H), MOE_BF16, scale / np.sqrt(H))
    targets = rng.integers(0, V, T).astype(np.int32)
    targets[rng.random(T) < 0.2] = -1
    dloss = rng.uniform(-1, 1, T).astype(np.float32)
    return x, xv, w, wv, targets, dloss


def run_loss(d, x, dtype, targets, V, stream=None):
    T = len(targets)
    loss, lse = Out((T,), MOE_F32), Out((T,), MOE_F32)
    xd, td = dev(x), dev(targets)
    d.lm_head_loss_device(xd, dtype, td, T, V, loss, lse, stream)
    lib().moe_synchronize(d.ctx) if stream is None else None
    return xd, td, loss, lse


def run_loss_backward(d, xd, dtype, td, lse, dloss, T, H, V, dx=True, dw=True):
    dx = Out((T, H), dtype) if dx else None
    dw = Out((V, H), dtype) if dw else None
    gd = dev(dloss)
    d.lm_head_loss_backward_device(xd, dtype, td, lse, gd, T, V, dx, dw)
    d.synchronize()
    return dx, dw


# T: one token, both sides of a 16-column tile, of a 128-row tile, more; H: one and several K-steps, tails
# of half a step; V: one row, odd, below and above a tile, not a multiple of 8
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,H,V", [(1, 32, 1), (1, 64, 257), (2, 96, 5), (15, 160, 130), (16, 64, 128), (17, 64, 129),
                                   (127, 32, 1000), (130, 544, 333), (300, 128, 777), (1, 2880, 1003), (33, 1024, 4099)])
def test_loss_and_gradient(dtype, T, H, V):
    x, xv, w, wv, targets, dloss = loss_case(dtype, T, H, V)
    want = ref.Loss(xv, wv, targets, dloss.astype(np.float64), dtype)
    d = context(H, w)
    try:
        xd, td, loss, lse = run_loss(d, x, dtype, targets, V)
        ref.assert_close(lse.get(), want.lse, want.lse_tol, "lse")
        ref.assert_close(loss.get(), want.loss, want.loss_tol, "loss")
        dx, dw = run_loss_backward(d, xd, dtype, td, lse, dloss, T, H, V)
        ref.assert_close(dx.get(), want.dx, want.dx_tol, "dx")
        ref.assert_close(dw.get(), want.dw, want.dw_tol, "dw")
    finally:
        d.close()


@pytest.mark.parametrize("dtype", TYPES)
def test_loss_gradient_against_differences(dtype):
    """A central difference of the sum of dloss * loss along one direction of x: off by the third
    derivative's step^2 / 6 (logits move by at most `move`) and by the losses' own errors."""
    T, H, V = 5, 64, 50
    x, xv, w, wv, targets, dloss = loss_case(MOE_F32, T, H, V, seed=1)
    rng = np.random.default_rng(2)
    direction = rng.standard_normal((T, H))
    step = 2.0 ** -6
    d = context(H, w)
    try:
        def total(v):
            _, _, loss, _ = run_loss(d, v.astype(np.float32), MOE_F32, targets, V)
            return float(loss.get() @ dloss)

        numeric = (total(xv + step * direction) - total(xv - step * direction)) / (2 * step)
        xd, td, loss, lse = run_loss(d, ref.store(x, dtype)[0], dtype, targets, V)
        dx, _ = run_loss_backward(d, xd, dtype, td, lse, dloss, T, H, V, dw=False)
        analytic = float((dx.get() * direction).sum())
    finally:
        d.close()
    move = np.abs(direction @ wv.T).max(1)  # of a logit per unit of step
    want = ref.Loss(xv, wv, targets, dloss.astype(np.float64), MOE_F32)
    tol = float((np.abs(dloss) * (move ** 3 * step ** 2 + 2 * (want.loss_tol + 2.0 ** -22 * 10) / step)).sum())
    if dtype == MOE_BF16:  # x itself is rounded: the gradient changes by at most |dloss| |move| (logits' change)
        tol += float((np.abs(dloss) * move * 2 * 2.0 ** -8 * (np.abs(xv) @ np.abs(wv).T).max(1)).sum())
        tol += float((np.abs(direction) * 2.0 ** -6 * np.abs(want.dx)).sum() + (np.abs(direction) * want.dx_tol).sum())
    else:
        tol += float((np.abs(direction) * want.dx_tol).sum())
    assert abs(numeric - analytic) <= tol, (numeric, analytic, tol)


@pytest.mark.parametrize("dtype", TYPES)
def test_loss_targets(dtype):
    """Ignored tokens have no loss and add nothing, whatever their rows hold; targets past the vocabulary
    give NaN; every token ignored gives zeros; dloss may be zero."""
    T, H, V = 20, 64, 40
    x, xv, w, wv, targets, dloss = loss_case(dtype, T, H, V, seed=3)
    targets[:] = np.arange(T) % V
    targets[[2, 5]] = -1
    targets[7] = -2**31
    dloss[9] = 0.0
    want = ref.Loss(xv, wv, targets, dloss.astype(np.float64), dtype)
    d = context(H, w)
    try:
        xd, td, loss, lse = run_loss(d, x, dtype, targets, V)
        ref.assert_close(loss.get(), want.loss, want.loss_tol, "loss")
        assert (loss.get()[[2, 5, 7]] == 0).all()
        dx, dw = run_loss_backward(d, xd, dtype, td, lse, dloss, T, H, V)
        ref.assert_close(dx.get(), want.dx, want.dx_tol, "dx")
        ref.assert_close(dw.get(), want.dw, want.dw_tol, "dw")
        assert (dx.get()[[2, 5, 7, 9]] == 0).all()
        for bad in (V, 2**31 - 1):
            t2 = targets.copy()
            t2[4] = bad
            xd, td, loss, lse = run_loss(d, x, dtype, t2, V)
            assert np.isnan(loss.get()[4]) and np.isnan(loss.get()).sum() == 1 and not np.isnan(lse.get()).any()
            dx, dw = run_loss_backward(d, xd, dtype, td, lse, dloss, T, H, V)
            assert np.isnan(dx.get()[4]).all() and not np.isnan(np.delete(dx.get(), 4, 0)).any()
            assert np.isnan(dw.get()).all()
        none = np.full(T, -1, np.int32)
        xd, td, loss, lse = run_loss(d, x, dtype, none, V)
        dx, dw = run_loss_backward(d, xd, dtype, td, lse, dloss, T, H, V)
        assert (loss.get() == 0).all() and (dx.get() == 0).all() and (dw.get() == 0).all()
    finally:
        d.close()


@pytest.mark.parametrize("dtype", TYPES)
def test_loss_gradient_of_tokens_that_do_not_count(dtype):
    """dloss of an ignored token may be anything: it moves nothing. Small dloss beside it keep their bits."""
    T, H, V = 30, 64, 200
    x, xv, w, wv, targets, dloss = loss_case(dtype, T, H, V, seed=11)
    dloss *= np.float32(2.0 ** -20)
    targets[[3, 8, 20, 29]] = -1
    want = ref.Loss(xv, wv, targets, np.where(targets < 0, 0.0, dloss.astype(np.float64)), dtype)
    dloss[[3, 8, 20, 29]] = 3e38, np.inf, np.nan, -np.inf
    d = context(H, w)
    try:
        xd, td, loss, lse = run_loss(d, x, dtype, targets, V)
        dx, dw = run_loss_backward(d, xd, dtype, td, lse, dloss, T, H, V)
        ref.assert_close(dx.get(), want.dx, want.dx_tol, "dx")
        ref.assert_close(dw.get(), want.dw, want.dw_tol, "dw")
    finally:
        d.close()


# Sizes at which each tile shape of the plan is taken by each of its products (the large ones in both
# types), with more than two steps and a tail of one
TILES_LOSS = [(1, 736, 4320, MOE_BF16), (33, 160, 2772, MOE_F32), (15, 224, 124, MOE_F32), (6, 224, 21505, MOE_F32),
              (2, 160, 38963, MOE_BF16), (6, 160, 34985, MOE_F32), (18, 160, 12710, MOE_BF16), (51, 160, 4593, MOE_F32),
              (1, 160, 21750, MOE_BF16), (22, 160, 16463, MOE_F32), (28, 160, 36238, MOE_F32), (37, 1472, 2076, MOE_F32),
              (163, 160, 37761, MOE_BF16), (22, 416, 26172, MOE_F32), (646, 160, 11029, MOE_F32), (257, 160, 30609, MOE_BF16),
              (257, 160, 30609, MOE_F32), (146, 416, 22646, MOE_BF16), (148, 160, 24214, MOE_F32), (7064, 1216, 136, MOE_BF16),
              (7064, 1216, 136, MOE_F32), (8021, 1600, 131, MOE_BF16), (8021, 1600, 131, MOE_F32), (171, 1056, 14315, MOE_F32),
              (1448, 1952, 3505, MOE_F32), (1058, 1440, 10839, MOE_BF16)]
TILES_BLOCK = [(27, 224, 296, MOE_F32), (6, 160, 80, MOE_F32), (3, 224, 4360, MOE_F32), (11, 160, 3224, MOE_F32),
               (26, 160, 6496, MOE_F32), (39, 160, 5176, MOE_BF16), (69, 160, 3800, MOE_F32), (36, 1280, 200, MOE_F32),
               (8587, 224, 112, MOE_BF16), (946, 32, 1064, MOE_F32), (347, 160, 5368, MOE_BF16), (619, 160, 808, MOE_BF16),
               (150, 288, 5648, MOE_BF16), (978, 160, 4368, MOE_F32), (6266, 160, 264, MOE_F32), (6596, 160, 616, MOE_BF16),
               (6451, 544, 72, MOE_BF16), (810, 224, 7048, MOE_BF16), (810, 224, 7048, MOE_F32), (7227, 2080, 528, MOE_BF16),
               (5000, 160, 2056, MOE_BF16), (1155, 160, 6904, MOE_F32), (11279, 160, 1168, MOE_BF16), (11819, 160, 1048, MOE_F32),
               (1, 224, 2056, MOE_BF16), (8, 160, 2568, MOE_BF16), (2, 96, 2056, MOE_F32)]


@pytest.mark.parametrize("T,H,V,dtype", TILES_LOSS)
def test_loss_tiles(T, H, V, dtype):
    test_loss_and_gradient(dtype, T, H, V)


@pytest.mark.parametrize("dtype", TYPES)
def test_loss_smaller_vocabulary_and_far_logits(dtype):
    """The first rows of a larger head; logits of hundreds, of one sign and the other."""
    T, H, V = 9, 64, 100
    x, xv, w, wv, targets, dloss = loss_case(dtype, T, H, 300, seed=4, scale=300.0)
    targets = np.where(targets >= 0, targets % V, -1).astype(np.int32)
    want = ref.Loss(xv, wv[:V], targets, dloss.astype(np.float64), dtype)
    d = context(H, w)
    try:
        xd, td, loss, lse = run_loss(d, x, dtype, targets, V)
        ref.assert_close(lse.get(), want.lse, want.lse_tol, "lse")
        ref.assert_close(loss.get(), want.loss, want.loss_tol, "loss")
        dx, dw = run_loss_backward(d, xd, dtype, td, lse, dloss, T, H, V)
        ref.assert_close(dx.get(), want.dx, want.dx_tol, "dx")
        ref.assert_close(dw.get(), want.dw, want.dw_tol, "dw")
    finally:
        d.close()


@pytest.mark.parametrize("dtype", TYPES)
def test_loss_not_finite(dtype):
    """A NaN or an infinity in a token's row makes that token's results NaN and leaves the others'."""
    T, H, V = 40, 64, 300
    x, xv, w, wv, targets, dloss = loss_case(dtype, T, H, V, seed=5)
    targets = np.abs(targets)
    clean = ref.Loss(xv, wv, targets, dloss.astype(np.float64), dtype)
    bits = x.view(np.uint32 if dtype == MOE_F32 else np.uint16)
    bits[3, 10], bits[8, 0] = (0x7FC00000, 0x7F800000) if dtype == MOE_F32 else (0x7FC0, 0x7F80)
    d = context(H, w)
    try:
        xd, td, loss, lse = run_loss(d, x, dtype, targets, V)
        got = loss.get()
        assert np.isnan(got[[3, 8]]).all()
        rest = np.delete(np.arange(T), [3, 8])
        ref.assert_close(got[rest], clean.loss[rest], clean.loss_tol[rest], "loss")
        targets[[3, 8]] = -1  # ignored, the same rows add nothing
        clean = ref.Loss(xv, wv, targets, dloss.astype(np.float64), dtype)
        xd, td, loss, lse = run_loss(d, x, dtype, targets, V)
        for with_dw in (False, True):
            dx, dw = run_loss_backward(d, xd, dtype, td, lse, dloss, T, H, V, dw=with_dw)
            assert (loss.get()[[3, 8]] == 0).all() and (dx.get()[[3, 8]] == 0).all()
            ref.assert_close(dx.get()[rest], clean.dx[rest], clean.dx_tol[rest], "dx")
        ref.assert_close(dw.get(), clean.dw, clean.dw_tol, "dw")
    finally:
        d.close()


@pytest.mark.parametrize("dtype,T,V", [(MOE_BF16, 8200, 33000), (MOE_F32, 8200, 11000)])
def test_loss_gradient_in_pieces(dtype, T, V):
    """More tokens and more vocabulary than one piece of the logits' gradient holds."""
    H = 32
    x, xv, w, wv, targets, dloss = loss_case(dtype, T, H, V, seed=6)
    d = context(H, w)
    try:
        xd, td, loss, lse = run_loss(d, x, dtype, targets, V)
        dx, dw = run_loss_backward(d, xd, dtype, td, lse, dloss, T, H, V)
        got = dict(loss=loss.get(), lse=lse.get(), dx=dx.get(), dw=dw.get())
    finally:
        d.close()
    dw_want, dw_tol = np.zeros((V, H)), np.zeros((V, H))
    for t in range(0, T, 820):
        part = ref.Loss(xv[t:t + 820], wv, targets[t:t + 820], dloss[t:t + 820].astype(np.float64), dtype)
        for name in ("loss", "lse", "dx"):
            ref.assert_close(got[name][t:t + 820], getattr(part, name), getattr(part, name + "_tol"), name)
        dw_want += part.dw
        dw_tol += part.dw_tol * (T / 820)  # the f32 sum is over all tokens, not the part's
    ref.assert_close(got["dw"], dw_want, dw_tol + ref.u(dtype) * np.abs(dw_want), "dw")


# ------------------------------------------------------------------ gated block


def block_case(dtype, T, H, I, seed=0, bias=True, scale=1.2):  # noqa: E741
    rng = np.random.default_rng([seed, T, H, I, dtype])
    c = dict(x=ref.rows(rng, (T, H), dtype), dy=ref.rows(rng, (T, H), dtype, 0.3),
             wgu=ref.rows(rng, (2 * I, H), MOE_BF16, scale / np.sqrt(H)), wd=ref.rows(rng, (H, I), MOE_BF16, 1 / np.sqrt(I)))
    c["bgu"] = (rng.standard_normal(2 * I) * 0.2 * bias).astype(np.float32)
    c["bd"] = (rng.standard_normal(H) * 0.2 * bias).astype(np.float32)
    return c


def block_ref(c, dtype, x_hat=None):
    return ref.Block(c["x"][1], c["wgu"][1], c["bgu"].astype(np.float64), c["wd"][1], c["bd"].astype(np.float64), c["dy"][1],
                     dtype, x_hat)


class BlockOnDevice:
    def __init__(self, c, bias=True):
        self.T, self.H = c["x"][0].shape
        self.I = c["wd"][0].shape[1]
        self.keep = {k: dev(c[k][0]) for k in ("x", "dy", "wgu", "wd")}
        self.keep.update(bgu=dev(c["bgu"]), bd=dev(c["bd"]))
        k = self.keep
        self.block = GatedFfn(self.I, k["wgu"].ptr, k["bgu"].ptr if bias else None, k["wd"].ptr, k["bd"].ptr if bias else None)

    def forward(self, d, dtype, x8=None, stream=None):
        y = Out((self.T, self.H), dtype)
        d.ffn_forward_device(self.block, self.keep["x"], dtype, self.T, y, x8=x8, stream=stream)
        return y

    def backward(self, d, dtype, x=None, x_type=None, skip=(), stream=None):
        H, I = self.H, self.I  # noqa: E741
        o = dict(x=Out((self.T, H), dtype), gate_up=Out((2 * I, H), dtype), gate_up_bias=Out((2 * I,), MOE_F32),
                 down=Out((H, I), dtype), down_bias=Out((H,), MOE_F32))
        for s in skip:
            o.pop(s)
        g = GatedFfnGrads(*(o[n].ptr if n in o else None for n in ("x", "gate_up", "gate_up_bias", "down", "down_bias")))
        d.ffn_backward_device(self.block, self.keep["x"] if x is None else x, dtype if x_type is None else x_type,
                              self.keep["dy"], dtype, self.T, g, stream)
        return o


NAMES = dict(x="dx", gate_up="dwgu", gate_up_bias="dbgu", down="dwd", down_bias="dbd")


def check_grads(got, want):
    for n, o in got.items():
        ref.assert_close(o.get(), getattr(want, NAMES[n]), getattr(want, NAMES[n] + "_tol"), n)


# T: as above; H and I: below, at and above the tiles, tails of K-steps (I = 8, 24, 200: not a multiple of 32)
BLOCKS = [(1, 32, 8), (1, 64, 64), (2, 96, 24), (15, 160, 200), (16, 64, 128), (17, 64, 136), (127, 32, 264), (130, 544, 72),
          (300, 128, 320), (1, 2880, 96), (37, 512, 1000), (257, 288, 520)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,H,I", BLOCKS)
def test_block(dtype, T, H, I):  # noqa: E741
    c = block_case(dtype, T, H, I)
    want = block_ref(c, dtype)
    d = context(H)
    try:
        b = BlockOnDevice(c)
        y = b.forward(d, dtype)
        grads = b.backward(d, dtype)
        d.synchronize()
        ref.assert_close(y.get(), want.y, want.y_tol, "y")
        check_grads(grads, want)
    finally:
        d.close()


@pytest.mark.parametrize("T,H,I,dtype", TILES_BLOCK)
def test_block_tiles(T, H, I, dtype):  # noqa: E741
    test_block(dtype, T, H, I)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,H,I", [(1, 64, 40), (50, 96, 72), (300, 128, 320), (257, 416, 1000), (1, 224, 2056)])
def test_block_from_checkpoint(dtype, T, H, I):  # noqa: E741
    """The forward pass keeps x in 8 bits, the backward pass reads that: the gradients are those at the
    values kept, to the operators' own tolerance."""
    c = block_case(dtype, T, H, I, seed=1)
    codes, scales, kept = ref.act8(c["x"][1])
    want = block_ref(c, dtype, x_hat=kept)
    d = context(H)
    try:
        b = BlockOnDevice(c)
        x8 = DeviceBuffer(d.act8_bytes(T, H))
        y = b.forward(d, dtype, x8=x8)
        grads = b.backward(d, dtype, x=x8, x_type=MOE_MXFP8)
        d.synchronize()
        got = x8.download(np.uint8, (T * H + T * H // 32,))
        assert np.array_equal(got[:T * H].reshape(T, H), codes) and np.array_equal(got[T * H:].reshape(scales.shape), scales)
        ref.assert_close(y.get(), want.y, want.y_tol, "y")
        check_grads(grads, want)
    finally:
        d.close()


@pytest.mark.parametrize("dtype", TYPES)
def test_block_clamps(dtype):
    """Gates and ups on, below and above the clamps, exactly: the rows of gate_up pick single values of x.
    At the limit the gradient passes, above it is 0."""
    T, H, I = 5, 32, 16  # noqa: E741
    c = block_case(dtype, T, H, I, seed=2, bias=False)
    wgu = np.zeros((2 * I, H), np.float32)
    for i in range(I):
        wgu[2 * i, i], wgu[2 * i + 1, 16 + i] = 1.0, 1.0
    c["wgu"] = ref.store(wgu, MOE_BF16)
    x = np.resize(np.array([7.0, 7.5, -7.0, 6.75, 0.0, -7.5, 100.0, -100.0, 8.0, 1.0, -1.0], np.float32), (T, H))
    c["x"] = ref.store(x, dtype)
    want = block_ref(c, dtype)
    assert (c["x"][1][:, :16] == 7).any() and (np.abs(c["x"][1][:, 16:]) == 7).any()
    d = context(H)
    try:
        b = BlockOnDevice(c, bias=False)
        y = b.forward(d, dtype)
        grads = b.backward(d, dtype)
        d.synchronize()
        ref.assert_close(y.get(), want.y, want.y_tol, "y")
        check_grads(grads, want)
    finally:
        d.close()


@pytest.mark.parametrize("dtype", TYPES)
def test_block_far_below_the_clamp(dtype):
    """Gates of -3e38 close: that token's h and gradients are 0, and the others' results are theirs alone."""
    T, H, I = 3, 32, 16  # noqa: E741
    c = block_case(dtype, T, H, I, seed=8, bias=False)
    wgu = np.zeros((2 * I, H), np.float32)
    for i in range(I):
        wgu[2 * i, i], wgu[2 * i + 1, 16 + i] = 1.0, 1.0
    c["wgu"] = ref.store(wgu, MOE_BF16)
    x = c["x"][1].astype(np.float32)
    x[1, :16] = -3e38
    c["x"] = ref.store(x, dtype)
    rest = [0, 2]
    want = block_ref(dict(c, x=(None, c["x"][1][rest]), dy=(None, c["dy"][1][rest])), dtype)
    want.dbd, want.dbd_tol = c["dy"][1].sum(0), (T + 1) * 2.0 ** -24 * np.abs(c["dy"][1]).sum(0)
    d = context(H)
    try:
        b = BlockOnDevice(c, bias=False)
        y, g = b.forward(d, dtype), b.backward(d, dtype)
        d.synchronize()
        assert (y.get()[1] == 0).all() and (g["x"].get()[1] == 0).all()
        ref.assert_close(y.get()[rest], want.y, want.y_tol, "y")
        ref.assert_close(g.pop("x").get()[rest], want.dx, want.dx_tol, "dx")
        check_grads(g, want)
    finally:
        d.close()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("skip", [("x",), ("gate_up", "gate_up_bias"), ("x", "gate_up", "gate_up_bias", "down"),
                                  ("x", "down", "down_bias"), ("x", "gate_up", "gate_up_bias", "down", "down_bias")])
def test_block_some_gradients(dtype, skip):
    c = block_case(dtype, 33, 64, 72, seed=3)
    want = block_ref(c, dtype)
    d = context(64)
    try:
        grads = BlockOnDevice(c).backward(d, dtype, skip=skip)
        d.synchronize()
        check_grads(grads, want)
    finally:
        d.close()


def test_block_not_finite_rows_stay_apart():
    """A NaN row gives NaN results for its token and its token alone (y and dx)."""
    c = block_case(MOE_F32, 40, 64, 72, seed=4)
    want = block_ref(c, MOE_F32)
    c["x"][0][6, 3] = np.nan
    d = context(64)
    try:
        b = BlockOnDevice(c)
        y, g = b.forward(d, MOE_F32), b.backward(d, MOE_F32)
        d.synchronize()
        rest = np.delete(np.arange(40), 6)
        assert np.isnan(y.get()[6]).all() and np.isnan(g["x"].get()[6]).all()
        ref.assert_close(y.get()[rest], want.y[rest], want.y_tol[rest], "y")
        ref.assert_close(g["x"].get()[rest], want.dx[rest], want.dx_tol[rest], "dx")
    finally:
        d.close()


@pytest.mark.parametrize("dtype", TYPES)
def test_block_gradient_against_differences(dtype):
    """Central differences of sum(dy * y) along directions of x and of the down weights, in 64 bits; y is
    smooth there (no clamp is reached), its third derivative along x at most 8 times the cube of the gate's
    and up's move times |dh|."""
    T, H, I = 4, 64, 40  # noqa: E741
    c = block_case(MOE_F32, T, H, I, seed=5, scale=0.8)
    rng = np.random.default_rng(6)
    direction, step = rng.standard_normal((T, H)), 2.0 ** -10
    dy = c["dy"][1]

    def total(xv):
        return float((ref.Block(xv, c["wgu"][1], c["bgu"].astype(np.float64), c["wd"][1], c["bd"].astype(np.float64), None,
                                MOE_F32).y * dy).sum())

    xv = c["x"][1]
    numeric = (total(xv + step * direction) - total(xv - step * direction)) / (2 * step)
    if dtype == MOE_BF16:
        return_to = {k: ref.store(c[k][0], MOE_BF16) for k in ("x", "dy")}
        c = dict(c, **return_to)
    want = block_ref(c, dtype)
    d = context(H)
    try:
        g = BlockOnDevice(c).backward(d, dtype)
        d.synchronize()
        analytic = float((g["x"].get() * direction).sum())
    finally:
        d.close()
    move = np.abs(direction @ c["wgu"][1].T).max(1)
    tol = float((np.abs(direction) * want.dx_tol).sum())
    tol += float((8 * move ** 3 * step ** 2 * np.abs(dy @ c["wd"][1]).sum(1)).sum())
    if dtype == MOE_BF16:
        exact = block_ref(dict(c, x=(None, xv), dy=(None, dy)), MOE_F32)
        tol += float((np.abs(direction) * np.abs(exact.dx - want.dx)).sum())
    assert abs(numeric - analytic) <= tol, (numeric, analytic, tol)


# ------------------------------------------------------------------ 8-bit checkpoints


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,cols", [(1, 32), (3, 64), (17, 160), (300, 2880), (1, 32 * 2000)])
def test_act8(dtype, T, cols):
    """Codes, scales and values bit for bit, over the whole range of exponents, with zeros, subnormals,
    ties, blocks whose maximum is 448, just above it and just below."""
    rng = np.random.default_rng([T, cols, dtype])
    x = rng.standard_normal((T, cols)) * 2.0 ** rng.integers(-140, 120, (T, cols // 32)).repeat(32, 1)
    special = np.array([0.0, -0.0, 448.0, 449.0, 447.9, -448.0, 1.0625, 1.1875, 2.0 ** -9, 2.0 ** -10, 3 * 2.0 ** -10, 5e-40,
                        -1e-45, 3e38, 464.0, 480.0])
    x.reshape(-1)[:16] = special
    if T * cols >= 96:
        x.reshape(-1)[32:64] = 0.0
        x.reshape(-1)[64:96] = np.where(np.arange(32) % 2, -448.0, 1.75 * np.arange(32))
    dv, v = ref.store(x.astype(np.float32), dtype)
    codes, scales, values = ref.act8(v)
    d = context(32)
    try:
        packed = DeviceBuffer.from_array(np.full(T * cols + T * cols // 32 + GUARD, 0xA5, np.uint8))
        xd = dev(dv)
        d.act8_pack_device(xd, dtype, T, cols, packed)
        f, b = Out((T, cols), MOE_F32), Out((T, cols), MOE_BF16)
        d.act8_unpack_device(packed, T, cols, f, MOE_F32)
        d.act8_unpack_device(packed, T, cols, b, MOE_BF16)
        d.synchronize()
        got = packed.download(np.uint8, (packed.nbytes,))
        assert (got[-GUARD:] == 0xA5).all()
        assert np.array_equal(got[:T * cols].reshape(T, cols), codes)
        assert np.array_equal(got[T * cols:-GUARD].reshape(scales.shape), scales)
        assert np.array_equal(f.get(), values)
        normal = np.abs(values) >= 2.0 ** -126
        assert np.array_equal(b.get()[normal | (values == 0)], values[normal | (values == 0)])
        # half a step: 2^-4 of the value where its code is normal, 2^-10 of the scale below
        assert (np.abs(values - v) <= np.maximum(2.0 ** -4 * np.abs(v), 2.0 ** (scales.astype(int) - 127 - 10.0).repeat(32, 1).reshape(v.shape))).all()
    finally:
        d.close()


@pytest.mark.parametrize("dtype", TYPES)
def test_act8_not_finite(dtype):
    rng = np.random.default_rng(7)
    x = rng.standard_normal((4, 96)).astype(np.float32)
    x[0, 5], x[1, 40], x[3, 95] = np.nan, np.inf, -np.inf
    bits = x if dtype == MOE_F32 else (x.view(np.uint32) >> 16).astype(np.uint16)
    v = x.astype(np.float64) if dtype == MOE_F32 else ref.from_bf16(bits).astype(np.float64)
    codes, scales, values = ref.act8(v)
    d = context(32)
    try:
        packed, out, xd = DeviceBuffer(d.act8_bytes(4, 96)), Out((4, 96), MOE_F32), dev(bits)
        d.act8_pack_device(xd, dtype, 4, 96, packed)
        d.act8_unpack_device(packed, 4, 96, out, MOE_F32)
        d.synchronize()
        assert np.array_equal(packed.download(np.uint8, (4 * 96 + 12,))[4 * 96:].reshape(4, 3), scales)
        assert np.array_equal(out.get(), values, equal_nan=True) and np.isnan(values).sum() == 96
    finally:
        d.close()


# ------------------------------------------------------------------ the largest sizes


def tail(buf, dtype, rows, cols, count):
    """The last `count` rows of a device matrix: (bits, values in 64 bits)."""
    el = 4 if dtype == MOE_F32 else 2
    out = np.empty((count, cols), np.float32 if dtype == MOE_F32 else np.uint16)
    check(lib().moe_memcpy_d2h(out.ctypes.data, buf.ptr + (rows - count) * cols * el, out.nbytes))
    return out, out.astype(np.float64) if dtype == MOE_F32 else ref.from_bf16(out).astype(np.float64)


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_past_32_bits(dtype):
    """2^20 tokens of 2080 values: offsets past 2^32 bytes and 2^31 values. Loss, block and their dx in the last rows."""
    T, H, V, I, n = 2**20, 2080, 24, 8, 70  # noqa: E741
    el = 4 if dtype == MOE_F32 else 2
    rng = np.random.default_rng(12)
    w, wv = ref.rows(rng, (V, H), MOE_BF16, 2 / np.sqrt(H))
    c = block_case(dtype, 1, H, I, seed=13)
    targets = rng.integers(-1, V, T).astype(np.int32)
    dloss = rng.uniform(-1, 1, T).astype(np.float32)
    d = context(H, w)
    try:
        x, out = DeviceBuffer(T * H * el), DeviceBuffer(T * H * el)
        check(lib().moe_synth_fill_device(x.ptr, T * H, 2 if dtype == MOE_F32 else 1, 1, 1.0, 0.0, None))
        check(lib().moe_synchronize(d.ctx))
        td, gd, loss, lse = dev(targets), dev(dloss), Out((T,), MOE_F32), Out((T,), MOE_F32)
        xv = tail(x, dtype, T, H, n)[1]
        want = ref.Loss(xv, wv, targets[-n:], dloss[-n:].astype(np.float64), dtype)
        d.lm_head_loss_device(x, dtype, td, T, V, loss, lse)
        d.lm_head_loss_backward_device(x, dtype, td, lse, gd, T, V, out, None)
        d.synchronize()
        ref.assert_close(lse.get()[-n:], want.lse, want.lse_tol, "lse")
        ref.assert_close(loss.get()[-n:], want.loss, want.loss_tol, "loss")
        ref.assert_close(tail(out, dtype, T, H, n)[1], want.dx, want.dx_tol, "dx")
        b = BlockOnDevice(c)
        c = dict(c, x=(None, xv), dy=(None, xv))
        want = block_ref(c, dtype)
        d.ffn_forward_device(b.block, x, dtype, T, out)
        d.synchronize()
        ref.assert_close(tail(out, dtype, T, H, n)[1], want.y, want.y_tol, "y")
        d.ffn_backward_device(b.block, x, dtype, x.ptr, dtype, T, GatedFfnGrads(out.ptr))
        d.synchronize()
        ref.assert_close(tail(out, dtype, T, H, n)[1], want.dx, want.dx_tol, "dx")
    finally:
        d.close()


@pytest.mark.parametrize("dtype", TYPES)
def test_most_tokens(dtype):
    """Every gradient over 2^20 tokens, ten of which have one: the others' dloss and dy are zero, so that the sums
    are those of ten."""
    T, H, V, I = 2**20, 32, 5, 8  # noqa: E741
    at = np.array([0, 1, 8191, 8192, 16384, 65535, 65536, 500000, T - 2, T - 1])
    x, xv, w, wv, targets, dloss = loss_case(dtype, T, H, V, seed=14)
    targets = np.abs(targets)
    dloss[np.isin(np.arange(T), at, invert=True)] = 0.0
    c = block_case(dtype, T, H, I, seed=15)
    dy = np.zeros((T, H), c["dy"][0].dtype)
    dy[at] = c["dy"][0][at]
    c["dy"] = (dy, None)
    d = context(H, w)
    try:
        xd, td, loss, lse = run_loss(d, x, dtype, targets, V)
        dx, dw = run_loss_backward(d, xd, dtype, td, lse, dloss, T, H, V)
        want = ref.Loss(xv[at], wv, targets[at], dloss[at].astype(np.float64), dtype)
        ref.assert_close(loss.get()[at], want.loss, want.loss_tol, "loss")
        ref.assert_close(dx.get()[at], want.dx, want.dx_tol, "dx")
        ref.assert_close(dw.get(), want.dw, want.dw_tol, "dw")
        b = BlockOnDevice(c)
        g = b.backward(d, dtype)
        d.synchronize()
        few = dict(c, x=(None, c["x"][1][at]), dy=(None, dy[at].astype(np.float64) if dtype == MOE_F32 else ref.from_bf16(dy[at]).astype(np.float64)))
        want = block_ref(few, dtype)
        ref.assert_close(g["x"].get()[at], want.dx, want.dx_tol, "dx")
        g.pop("x")
        check_grads(g, want)
    finally:
        d.close()


# ------------------------------------------------------------------ refusals


def refused(code, f, *a, **k):
    with pytest.raises(MoeError) as e:
        f(*a, **k)
    assert e.value.code == code, e.value
    return str(e.value)


def test_refusals():
    """Arguments are checked on the host before anything is enqueued; a refused call leaves the outputs."""
    from silentotithrandousha_amd import _ffi as ffi
    T, H, V, I = 4, 64, 40, 24  # noqa: E741
    x, _, w, _, targets, dloss = loss_case(MOE_F32, T, H, V)
    d = context(H)
    try:
        xd, td, gd = dev(x), dev(targets), dev(dloss)
        loss, lse, dx, dw = Out((T,), MOE_F32), Out((T,), MOE_F32), Out((T, H), MOE_F32), Out((V, H), MOE_F32)
        inv, state = ffi.MOE_ERR_INVALID, ffi.MOE_ERR_STATE

        def forward(**k):
            a = dict(x=xd, dtype=MOE_F32, targets=td, n_tokens=T, vocab_size=V, loss=loss, lse=lse)
            a.update(k)
            d.lm_head_loss_device(**a)

        def backward(**k):
            a = dict(x=xd, dtype=MOE_F32, targets=td, lse=lse, dloss=gd, n_tokens=T, vocab_size=V, dx=dx, dw=dw)
            a.update(k)
            d.lm_head_loss_backward_device(**a)

        assert "init_lm_head_bf16" in refused(state, forward)
        d.init_lm_head(np.zeros((V, H), np.float32), V)
        assert "bf16" in refused(state, forward)
        d.init_lm_head_bf16(w, V)
        for f in (forward, backward):
            refused(inv, f, dtype=MOE_MXFP8)
            refused(inv, f, dtype=7)
            refused(inv, f, vocab_size=0)
            refused(inv, f, vocab_size=V + 1)
            refused(inv, f, n_tokens=2**20 + 1)
            refused(inv, f, x=None)
            refused(inv, f, targets=None)
            refused(inv, f, x=xd.ptr + 4)
        refused(inv, forward, loss=None)
        refused(inv, forward, lse=None)
        refused(inv, forward, loss=lse)
        refused(inv, backward, lse=None)
        refused(inv, backward, dloss=None)
        refused(inv, backward, dx=xd)
        refused(inv, backward, dx=dw)
        refused(inv, backward, dx=dx.ptr + 8)
        forward(n_tokens=0, x=None, targets=None)
        refused(inv, backward, n_tokens=0, x=None, targets=None, dw=dx)

        c = block_case(MOE_F32, T, H, I)
        b = BlockOnDevice(c)
        k = b.keep
        y, x8 = Out((T, H), MOE_F32), DeviceBuffer(d.act8_bytes(T, H))

        def ffn(block=b.block, x=k["x"], dtype=MOE_F32, n=T, y=y, x8=None):
            d.ffn_forward_device(block, x, dtype, n, y, x8=x8)

        def grad(block=b.block, x=k["x"], x_type=MOE_F32, dy=k["dy"], dtype=MOE_F32, n=T, grads=GatedFfnGrads(dx.ptr)):
            d.ffn_backward_device(block, x, x_type, dy, dtype, n, grads)

        bad_blocks = [GatedFfn(0, k["wgu"].ptr, None, k["wd"].ptr, None), GatedFfn(12, k["wgu"].ptr, None, k["wd"].ptr, None),
                      GatedFfn(I, None, None, k["wd"].ptr, None), GatedFfn(I, k["wgu"].ptr, None, None, None),
                      GatedFfn(I, k["wgu"].ptr + 2, None, k["wd"].ptr, None), GatedFfn(2**21, k["wgu"].ptr, None, k["wd"].ptr, None)]
        for f in (ffn, grad):
            for bad in bad_blocks:
                refused(inv, f, block=bad)
            refused(inv, f, dtype=MOE_MXFP8)
            refused(inv, f, x=None)
            refused(inv, f, n=2**20 + 1)
        refused(inv, ffn, y=None)
        refused(inv, ffn, y=k["x"])
        refused(inv, ffn, x8=x8.ptr + 8)
        refused(inv, grad, dy=None)
        refused(inv, grad, x_type=MOE_BF16)
        refused(inv, grad, grads=GatedFfnGrads(k["dy"].ptr))
        refused(inv, grad, grads=GatedFfnGrads(dx.ptr, dx.ptr))
        assert lib().moe_ffn_forward_device(d.ctx, None, k["x"].ptr, 0, T, y.ptr, None, None) == inv
        assert lib().moe_ffn_backward_device(d.ctx, ctypes.byref(b.block), k["x"].ptr, 0, k["dy"].ptr, 0, T, None, None) == inv

        for cols in (0, 33, 2**21):
            refused(inv, d.act8_pack_device, k["x"], MOE_F32, 1, cols, x8)
            refused(inv, d.act8_unpack_device, x8, 1, cols, y, MOE_F32)
        refused(inv, d.act8_pack_device, k["x"], MOE_MXFP8, T, H, x8)
        refused(inv, d.act8_pack_device, None, MOE_F32, T, H, x8)
        refused(inv, d.act8_pack_device, x8, MOE_F32, T, H, x8)
        d.act8_pack_device(None, MOE_F32, 0, H, None)
        d.synchronize()
        for o in (loss, lse, dx, dw, y):
            assert (o.buf.download(np.uint8, (o.n + GUARD,)) == 0xA5).all()
    finally:
        d.close()


@pytest.mark.parametrize("dtype", TYPES)
def test_no_tokens(dtype):
    """No tokens: nothing is written forward, the weights' gradients are zero backward."""
    H, V, I = 64, 41, 24  # noqa: E741
    w = loss_case(dtype, 1, H, V)[2]
    d = context(H, w)
    try:
        dw = Out((V, H), dtype)
        d.lm_head_loss_backward_device(None, dtype, None, None, None, 0, V, None, dw)
        c = block_case(dtype, 1, H, I)
        b = BlockOnDevice(c)
        b.T = 0
        g = b.backward(d, dtype)
        d.synchronize()
        assert (dw.get() == 0).all()
        for n, o in g.items():
            assert (o.get() == 0).all(), n
    finally:
        d.close()


# ------------------------------------------------------------------ graphs, streams, workspaces


class Step:
    """One training step over device buffers: block forward with a checkpoint, loss, both gradients."""

    def __init__(self, d, dtype, T, H, I, V, seed):  # noqa: E741
        self.d, self.dtype, self.T, self.V = d, dtype, T, V
        c = block_case(dtype, T, H, I, seed=seed)
        self.b = BlockOnDevice(c)
        rng = np.random.default_rng(seed)
        self.targets, self.dloss = dev(rng.integers(-1, V, T).astype(np.int32)), dev(rng.random(T).astype(np.float32))
        self.x8 = DeviceBuffer(d.act8_bytes(T, H))
        self.out = dict(y=Out((T, H), dtype), loss=Out((T,), MOE_F32), lse=Out((T,), MOE_F32), dy=Out((T, H), dtype),
                        dw=Out((V, H), dtype), x=Out((T, H), dtype), gate_up=Out((2 * I, H), dtype),
                        gate_up_bias=Out((2 * I,), MOE_F32), down=Out((H, I), dtype), down_bias=Out((H,), MOE_F32))
        self.grads = GatedFfnGrads(*(self.out[n].ptr for n in ("x", "gate_up", "gate_up_bias", "down", "down_bias")))

    def enqueue(self, stream=None):
        d, o, T, V, dt = self.d, self.out, self.T, self.V, self.dtype
        d.ffn_forward_device(self.b.block, self.b.keep["x"], dt, T, o["y"], x8=self.x8, stream=stream)
        d.lm_head_loss_device(o["y"], dt, self.targets, T, V, o["loss"], o["lse"], stream)
        d.lm_head_loss_backward_device(o["y"], dt, self.targets, o["lse"], self.dloss, T, V, o["dy"], o["dw"], stream)
        d.ffn_backward_device(self.b.block, self.x8, MOE_MXFP8, o["dy"], dt, T, self.grads, stream)

    def get(self):
        return {n: o.get() for n, o in self.out.items()}

    def clear(self):
        for o in self.out.values():
            check(lib().moe_memset_device(o.ptr, 0xEE, o.n))


class Capture:
    """Captures the context's stream into a graph. No garbage is collected meanwhile: a buffer freed by the
    collector (hipFree) would end the capture."""

    def __init__(self, d):
        self.d, self.graph = d, ctypes.c_void_p()

    def __enter__(self):
        gc.collect()
        gc.disable()
        check(lib().moe_graph_begin(self.d.ctx))
        return self

    def __exit__(self, *exc):
        rc = lib().moe_graph_end(self.d.ctx, ctypes.byref(self.graph))
        gc.enable()
        if exc[0] is None:
            check(rc)


def same(a, b):
    return all(np.array_equal(a[n], b[n], equal_nan=True) for n in a)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("H,I,V,tokens", [(64, 72, 300, (20, 33, 150)), (160, 520, 1500, (130, 3, 600))])
def test_steps_in_graphs(dtype, H, I, V, tokens):  # noqa: E741
    """Two captured steps of different sizes on one context, replayed in turn with eager work between them
    and with the workspace grown after their capture: every replay gives the eager bits."""
    w = loss_case(dtype, 1, H, V)[2]
    d = context(H, w)
    graphs = []
    try:
        steps = [Step(d, dtype, tokens[0], H, I, V, 1), Step(d, dtype, tokens[1], H, I, V, 2)]
        refused_first = Step(d, dtype, tokens[0], H, I, V, 1)
        with pytest.raises(MoeError) as e:  # the workspace has no size yet
            with Capture(d) as g:
                refused_first.enqueue()
        assert "workspace" in str(e.value)
        if g.graph.value:
            lib().moe_graph_destroy(g.graph)
        eager = []
        for s in steps:
            s.enqueue()
            d.synchronize()
            eager.append(s.get())
        for s in steps:
            with Capture(d) as g:
                s.enqueue()
            graphs.append(g.graph)
        large = Step(d, dtype, tokens[2], H, I, V, 3)
        for rep in range(3):
            for s, g, want in zip(steps, graphs, eager):
                s.clear()
                check(lib().moe_graph_launch(d.ctx, g))
                d.synchronize()
                assert same(s.get(), want), rep
            large.enqueue()  # grows the workspace in the first round
            d.synchronize()
    finally:
        for g in graphs:
            lib().moe_graph_destroy(g)
        d.close()


def test_caller_stream_and_contexts():
    """The same step on a stream that is not the context's, and in another context: the same bits."""
    H, I, V, T = 64, 72, 300, 40  # noqa: E741
    w = loss_case(MOE_F32, 1, H, V)[2]
    d, other = context(H, w), context(H, w)
    try:
        a, b, c = (Step(x, MOE_F32, T, H, I, V, 4) for x in (d, d, other))
        a.enqueue()
        d.synchronize()
        b.enqueue(stream=lib().moe_stream(other.ctx))
        other.synchronize()
        c.enqueue()
        other.synchronize()
        assert same(a.get(), b.get()) and same(a.get(), c.get())
    finally:
        d.close()
        other.close()


# ------------------------------------------------------------------ together


def test_layer_block_and_loss_together(orc):
    """A prompt through the MXFP4 layer with its norm (f32 rows), the dense block with an 8-bit checkpoint,
    the loss over the LM head, and back to the block's input: each operator against 64 bits from the rows
    that the one before it returned."""
    T, H, I, V = 50, 128, 96, 500  # noqa: E741
    L = syn.make_layer(H, 64, 4, seed=11, scale_lo=117, scale_hi=121)
    w, wv = ref.rows(np.random.default_rng(12), (V, H), MOE_BF16, 2 / np.sqrt(H))
    d = context(H, w, inter=64)
    try:
        d.preload_layer(0, L)
        d.preload_norm(0, np.ones(H, np.float32))
        x0 = dev(syn.hidden(T, H, seed=13))
        s = Step(d, MOE_F32, T, H, I, V, 14)
        s.b.block.down_bias = None
        rows_in = s.b.keep["x"]
        d.block_forward_device(0, x0, T, 2, rows_in)
        s.enqueue()
        d.synchronize()
        got = s.get()
        x = rows_in.download(np.float32, (T, H)).astype(np.float64)
        c = block_case(MOE_F32, T, H, I, seed=14)
        kept = ref.act8(x)[2]
        c["x"], c["dy"], c["bd"] = (None, x), (None, got["dy"]), np.zeros(H, np.float32)
        want = block_ref(c, MOE_F32, x_hat=kept)
        ref.assert_close(got["y"], want.y, want.y_tol, "y")
        targets, dloss = s.targets.download(np.int32, (T,)), s.dloss.download(np.float32, (T,)).astype(np.float64)
        loss = ref.Loss(got["y"], wv, targets, dloss, MOE_F32)
        ref.assert_close(got["loss"], loss.loss, loss.loss_tol, "loss")
        ref.assert_close(got["dy"], loss.dx, loss.dx_tol, "dy")
        ref.assert_close(got["dw"], loss.dw, loss.dw_tol, "dw")
        check_grads({n: s.out[n] for n in NAMES}, want)
        assert np.isfinite(got["x"]).all()
    finally:
        d.close()
