"""The serving operators (include/moe_serve.h) against 64-bit results with derived tolerances (tests/serve_ref.py): MXFP4
quantisation and product, routing rules and their gradient, sampling; their refusals, graphs, streams and workspaces; and a
run of them together."""
import ctypes

import numpy as np
import pytest

from silentotithrandousha_amd import (MOE_BF16, MOE_F32, MOE_GROUP_MAX, MOE_GROUP_TOP2, MOE_MXFP4, MOE_MXFP8, MOE_SCORE_SIGMOID,
                                      MOE_SCORE_SOFTMAX, DeviceBuffer, GpuMoeDispatcher, MoeError, Routing, Sampling)
from tests import dense_ref, serve_ref as ref

pytestmark = pytest.mark.gpu

GUARD = 64  # bytes behind each output that must stay as they were


class Out:
    """An output of `shape`, filled with 0xA5 and followed by guard bytes."""

    def __init__(self, shape, dtype):
        self.shape, self.dtype = shape, np.dtype(dtype)
        self.n = int(np.prod(shape)) * self.dtype.itemsize
        self.buf = DeviceBuffer.from_array(np.full(self.n + GUARD, 0xA5, np.uint8))
        self.ptr = self.buf.ptr

    def get(self):
        raw = self.buf.download(np.uint8, (self.n + GUARD,))
        assert (raw[self.n:] == 0xA5).all(), "written behind the output"
        return raw[:self.n].view(self.dtype).reshape(self.shape)


def dev(a):
    return None if a is None else DeviceBuffer.from_array(np.ascontiguousarray(a))


def ptr(b):
    return None if b is None else b.ptr


@pytest.fixture(scope="module")
def d():
    return GpuMoeDispatcher(32, 32)


# ------------------------------------------------------------------ quantisation


def rows(seed, T, C, dtype, scale=1.0):
    rng = np.random.default_rng([seed, T, C, dtype])
    x = rng.standard_normal((T, C)) * np.exp(0.5 * rng.standard_normal(C)) * scale
    return dense_ref.store(x.astype(np.float32), dtype)


def quantize(d, x, dtype, T, C):
    blocks, scales = Out((T, C // 32, 16), np.uint8), Out((T, C // 32), np.uint8)
    d.mxfp4_quantize_device(dev(x), dtype, T, C, blocks, scales)
    d.synchronize()
    return blocks, scales


@pytest.mark.parametrize("dtype", [MOE_F32, MOE_BF16])
@pytest.mark.parametrize("T,C", [(1, 32), (1, 2880), (3, 96), (17, 1056), (250, 416)])
def test_quantize(d, T, C, dtype):
    x, v = rows(1, T, C, dtype)
    blocks, scales = quantize(d, x, dtype, T, C)
    want = ref.mx4(v)
    assert np.array_equal(scales.get(), want[1]) and np.array_equal(blocks.get(), want[0])
    out = Out((T, C), np.float32)
    d.mxfp4_dequant_device(blocks, scales, T, C, out)
    d.synchronize()
    assert np.array_equal(out.get(), want[2].astype(np.float32))


@pytest.mark.parametrize("dtype", [MOE_F32, MOE_BF16])
def test_quantize_edges(d, dtype):
    """Every border between codes under scales from the smallest to the largest, subnormals, zeros, infinities and NaN."""
    grid = np.concatenate((ref.E2M1, (ref.E2M1[1:] + ref.E2M1[:-1]) / 2, [6.5, 7, 7.5, 7.75]))
    near = np.concatenate([grid * (1 + s * 2.0 ** -7) for s in (-1, 0, 1)])
    near = near[near < 8]
    near = np.resize(near, 31 * 2)
    x = []
    for e in (-140, -130, -127, -126, -100, -1, 0, 50, 120, 124):
        for half in (near[:31], near[31:]):
            for sign in (1, -1):
                x.append(np.append(half, 4.0) * sign * 2.0 ** e)
    x += [np.zeros(32), -np.zeros(32), np.append(np.ones(31), np.inf), np.append(np.ones(31), np.nan), np.append(-np.inf, np.ones(31)),
          np.full(32, 3.3e38), np.append(np.full(31, 1e-45), 0.0)]
    stored, v = dense_ref.store(np.array(x, np.float32), dtype)
    blocks, scales = quantize(d, stored, dtype, len(x), 32)
    want = ref.mx4(v)
    assert np.array_equal(scales.get(), want[1])
    got, exp = blocks.get(), want[0]
    nib = [np.stack((b & 15, b >> 4), -1) for b in (got, exp)]
    nib = [np.where(n == 8, 0, n) for n in nib]  # (a zero's sign says nothing)
    assert np.array_equal(*nib)


def test_quantize_empty(d):
    blocks, scales = quantize(d, np.zeros((1, 32), np.float32), MOE_F32, 0, 32)
    assert (blocks.buf.download(np.uint8, (GUARD,)) == 0xA5).all()


# ------------------------------------------------------------------ product


def weights(seed, R, C, lo=118, hi=126):
    rng = np.random.default_rng([seed, R, C])
    return rng.integers(0, 256, (R, C // 32, 16), dtype=np.uint8), rng.integers(lo, hi, (R, C // 32), dtype=np.uint8)


def resident(d, blocks, scales):
    R, C = blocks.shape[0], blocks.shape[1] * 32
    packed = DeviceBuffer(d.mxfp4_packed_size(R, C))
    b, s = dev(blocks), dev(scales)
    d.mxfp4_pack_device(b, s, R, C, packed)
    d.synchronize()
    return packed


def matmul(d, packed, R, C, bias, stored, x_type, x_scales, T, dtype, stream=None):
    y = Out((T, R), np.float32 if dtype == MOE_F32 else np.uint16)
    keep = [dev(bias), dev(stored), dev(x_scales)]
    d.mxfp4_matmul_device(packed, R, C, keep[0], keep[1], x_type, keep[2], T, y, dtype, stream)
    d.synchronize()
    got = y.get()
    return got.astype(np.float64) if dtype == MOE_F32 else dense_ref.from_bf16(got).astype(np.float64)


SIZES = [(1, 16, 32), (1, 64, 2880), (2, 80, 96), (15, 16, 160), (16, 32, 128), (17, 144, 416), (33, 2064, 64), (64, 256, 512), (65, 48, 544),
         (129, 272, 288), (255, 512, 128), (300, 528, 1056), (1024, 256, 256), (1030, 592, 352), (2100, 272, 96), (1, 2064, 8224), (40, 112, 4512), (2, 48, 2880), (3, 32, 1056), (4, 2064, 32), (5, 16, 64)]
# tiles of 64 x 64, of 128 x 128 and of 192 x 256
LARGE = [(333, 2064, 96), (400, 1600, 544), (1100, 2064, 288), (4001, 2896, 96), (3900, 3008, 544)]


@pytest.mark.parametrize("x_type", [MOE_F32, MOE_BF16, MOE_MXFP8, MOE_MXFP4])
@pytest.mark.parametrize("T,R,C", SIZES + LARGE)
def test_matmul(d, T, R, C, x_type):
    blocks, scales = weights(2, R, C)
    rng = np.random.default_rng([3, T, R, C])
    x = (rng.standard_normal((T, C)) * np.exp(rng.standard_normal(C))).astype(np.float32)
    x[0, 0] = 300.0  # an outlier beside ordinary values
    bias = rng.standard_normal(R).astype(np.float32)
    stored, x_scales, values = ref.x_forms(x, x_type)
    w = ref.mx4_values(blocks, scales)
    packed = resident(d, blocks, scales)
    for dtype in (MOE_F32, MOE_BF16):
        for b in (bias, None) if (T, R, C) not in LARGE else ((bias,) if dtype == MOE_F32 else (None,)):
            got = matmul(d, packed, R, C, b, stored, x_type, x_scales, T, dtype)
            want, tol = ref.matmul(values, x_type, w, b if b is not None else np.zeros(R), dtype)
            assert (np.abs(got - want) <= tol).all(), (dtype, np.max(np.abs(got - want) / tol))


# ------------------------------------------------------------------ routing


def rule(score=MOE_SCORE_SOFTMAX, k=4, groups=0, top_groups=0, two=False, normalize=True, scale=1.0, bias=None):
    return Routing(score=score, normalize=int(normalize), top_k=k, n_groups=groups, top_groups=top_groups,
                   group_score=MOE_GROUP_TOP2 if two else MOE_GROUP_MAX, scale=scale, bias=ptr(bias))


def route(d, r, logits, counts=True):
    T, E = logits.shape
    idx, w, n = Out((T, r.top_k), np.int32), Out((T, r.top_k), np.float32), Out((E,), np.int32)
    x = dev(logits)
    d.route_device(r, x, T, E, idx, w, n if counts else None)
    d.synchronize()
    return idx.get(), w.get(), n.get()


RULES = [dict(), dict(k=1), dict(normalize=False), dict(score=MOE_SCORE_SIGMOID, normalize=False), dict(score=MOE_SCORE_SIGMOID, scale=2.5),
         dict(score=MOE_SCORE_SIGMOID, scale=2.5, groups=4, top_groups=2, two=True), dict(groups=4, top_groups=3, k=3),
         dict(groups=2, top_groups=1, two=True, normalize=False, scale=16.0)]


@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("r", range(len(RULES)))
@pytest.mark.parametrize("T,E", [(1, 8), (5, 32), (64, 64), (65, 72), (333, 128), (200, 256), (70, 512), (9, 1024), (33, 520)])
def test_route(d, T, E, r, biased):
    rng = np.random.default_rng([4, T, E, r, biased])
    logits = (rng.standard_normal((T, E)) * 2).astype(np.float32)
    logits[rng.random((T, E)) < 0.3] = np.round(logits[rng.random((T, E)) < 0.3].mean())  # ties
    bias = (rng.standard_normal(E) * 0.05).astype(np.float32) if biased else None
    if biased:
        bias[:E // 2] = bias[0]
    b = dev(bias)
    R = rule(**RULES[r], bias=b)
    idx, w, n = route(d, R, logits)
    want = ref.route(logits, R, bias)
    assert np.array_equal(idx, want[0]) and np.array_equal(n, want[2])
    assert (np.abs(w - want[1]) <= 2.0 ** -24 * np.abs(want[1]) * 1.001 + 1e-45).all()
    dw = rng.standard_normal(w.shape).astype(np.float32)
    dl = Out((T, E), np.float32)
    keep = [dev(logits), dev(idx), dev(dw)]
    d.route_backward_device(R, *keep, T, E, dl)
    d.synchronize()
    grad, tol = ref.route_backward(logits, idx, dw, R)
    assert (np.abs(dl.get() - grad) <= tol).all()


# ------------------------------------------------------------------ sampling


def sample(d, logits, u, ld=None, V=None, logprob=True, **settings):
    T = logits.shape[0]
    V = V or logits.shape[1]
    bufs = {k: dev(np.asarray(v, np.int32 if k == "top_k" else np.float32)) for k, v in settings.items() if v is not None}
    r = Sampling(*(ptr(bufs.get(k)) for k in ("temperature", "top_k", "top_p", "min_p")))
    tokens, lp = Out((T,), np.int32), Out((T,), np.float32)
    x, uu = dev(logits), dev(np.asarray(u, np.float32))
    d.sample_device(r, x, ld or logits.shape[1], uu, T, V, tokens, lp if logprob else None)
    d.synchronize()
    return tokens.get(), lp.get()


def check_sample(d, logits, u, **settings):
    got, lp = sample(d, logits, u, **settings)
    want, wlp, room = ref.sample(logits, np.asarray(u, np.float32), **settings)
    assert (room > 2.0 ** -40).all(), "a draw too near a border for the test"
    assert np.array_equal(got, want), np.nonzero(got != want)
    live = ~np.isnan(wlp)
    assert np.array_equal(np.isnan(lp), ~live)
    # log(e / S): an f32 rounding, S to 2^-40, the temperature's exponent to 2^-50 of its size
    assert (np.abs(lp - wlp)[live] <= 2.0 ** -24 * np.abs(wlp[live]) * 1.001 + 2.0 ** -40).all()


def settings(rng, T, which):
    s = {}
    if which in ("temperature", "all", "mixed"):
        s["temperature"] = rng.uniform(0.3, 2.0, T).astype(np.float32)
    if which in ("top_k", "all", "mixed"):
        s["top_k"] = rng.integers(1, 60, T).astype(np.int32)
    if which in ("top_p", "all", "mixed"):
        s["top_p"] = rng.uniform(0.2, 0.99, T).astype(np.float32)
    if which in ("min_p", "all", "mixed"):
        s["min_p"] = rng.uniform(0.001, 0.2, T).astype(np.float32)
    if which == "mixed":
        for k, off in (("temperature", 0.0), ("top_k", 0), ("top_p", 1.0), ("min_p", 0.0)):
            s[k][rng.random(T) < 0.4] = off
    return s


@pytest.mark.parametrize("which", ["none", "temperature", "top_k", "top_p", "min_p", "all", "mixed"])
@pytest.mark.parametrize("T,V", [(1, 1), (3, 2), (8, 37), (33, 1000), (5, 8192), (4, 8193), (20, 32003), (2, 201088)])
def test_sample(d, T, V, which):
    rng = np.random.default_rng([5, T, V, len(which), ord(which[-1])])
    logits = (rng.standard_normal((T, V)) * 3).astype(np.float32)
    check_sample(d, logits, rng.random(T).astype(np.float32), **settings(rng, T, which))
