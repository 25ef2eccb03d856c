"""The serving operators where a call can go wrong: refusals, values that are not finite, ties, borders, streams, graphs,
workspaces; and a run of them together."""
import ctypes

import numpy as np
import pytest

from oracle import orc
from silentotithrandousha_amd import (MOE_BF16, MOE_F32, MOE_MXFP4, MOE_MXFP8, MOE_SCORE_SIGMOID, MOE_SCORE_SOFTMAX, DeviceBuffer, GpuMoeDispatcher, MoeError,
                                      Routing, Sampling, _ffi)
from silentotithrandousha_amd import synthetic as syn
from silentotithrandousha_amd._ffi import check, lib
from tests import dense_ref, serve_ref as ref
from tests.test_gpu_dense import Capture
from tests.test_gpu_serve import Out, check_sample, d, dev, matmul, quantize, resident, route, rule, sample, settings, weights  # noqa: F401

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------ refusals


def test_refusals(d):  # noqa: F811
    x, y, s = DeviceBuffer(4096), DeviceBuffer(4096), DeviceBuffer(4096)
    off = x.ptr + 4
    r = rule(k=2)
    sm = Sampling()

    def routing(**k):
        return Routing(**dict(dict(top_k=2, scale=1.0), **k))

    calls = [
        lambda: d.mxfp4_quantize_device(x, 2, 1, 32, y, s),
        lambda: d.mxfp4_quantize_device(x, 0, 1, 33, y, s),
        lambda: d.mxfp4_quantize_device(x, 0, 1, 0, y, s),
        lambda: d.mxfp4_quantize_device(x, 0, 2**24 + 1, 32, y, s),
        lambda: d.mxfp4_quantize_device(off, 0, 1, 32, y, s),
        lambda: d.mxfp4_quantize_device(x, 0, 1, 32, off, s),
        lambda: d.mxfp4_quantize_device(x, 0, 1, 32, x, s),
        lambda: d.mxfp4_quantize_device(x, 0, 1, 32, y, y),
        lambda: d.mxfp4_quantize_device(None, 0, 1, 32, y, s),
        lambda: d.mxfp4_quantize_device(x, 0, 1, 32, y, None),
        lambda: d.mxfp4_matmul_device(s, 16, 32, None, x, 4, None, 1, y, 0),
        lambda: d.mxfp4_matmul_device(s, 16, 32, None, x, -1, None, 1, y, 0),
        lambda: d.mxfp4_matmul_device(s, 16, 32, None, x, 0, None, 1, y, 2),
        lambda: d.mxfp4_matmul_device(s, 15, 32, None, x, 0, None, 1, y, 0),
        lambda: d.mxfp4_matmul_device(s, 0, 32, None, x, 0, None, 1, y, 0),
        lambda: d.mxfp4_matmul_device(s, 16, 48, None, x, 0, None, 1, y, 0),
        lambda: d.mxfp4_matmul_device(s, 16, 2**20 + 32, None, x, 0, None, 1, y, 0),
        lambda: d.mxfp4_matmul_device(s, 2**24 + 16, 32, None, x, 0, None, 1, y, 0),
        lambda: d.mxfp4_matmul_device(s, 16, 32, None, x, 0, None, 2**20 + 1, y, 0),
        lambda: d.mxfp4_matmul_device(s, 16, 32, None, x, MOE_MXFP4, None, 1, y, 0),
        lambda: d.mxfp4_matmul_device(None, 16, 32, None, x, 0, None, 1, y, 0),
        lambda: d.mxfp4_matmul_device(s, 16, 32, None, x, 0, None, 1, x, 0),
        lambda: d.mxfp4_matmul_device(s, 16, 32, None, off, 0, None, 1, y, 0),
        lambda: d.mxfp4_matmul_device(s, 16, 32, off, x, 0, None, 1, y, 0),
        lambda: d.route_device(routing(top_k=0), x, 1, 8, y, s),
        lambda: d.route_device(routing(top_k=33), x, 1, 64, y, s),
        lambda: d.route_device(routing(top_k=9), x, 1, 8, y, s),
        lambda: d.route_device(routing(score=2), x, 1, 8, y, s),
        lambda: d.route_device(routing(scale=float("nan")), x, 1, 8, y, s),
        lambda: d.route_device(routing(n_groups=3, top_groups=1), x, 1, 8, y, s),
        lambda: d.route_device(routing(n_groups=65, top_groups=1), x, 1, 130, y, s),
        lambda: d.route_device(routing(n_groups=4, top_groups=0), x, 1, 8, y, s),
        lambda: d.route_device(routing(n_groups=4, top_groups=5), x, 1, 8, y, s),
        lambda: d.route_device(routing(n_groups=4, top_groups=1, top_k=3), x, 1, 8, y, s),
        lambda: d.route_device(routing(n_groups=4, top_groups=1, group_score=2), x, 1, 8, y, s),
        lambda: d.route_device(r, x, 1, 0, y, s),
        lambda: d.route_device(r, x, 1, 1025, y, s),
        lambda: d.route_device(r, x, 2**20 + 1, 8, y, s),
        lambda: d.route_device(r, x.ptr + 2, 1, 8, y, s),
        lambda: d.route_device(r, x, 1, 8, y, y),
        lambda: d.route_device(r, x, 1, 8, x, s),
        lambda: d.route_device(r, None, 1, 8, y, s),
        lambda: d.route_backward_device(r, x, y, s, 1, 8, None),
        lambda: d.route_backward_device(r, x, y, s, 1, 8, s),
        lambda: d.sample_device(sm, x, 7, y, 1, 8, s),
        lambda: d.sample_device(sm, x, 8, y, 1, 0, s),
        lambda: d.sample_device(sm, x, 2**28 + 1, y, 1, 2**28 + 1, s),
        lambda: d.sample_device(sm, x, 8, y, 2**20 + 1, 8, s),
        lambda: d.sample_device(sm, x, 8, None, 1, 8, s),
        lambda: d.sample_device(sm, x, 8, y, 1, 8, y),
        lambda: d.sample_device(sm, x, 8, y, 1, 8, s, s),
        lambda: d.sample_device(sm, x.ptr + 2, 8, y, 1, 8, s),
    ]
    for i, call in enumerate(calls):
        with pytest.raises(MoeError) as e:
            call()
        assert e.value.code == _ffi.MOE_ERR_INVALID, i
    L = lib()
    assert L.moe_route_device(d.ctx, None, x.ptr, 1, 8, y.ptr, s.ptr, None, None) == _ffi.MOE_ERR_INVALID
    assert L.moe_sample_device(d.ctx, None, x.ptr, 8, y.ptr, 1, 8, s.ptr, None, None) == _ffi.MOE_ERR_INVALID
    # nothing to do is no error
    d.mxfp4_matmul_device(None, 16, 32, None, None, 0, None, 0, None, 0)
    d.sample_device(sm, None, 8, None, 0, 8, None)
    d.route_backward_device(r, None, None, None, 0, 8, None)
    n = Out((8,), np.int32)
    d.route_device(r, None, 0, 8, None, None, n)
    d.synchronize()
    assert (n.get() == 0).all()


# ------------------------------------------------------------------ product


@pytest.mark.parametrize("x_type", [MOE_F32, MOE_BF16, MOE_MXFP8, MOE_MXFP4])
@pytest.mark.parametrize("T,R", [(2, 32), (40, 48), (333, 2064)])
def test_matmul_not_finite(d, T, R, x_type):  # noqa: F811
    """A row with a value that is not finite is NaN, the others are what they were; so are a scale of 255 in the weights and a
    scale of 0."""
    C = 160
    blocks, scales = weights(7, R, C)
    scales[3, 2], scales[5, 1] = 255, 0
    x = np.random.default_rng(7).standard_normal((T, C)).astype(np.float32)
    stored, x_scales, values = ref.x_forms(x, x_type)
    packed = resident(d, blocks, scales)
    bad = {0: np.inf, T // 2: np.nan, T - 1: -np.inf}
    y = x.copy()
    for t, v in bad.items():
        y[t, 37] = v
    stored, x_scales, _ = ref.x_forms(y, x_type)
    got = matmul(d, packed, R, C, None, stored, x_type, x_scales, T, MOE_F32)
    w = ref.mx4_values(blocks, scales)
    want, tol = ref.matmul(values, x_type, np.nan_to_num(w), np.zeros(R), MOE_F32)
    nan = np.zeros((T, R), bool)
    nan[list(bad)] = True
    nan[:, 3] = True
    assert np.array_equal(np.isnan(got), nan)
    assert (np.abs(got - want) <= tol)[~nan].all()


@pytest.mark.parametrize("x_type", [MOE_F32, MOE_BF16])
@pytest.mark.parametrize("T", [1, 20, 70])
@pytest.mark.parametrize("scale", [2.0 ** -120, 2.0 ** -60, 2.0 ** 100])
def test_matmul_far_scales(d, T, x_type, scale):  # noqa: F811
    R, C = 32, 96
    blocks, scales = weights(8, R, C, 126, 129)
    x = (np.random.default_rng(8).standard_normal((T, C)) * scale).astype(np.float32)
    stored, x_scales, values = ref.x_forms(x, x_type)
    got = matmul(d, resident(d, blocks, scales), R, C, None, stored, x_type, x_scales, T, MOE_F32)
    want, tol = ref.matmul(values, x_type, ref.mx4_values(blocks, scales), np.zeros(R), MOE_F32)
    assert (np.abs(got - want) <= tol + 1e-38 * (scale < 2.0 ** -100)).all()  # (sums below the normal numbers may be 0)


def test_matmul_scales_behind_the_codes(d):  # noqa: F811
    T, R, C = 70, 64, 96
    blocks, scales = weights(9, R, C)
    x = np.random.default_rng(9).standard_normal((T, C)).astype(np.float32)
    codes, x_scales, _ = ref.x_forms(x, MOE_MXFP8)
    packed = resident(d, blocks, scales)
    a = matmul(d, packed, R, C, None, codes, MOE_MXFP8, x_scales, T, MOE_F32)
    b = matmul(d, packed, R, C, None, np.concatenate((codes.ravel(), x_scales.ravel())), MOE_MXFP8, None, T, MOE_F32)
    kept = DeviceBuffer(d.act8_bytes(T, C))
    y = Out((T, R), np.float32)
    d.act8_pack_device(dev(x), MOE_F32, T, C, kept)
    d.mxfp4_matmul_device(packed, R, C, None, kept, MOE_MXFP8, None, T, y, MOE_F32)
    d.synchronize()
    assert np.array_equal(a, b) and np.array_equal(a, y.get().astype(np.float64))


# ------------------------------------------------------------------ routing


def test_route_masked(d):  # noqa: F811
    inf, nan = np.inf, np.nan
    logits = np.array([[-inf] * 8, [nan] * 8, [1, -inf, 2, nan, -inf, -inf, -inf, -inf], [inf, 1, inf, 0, -inf, 3, 2, inf],
                       [5, 5, 5, 5, 5, 5, 5, 5], [0.0, -0.0, 0.0, -0.0, -1, -1, -1, -1], [3e38, -3e38, 0, 1, 2, 3, 4, 5],
                       [-1e30] * 8], np.float32)
    for kw in (dict(k=4), dict(k=4, normalize=False), dict(score=MOE_SCORE_SIGMOID, k=3), dict(score=MOE_SCORE_SIGMOID, k=2, normalize=False),
               dict(k=2, groups=4, top_groups=2, two=True), dict(k=3, groups=2, top_groups=1), dict(k=8)):
        for bias in (None, np.array([0, 0.1, 0.1, nan, -inf, 0, 0, inf], np.float32)):
            b = dev(bias)
            r = rule(**kw, bias=b)
            idx, w, n = route(d, r, logits)
            want = ref.route(logits, r, bias)
            assert np.array_equal(idx, want[0]), (kw, bias is None)
            assert np.allclose(w, want[1], rtol=1e-7, atol=0, equal_nan=True) and np.array_equal(n, want[2])


def test_route_keys_closer_than_f32(d):  # noqa: F811
    """Scores and biases whose sums differ by 2^-30 to 2^-45, in both directions, ties among them: the order of 64 bits."""
    rng = np.random.default_rng(11)
    T, E = 200, 64
    logits = rng.standard_normal((T, E)).astype(np.float32)
    # the bias makes all keys of row 0 nearly the same
    s = ref.scores(logits[:1], MOE_SCORE_SIGMOID)[0]
    bias = (1.0 - s).astype(np.float32)
    logits[1:] = logits[0] + (rng.standard_normal((T - 1, E)) * 1e-6).astype(np.float32)
    logits[100:] = logits[0]
    logits[100:, ::2] = logits[0, 0]
    bias[::2] = bias[0]
    b = dev(bias)
    for kw in (dict(k=8), dict(k=8, groups=8, top_groups=3, two=True), dict(k=5, groups=4, top_groups=2)):
        r = rule(score=MOE_SCORE_SIGMOID, bias=b, **kw)
        idx, w, _ = route(d, r, logits)
        want = ref.route(logits, r, bias)
        key = ref.scores(logits, MOE_SCORE_SIGMOID) + bias.astype(np.float64)
        other = np.nonzero((idx != want[0]).any(1))[0]
        # (two libraries' exponentials differ in the last bit of 64: keys that close may change places)
        for t in other:
            assert np.abs(key[t][idx[t]] - key[t][want[0][t]]).max() < 2.0 ** -50 or kw.get("groups"), (kw, t)
        assert len(other) <= 2, kw


@pytest.mark.parametrize("E,kw", [(256, dict(k=8, groups=8, top_groups=4, two=True)), (256, dict(k=5)), (250, dict(k=32)), (128, dict(k=6, groups=4, top_groups=2)),
                                  (128, dict(k=3, groups=16, top_groups=16)), (96, dict(k=4, groups=3, top_groups=2, two=True)), (72, dict(k=9, groups=8, top_groups=3)),
                                  (64, dict(k=8, groups=2, top_groups=1, scale=2.5)), (40, dict(k=2, normalize=False)), (2, dict(k=2)), (7, dict(k=1))])
@pytest.mark.parametrize("score", [MOE_SCORE_SOFTMAX, MOE_SCORE_SIGMOID])
def test_route_many(d, score, E, kw):  # noqa: F811
    """Many tokens with a bias: ordinary ones, masked, equal, infinite and with keys closer than an f32 tells apart, side by side."""
    rng = np.random.default_rng([25, E, score])
    T, n = 4097, 241
    x = (rng.standard_normal((n, E)) * 1.5).astype(np.float32)
    x[5:40][rng.random((35, E)) < 0.6] = -np.inf
    x[40] = -np.inf
    x[41] = np.nan
    x[42, ::3] = np.inf
    x[43:60] = x[43]
    x[60:80] = np.round(x[60:80])
    bias = (rng.standard_normal(E) * 0.1).astype(np.float32)
    bias[E // 2:] = bias[0]
    near = (1.0 - ref.scores(x[100:101], score)[0]).astype(np.float32)  # all keys of rows 100 .. nearly the same
    x[100:120] = x[100] + (rng.standard_normal((20, E)) * 1e-6).astype(np.float32)
    for b in (bias, near):
        if b is bias and E > 6:
            b[3], b[4] = np.nan, -np.inf
        keep = dev(b)
        r = rule(score=score, bias=keep, **kw)
        want = ref.route(x, r, b)
        at = rng.integers(0, n, T)
        at[:n] = np.arange(n)
        idx, w, count = route(d, r, x[at])
        key = ref.scores(x, score) + b.astype(np.float64)
        other = np.nonzero((idx != want[0][at]).any(1))[0]
        for t in other:  # (two libraries' exponentials differ in the last bit of 64)
            assert np.abs(key[at[t]][idx[t]] - key[at[t]][want[0][at[t]]]).max() < 2.0 ** -50, t
        assert len(other) <= T // 100
        same = np.setdiff1d(np.arange(T), other)
        assert (np.abs(w - want[1][at])[same] <= 2.0 ** -24 * np.abs(want[1][at])[same] * 1.001 + 1e-45).all()
        assert np.array_equal(count, np.bincount(idx[idx >= 0], minlength=E))


def test_route_is_the_paths_own(d):  # noqa: F811
    """Without bias or groups, normalised: what moe_router_topk chooses."""
    H = 64
    c = GpuMoeDispatcher(H, 32)
    layer = syn.make_layer(H, 32, 40, seed=3, router_sigma=0.5)
    c.preload_layer(0, layer)
    x = syn.hidden(30, H, seed=4)
    idx, w, logits = c.router_topk(0, x, 4, want_logits=True, n_experts=40)
    got = route(d, rule(k=4), logits)
    assert np.array_equal(got[0], idx) and np.allclose(got[1], w, rtol=1e-6)


def test_route_backward_strange_choices(d):  # noqa: F811
    """Slots without an expert, outside the experts, and one expert twice."""
    rng = np.random.default_rng(13)
    logits = rng.standard_normal((5, 10)).astype(np.float32)
    logits[3, 2] = -np.inf
    idx = np.array([[0, 1, 2], [-1, 3, -1], [10, 4, 1 << 30], [2, 5, 6], [7, 7, 7]], np.int32)
    dw = rng.standard_normal((5, 3)).astype(np.float32)
    dw[1, 0] = dw[2, 0] = np.nan  # (of slots that are left out)
    for kw in (dict(), dict(normalize=False), dict(score=MOE_SCORE_SIGMOID), dict(score=MOE_SCORE_SIGMOID, normalize=False)):
        r = rule(k=3, **kw)
        dl = Out((5, 10), np.float32)
        keep = [dev(logits), dev(idx), dev(dw)]
        d.route_backward_device(r, *keep, 5, 10, dl)
        d.synchronize()
        grad, tol = ref.route_backward(logits, idx, dw, r)
        assert (np.abs(dl.get() - grad) <= tol).all(), kw


# ------------------------------------------------------------------ sampling


def test_sample_masked(d):  # noqa: F811
    inf, nan = np.inf, np.nan
    V = 600
    logits = np.full((9, V), -inf, np.float32)
    logits[1, 5] = 3.0
    logits[2, ::7] = inf
    logits[3] = nan
    logits[4, 100:200] = 2.0
    logits[4, 150] = nan
    logits[5] = np.float32(-3e38)
    logits[6, 3], logits[6, 4] = 3e38, -3e38
    logits[7, 599] = -1e30
    logits[8] = np.linspace(-5, 5, V)
    u = np.full(9, 0.4, np.float32)
    for kw in (dict(), dict(temperature=np.full(9, 0.7)), dict(top_k=np.full(9, 3)), dict(top_p=np.full(9, 0.6)), dict(min_p=np.full(9, 0.3)),
               dict(temperature=np.zeros(9)), dict(temperature=np.full(9, nan)), dict(temperature=np.full(9, -1.0)), dict(temperature=np.full(9, inf)),
               dict(temperature=np.full(9, inf), top_p=np.full(9, 0.6)), dict(temperature=np.full(9, 1e-38), top_k=np.full(9, 50)),
               dict(top_k=np.full(9, 5), top_p=np.full(9, 0.5), min_p=np.full(9, 0.1))):
        tokens, lp = sample(d, logits, u, **kw)
        f = {k: np.asarray(v, np.int32 if k == "top_k" else np.float32) for k, v in kw.items()}
        want, wlp, room = ref.sample(logits, u, **f)
        sure = room > 2.0 ** -40
        assert np.array_equal(tokens[sure], want[sure]), kw
        assert np.allclose(lp[sure], wlp[sure], rtol=2e-7, atol=1e-9, equal_nan=True), kw
        assert tokens[0] == tokens[3] == -1 and np.isnan(lp[[0, 3]]).all()


def test_sample_random_number_at_its_ends(d):  # noqa: F811
    V = 5000
    logits = np.random.default_rng(15).standard_normal((8, V)).astype(np.float32)
    u = np.array([0, -1, np.nan, -0.0, 1, 2, np.inf, np.nextafter(np.float32(1), np.float32(0))], np.float32)
    tokens, _ = sample(d, logits, u)
    assert (tokens[:4] == 0).all() and (tokens[4:7] == V - 1).all() and tokens[7] >= V - 2
    tokens, _ = sample(d, logits, u, top_k=np.full(8, 3))
    for t in range(8):
        left = np.sort(np.argsort(-logits[t], kind="stable")[:3])
        assert tokens[t] == (left[0] if t < 4 else left[2])


@pytest.mark.parametrize("top_k,top_p", [(1, 1.0), (0, 0.0), (0, 1e-9), (5, 0.0)])
def test_sample_leaves_one(d, top_k, top_p):  # noqa: F811
    logits = np.random.default_rng(16).standard_normal((6, 3000)).astype(np.float32)
    logits[0, [7, 2900]] = 9.0  # of two largest the first
    tokens, lp = sample(d, logits, np.full(6, 0.999), top_k=np.full(6, top_k), top_p=np.full(6, top_p))
    assert np.array_equal(tokens, logits.argmax(1)) and (lp == 0).all()


def test_sample_min_p_above_one(d):  # noqa: F811
    logits = np.zeros((2, 100), np.float32)
    logits[:, [20, 40]] = 1.0
    tokens, lp = sample(d, logits, [0.2, 0.8], min_p=[1.5, 1.0])
    assert tokens.tolist() == [20, 40] and np.allclose(lp, np.log(0.5))


@pytest.mark.parametrize("V", [6000, 20000])
@pytest.mark.parametrize("which", ["top_k", "top_p", "all"])
def test_sample_flat_rows(d, V, which):  # noqa: F811
    """Logits that are equal, or so near that more of them lie at the border than a row's list holds."""
    rng = np.random.default_rng([17, V])
    T = 6
    logits = np.zeros((T, V), np.float32)
    logits[1] = (rng.standard_normal(V) * 1e-3).astype(np.float32)
    logits[2] = np.round(rng.standard_normal(V) * 2) / 2
    logits[3] = (rng.standard_normal(V) * 1e-3).astype(np.float32) - 1
    logits[3, :50] = np.linspace(0, 1, 50)
    logits[4] = 100.0
    logits[5] = rng.choice(np.array([1.0, 1.0000001, 0.9999999], np.float32), V)
    s = dict(top_k=np.full(T, V // 3 + 1), top_p=np.full(T, 0.4137), min_p=np.full(T, 0.2), temperature=rng.uniform(0.5, 1.5, T))
    f = {k: np.asarray(v, np.int32 if k == "top_k" else np.float32) for k, v in s.items() if which == "all" or k == which}
    check_sample(d, logits, rng.random(T).astype(np.float32), **f)


@pytest.mark.parametrize("V", [2048, 20000, 32003, 300000])
@pytest.mark.parametrize("k", [1, 4, 30, 60, 580])
def test_sample_few_of_many(d, k, V):  # noqa: F811
    """top-k below and above half of the row's pieces of 256 logits: ordinary rows, rows whose largest lie side by side, whose
    pieces are nearly all masked, whose logits are equal or few values."""
    rng = np.random.default_rng([21, k, V])
    T = 8
    logits = (rng.standard_normal((T, V)) * 3).astype(np.float32)
    logits[1] = np.sort(logits[1])
    logits[2, 700:] = -np.inf
    logits[3, :] = -np.inf
    logits[3, 5::256] = np.linspace(0, 3, len(logits[3, 5::256]))
    logits[4] = 1.0
    logits[5] = np.round(logits[5])
    logits[6, rng.random(V) < 0.5] = np.nan
    logits[7] *= 1e-4
    logits = np.tile(logits, (-(-800 // (T * -(-V // 2048))), 1))  # enough rows that their pieces are looked at
    T = len(logits)
    u = rng.random(T).astype(np.float32)
    check_sample(d, logits, u, top_k=np.full(T, k, np.int32))
    check_sample(d, logits, u, top_k=np.where(np.arange(T) % 2 == 0, k, 0).astype(np.int32), top_p=np.full(T, 0.813, np.float32),
                 temperature=rng.uniform(0.4, 1.6, T).astype(np.float32), min_p=np.full(T, 0.01, np.float32))


@pytest.mark.parametrize("temperature", [1e-4, 0.05, 30.0, 1e6, 1e30, np.inf])
def test_sample_far_temperatures(d, temperature):  # noqa: F811
    rng = np.random.default_rng(18)
    logits = (rng.standard_normal((6, 4000)) * 4).astype(np.float32)
    logits[3] *= 1e30
    for kw in (dict(), dict(top_k=np.full(6, 40, np.int32)), dict(top_p=np.full(6, 0.7, np.float32))):
        check_sample(d, logits, rng.random(6).astype(np.float32), temperature=np.full(6, temperature, np.float32), **kw)


def test_sample_rows_apart(d):  # noqa: F811
    """Rows with a stride, at an address that is a multiple of 4 alone, with larger logits between them."""
    rng = np.random.default_rng(19)
    T, V, ld = 7, 3001, 3010
    x = np.full((T, ld), 50.0, np.float32)
    x[:, :V] = rng.standard_normal((T, V)) * 3
    flat = np.concatenate(([99.0], x.ravel())).astype(np.float32)
    buf, u = dev(flat), rng.random(T).astype(np.float32)
    s = settings(rng, T, "all")
    bufs = {k: dev(v) for k, v in s.items()}
    tokens, lp = Out((T,), np.int32), Out((T,), np.float32)
    d.sample_device(Sampling(*(bufs[k].ptr for k in ("temperature", "top_k", "top_p", "min_p"))), buf.ptr + 4, ld, dev(u), T, V, tokens, lp)
    d.synchronize()
    want, wlp, room = ref.sample(x[:, :V], u, **s)
    assert (room > 2.0 ** -40).all() and np.array_equal(tokens.get(), want) and np.allclose(lp.get(), wlp, rtol=2e-7, atol=1e-9)


def test_sample_wide_vocabulary_and_many_rows(d):  # noqa: F811
    """A vocabulary of 2^21 + 3 (masses of fewer bits, sums of chunks beside LDS), and rows in more than one piece."""
    rng = np.random.default_rng(20)
    check_sample(d, (rng.standard_normal((2, 2**21 + 3)) * 4).astype(np.float32), rng.random(2).astype(np.float32), **settings(rng, 2, "all"))
    check_sample(d, (rng.standard_normal((2, 2**21 + 3)) * 4).astype(np.float32), rng.random(2).astype(np.float32), **settings(rng, 2, "top_p"))
    T = 4100
    s = settings(rng, T, "mixed")
    logits = (rng.standard_normal((T, 50)) * 3).astype(np.float32)
    check_sample(d, logits, rng.random(T).astype(np.float32), **s)


def test_sample_keeps_nothing_between_calls(d):  # noqa: F811
    """The same rows in another order, after a call whose workspace lay elsewhere, give the same tokens."""
    rng = np.random.default_rng(21)
    T, V = 40, 9000
    logits, u, s = (rng.standard_normal((T, V)) * 3).astype(np.float32), rng.random(T).astype(np.float32), settings(rng, T, "mixed")
    a = sample(d, logits, u, **s)
    sample(d, logits[:3, :100].copy(), u[:3])
    p = rng.permutation(T)
    b = sample(d, logits[p], u[p], **{k: v[p] for k, v in s.items()})
    assert np.array_equal(a[0][p], b[0]) and np.array_equal(a[1][p], b[1])


# ------------------------------------------------------------------ offsets past 32 bits


class Large:
    """A buffer of zeros, written and read in parts."""

    def __init__(self, n):
        self.buf = DeviceBuffer(n)
        self.ptr, self.n = self.buf.ptr, n
        check(lib().moe_memset_device(self.ptr, 0, n))

    def put(self, at, a):
        a = np.ascontiguousarray(a)
        check(lib().moe_memcpy_h2d(self.ptr + at, a.ctypes.data, a.nbytes))

    def get(self, at, shape, dtype):
        a = np.empty(shape, dtype)
        check(lib().moe_memcpy_d2h(a.ctypes.data, self.ptr + at, a.nbytes))
        return a


def test_quantize_past_32_bits(d):  # noqa: F811
    T, C = 2**17 + 3, 2**15
    x = np.random.default_rng(22).standard_normal((2, C)).astype(np.float32)
    stored, v = dense_ref.store(x, MOE_BF16)
    src, blocks, scales = Large(T * C * 2), Large(T * C // 2), Large(T * C // 32)
    src.put((T - 2) * C * 2, stored)
    d.mxfp4_quantize_device(src, MOE_BF16, T, C, blocks, scales)
    d.synchronize()
    want = ref.mx4(v)
    assert np.array_equal(blocks.get((T - 2) * C // 2, (2, C // 32, 16), np.uint8), want[0])
    assert np.array_equal(scales.get((T - 2) * C // 32, (2, C // 32), np.uint8), want[1])
    assert (scales.get((T - 3) * C // 32, (C // 32,), np.uint8) == 1).all()


def test_matmul_past_32_bits(d):  # noqa: F811
    """More than one piece of tokens, more than 4 GB of results."""
    T, R, C = 66000, 16416, 32
    blocks, scales = weights(23, R, C)
    packed = resident(d, blocks, scales)
    x = np.random.default_rng(23).standard_normal((T, C)).astype(np.float32)
    y = Large(T * R * 4)
    d.mxfp4_matmul_device(packed, R, C, None, dev(x), MOE_F32, None, T, y, MOE_F32)
    d.synchronize()
    for t in (0, 40000, 65400, 65535, 65536, T - 1):
        want, tol = ref.matmul(x[t:t + 1], MOE_F32, ref.mx4_values(blocks, scales), np.zeros(R), MOE_F32)
        assert (np.abs(y.get(t * R * 4, (1, R), np.float32) - want) <= tol).all(), t


def test_sample_past_32_bits(d):  # noqa: F811
    T, V = 2100, 2**19 + 1
    rng = np.random.default_rng(24)
    last = (rng.standard_normal((2, V)) * 3).astype(np.float32)
    logits = Large(T * V * 4)
    logits.put((T - 2) * V * 4, last)
    u = rng.random(T).astype(np.float32)
    for top_k, top_p in ((0, 1.0), (50, 1.0), (0, 0.9)):
        k, p = np.zeros(T, np.int32), np.ones(T, np.float32)
        k[-2:], p[-2:] = top_k, top_p
        bufs = [dev(k), dev(p), dev(u)]
        tokens = Out((T,), np.int32)
        d.sample_device(Sampling(None, bufs[0].ptr, bufs[1].ptr, None), logits, V, bufs[2], T, V, tokens)
        d.synchronize()
        got = tokens.get()
        want, _, room = ref.sample(last, u[-2:], top_k=k[-2:], top_p=p[-2:])
        assert (room > 2.0 ** -40).all() and np.array_equal(got[-2:], want)
        assert (np.abs(got[:-2] - u[:-2].astype(np.float64) * V) <= 1).all()  # (equal logits)


# ------------------------------------------------------------------ streams, graphs, workspaces, together


class Step:
    """A decode step's calls on buffers of their own: rows -> product -> experts and their gradient; logits -> tokens."""

    def __init__(self, T, H, E, V, x_type):
        rng = np.random.default_rng([30, T, H, E, V, x_type])
        self.T, self.H, self.E, self.V, self.x_type = T, H, E, V, x_type
        dtype = MOE_BF16 if x_type == MOE_BF16 else MOE_F32
        self.dtype = dtype
        stored, self.x = dense_ref.store(rng.standard_normal((T, H)).astype(np.float32), dtype)
        wr, wv = (dense_ref.store((rng.standard_normal((n, H)) / np.sqrt(H) * 2).astype(np.float32), MOE_BF16) for n in (E, V))
        self.w = [wr[1], wv[1]]
        self.u = rng.random(T).astype(np.float32)
        self.s = settings(rng, T, "all")
        self.buf = dict(x=dev(stored), wr=dev(wr[0]), wv=dev(wv[0]), u=dev(self.u), dw=dev(np.ones((T, 2), np.float32)), **{k: dev(v) for k, v in self.s.items()})
        for n, size in (("xb", T * H // 2), ("xs", T * H // 32), ("rb", E * H // 2), ("rs", E * H // 32), ("vb", V * H // 2), ("vs", V * H // 32),
                        ("rp", lib().moe_mxfp4_packed_size(E, H)), ("vp", lib().moe_mxfp4_packed_size(V, H))):
            self.buf[n] = DeviceBuffer(size)
        self.out = dict(route=Out((T, E), np.float32), logits=Out((T, V), np.float32), idx=Out((T, 2), np.int32), weights=Out((T, 2), np.float32),
                        counts=Out((E,), np.int32), dl=Out((T, E), np.float32), tokens=Out((T,), np.int32), lp=Out((T,), np.float32))

    def prepare(self, d):  # noqa: F811
        b = self.buf
        for n, rows, w in (("r", self.E, "wr"), ("v", self.V, "wv")):
            d.mxfp4_quantize_device(b[w], MOE_BF16, rows, self.H, b[n + "b"], b[n + "s"])
            d.mxfp4_pack_device(b[n + "b"], b[n + "s"], rows, self.H, b[n + "p"])
        d.synchronize()

    def run(self, d, stream=None):  # noqa: F811
        b, o, T, H = self.buf, self.out, self.T, self.H
        x, xs = b["x"], None
        if self.x_type == MOE_MXFP4:
            d.mxfp4_quantize_device(x, self.dtype, T, H, b["xb"], b["xs"], stream)
            x, xs = b["xb"], b["xs"]
        d.mxfp4_matmul_device(b["rp"], self.E, H, None, x, self.x_type, xs, T, o["route"], MOE_F32, stream)
        r = Routing(top_k=2, scale=1.0, normalize=1)
        d.route_device(r, o["route"], T, self.E, o["idx"], o["weights"], o["counts"], stream)
        d.route_backward_device(r, o["route"], o["idx"], b["dw"], T, self.E, o["dl"], stream)
        d.mxfp4_matmul_device(b["vp"], self.V, H, None, x, self.x_type, xs, T, o["logits"], MOE_F32, stream)
        d.sample_device(Sampling(*(b[k].ptr for k in ("temperature", "top_k", "top_p", "min_p"))), o["logits"], self.V, b["u"], T, self.V,
                        o["tokens"], o["lp"], stream)

    def get(self):
        return {n: v.get().copy() for n, v in self.out.items()}

    def clear(self):
        for v in self.out.values():
            check(lib().moe_memset_device(v.ptr, 0xA5, v.n))


@pytest.mark.parametrize("x_type", [MOE_F32, MOE_BF16, MOE_MXFP4])
@pytest.mark.parametrize("T,H,E,V", [(1, 64, 16, 304), (20, 96, 32, 2000), (150, 160, 64, 9008)])
def test_together(d, T, H, E, V, x_type):  # noqa: F811
    step = Step(T, H, E, V, x_type)
    step.prepare(d)
    step.run(d)
    d.synchronize()
    o = step.get()
    x = ref.mx4(step.x)[2] if x_type == MOE_MXFP4 else step.x
    for name, w in (("route", step.w[0]), ("logits", step.w[1])):
        want, tol = ref.matmul(x, x_type, ref.mx4(w)[2], np.zeros(w.shape[0]), MOE_F32)
        assert (np.abs(o[name] - want) <= tol).all(), name
    r = Routing(top_k=2, scale=1.0, normalize=1)
    want = ref.route(o["route"], r)
    assert np.array_equal(o["idx"], want[0]) and np.array_equal(o["counts"], want[2])
    tokens, lp, room = ref.sample(o["logits"], step.u, **step.s)
    assert np.array_equal(o["tokens"][room > 2.0 ** -40], tokens[room > 2.0 ** -40])


def test_steps_in_graphs_and_streams():
    """Captured steps of two sizes on one context, replayed in turn with eager work and a grown workspace between them, and the same
    on another stream: always the eager bits."""
    c = GpuMoeDispatcher(32, 32)
    steps = [Step(20, 96, 32, 2000, MOE_MXFP4), Step(150, 160, 64, 9008, MOE_BF16), Step(1, 64, 16, 304, MOE_F32)]
    eager, graphs = [], []
    for s in steps:
        s.prepare(c)
        s.run(c)
        c.synchronize()
        eager.append(s.get())
    for s in steps:
        with Capture(c) as g:
            s.run(c)
        graphs.append(g.graph)
    big = Step(400, 160, 64, 9008, MOE_F32)
    big.prepare(c)
    for _ in range(3):
        for s, g, want in zip(steps, graphs, eager):
            s.clear()
            check(lib().moe_graph_launch(c.ctx, g))
            c.synchronize()
            got = s.get()
            assert all(np.array_equal(got[n], want[n], equal_nan=True) for n in want)
            big.run(c)
            c.synchronize()
    other = GpuMoeDispatcher(32, 32)
    for s, want in zip(steps, eager):
        s.clear()
        s.run(c, stream=lib().moe_stream(other.ctx))
        other.synchronize()
        got = s.get()
        assert all(np.array_equal(got[n], want[n], equal_nan=True) for n in want)
    for g in graphs:
        check(lib().moe_graph_destroy(g))


def test_capture_does_not_grow_the_workspace():
    c = GpuMoeDispatcher(32, 32)
    s = Step(50, 96, 32, 2000, MOE_BF16)
    s.prepare(c)
    with pytest.raises(MoeError) as e:
        with Capture(c) as g:
            s.run(c)
    assert e.value.code == _ffi.MOE_ERR_STATE
    if g.graph.value:
        lib().moe_graph_destroy(g.graph)
    s.run(c)
    c.synchronize()


def test_two_contexts_at_once():
    """Calls of two contexts interleave on their own streams."""
    c = [GpuMoeDispatcher(32, 32) for _ in range(2)]
    steps = [Step(150, 160, 64, 9008, MOE_BF16), Step(140, 96, 32, 9008, MOE_F32)]
    want = []
    for k, s in zip(c, steps):
        s.prepare(k)
        s.run(k)
        k.synchronize()
        want.append(s.get())
        s.clear()
    for _ in range(5):
        for k, s in zip(c, steps):
            s.run(k)
    for k in c:
        k.synchronize()
    for s, w in zip(steps, want):
        got = s.get()
        assert all(np.array_equal(got[n], w[n], equal_nan=True) for n in w)


def test_experts_quantised_here():
    """A bf16 layer quantised by the operator and preloaded from the device runs as the oracle runs its codes."""
    H, I, E = 64, 96, 8  # noqa: E741
    rng = np.random.default_rng(40)
    c = GpuMoeDispatcher(H, I)
    layer = syn.make_layer(H, I, E, seed=41)
    bufs = {}
    for name, rows, cols in (("gu", 2 * I, H), ("d", H, I)):
        w, v = dense_ref.store((rng.standard_normal((E * rows, cols)) / np.sqrt(cols)).astype(np.float32), MOE_BF16)
        blocks, scales = quantize(c, w, MOE_BF16, E * rows, cols)
        bufs[name] = blocks, scales
        want = ref.mx4(v)
        layer[name + "_blocks"] = want[0].reshape(E, rows, cols // 32, 16)
        layer[name + "_scales"] = want[1].reshape(E, rows, cols // 32)
    gb, db = dev(layer["gu_bias"]), dev(layer["d_bias"])
    check(lib().moe_preload_layer_device(c.ctx, 0, E, bufs["gu"][0].ptr, bufs["gu"][1].ptr, gb.ptr, bufs["d"][0].ptr, bufs["d"][1].ptr, db.ptr, None))
    check(lib().moe_preload_router(c.ctx, 0, E, ctypes.c_void_p(layer["router_w"].ctypes.data), ctypes.c_void_p(layer["router_b"].ctypes.data)))
    x = syn.hidden(5, H, seed=42)
    got = c.layer_forward(0, x, 4)
    want = orc.moe_layer(x, layer, 4)[0]
    assert np.linalg.norm(got - want) < 1e-3 * np.linalg.norm(want)
