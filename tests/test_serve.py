"""CPU checks of the serving operators: refusals that need no device, and the 64-bit results that the GPU tests compare
with."""
import ctypes
import subprocess

import numpy as np
import pytest

from silentotithrandousha_amd import (MOE_BF16, MOE_F32, MOE_GROUP_TOP2, MOE_MXFP4, MOE_MXFP8, MOE_SCORE_SIGMOID, MOE_SCORE_SOFTMAX, Routing,
                                      Sampling, _ffi)
from tests import dense_ref, serve_ref as ref
from tests.test_dense_calls import build


def test_null_context():
    L = _ffi.lib()
    r, s = Routing(top_k=1, scale=1.0), Sampling()
    calls = [lambda: L.moe_mxfp4_quantize_device(None, None, 0, 1, 32, None, None, None),
             lambda: L.moe_mxfp4_matmul_device(None, None, 16, 32, None, None, 0, None, 1, None, 0, None),
             lambda: L.moe_route_device(None, ctypes.byref(r), None, 1, 8, None, None, None, None),
             lambda: L.moe_route_backward_device(None, ctypes.byref(r), None, None, None, 1, 8, None, None),
             lambda: L.moe_sample_device(None, ctypes.byref(s), None, 8, None, 1, 8, None, None, None)]
    for call in calls:
        assert call() == _ffi.MOE_ERR_INVALID
        assert b"null context" in L.moe_last_error()


@pytest.fixture(scope="module")
def calls(tmp_path_factory):
    return build(tmp_path_factory.mktemp("serve"), "serve_calls_test", "serve_api.cpp")


@pytest.mark.parametrize("what", ["refusals", "calls"])
def test_calls_on_the_host(calls, what):
    """csrc/serve_api.cpp over launches that only note what they read and write (tests/cpp/serve_calls_test.cpp)."""
    r = subprocess.run([calls, what], capture_output=True, text=True, timeout=100)
    assert r.returncode == 0, r.stdout


def test_mx4_reference():
    """Every value under every scale is its own code; nothing nearer exists; the OCP scale."""
    for e in (-126, -100, -1, 0, 5, 100, 125):
        x = np.zeros((1, 32))
        x[0, :8], x[0, 8:16], x[0, 16] = ref.E2M1, -ref.E2M1, 6.0
        blocks, scales, values = ref.mx4(x * 2.0 ** e)
        assert scales[0, 0] == e + 127 and np.array_equal(values, x * 2.0 ** e)
        assert np.array_equal(blocks[0, 0, :4], [0x10, 0x32, 0x54, 0x76])
        assert np.array_equal(ref.mx4_values(blocks, scales), values)
    rng = np.random.default_rng(1)
    x = rng.standard_normal((50, 320)) * np.exp(2 * rng.standard_normal((50, 320)))
    _, scales, values = ref.mx4(x)
    s = 2.0 ** (scales.astype(int) - 127.0)
    top = np.abs(x).reshape(50, -1, 32).max(-1)
    assert (top >= 4 * s).all() and (top < 8 * s).all()
    grid = np.concatenate((-ref.E2M1[::-1], ref.E2M1))
    nearest = np.abs(x.reshape(50, -1, 32, 1) / s[..., None, None] - grid).min(-1)
    assert np.allclose(np.abs(x - values).reshape(50, -1, 32) / s[..., None], nearest, rtol=0, atol=1e-12)


@pytest.mark.parametrize("x_type", [MOE_F32, MOE_BF16, MOE_MXFP8, MOE_MXFP4])
def test_x_forms(x_type):
    rng = np.random.default_rng(2)
    x = rng.standard_normal((4, 64)).astype(np.float32)
    stored, scales, values = ref.x_forms(x, x_type)
    assert values.shape == x.shape and np.abs(values - x).max() < {MOE_F32: 1e-9, MOE_BF16: 2e-2, MOE_MXFP8: 0.15, MOE_MXFP4: 0.6}[x_type]
    assert (scales is None) == (x_type in (MOE_F32, MOE_BF16))


RULES = [dict(score=s, normalize=n, n_groups=g, top_groups=2, group_score=MOE_GROUP_TOP2)
         for s in (MOE_SCORE_SOFTMAX, MOE_SCORE_SIGMOID) for n in (0, 1) for g in (0, 4)]


@pytest.mark.parametrize("r", range(len(RULES)))
def test_route_reference(r):
    """The gradient's formula against differences of the weights."""
    rule = Routing(top_k=3, scale=1.7, **RULES[r])
    rng = np.random.default_rng([3, r])
    logits = rng.standard_normal((6, 16)).astype(np.float32)
    logits[1, :5] = -np.inf
    idx, w, counts = ref.route(logits, rule, rng.standard_normal(16).astype(np.float32) * 0.1)
    assert counts.sum() == 18 and np.allclose(w, ref.route_weights(logits, idx, rule), rtol=1e-12)
    if rule.normalize:
        assert np.allclose(w.sum(1), 1.7)
    dw = rng.standard_normal(w.shape)
    grad, _ = ref.route_backward(logits, idx, dw, rule)
    z, h = logits.astype(np.float64), 1e-6
    for e in range(16):
        live = logits[:, e] > -np.inf
        up, down = z.copy(), z.copy()
        up[:, e] += h
        down[:, e] -= h
        numeric = ((ref.route_weights(up, idx, rule) - ref.route_weights(down, idx, rule)) * dw).sum(1) / (2 * h)
        assert np.abs(numeric - grad[:, e])[live].max() < 1e-8  # (third derivatives below 100, 16 digits)


def test_route_reference_groups():
    rule = Routing(top_k=2, scale=1.0, normalize=1, n_groups=3, top_groups=1, group_score=MOE_GROUP_TOP2)
    logits = np.log(np.array([[5, 1, 4, 3, 4.5, 1]], np.float32))  # sums 6, 7, 5.5
    assert ref.route(logits, rule)[0].tolist() == [[2, 3]]
    rule.group_score = 0  # largest 5, 4, 4.5
    assert ref.route(logits, rule)[0].tolist() == [[0, 1]]


def test_sample_reference():
    """The share of draws that take a token is its probability among those left."""
    logits = np.log(np.array([[0.05, 0.4, 0.1, 0.25, 0.2]], np.float32))
    u = (np.arange(1000) + 0.5).astype(np.float32) / 1000
    rows = np.repeat(logits, 1000, 0)

    def share(**s):
        tokens = ref.sample(rows, u, **{k: np.full(1000, v, np.float32) for k, v in s.items()})[0]
        return np.bincount(tokens, minlength=5) / 1000

    assert np.allclose(share(), [0.05, 0.4, 0.1, 0.25, 0.2], atol=2e-3)
    assert np.allclose(share(top_k=2), [0, 0.4 / 0.65, 0, 0.25 / 0.65, 0], atol=2e-3)
    assert np.allclose(share(top_p=0.7), [0, 0.4 / 0.85, 0, 0.25 / 0.85, 0.2 / 0.85], atol=2e-3)
    assert np.allclose(share(top_k=3, top_p=0.7), [0, 0.4 / 0.65, 0, 0.25 / 0.65, 0], atol=2e-3)  # 0.4 + 0.25 of 0.85
    assert np.allclose(share(min_p=0.3), [0, 0.4 / 0.85, 0, 0.25 / 0.85, 0.2 / 0.85], atol=2e-3)
    assert np.allclose(share(temperature=0.0), [0, 1, 0, 0, 0])
    p = np.array([0.05, 0.4, 0.1, 0.25, 0.2]) ** 2
    assert np.allclose(share(temperature=0.5), p / p.sum(), atol=2e-3)


def test_matmul_tolerances_count_lost_terms():
    """A product whose rows lost half of their terms, or whose scales were taken from the next block, is outside."""
    rng = np.random.default_rng(5)
    T, R, C = 4, 16, 256
    blocks, scales = rng.integers(0, 256, (R, C // 32, 16), dtype=np.uint8), rng.integers(120, 126, (R, C // 32), dtype=np.uint8)
    w = ref.mx4_values(blocks, scales)
    x = rng.standard_normal((T, C)).astype(np.float32)
    for x_type, bits in ((MOE_F32, 14), (MOE_BF16, 5)):
        values = dense_ref.store(x, x_type)[1]
        y, tol = ref.matmul(values, x_type, w, np.zeros(R), MOE_F32)
        cut = np.round(values * 2.0 ** bits) / 2.0 ** bits
        assert (np.abs(cut @ w.T - y) > tol).any()
        wrong = ref.mx4_values(blocks, np.roll(scales, 1, 1))
        assert (np.abs(values @ wrong.T - y) > tol).any()
