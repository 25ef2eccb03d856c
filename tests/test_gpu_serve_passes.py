"""Routing rules (include/moe_serve.h) with more tokens than one pass of a kernel's workgroups takes: what a pass leaves in registers and
LDS must not reach the next. 256 workgroups take 8192 tokens a pass under a bias (up to 256 experts), 4096, 2048 or 1024 otherwise (up to 256, 512,
1024 experts); of the gradient 4096 workgroups take 16384."""
import numpy as np
import pytest

from silentotithrandousha_amd import MOE_SCORE_SIGMOID, MOE_SCORE_SOFTMAX
from tests import serve_ref as ref
from tests.test_gpu_serve import Out, d, dev, route, rule  # noqa: F401

pytestmark = pytest.mark.gpu


def distinct(rng, E, score, n=149):
    """(rows, biases): ordinary rows, masked ones, equal ones, infinities, and rows whose keys lie closer than an f32 tells apart under the
    second bias."""
    x = (rng.standard_normal((n, E)) * 1.5).astype(np.float32)
    x[5:25][rng.random((20, E)) < 0.6] = -np.inf
    x[25], x[26] = -np.inf, np.nan
    x[27, ::3] = np.inf
    x[28:40] = np.round(x[28:40])
    bias = (rng.standard_normal(E) * 0.1).astype(np.float32)
    bias[E // 2:] = bias[0]
    near = (1.0 - ref.scores(x[40:41], score)[0]).astype(np.float32)
    x[40:60] = x[40] + (rng.standard_normal((20, E)) * 1e-6).astype(np.float32)
    return x, (bias, near)


@pytest.mark.parametrize("T,E,biased,kw", [
    (8193, 256, True, dict(k=8, groups=8, top_groups=4, two=True)), (16417, 256, True, dict(k=7)), (24577, 64, True, dict(k=5, groups=4, top_groups=2)),
    (16385, 128, True, dict(k=32)), (4099, 64, False, dict(k=6)), (8195, 200, False, dict(k=4, normalize=False)),
    (4500, 256, False, dict(k=8, groups=8, top_groups=3)), (4500, 160, True, dict(k=6, groups=8, top_groups=3)),
    (2051, 512, True, dict(k=8, groups=8, top_groups=4, two=True)), (4100, 384, True, dict(k=8)), (2053, 512, False, dict(k=3)),
    (1029, 1024, True, dict(k=9, groups=16, top_groups=5)), (2050, 777, False, dict(k=32, normalize=False))])
@pytest.mark.parametrize("score", [MOE_SCORE_SOFTMAX, MOE_SCORE_SIGMOID])
def test_route_passes(d, score, T, E, biased, kw):  # noqa: F811
    rng = np.random.default_rng([71, T, E, score])
    x, biases = distinct(rng, E, score)
    n = len(x)
    at = rng.integers(0, n, T)
    at[-n:] = rng.permutation(n)  # the last pass holds every kind
    at[::97] = 40 + at[::97] % 20  # and each one rows that are chosen again in 64 bits
    for b in biases if biased else (None,):
        keep = dev(b)
        r = rule(score=score, bias=keep, **kw)
        want = ref.route(x, r, b)
        idx, w, count = route(d, r, x[at])
        key = ref.scores(x, score) + (b.astype(np.float64) if biased else 0.0)
        other = np.nonzero((idx != want[0][at]).any(1))[0]
        for t in other:  # (two libraries' exponentials differ in the last bit of 64)
            assert biased and np.abs(key[at[t]][idx[t]] - key[at[t]][want[0][at[t]]]).max() < 2.0 ** -50, t
        assert len(set(at[other])) <= 2
        same = np.setdiff1d(np.arange(T), other)
        assert (np.abs(w - want[1][at])[same] <= 2.0 ** -24 * np.abs(want[1][at])[same] * 1.001 + 1e-45).all()
        assert np.array_equal(count, np.bincount(idx[idx >= 0], minlength=E))
        if len(other):  # a token's choice is the same wherever it stands
            for row in set(at[other]):
                assert (idx[at == row] == idx[at == row][0]).all()


@pytest.mark.parametrize("T,E,k", [(16389, 64, 4), (16387, 256, 8), (33001, 40, 32), (16399, 520, 6)])
@pytest.mark.parametrize("normalize", [True, False])
@pytest.mark.parametrize("score", [MOE_SCORE_SOFTMAX, MOE_SCORE_SIGMOID])
def test_route_backward_passes(d, score, normalize, T, E, k):  # noqa: F811
    """Some rows name an expert twice, some leave slots out."""
    rng = np.random.default_rng([72, T, E, score, normalize])
    n = 127
    x = (rng.standard_normal((n, E)) * 2).astype(np.float32)
    x[:20][rng.random((20, E)) < 0.3] = -np.inf
    idx = np.argsort(rng.random((n, E)), 1)[:, :k].astype(np.int32)
    idx[10:30, 1] = idx[10:30, 0]
    idx[25:40, 2] = -1
    idx[35:40, 0] = E
    dw = rng.standard_normal((n, k)).astype(np.float32)
    at = rng.integers(0, n, T)
    at[-n:] = rng.permutation(n)
    r = rule(score=score, k=k, normalize=normalize, scale=1.5)
    dl = Out((T, E), np.float32)
    keep = [dev(x[at]), dev(idx[at]), dev(dw[at])]
    d.route_backward_device(r, *keep, T, E, dl)
    d.synchronize()
    grad, tol = ref.route_backward(x, idx, dw, r)
    assert (np.abs(dl.get() - grad[at]) <= tol[at]).all()
