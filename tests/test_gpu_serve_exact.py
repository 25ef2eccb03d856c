"""The serving operators (include/moe_serve.h) where values of far sizes meet: each result against 64 bits, with tolerances that
hold what f32 sums lose and nothing else."""
import numpy as np
import pytest

from silentotithrandousha_amd import MOE_BF16, MOE_F32, MOE_MXFP8, MOE_SCORE_SIGMOID, MOE_SCORE_SOFTMAX
from tests import dense_ref, serve_ref as ref
from tests.test_gpu_serve import Out, d, dev, matmul, resident, route, rule, sample, weights  # noqa: F401

pytestmark = pytest.mark.gpu

# e4m3: subnormals, then 15 binades of 8; the last code is NaN
E4M3 = np.array([m / 8 * 2.0 ** -6 for m in range(8)] + [(1 + m / 8) * 2.0 ** (k - 7) for k in range(1, 16) for m in range(8)][:119])

# one, two and more tiles of few rows; tiles of 64 x 64, 128 x 128, 192 x 256
FORMS = [(1, 16, 128), (3, 2064, 2880), (20, 64, 416), (70, 48, 416), (128, 5760, 512), (333, 2064, 416), (1100, 2064, 288), (3900, 3008, 544)]


@pytest.mark.parametrize("T,R,C", FORMS)
def test_mxfp8_large_values_that_cancel(d, T, R, C):  # noqa: F811
    """Two neighbours of 448 and -448 under the same weight leave what their neighbours below 2 sum up to, to the last bit: multiples of
    2^-10 (2^-9 x 0.5), whose sums stay below 2^14."""
    rng = np.random.default_rng([41, T, R, C])
    codes = (rng.integers(0, 64, (T, C)) | rng.integers(0, 2, (T, C)) << 7).astype(np.uint8)
    codes[:, 0::8], codes[:, 1::8] = 0x7E, 0xFE
    blocks = rng.integers(0, 256, (R, C // 32, 16), dtype=np.uint8)
    blocks[..., 0::4] = (blocks[..., 0::4] & 15) * 17  # (values 8 i and 8 i + 1)
    x = np.where(codes & 128, -1.0, 1.0) * E4M3[codes & 127]
    want = x @ ref.mx4_values(blocks, np.full((R, C // 32), 127, np.uint8)).T
    assert np.abs(want).max() < 2.0 ** 14 and np.array_equal(want, want.astype(np.float32))
    ones = np.full((T, C // 32), 127, np.uint8)
    got = matmul(d, resident(d, blocks, np.full((R, C // 32), 127, np.uint8)), R, C, None, codes, MOE_MXFP8, ones, T, MOE_F32)
    assert np.array_equal(got, want), np.abs(got - want).max()


@pytest.mark.parametrize("dtype", [MOE_F32, MOE_BF16])
@pytest.mark.parametrize("T,R,C", FORMS)
def test_mxfp8_products_are_exact(d, T, R, C, dtype):  # noqa: F811
    """Codes of all sizes side by side, every product counted: 8 roundings an MFMA in its sums (2 MFMAs a step of 128), then the
    joins' and the output's. (2^-13 of the largest of 8 neighbours, 7 times, would be 700 times that.)"""
    rng = np.random.default_rng([42, T, R, C])
    codes = (rng.integers(0, 127, (T, C)) | rng.integers(0, 2, (T, C)) << 7).astype(np.uint8)
    x_scales = rng.integers(118, 130, (T, C // 32), dtype=np.uint8)
    blocks, scales = weights(43, R, C)
    bias = rng.standard_normal(R).astype(np.float32)
    x = np.where(codes & 128, -1.0, 1.0) * E4M3[codes & 127] * 2.0 ** (x_scales.repeat(32, 1).astype(np.float64) - 127)
    w = ref.mx4_values(blocks, scales)
    want, mag = x @ w.T + bias, np.abs(x) @ np.abs(w).T
    tol = (2 * -(-C // 128) + 8) * 2.0 ** -23 * mag + 2.0 ** -23 * (np.abs(want) + np.abs(bias)) + (dense_ref.u(dtype) + 2.0 ** -24) * np.abs(want)
    got = matmul(d, resident(d, blocks, scales), R, C, bias, codes, MOE_MXFP8, x_scales, T, dtype)
    assert (np.abs(got - want) <= tol).all(), np.max(np.abs(got - want) / tol)


# ------------------------------------------------------------------ bf16 rows


BF16_FORMS = FORMS + [(700, 2064, 160), (2000, 2880, 96), (5, 80, 1056), (16, 5760, 2880), (2, 16, 32), (1, 32768, 96), (4, 64, 8224), (17, 16, 96)]


def bf16_rows(x):
    """(bits, values)"""
    return dense_ref.store(np.asarray(x, np.float32), MOE_BF16)


@pytest.mark.parametrize("dtype", [MOE_F32, MOE_BF16])
@pytest.mark.parametrize("T,R,C", BF16_FORMS)
def test_bf16_rows_enter_as_they_are(d, T, R, C, dtype):  # noqa: F811
    """Beside each block's one huge value, whose weight is 0, its neighbours of all sizes count in full: what is left are an f32 sum's
    roundings, 8 an MFMA (4 MFMAs a step of 128), then the joins' and the output's."""
    rng = np.random.default_rng([44, T, R, C])
    x = rng.standard_normal((T, C)) * 2.0 ** rng.integers(-12, 3, (T, C))
    at = 32 * np.arange(C // 32) + rng.integers(0, 32, C // 32)
    x[:, at] = rng.choice([-1.0, 1.0], (T, C // 32)) * 2.0 ** rng.integers(8, 60, (T, C // 32))
    stored, x = bf16_rows(x)
    blocks, scales = weights(45, R, C)
    byte = blocks.reshape(R, -1)
    byte[:, at // 2] &= np.where(at % 2, 0x0F, 0xF0).astype(np.uint8)
    w = ref.mx4_values(blocks, scales)
    assert (w[:, at] == 0).all()
    bias = rng.standard_normal(R).astype(np.float32)
    want, mag = x @ w.T + bias, np.abs(x) @ np.abs(w).T
    tol = (4 * -(-C // 128) + 8) * 2.0 ** -23 * mag + 2.0 ** -23 * (np.abs(want) + np.abs(bias)) + (dense_ref.u(dtype) + 2.0 ** -24) * np.abs(want)
    got = matmul(d, resident(d, blocks, scales), R, C, bias, stored, MOE_BF16, None, T, dtype)
    assert (np.abs(got - want) <= tol).all(), np.max(np.abs(got - want) / tol)


@pytest.mark.parametrize("T", [16, 64, 333])
def test_bf16_products_of_far_numbers(d, T):  # noqa: F811
    """One value by one weight, exactly, from the smallest numbers of either to the largest: results below the normal numbers may be 0, above
    the largest infinite."""
    C = 32
    R = 16 * 8 if T < 333 else 16 * 129
    byte = np.array([0, 1, 2, 3, 127, 240, 252, 253])[np.arange(R) // 16 % 8].astype(np.uint8)
    blocks = np.zeros((R, 1, 16), np.uint8)
    blocks[:, 0, 3] = np.arange(R) % 16 << 4  # value 7
    scales = byte[:, None]
    numbers = [2.0 ** -133, 3 * 2.0 ** -133, 127 * 2.0 ** -133, 2.0 ** -126, 255 * 2.0 ** -133, 2.0 ** -100, 2.0 ** -20, 1.0, -1.9921875, 2.0 ** 50, 255 * 2.0 ** 120, -(2.0 ** -130)]
    v = np.resize(np.array(numbers), T)
    x = np.zeros((T, C))
    x[:, 7] = v
    x[:, 8] = 2.0 ** 90  # its weights are 0
    stored, x = bf16_rows(x)
    assert np.array_equal(x[:, 7], v)
    got = matmul(d, resident(d, blocks, scales), R, C, None, stored, MOE_BF16, None, T, MOE_F32)
    w = ref.mx4_values(blocks, scales)[:, 7]
    want = v[:, None] * w
    over = (np.abs(w) >= 2.0 ** 128)[None, :] | (np.abs(want) >= 2.0 ** 128)
    assert not np.isfinite(got[over]).any()
    small = np.abs(want) < 2.0 ** -126
    assert np.array_equal(got[~over & ~small], want[~over & ~small])
    assert (np.abs(got - want)[small & ~over] <= np.abs(want)[small & ~over]).all()


@pytest.mark.parametrize("T,R", [(1, 16), (16, 48), (33, 32), (333, 2064), (1100, 2064), (2000, 2880), (3900, 3008)])
def test_bf16_rows_that_are_not_finite(d, T, R):  # noqa: F811
    """NaN, whatever the signs of what an infinity meets, and nothing of it in the other rows."""
    C = 160
    blocks = np.full((R, C // 32, 16), 0x22, np.uint8)  # all weights are 1
    scales = np.full((R, C // 32), 127, np.uint8)
    scales[5, 1] = 255
    rng = np.random.default_rng([46, T])
    x = np.abs(rng.integers(1, 5, (T, C))).astype(np.float64)
    bad = {0: np.inf, T - 1: -np.inf, T // 2: np.nan}
    clean = x.copy()
    for t, v in bad.items():
        x[t, rng.integers(0, C)] = v
    got = matmul(d, resident(d, blocks, scales), R, C, None, bf16_rows(x)[0], MOE_BF16, None, T, MOE_F32)
    want = np.broadcast_to(clean.sum(1)[:, None], (T, R)).copy()
    want[list(bad)] = np.nan
    want[:, 5] = np.nan
    assert np.array_equal(got, want, equal_nan=True)


# ------------------------------------------------------------------ sampling


def check_wide(d, logits, u, **s):  # noqa: F811
    """Rows whose masses sum up to nearly as much as 64 bits hold. A mass is a multiple of 2^-s of the largest, s at least 34, off by half
    of that: sums over V of them by at most 2^-s-1 V, relative to a sum of nearly V 2^-35, and each border by as much."""
    s = {k: np.asarray(v, np.int32 if k == "top_k" else np.float32) for k, v in s.items()}
    u = np.asarray(u, np.float32)
    got, lp = sample(d, logits, u, **s)
    want, wlp, room = ref.sample(logits, u, **s)
    assert (room > 2.0 ** -33).all(), "a draw too near a border for the test"
    assert np.array_equal(got, want), (got, want)
    assert (np.abs(lp - wlp) <= 2.0 ** -24 * np.abs(wlp) * 1.001 + 2.0 ** -33).all(), (lp, wlp)


U = [0.0101, 0.3337, 0.5003, 0.9871]


@pytest.mark.parametrize("V", [2**18 + 1, 2**20 - 1, 2**20, 2**20 + 1, 1200000, 2**21 + 3])
@pytest.mark.parametrize("rows", ["equal", "near", "hot"])
def test_sample_flat_wide_rows(d, V, rows):  # noqa: F811
    """Equal logits, logits within 1e-3, and ordinary ones under a temperature of 1e30: all tokens' masses count."""
    rng = np.random.default_rng([51, V])
    u = U if V <= 2**20 else U[V % 2::2]
    T = len(u)
    x = np.full((T, V), 1.25, np.float32)
    if rows != "equal":
        x = (x + rng.standard_normal((T, V)) * (2e-4 if rows == "near" else 1)).astype(np.float32)
    s = dict(temperature=np.full(T, 1e30)) if rows == "hot" else {}
    check_wide(d, x, u, **s)
    check_wide(d, x, u, min_p=np.full(T, 0.5), **s)
    check_wide(d, x, u, top_p=np.full(T, 0.6), **s)
    check_wide(d, x, u, top_k=np.full(T, V - 5000), **s)


def test_sample_flat_rows_of_16_million(d):  # noqa: F811
    V = 2**24 + 7
    x = (np.float32(-3.5) + np.random.default_rng(52).standard_normal((1, V)) * 1e-4).astype(np.float32)
    check_wide(d, x, [0.87654])
    check_wide(d, x, [0.41234], top_p=[0.6])


# ------------------------------------------------------------------ routing: scores that 64 bits hold badly or not at all


def log_form(z, idx, dw, rule):
    """(weights, dlogits, its magnitude) by logarithms of the scores. A softmax whose chosen scores all lie below 2^-1075: uniform, and
    without a gradient."""
    T, k = idx.shape
    sigmoid = rule.score == MOE_SCORE_SIGMOID
    if sigmoid:
        ls, rest = np.minimum(z, 0) - np.log1p(np.exp(-np.abs(z))), np.exp(np.minimum(-z, 0) - np.log1p(np.exp(-np.abs(z))))
    else:
        top = z.max(1, keepdims=True)
        ls = z - top - np.log(np.exp(z - top).sum(1, keepdims=True))
    live = idx >= 0
    at = np.where(live, idx, 0)
    lw = np.where(live, np.take_along_axis(ls, at, 1), -np.inf)
    gone = np.zeros(T, bool)
    if rule.normalize:
        best = lw.max(1, keepdims=True)
        gone = (best[:, 0] < np.log(2) * -1075) & (not sigmoid)
        w = np.exp(lw - best)
        w[gone] = live[gone]
        w = w / w.sum(1, keepdims=True)
    else:
        w = np.exp(lw)
    w = w * rule.scale
    g = dw * w
    size = np.abs(g)
    if rule.normalize:
        part = w / rule.scale
        g, size = g - part * g.sum(1, keepdims=True), size + part * size.sum(1, keepdims=True)
    out, mag = np.zeros_like(z), np.zeros_like(z)
    for t in range(T):
        for j in range(k):
            if live[t, j] and not gone[t]:
                f = rest[t, idx[t, j]] if sigmoid else 1.0
                out[t, idx[t, j]] += g[t, j] * f
                mag[t, idx[t, j]] += size[t, j] * f
    if not sigmoid and not rule.normalize:
        s = np.exp(ls)
        out -= s * g.sum(1, keepdims=True)
        mag += s * size.sum(1, keepdims=True)
    return w, out, mag


FAR = [[-720, -720.5, -719.25], [-600.5, -601, -640], [-599.5, -640, -720], [-650, -700, -743], [-744.5, -745.5, -746], [-800, -900, -801],
       [-1e9, -1e9, -1e9], [-1e30, -1e30, -1.5e30], [-1e30, -3e38, -1e9], [-20, -700, -1], [3, -700, -1e30], [-590, -720.5, -1e30], [-708, -709.5, -710]]


@pytest.mark.parametrize("T", [13, 70, 4099])
@pytest.mark.parametrize("E", [8, 200, 520])
@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("score", [MOE_SCORE_SOFTMAX, MOE_SCORE_SIGMOID])
def test_route_far_scores(d, score, biased, E, T):  # noqa: F811
    """Rows whose chosen logits all lie far below 0 (sigmoid) or below a logit that is not chosen (softmax): a masked token, a token under
    a strong bias. Weights and gradient are finite and what the formula says."""
    rng = np.random.default_rng([61, E, T])
    k = 3
    places = [E // 2, E // 2 + 1, E - 1]
    logits = np.full((T, E), -np.inf, np.float32)
    logits[:, places] = np.array(FAR, np.float32)[np.arange(T) % len(FAR)]
    bias = None
    if biased:  # the largest logit of a softmax, 0, is not among the chosen
        bias = np.ones(E, np.float32)
        bias[1] = -9
        if score == MOE_SCORE_SOFTMAX:
            logits[:, 1] = np.maximum(0, logits[:, places].max(1) + 1)
    b = dev(bias)
    dw = rng.standard_normal((T, k)).astype(np.float32)
    for normalize in (True, False):
        r = rule(score=score, k=k, normalize=normalize, scale=2.5, bias=b)
        idx, w, _ = route(d, r, logits)
        assert np.array_equal(np.sort(idx, 1), np.broadcast_to(places, (T, k)))
        dl = Out((T, E), np.float32)
        keep = [dev(logits), dev(idx), dev(dw)]
        d.route_backward_device(r, *keep, T, E, dl)
        d.synchronize()
        want, grad, mag = log_form(logits.astype(np.float64), idx, dw.astype(np.float64), r)
        # (logarithms of up to 1000 are off by 2^-43, their exponentials by as much)
        assert (np.abs(w - want) <= (2.0 ** -24 + 2.0 ** -40) * np.abs(want) + 1e-45).all(), normalize
        assert (np.abs(dl.get() - grad) <= 2.0 ** -24 * np.abs(grad) + 2.0 ** -38 * mag + 1e-45).all(), normalize
