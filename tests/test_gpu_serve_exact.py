"""The serving operators (include/moe_serve.h) where values of far sizes meet: each result against 64 bits, with tolerances that
hold what f32 sums lose and nothing else."""
import numpy as np
import pytest

from silentotithrandousha_amd import MOE_BF16, MOE_F32, MOE_MXFP8
from tests import dense_ref, serve_ref as ref
from tests.test_gpu_serve import d, matmul, resident, sample, weights  # noqa: F401

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
