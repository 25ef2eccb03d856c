"""The dense product's operand tiles replayed on the CPU (csrc/dense_gemm.hpp, DenseTile): every LDS-DMA
reads inside the operand, and the fragments that the wavefronts read back from LDS are the rows and k
values that the product needs, zeros past K; with a planted mistake the replay fails."""
import numpy as np
import pytest

STEP = 64
HALF = 32


def piece(q, k, pairs):
    mask = np.where((q | 3) < pairs, 3, 0) if pairs >= 4 else 1 if pairs >= 2 else 0
    return q ^ (k & mask)


def load(mem, base, ld, R, W, transposed, rows, left, clamp=True):
    """LDS image (bf16 elements) of one step: mem is the operand's memory, base the tile's first element."""
    lds = np.full(R * STEP, -1.0)
    dmas = R // 8
    lane = np.arange(64)
    for wave in range(W):
        for i in range(-(-dmas // W)):
            dma = (i * W + wave) % dmas
            c = dma * 64 + lane
            part = k_of(c, R, transposed)
            if not transposed:
                at = np.minimum(c >> 3, rows - 1) * ld + part
                back = part
            else:
                pos = c % (R // 8)
                col = piece(pos >> 1, part, R // 16) * 16 + (pos & 1) * 8
                col = np.where(col >= rows, 0, col)
                at = part * ld + col
                back = (part - (left - 1)) * ld
            if left < STEP and clamp:
                at = at - np.where(part >= left, back, 0)
            at = base + at
            assert at.min() >= 0 and at.max() + 8 <= mem.size, "a load outside the operand"
            for j in range(8):
                lds[dma * 512 + lane * 8 + j] = mem[at + j]
    assert (lds != -1.0).all()
    return lds


def k_of(c, R, transposed):
    return c // (R // 8) if transposed else ((c & 7) ^ ((c >> 3) & 7)) * 8


def zero_tail(lds, R, transposed, left):
    for c in range(R * 8):
        if k_of(c, R, transposed) >= left:
            lds[c * 8:c * 8 + 8] = 0


def frag(lds, R, transposed, row0, half):
    """[64 lanes][8]: what the lanes hold of 16 rows and a half step's 32 k values."""
    out = np.empty((64, 8))
    lane = np.arange(64)
    if not transposed:
        row, ch = row0 + (lane & 15), half * 4 + (lane >> 4)
        at = row * 64 + (ch ^ (row & 7)) * 8
        for j in range(8):
            out[:, j] = lds[at + j]
        return out
    i, q = lane & 15, row0 >> 4
    k = (lane >> 4) * 8 + (i >> 2)
    for part in range(2):
        kh = k + 4 * part
        at = (half * HALF + kh) * R + piece(np.full(64, q), kh, R // 16) * 16 + (i & 3) * 4
        for j in range(4):  # lane l gets element l % 4 of the lane j * 4 + l / 4 of its 16
            src = (lane & 48) + j * 4 + (i >> 2)
            out[:, part * 4 + j] = lds[at[src] + (i & 3)]
    return out


def tile_of(b, tiles_m, tiles_n):
    total = tiles_m * tiles_n
    x, q, r = b & 7, total >> 3, total & 7
    t = x * q + min(x, r) + (b >> 3)
    group = t // (tiles_m * 8)
    n0 = group * 8
    width, inside = min(8, tiles_n - n0), t - group * tiles_m * 8
    return inside // width, n0 + inside % width


@pytest.mark.parametrize("tiles_m,tiles_n", [(1, 1), (3, 2), (15, 16), (1048, 3), (7, 9), (23, 17), (2, 100), (8, 8)])
def test_every_tile_is_computed_once(tiles_m, tiles_n):
    got = {tile_of(b, tiles_m, tiles_n) for b in range(tiles_m * tiles_n)}
    assert got == {(m, n) for m in range(tiles_m) for n in range(tiles_n)}


# rows of a tile, wavefronts that load it
TILES = [(16, 2), (16, 4), (32, 2), (32, 4), (64, 4), (128, 4), (64, 8), (96, 4), (128, 8), (192, 8), (256, 8), (288, 8)]


@pytest.mark.parametrize("R,W", TILES)
@pytest.mark.parametrize("transposed", [False, True])
def test_tiles(R, W, transposed):
    rng = np.random.default_rng(R + W)
    for rows_all in (1, 7, 8, R - 3, R, R + 5, 2 * R + 9):
        for K in (1, 8, 31, 32, 56, 64, 72, 130):
            if not transposed:
                ld = (K + 7) // 8 * 8
                mat = rng.standard_normal((rows_all, ld))
                value = lambda r, k: mat[r, k]  # noqa: E731
            else:
                ld = (rows_all + 7) // 8 * 8
                mat = rng.standard_normal((K, ld))
                value = lambda r, k: mat[k, r]  # noqa: E731
            mem = mat.reshape(-1)
            for r0 in range(0, rows_all, R):
                for k0 in range(0, K, STEP):
                    base = k0 * ld + r0 if transposed else r0 * ld + k0
                    left = K - k0
                    lds = load(mem, base, ld, R, W, transposed, rows_all - r0, left)
                    if left < STEP:
                        zero_tail(lds, R, transposed, left)
                    for row0 in range(0, R, 16):
                        for half in range(2):
                            got = frag(lds, R, transposed, row0, half)
                            for lane in range(0, 64, 5):
                                r, k = r0 + row0 + (lane & 15), k0 + half * HALF + (lane >> 4) * 8
                                if r >= rows_all:
                                    continue
                                # (K-contiguous values between K and its next multiple of 8 are the operand's own)
                                top = K if transposed else ld
                                want = [value(r, k + j) if k + j < top else 0.0 for j in range(8)]
                                assert np.array_equal(got[lane], want), (rows_all, K, r0, k0, row0, half, lane)


def test_a_planted_overflow_is_found():
    mem = np.zeros(100 * 72)
    with pytest.raises(AssertionError, match="outside"):
        load(mem, 64 + 99 * 72, 72, 128, 4, False, 1, 8, clamp=False)
    with pytest.raises(AssertionError, match="outside"):
        load(mem, 96 * 72, 72, 64, 4, True, 64, 4, clamp=False)
