"""Inputs of the dense operators whose f32 results show every bit of the f32 rows: rows of 24 significant bits meet weights
of one +-1 a row, so that a product is one value of theirs, and sums have the few terms that are counted here. Tolerances
count those terms: a row's value less its last 8 bits (two bf16 terms in place of three, 2^-17 of it) is outside them, as
is a weight gradient without one of its products of terms (2^-16 to 2^-18)."""
import numpy as np

from tests import dense_ref as ref
from tests.dense_ref import ALPHA

U = 2.0 ** -24


def bits24(rng, shape, top=1.0):
    """Values in [top / 2, top) with 24 significant bits, the last one set."""
    return ((rng.integers(2 ** 22, 2 ** 23, shape) * 2 + 1) * (top * U)).astype(np.float32)


def signs(rng, shape):
    return rng.choice([-1.0, 1.0], shape).astype(np.float32)


def by_one(a, b):
    """sum_t a[t, i] b[t, j] in 64 bits, and of the magnitudes; the number of terms that are not 0."""
    return a.T @ b, np.abs(a).T @ np.abs(b), (a != 0).astype(np.float64).T @ (b != 0).astype(np.float64)


def gradient_tol(magnitude, terms):
    """A weight gradient's error: of each term 6 products of bf16 terms added one by one in f32 and three of at most 2^-24
    together left out, then the sum's own additions and the result's rounding."""
    return (12.0 * terms + 4.0) * U * magnitude


class Loss:
    """Row v_c of the head is +-e_c, every other row 0; a token's largest logit is above 128, the others below 1, so that
    their exponentials are 0 in f32. The log-sum-exp is the largest logit, off by half a step of the base 2 logarithm
    that exponentials are taken against (2^-24 of it) and by its own rounding. Given the exact one, dx is exact, and dw sums
    the tokens whose largest logit or target a row is."""

    def __init__(self, T, H, V, seed=41):
        rng = np.random.default_rng([seed, T, H, V])
        m = min(H, V)
        self.row = rng.permutation(V)[:m]  # of column c
        sign = signs(rng, m)
        w = np.zeros((V, H), np.float32)
        w[self.row, np.arange(m)] = sign
        x = bits24(rng, (T, H)) * signs(rng, (T, H))
        t, c = np.arange(T), (np.arange(T) * 7 + seed) % m
        top = bits24(rng, T, 256.0)
        x[t, c] = top * sign[c]
        targets = rng.integers(0, V, T).astype(np.int32)
        targets[rng.random(T) < 0.1] = -1
        dloss = bits24(rng, T) * signs(rng, T)
        self.x, self.w, self.targets, self.dloss = x, w, targets, dloss
        live = targets >= 0
        self.lse = top.astype(np.float64)
        picked = (x * w[np.where(live, targets, 0)]).sum(1)  # (one term: exact)
        self.loss = np.where(live, top - picked, np.float32(0)).astype(np.float64)
        scale = np.abs(dloss[live]).max() if live.any() else np.float32(1)
        d = (dloss / scale).astype(np.float32) * live  # over the largest dloss, and times it again behind the product
        d[targets == self.row[c]] = 0.0
        back = (d * scale).astype(np.float32)
        self.d, self.scale, self.best = d, scale, self.row[c]
        self.dx = np.zeros((T, H))
        self.dx[t, c] += back * sign[c]
        column = np.full(V, -1)
        column[self.row] = np.arange(m)
        at = column[np.where(live, targets, 0)]
        k = live & (at >= 0) & (d != 0)
        self.dx[t[k], at[k]] -= back[k] * sign[at[k]]
        self.dw, magnitude, terms = np.zeros((V, H)), np.zeros((V, H)), np.zeros(V)
        dt = d.astype(np.float64) * np.float64(scale)
        one = x.astype(np.float64)
        for rows, s in ((self.best, 1.0), (np.where(live, targets, 0), -1.0)):
            np.add.at(self.dw, rows, s * dt[:, None] * one)
            np.add.at(magnitude, rows, np.abs(dt[:, None] * one))
            np.add.at(terms, rows, d != 0)
        self.dw_tol = gradient_tol(magnitude, terms[:, None])

    def check(self, got):
        """dx and dw: with self.lse for the log-sum-exp."""
        lse_tol = 2 * U * np.abs(self.lse)
        ref.assert_close(got["lse"], self.lse, lse_tol, "lse")
        ref.assert_close(got["loss"], self.loss, np.where(self.targets < 0, 0.0, lse_tol + U * np.abs(self.loss)), "loss")
        assert np.array_equal(got["dx"], self.dx), np.abs(got["dx"] - self.dx).max()
        ref.assert_close(got["dw"], self.dw, self.dw_tol, "dw")


class Block:
    """Gate i is +-x[a_i], up i x[b_i], output j +-h[i_j]; x is positive and below 4 (no clamp is reached, no sum cancels).
    dy has a few values a column, so that every sum over the tokens has a few terms."""

    def __init__(self, T, H, I, seed=42, kept=False):  # noqa: E741
        rng = np.random.default_rng([seed, T, H, I])
        i = np.arange(I)
        a, b, sg = i % H, (i * 5 + 3) % H, signs(rng, I)
        wgu = np.zeros((2 * I, H), np.float32)
        wgu[2 * i, a], wgu[2 * i + 1, b] = sg, 1.0
        j = np.arange(H)
        at, sd = j % I, signs(rng, H)
        wd = np.zeros((H, I), np.float32)
        wd[j, at] = sd
        x = bits24(rng, (T, H), 4.0) * 2.0 ** -rng.integers(0, 3, (T, H)).astype(np.float32)
        dy = bits24(rng, (T, H)) * signs(rng, (T, H))
        if T > 4:
            dy[rng.random((T, H)) > 3.0 / T] = 0.0
        self.x, self.dy, self.wgu, self.wd = x, dy, wgu, wd
        f = np.float64
        h, h_tol = self.gate(x.astype(f), a, b, sg)[3:]
        self.y, self.y_tol = h[:, at] * sd, h_tol[:, at] + 2 * U * np.abs(h[:, at])
        xh = ref.act8(x.astype(f))[2] if kept else x.astype(f)
        G, Up, s, h, h_tol = self.gate(xh, a, b, sg)
        dh, dh_sum = np.zeros((T, I)), np.zeros((T, I))
        np.add.at(dh, (slice(None), at), dy.astype(f) * sd)
        np.add.at(dh_sum, (slice(None), at), np.abs(dy.astype(f)))
        dh_tol = (-(-H // I) - 1) * U * dh_sum
        A = s * (1.0 + ALPHA * G * (1.0 - s))
        d, d_tol = np.zeros((T, 2 * I)), np.zeros((T, 2 * I))
        d[:, 0::2], d[:, 1::2] = dh * (Up + 1.0) * A, dh * G * s
        d_tol[:, 0::2] = dh_tol * (Up + 1.0) * 1.1 + np.abs(dh) * 2.0 ** -20 * (Up + 1.0) * (1.0 + np.abs(G) * s)
        d_tol[:, 1::2] = dh_tol * np.abs(G * s) + np.abs(dh) * 2.0 ** -20 * np.abs(G * s)
        terms = (d != 0).sum(0)
        self.gate_up_bias, self.gate_up_bias_tol = d.sum(0), d_tol.sum(0) + terms * U * np.abs(d).sum(0)
        self.down_bias, self.down_bias_tol = dy.astype(f).sum(0), ((dy != 0).sum(0) + 1) * U * np.abs(dy.astype(f)).sum(0)
        col, sign = np.stack((a, b), 1).reshape(-1), np.stack((sg, np.ones(I)), 1).reshape(-1)
        self.dx, size, tol, count = (np.zeros((T, H)) for _ in range(4))
        for out, v in ((self.dx, d * sign), (size, np.abs(d)), (tol, d_tol), (count, (d != 0).astype(f))):
            order = np.argsort(col, kind="stable")
            sums = np.add.reduceat(v[:, order], np.unique(col[order], return_index=True)[1], axis=1)
            out[:, np.unique(col)] = sums
        self.dx_tol = tol + (3.0 * count + 2.0) * U * size
        self.gate_up, size, count = by_one(d, xh)
        self.gate_up_tol = d_tol.T @ np.abs(xh) + gradient_tol(size, count)
        self.down, size, count = by_one(dy.astype(f), h)
        self.down_tol = np.abs(dy.astype(f)).T @ h_tol + gradient_tol(size, count)

    @staticmethod
    def gate(x, a, b, sg):
        """(gate, up, sigmoid, h, h's error): exp, reciprocal and three products in f32."""
        G, Up = x[:, a] * sg, x[:, b]
        s = 1.0 / (1.0 + np.exp(-ALPHA * G))
        h = (Up + 1.0) * G * s
        return G, Up, s, h, 2.0 ** -20 * (Up + 1.0) * np.abs(G * s)

    def check(self, got):
        for n, v in got.items():
            name = "dx" if n == "x" else n
            ref.assert_close(v, getattr(self, name), getattr(self, name + "_tol"), n)
