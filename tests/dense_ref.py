"""The dense operators in 64 bits, with the error that each result may have.

u(t) is half a step of a type relative to the value: bf16 2^-8, f32 2^-24 (an output's rounding, and that
of the logits' gradient, of h and of d(gate, up) before the products after them, which enter in the
activations' type). An f32 sum of n products is within n 2^-24 of the sum of their magnitudes, plus 2^-22
of it for f32 activations, whose three bf16 terms and left-out cross terms keep 2^-24 each. exp, reciprocal
and their arguments add a few 2^-24: 2^-20 covers them."""
import numpy as np

from silentotithrandousha_amd import MOE_BF16, MOE_F32

CLAMP = 7.0
ALPHA = 1.702


def to_bf16(x):
    """Bits of x rounded to the nearest bf16, ties to even (finite values)."""
    u = np.ascontiguousarray(x, np.float32).view(np.uint32)
    r = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), r)


def from_bf16(b):
    return (np.asarray(b, np.uint16).astype(np.uint32) << 16).view(np.float32)


def rows(rng, shape, dtype, scale=1.0):
    """(what the device gets, its values in 64 bits) of random rows."""
    x = (rng.standard_normal(shape) * scale).astype(np.float32)
    return store(x, dtype)


def store(x, dtype):
    if dtype == MOE_F32:
        x = np.ascontiguousarray(x, np.float32)
        return x, x.astype(np.float64)
    b = to_bf16(x)
    return b, from_bf16(b).astype(np.float64)


def load(buf, dtype, shape):
    if dtype == MOE_F32:
        return buf.download(np.float32, shape).astype(np.float64)
    return from_bf16(buf.download(np.uint16, shape)).astype(np.float64)


def u(dtype):
    return 2.0 ** -24 if dtype == MOE_F32 else 2.0 ** -8


def sums(n, magnitude, dtype):
    """Error of sums of n products whose magnitudes add up to `magnitude`."""
    passes = 6 if dtype == MOE_F32 else 1
    return (n * passes * 2.0 ** -24 + (2.0 ** -22 if dtype == MOE_F32 else 0.0)) * magnitude


# Factors below the smallest normal number of bf16 and f32, 2^-126 (exponentials of far logits, the lower
# terms of a small f32 value) may enter a product as 0: each of up to 3 x 2^12 products of a sum then loses
# at most 2^-126 times its other factor, which is below 4 here. Together below 2^-110.
TINY = 2.0 ** -110


def assert_close(got, want, tol, what):
    assert got.shape == want.shape, what
    assert np.array_equal(np.isnan(got), np.isnan(want)), f"{what}: NaN in other places"
    ok = ~np.isnan(want)
    off = np.abs(got - want)[ok] - np.broadcast_to(tol, want.shape)[ok] - TINY
    if off.size:
        i = int(np.argmax(off))
        assert off[i] <= 0, f"{what}: {got[ok][i]!r} against {want[ok][i]!r}, tolerance {np.broadcast_to(tol, want.shape)[ok][i]:.3e}"


class Loss:
    """Loss of x [T, H] over w [V, H] (64 bits), its gradient, and their tolerances."""

    def __init__(self, x, w, targets, dloss, dtype):
        T, H = x.shape
        V = w.shape[0]
        logits, mag = x @ w.T, np.abs(x) @ np.abs(w).T
        dl = sums(H, mag, dtype)  # of a logit
        top = logits.max(1)
        self.lse = top + np.log(np.exp(logits - top[:, None]).sum(1))
        live, invalid = targets >= 0, targets >= V
        at = np.where(live & ~invalid, targets, 0)
        t = np.arange(T)
        self.loss = np.where(live, self.lse - logits[t, at], 0.0)
        self.loss[invalid] = np.nan
        # a sum of V positive terms, each off by its logit's error and 2^-20, in f32
        self.lse_tol = dl.max(1) + 2.0 ** -20 + V * 2.0 ** -24 + 2.0 ** -22 * np.abs(self.lse)
        self.loss_tol = self.lse_tol + dl[t, at] + 2.0 ** -23 * np.abs(self.loss)
        # the logits' gradient, from the log-sum-exp that the loss returned
        p = np.exp(logits - self.lse[:, None])
        hot = np.zeros_like(p)
        hot[t[live & ~invalid], at[live & ~invalid]] = 1.0
        g = (p - hot) * (dloss * live)[:, None]
        g_tol = np.abs(dloss * live)[:, None] * (p * (dl + self.lse_tol[:, None] + 2.0 ** -20)) + (u(dtype) + 2.0 ** -22) * np.abs(g)
        self.dx = g @ w
        self.dx_tol = g_tol @ np.abs(w) + sums(V, np.abs(g) @ np.abs(w), dtype) + u(dtype) * np.abs(self.dx)
        self.dx[invalid] = np.nan
        self.dw = g.T @ x
        self.dw_tol = g_tol.T @ np.abs(x) + sums(T, np.abs(g).T @ np.abs(x), dtype) + u(dtype) * np.abs(self.dw)
        if invalid.any():
            self.dw[:] = np.nan


class Block:
    """Gated block of x [T, H] (64 bits), its gradients, and their tolerances. x_hat: the values that the
    backward pass takes in x's place."""

    def __init__(self, x, wgu, bgu, wd, bd, dy, dtype, x_hat=None):
        self.dtype, self.wgu, self.bgu, self.wd = dtype, wgu, bgu, wd
        h, h_tol = self._gate(x)[4:6]
        I = wd.shape[1]  # noqa: E741
        h_tol = h_tol + u(dtype) * np.abs(h)
        self.y = h @ wd.T + bd
        self.y_tol = (h_tol @ np.abs(wd).T + sums(I + 1, np.abs(h) @ np.abs(wd).T + np.abs(bd), dtype)
                      + (u(dtype) + 2.0 ** -24) * np.abs(self.y))
        if dy is not None:
            self._backward(x if x_hat is None else x_hat, dy)

    def _gate(self, x):
        H = x.shape[1]
        gu = x @ self.wgu.T + self.bgu
        tol = sums(H + 1, np.abs(x) @ np.abs(self.wgu).T + np.abs(self.bgu), self.dtype)
        g, up, dg, du = gu[:, 0::2], gu[:, 1::2], tol[:, 0::2], tol[:, 1::2]
        # no value so near a clamp that 32 bits may see it on the other side, except on it exactly
        for v, d in ((g - CLAMP, dg), (np.abs(up) - CLAMP, du)):
            assert not ((np.abs(v) <= d) & (v != 0)).any(), "the inputs put a value next to a clamp"
        G, U = np.minimum(g, CLAMP), np.clip(up, -CLAMP, CLAMP)
        s = 1.0 / (1.0 + np.exp(-ALPHA * G))
        h = (U + 1.0) * G * s
        # |d(G s)/dG| <= 1.1
        h_tol = np.abs(U + 1.0) * 1.1 * dg + np.abs(G * s) * du + 2.0 ** -20 * (np.abs(U) + 1.0) * np.abs(G * s)
        return g, up, (G, U, s), (dg, du), h, h_tol

    def _backward(self, x, dy):
        dt = self.dtype
        T, H = x.shape
        g, up, (G, U, s), (eg, eu), h, h_tol = self._gate(x)
        dh, dh_tol = dy @ self.wd, sums(H, np.abs(dy) @ np.abs(self.wd), dt)
        A = s * (1.0 + ALPHA * G * (1.0 - s))  # d(G s)/dG, at most 1.1; its slope is below 0.9
        in_g, in_u = g <= CLAMP, np.abs(up) <= CLAMP
        dg, du = dh * (U + 1.0) * A * in_g, dh * G * s * in_u
        dg_tol = (dh_tol * np.abs(U + 1.0) * 1.1 + np.abs(dh) * (eu * 1.1 + np.abs(U + 1.0) * 0.9 * eg
                  + 2.0 ** -20 * (np.abs(U) + 1.0) * (1.0 + np.abs(G) * s))) * in_g
        du_tol = (dh_tol * np.abs(G * s) + np.abs(dh) * (1.1 * eg + 2.0 ** -20 * np.abs(G * s))) * in_u
        d, d_tol = np.stack((dg, du), -1).reshape(T, -1), np.stack((dg_tol, du_tol), -1).reshape(T, -1)
        self.dbgu, self.dbgu_tol = d.sum(0), d_tol.sum(0) + T * 2.0 ** -24 * np.abs(d).sum(0)
        d_tol = d_tol + u(dt) * np.abs(d)
        h_tol = h_tol + u(dt) * np.abs(h)

        def product(a, a_tol, b, b_tol, n):
            want, m = a.T @ b, np.abs(a).T @ np.abs(b)
            tol = np.abs(a).T @ b_tol + a_tol.T @ np.abs(b) + a_tol.T @ b_tol + sums(n, m, dt) + u(dt) * np.abs(want)
            return want, tol

        zero = np.zeros_like
        self.dx, self.dx_tol = product(d.T, d_tol.T, self.wgu, zero(self.wgu), d.shape[1])
        self.dwgu, self.dwgu_tol = product(d, d_tol, x, zero(x), T)
        self.dwd, self.dwd_tol = product(dy, zero(dy), h, h_tol, T)
        self.dbd, self.dbd_tol = dy.sum(0), (T + 1) * 2.0 ** -24 * np.abs(dy).sum(0)


def act8(x):
    """(codes, scale bytes, values in 64 bits) of the 8-bit form of f32 rows x [n, cols], by its definition."""
    pos = np.array([m / 8 * 2.0 ** -6 for m in range(8)]
                   + [(1 + m / 8) * 2.0 ** (k - 7) for k in range(1, 16) for m in range(8)])[:127]
    b = np.asarray(x, np.float64).reshape(x.shape[0], -1, 32)
    bad = ~np.isfinite(b).all(-1)
    top = np.where(bad, 0.0, np.abs(np.where(np.isfinite(b), b, 0.0)).max(-1))
    e = np.full(top.shape, -127)
    for k in range(-127, 121):
        e = np.where(top > 448.0 * 2.0 ** k, k + 1, e)
    v = np.abs(np.where(np.isfinite(b), b, 0.0)) / 2.0 ** e[..., None]
    hi = np.minimum(np.searchsorted(pos, v), 126)
    lo = np.maximum(hi - 1, 0)
    down, up = v - pos[lo], pos[hi] - v
    code = np.where((down < up) | ((down == up) & (lo % 2 == 0)), lo, hi)
    values = pos[code] * np.where(np.signbit(b), -1.0, 1.0) * 2.0 ** e[..., None]
    codes = (code | np.where(np.signbit(b), 128, 0)).astype(np.uint8)
    codes[bad] = 0x7F
    values[bad] = np.nan
    scales = np.where(bad, 255, e + 127).astype(np.uint8)
    return codes.reshape(x.shape), scales, values.reshape(x.shape)
