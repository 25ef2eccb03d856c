"""64-bit results of the serving operators (include/moe_serve.h) and what an f32 kernel may be off by."""
import numpy as np

from silentotithrandousha_amd import MOE_BF16, MOE_F32, MOE_GROUP_TOP2, MOE_MXFP4, MOE_MXFP8, MOE_SCORE_SIGMOID
from tests import dense_ref

E2M1 = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])


def mx4(x):
    """(blocks [n, cols / 32, 16], scales [n, cols / 32], values) of rows x [n, cols]."""
    b = np.asarray(x, np.float64).reshape(x.shape[0], -1, 32)
    with np.errstate(invalid="ignore"):
        top = np.abs(b).max(-1)
    bad = ~np.isfinite(b).all(-1)
    _, e = np.frexp(np.where(bad, 1.0, top))
    e = np.maximum(np.where(top > 0, e - 3, -126), -126)
    v = np.abs(np.where(bad[..., None], 0.0, b)) * 2.0 ** -e[..., None].astype(np.float64)
    hi = np.minimum(np.searchsorted(E2M1, v), 7)
    lo = np.maximum(hi - 1, 0)
    down, up = v - E2M1[lo], E2M1[hi] - v
    code = np.where((down < up) | ((down == up) & (lo % 2 == 0)), lo, hi)
    values = np.where(bad[..., None], np.nan, E2M1[code] * np.sign(b) * 2.0 ** e[..., None].astype(np.float64))
    code = np.where(bad[..., None], 0, code + 8 * np.signbit(b)).astype(np.uint8)
    return code[..., 0::2] | code[..., 1::2] << 4, np.where(bad, 255, e + 127).astype(np.uint8), values.reshape(x.shape)


def mx4_values(blocks, scales):
    """What MXFP4 blocks stand for in a product: a scale byte of 0 is 2^-127, of 255 NaN."""
    code = np.stack((blocks & 15, blocks >> 4), -1).reshape(*blocks.shape[:2], 32)
    s = np.where(scales == 255, np.nan, 2.0 ** (scales.astype(np.float64) - 127.0))
    v = E2M1[code & 7] * np.where(code & 8, -1.0, 1.0) * s[..., None]
    return v.reshape(blocks.shape[0], -1)


def matmul(x, x_type, w, bias, dtype):
    """(y, tolerance) of rows' values x and weights' values w.

    Entering: f32 rows are off by 2^-29, bf16 rows by 2^-19 of their block's largest magnitude (and 2^-129), microscaled rows by
    nothing; in the mean over a block far less, but a result may hang on one value. Sums: an MFMA adds 128 products to
    its accumulator, each of its roundings at most 2^-23 (f32, truncated or not) of the magnitudes' sum; counted as 8 an
    MFMA for its 128 products and 1 for the accumulator. Then the bias and the output's rounding.

    The products of e4m3 with E2M1 lie up to 2^24 apart (448 x 6 to 2^-9 x 0.5). The MFMA aligns 8 neighbours to the
    largest and drops what lies more than 13 bits below its leading bit (measured: beside 256 a 2^-5 is kept, a 2^-6 lost; none is
    lost outside the 8): each of the other 7 may lose up to 2^-13 of it. Products of E2M3 and E2M1 (45 to 2^-4) and of two E2M1
    lie within 10 bits: nothing is dropped."""
    x = np.asarray(x, np.float64)
    y = x @ w.T + bias
    mag = np.abs(x) @ np.abs(w).T
    terms = {MOE_F32: 6, MOE_BF16: 4}.get(x_type, 1)
    steps = -(-x.shape[1] // 128)
    tol = (steps * terms + 8) * 2.0 ** -23 * mag
    if x_type == MOE_MXFP8:
        gx, gw = (np.abs(v).reshape(v.shape[0], -1, 8).max(-1) for v in (x, w))  # (no product is above those of these)
        tol += 7 * 2.0 ** -13 * (gx @ gw.T)
    if terms > 1:
        top = np.abs(x).reshape(x.shape[0], -1, 32).max(-1)
        off = np.where(top < 2.0 ** -99, 2.0 ** -129, 2.0 ** (-29 if x_type == MOE_F32 else -19) * top)
        if x_type == MOE_BF16:  # values of bf16 down to 2^-11 of the largest enter exactly
            small = np.abs(x).reshape(*top.shape, 32) < 2.0 ** -11 * top[..., None]
            # (a block whose largest is below 2^-99: terms have scales of at least 2^-126 and steps of 2^-3 of those, so that a bf16
            # between 2^-k and 2^(1 - k), whose step is 2^-(k + 7), is off by up to 2^-130 from k = 123 on, whatever the block's
            # largest; the last term's rounding counted as 2^-129 as for f32)
            small |= (top < 2.0 ** -99)[..., None]
            tol += (off[..., None] * small).reshape(x.shape) @ np.abs(w).T
        else:
            tol += off.repeat(32, -1) @ np.abs(w).T
    return y, tol + 2 * 2.0 ** -24 * (np.abs(y) + np.abs(bias)) + (dense_ref.u(dtype) + 2.0 ** -24) * np.abs(y)


def x_forms(x, x_type):
    """(what a product takes: codes, scales or None; the values that they stand for) of rows x."""
    if x_type == MOE_MXFP4:
        blocks, scales, values = mx4(x)
        return blocks, scales, values
    if x_type == MOE_MXFP8:
        codes, scales, values = dense_ref.act8(np.asarray(x, np.float64))
        return codes, scales, values
    stored, values = dense_ref.store(x, x_type)
    return stored, None, values


def scores(logits, score):
    z = np.asarray(logits, np.float64)
    z = np.where(np.isnan(z), -np.inf, z)
    if score == MOE_SCORE_SIGMOID:
        with np.errstate(over="ignore"):
            return 1.0 / (1.0 + np.exp(-z))
    top = z.max(1, keepdims=True)
    with np.errstate(invalid="ignore"):
        e = np.where(z == top, 1.0, np.exp(z - top))
    e = np.where(z == -np.inf, 0.0, e)
    total = e.sum(1, keepdims=True)
    return e / np.where(total > 0, total, 1.0)


def route(logits, rule, bias=None):
    """(idx, weights, counts), token by token."""
    T, E = logits.shape
    s = scores(logits, rule.score)
    idx, w = np.full((T, rule.top_k), -1, np.int32), np.zeros((T, rule.top_k))
    for t in range(T):
        dead = np.isnan(logits[t]) | (logits[t] == -np.inf)
        key = s[t] + (np.asarray(bias, np.float64) if bias is not None else 0.0)
        dead |= np.isnan(key) | (key == -np.inf)
        key = np.where(dead, -np.inf, key)
        order_by = key if bias is not None else np.where(dead, -np.inf, logits[t].astype(np.float64))
        if rule.n_groups > 1:
            per = np.sort(key.reshape(rule.n_groups, -1), 1)[:, ::-1]
            g = per[:, 0].copy()
            if rule.group_score == MOE_GROUP_TOP2 and per.shape[1] > 1:
                g = np.where(per[:, 1] > -np.inf, per[:, 0] + np.where(per[:, 1] > -np.inf, per[:, 1], 0), g)
            kept = np.argsort(-g, kind="stable")[:rule.top_groups]
            dead |= ~np.isin(np.arange(E) // (E // rule.n_groups), kept)
        order = [e for e in np.argsort(-np.where(dead, -np.inf, order_by), kind="stable") if not dead[e]][:rule.top_k]
        n = len(order)
        v = s[t][order]
        if rule.normalize and n:
            v = v / v.sum() if v.sum() > 0 else np.full(n, 1.0 / n)
        idx[t, :n], w[t, :n] = order, v * np.float64(rule.scale)
    return idx, w, np.bincount(idx[idx >= 0], minlength=E).astype(np.int32)


def route_weights(logits, idx, rule):
    """The weights as a function of the logits, the choice fixed."""
    s = scores(logits, rule.score)
    live = (idx >= 0) & (idx < logits.shape[1])
    v = np.where(live, np.take_along_axis(s, np.where(live, idx, 0), 1), 0.0)
    if rule.normalize:
        total = v.sum(1, keepdims=True)
        v = np.where(total > 0, v / np.where(total > 0, total, 1.0), 0.0)
    return v * np.float64(rule.scale)


def route_backward(logits, idx, dweights, rule):
    """(dlogits, tolerance): by the chain rule of the logarithms, log w = log s - log S."""
    z = np.asarray(logits, np.float64)
    s = scores(logits, rule.score)
    live = (idx >= 0) & (idx < z.shape[1])
    w = route_weights(logits, idx, rule)
    g = np.where(live, dweights * w, 0.0)
    size = np.abs(g)
    if rule.normalize:
        part = w / np.float64(rule.scale) if rule.scale else 0.0 * w
        g = g - part * g.sum(1, keepdims=True)
        size = size + part * size.sum(1, keepdims=True)
    out, mag = np.zeros_like(z), np.zeros_like(z)
    for j in range(idx.shape[1]):
        at = np.where(live[:, j], idx[:, j], 0)[:, None]
        f = (1.0 - np.take_along_axis(s, at, 1)[:, 0]) if rule.score == MOE_SCORE_SIGMOID else 1.0
        np.put_along_axis(out, at, np.take_along_axis(out, at, 1) + (g[:, j] * f * live[:, j])[:, None], 1)
        np.put_along_axis(mag, at, np.take_along_axis(mag, at, 1) + (size[:, j] * f * live[:, j])[:, None], 1)
    if rule.score != MOE_SCORE_SIGMOID and not rule.normalize:
        out -= s * g.sum(1, keepdims=True)
        mag += s * size.sum(1, keepdims=True)
    return out, 2.0 ** -24 * np.abs(out) + 2.0 ** -44 * mag + 1e-45


def sample(logits, u, temperature=None, top_k=None, top_p=None, min_p=None):
    """(tokens, logprob, room): room says how far u lies from the nearest border between two tokens, and top_p from
    the sums at its own, relative to the sums' scale; below 2^-40 a kernel whose masses are whole numbers may differ."""
    T, V = logits.shape
    tokens, logprob, room = np.full(T, -1, np.int64), np.full(T, np.nan), np.ones(T)
    for t in range(T):
        row = np.where(np.isnan(logits[t]), -np.inf, logits[t].astype(np.float64))
        m = row.max()
        if m == -np.inf:
            continue
        tau = 1.0 if temperature is None else float(temperature[t])
        order = np.argsort(-row, kind="stable")
        if not tau > 0:
            tokens[t], logprob[t] = order[0], 0.0
            continue
        with np.errstate(invalid="ignore"):
            z = np.where(row == m, 0.0, np.where(row == -np.inf, -np.inf, (row - m) / tau))
        e = np.exp(z)[order]
        k = V if top_k is None or top_k[t] < 1 else min(int(top_k[t]), V)
        p = 1.0 if top_p is None else float(top_p[t])
        least = 0.0 if min_p is None or not min_p[t] > 0 else float(min_p[t])
        e[k:] = 0.0
        if p < 1:
            before = np.concatenate(([0.0], np.cumsum(e)[:-1]))
            target = max(p, 0.0) * e.sum()
            keep = before < target
            keep[0] = True
            room[t] = min(room[t], np.abs(before[1:k] - target).min(initial=1.0) / e.sum())
            e = np.where(keep, e, 0.0)
        e = np.where((e >= least) | (row[order] == m), e, 0.0)
        mass = np.zeros(V)
        mass[order] = e
        run = np.cumsum(mass)
        uu = min(max(0.0 if np.isnan(u[t]) else float(u[t]), 0.0), 1.0)
        at = min(int(np.searchsorted(run, uu * run[-1], side="right")), V - 1)
        if uu >= 1:
            at = int(np.nonzero(mass > 2.0 ** -45)[0][-1])
        else:
            room[t] = min(room[t], np.abs(run[mass > 0] - uu * run[-1]).min() / run[-1])
        tokens[t], logprob[t] = at, np.log(mass[at] / run[-1])
    return tokens, logprob, room
