"""The exact cases (tests/dense_exact.py) against the operators' f32 arithmetic, emulated with bf16 terms in 64 bits: three
terms a value pass, and every mistake with a term is found. (The tolerances of tests/dense_ref.py, which count the roundings
of sums over thousands of products, do not see two terms in place of three.)"""
import numpy as np
import pytest

from silentotithrandousha_amd import MOE_F32
from tests import dense_exact as exact
from tests import dense_ref as ref
from tests.dense_ref import ALPHA

PAIRS = [(0, 0), (0, 1), (1, 0), (1, 1), (0, 2), (2, 0)]


def terms(v):
    """v as three bf16 values."""
    out, rest = [], np.asarray(v, np.float32)
    for _ in range(3):
        out.append(ref.from_bf16(ref.to_bf16(rest)))
        rest = (rest - out[-1]).astype(np.float32)
    return [t.astype(np.float64) for t in out]


class Arithmetic:
    """f32 rows as `count` of their terms (of the operand `only`, or of all), weight gradients of `pairs` of them; `swap`: the
    operand whose last two terms change places in the pairs."""

    def __init__(self, count=3, only=None, pairs=PAIRS, swap=None):
        self.count, self.only, self.pairs, self.swap = count, only, pairs, swap

    def terms(self, v, name):
        n = self.count if self.only in (None, name) else 3
        return [t * (k < n) for k, t in enumerate(terms(v))]

    def rows(self, v, name):
        return sum(self.terms(v, name))

    def gradient(self, a, b, names):
        a, b = self.terms(a, names[0]), self.terms(b, names[1])
        for v, n in ((a, names[0]), (b, names[1])):
            if n == self.swap:
                v[1], v[2] = v[2], v[1]
        return sum(a[i].T @ b[j] for i, j in self.pairs)


def f32(v):
    return v.astype(np.float32).astype(np.float64)


def loss(c, m):
    logits = m.rows(c.x, "x") @ c.w.T.astype(np.float64)
    t = np.arange(len(c.x))
    lse = f32(logits.max(1) + np.log(f32(np.exp(logits - logits.max(1)[:, None]).sum(1))))
    live = c.targets >= 0
    at = np.where(live, c.targets, 0)
    out = dict(lse=lse, loss=f32(np.where(live, lse - logits[t, at], 0.0)))
    p = np.exp(logits - c.lse[:, None])
    p[p < 2.0 ** -126] = 0.0
    hot = np.zeros_like(p)
    hot[t[live], at[live]] = 1.0
    q = np.where(live, (c.dloss / c.scale).astype(np.float32), np.float32(0))
    d = ((p - hot) * q[:, None]).astype(np.float32)
    out["dx"] = f32(f32(m.rows(d, "d") @ c.w.astype(np.float64)) * np.float64(c.scale))
    out["dw"] = f32(m.gradient(d, c.x, "dx") * np.float64(c.scale))
    return out


def block(c, m, kept=False):
    w, wd = c.wgu.astype(np.float64), c.wd.astype(np.float64)

    def gates(x):
        gu = f32(x @ w.T)
        G, U = gu[:, 0::2], gu[:, 1::2]
        s = 1.0 / (1.0 + np.exp(-ALPHA * G))
        return G, U, s, f32((U + 1.0) * G * s)

    out = dict(y=f32(m.rows(gates(m.rows(c.x, "x"))[3], "h") @ wd.T))
    xh = ref.act8(c.x.astype(np.float64))[2]
    G, U, s, h = gates(xh if kept else m.rows(c.x, "x"))
    dh = f32(m.rows(c.dy, "dy") @ wd)
    d = np.stack((f32(dh * (U + 1.0) * s * (1.0 + ALPHA * G * (1.0 - s))), f32(dh * G * s)), -1).reshape(len(c.x), -1)
    out["x"] = f32(m.rows(d, "d") @ w)
    out["gate_up"] = f32(m.rows(d, "d").T @ xh if kept else m.gradient(d, c.x, ("d", "x")))
    out["gate_up_bias"] = f32(d.sum(0))
    out["down"] = f32(m.gradient(c.dy, h, ("dy", "h")))
    return out


LOSSES = [(4, 64, 257), (12, 96, 300), (130, 64, 333)]  # (of one token d is +-1: its dloss is the largest)
BLOCKS = [(1, 64, 40), (3, 32, 200), (40, 96, 72), (300, 64, 128)]
DROPPED = [[p for p in PAIRS if p != drop] for drop in PAIRS]


@pytest.mark.parametrize("T,H,V", LOSSES)
def test_loss(T, H, V):
    c = exact.Loss(T, H, V)
    c.check(loss(c, Arithmetic()))
    for wrong in ([Arithmetic(n) for n in (1, 2)] + [Arithmetic(2, o) for o in "dx"] + [Arithmetic(pairs=p) for p in DROPPED]
                  + [Arithmetic(swap=o) for o in "dx"]):
        with pytest.raises(AssertionError):
            c.check(loss(c, wrong))


@pytest.mark.parametrize("kept", [False, True])
@pytest.mark.parametrize("T,H,I", BLOCKS)
def test_block(T, H, I, kept):  # noqa: E741
    c = exact.Block(T, H, I, kept=kept)
    c.check(block(c, Arithmetic(), kept))
    for wrong in ([Arithmetic(n) for n in (1, 2)] + [Arithmetic(2, o) for o in ("x", "h", "dy", "d")] + [Arithmetic(pairs=p) for p in DROPPED]
                  + [Arithmetic(swap=o) for o in ("dy", "h", *(("d", "x") * (not kept)))]):
        with pytest.raises(AssertionError):
            c.check(block(c, wrong, kept))


def test_the_summed_tolerances_do_not_see_it():
    """What these cases are for: two terms a value are inside the tolerances of sums of many products."""
    rng = np.random.default_rng(1)
    x, w = rng.standard_normal((20, 544)).astype(np.float32), ref.rows(rng, (300, 544), 1, 2 / np.sqrt(544))[1]
    targets, dloss = rng.integers(0, 300, 20).astype(np.int32), rng.uniform(-1, 1, 20)
    want = ref.Loss(x.astype(np.float64), w, targets, dloss, MOE_F32)
    two = ref.Loss(sum(terms(x)[:2]), w, targets, dloss, MOE_F32)
    ref.assert_close(two.lse, want.lse, want.lse_tol, "lse")
    ref.assert_close(two.dx, want.dx, want.dx_tol, "dx")
