"""The dense operators at the far ends of f32's range: logits, gates and clamps whose exponents overflow a
factor log2 e, against 64-bit results (tests/dense_ref.py)."""
import numpy as np
import pytest

from silentotithrandousha_amd import MOE_BF16, MOE_F32, GpuMoeDispatcher
from tests import dense_ref as ref
from tests.test_gpu_dense import BlockOnDevice, block_case, block_ref, check_grads, context, run_loss, run_loss_backward

pytestmark = pytest.mark.gpu

TYPES = [MOE_F32, MOE_BF16]
FAR = 1.5 * 2.0 ** 127  # its product with log2 e is above the largest f32


def far_loss_case(dtype, T, V, first, seed):
    """Rows `first` to `first` + 400 of the head are minus the first unit vector: their logits are -x[t, 0]."""
    H = 64
    rng = np.random.default_rng([seed, T, V, dtype])
    x = rng.standard_normal((T, H)).astype(np.float32)
    x[:, 0] = 0.0
    w = (rng.standard_normal((V, H)) * 2 / np.sqrt(H)).astype(np.float32)
    w[:, 0] = 0.0
    far = np.arange(first, first + 400)
    w[far] = 0.0
    w[far, 0] = -1.0
    rest = np.setdiff1d(np.arange(V), far)
    targets = rng.choice(rest, T).astype(np.int32)
    dloss = rng.uniform(-1, 1, T).astype(np.float32)
    return H, x, w, far, rest, targets, dloss


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,V,first", [(1, 1000, 0), (5, 1000, 300), (40, 5000, 4600), (300, 1000, 0)])
def test_loss_far_below(dtype, T, V, first):
    """Logits of -2.6e38 beside ones of order one, in tiles of their own and in shared ones: they count as 0, and the
    results are those of the other rows."""
    H, x, w, far, rest, targets, dloss = far_loss_case(dtype, T, V, first, seed=1)
    x[T // 2, 0] = FAR
    dloss[T // 2] = 0.5
    x, xv = ref.store(x, dtype)
    wb, wv = ref.store(w, MOE_BF16)
    at = np.searchsorted(rest, targets).astype(np.int32)
    bounded = xv.copy()
    bounded[:, 0] = 0.0  # (no row of `rest` reads it)
    want = ref.Loss(bounded, wv[rest], at, dloss.astype(np.float64), dtype)
    # without the far rows only the other tokens' rows have logits of 0 there: those tokens have 400 more terms of exp(0)
    near = np.delete(np.arange(T), T // 2)
    whole = ref.Loss(bounded[near], wv, targets[near], dloss[near].astype(np.float64), dtype) if T > 1 else None
    d = context(H, wb)
    try:
        xd, td, loss, lse = run_loss(d, x, dtype, targets, V)
        t = T // 2
        ref.assert_close(lse.get()[t], want.lse[t], want.lse_tol[t], "lse")
        ref.assert_close(loss.get()[t], want.loss[t], want.loss_tol[t], "loss")
        dx, dw = run_loss_backward(d, xd, dtype, td, lse, dloss, T, H, V)
        ref.assert_close(dx.get()[t], want.dx[t], want.dx_tol[t], "dx")
        if whole is not None:
            ref.assert_close(lse.get()[near], whole.lse, whole.lse_tol, "lse")
            ref.assert_close(loss.get()[near], whole.loss, whole.loss_tol, "loss")
            ref.assert_close(dx.get()[near], whole.dx, whole.dx_tol, "dx")
        assert np.isfinite(dw.get()).all()
    finally:
        d.close()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,V,first", [(1, 1000, 0), (40, 5000, 4600), (300, 1000, 300)])
def test_loss_far_above(dtype, T, V, first):
    """Logits of 2.6e38: the log-sum-exp is their maximum, within the f32 that it is returned in; the gradients are finite."""
    H, x, w, far, rest, targets, dloss = far_loss_case(dtype, T, V, first, seed=2)
    t = T // 2
    x[t, 0] = -FAR
    dloss[t] = 2.0 ** -12
    x, _ = ref.store(x, dtype)
    wb, _ = ref.store(w, MOE_BF16)
    d = context(H, wb)
    try:
        xd, td, loss, lse = run_loss(d, x, dtype, targets, V)
        assert lse.get()[t] == FAR and loss.get()[t] == FAR  # (log 400 and the target's logit are below its half step)
        dx, dw = run_loss_backward(d, xd, dtype, td, lse, dloss, T, H, V)
        assert np.isfinite(dx.get()).all() and np.isfinite(dw.get()).all()
    finally:
        d.close()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T", [1, 5, 40, 300])
def test_block_far_clamp(dtype, T, monkeypatch):
    """A clamp of 3e38 and gates of +-2.6e38 below it (ups of -1/2, so that h stays in range): h is (U + 1) G there and 0
    for the negative ones, the gate's gradient dh (U + 1) and 0."""
    H, I = 32, 16  # noqa: E741
    monkeypatch.setattr(ref, "CLAMP", 3e38)
    c = block_case(dtype, T, H, I, seed=3, bias=False)
    wgu = np.zeros((2 * I, H), np.float32)
    for i in range(I):
        wgu[2 * i, i], wgu[2 * i + 1, 16 + i] = 1.0, 1.0
    c["wgu"] = ref.store(wgu, MOE_BF16)
    c["wd"] = ref.store((ref.from_bf16(c["wd"][0]) * 2.0 ** -30).astype(np.float32), MOE_BF16)
    c["dy"] = ref.store((c["dy"][1] * 2.0 ** -30).astype(np.float32), dtype)
    x = np.array(c["x"][1], np.float32)
    x[:, 16:] = -0.5
    x[T // 2, :16] = np.where(np.arange(16) % 2, FAR, -FAR)
    c["x"] = ref.store(x, dtype)
    with np.errstate(over="ignore"):  # exp of 1.702 times the far negative gates
        want = block_ref(c, dtype)
    d = GpuMoeDispatcher(H, 32, 3e38)
    try:
        b = BlockOnDevice(c, bias=False)
        y, g = b.forward(d, dtype), b.backward(d, dtype)
        d.synchronize()
        ref.assert_close(y.get(), want.y, want.y_tol, "y")
        # an up's gradient times the far x is past f32's range (dh of 2^-60 times 2^254): those entries are not compared
        inside, got = np.abs(want.dwgu) < 2.0 ** 127, g.pop("gate_up").get()
        assert not inside.all() and inside.mean() > 0.5
        ref.assert_close(got[inside], want.dwgu[inside], want.dwgu_tol[inside], "gate_up")
        check_grads(g, want)
    finally:
        d.close()
