"""The dense operators at the sizes of tests/dense_sizes.py, which take the forms of launch that the other tests do not,
against 64 bits. Of large sizes sampled tokens and sampled rows of the vocabulary (or inner columns) are compared, the
first, the last and those at the ends of a piece among them; of the others everything."""
import numpy as np
import pytest

from silentotithrandousha_amd import MOE_MXFP8, DeviceBuffer
from tests import dense_ref as ref
from tests import dense_sizes as sizes
from tests.test_gpu_dense import NAMES, BlockOnDevice, block_case, check_grads, context, loss_case, run_loss, run_loss_backward

pytestmark = pytest.mark.gpu

WHOLE = 1.5e9  # T H V (T H I) up to which everything is compared


def some(n, most, ends, seed):
    """Sampled indices below n."""
    if n <= most:
        return np.arange(n)
    at = [i for i in (0, 1, 15, 16, n // 2, n - 17, n - 2, n - 1, *ends) if 0 <= i < n]
    return np.unique(np.append(at, np.random.default_rng(seed).integers(0, n, most - len(at))))


def check_loss(T, H, V, dtype, with_dw=True):
    x, xv, w, wv, targets, dloss = loss_case(dtype, T, H, V, seed=31)
    d = context(H, w)
    try:
        xd, td, loss, lse = run_loss(d, x, dtype, targets, V)
        dx, dw = run_loss_backward(d, xd, dtype, td, lse, dloss, T, H, V, dw=with_dw)
        got = {n: o.get() for n, o in dict(loss=loss, lse=lse, dx=dx, dw=dw).items() if o is not None}
    finally:
        d.close()
    dl = dloss.astype(np.float64)
    if T * H * V <= WHOLE:
        want = ref.Loss(xv, wv, targets, dl, dtype)
        for n in got:
            ref.assert_close(got[n], getattr(want, n), getattr(want, n + "_tol"), n)
        return
    at = some(T, 40, (8191, 8192), 1)
    want = ref.Loss(xv[at], wv, targets[at], dl[at], dtype)
    for n in ("loss", "lse", "dx"):
        ref.assert_close(got[n][at], getattr(want, n), getattr(want, n + "_tol"), n)
    assert all(np.isfinite(g).all() for g in got.values())
    if not with_dw:
        return
    # rows of dw, from the log-sum-exp that the call was given
    rows = some(V, 40, (255, 256, V // 2 - 1, V // 2, V // 2 + 128), 2)
    logits, error = xv @ wv[rows].T, ref.sums(H, np.abs(xv) @ np.abs(wv[rows]).T, dtype)
    p, weight = np.exp(logits - got["lse"][:, None]), (dl * (targets >= 0))[:, None]
    g = (p - (targets[:, None] == rows[None, :])) * weight
    g_tol = np.abs(weight) * p * (error + 2.0 ** -20) + (ref.u(dtype) + 2.0 ** -22) * np.abs(g)
    dw_want = g.T @ xv
    tol = g_tol.T @ np.abs(xv) + ref.sums(T, np.abs(g).T @ np.abs(xv), dtype) + ref.u(dtype) * np.abs(dw_want)
    ref.assert_close(got["dw"][rows], dw_want, tol, "dw")


def check_block(T, H, I, dtype, kept=False):  # noqa: E741
    c = block_case(dtype, T, H, I, seed=32)
    xv, dyv, wgu, wd = (c[n][1] for n in ("x", "dy", "wgu", "wd"))
    bgu, bd = c["bgu"].astype(np.float64), c["bd"].astype(np.float64)
    d = context(H)
    try:
        b = BlockOnDevice(c)
        x8 = DeviceBuffer(d.act8_bytes(T, H)) if kept else None
        y = b.forward(d, dtype, x8=x8)
        grads = b.backward(d, dtype, x=x8, x_type=MOE_MXFP8) if kept else b.backward(d, dtype)
        d.synchronize()
        if T * H * I <= WHOLE:
            want = ref.Block(xv, wgu, bgu, wd, bd, dyv, dtype, ref.act8(xv)[2] if kept else None)
            ref.assert_close(y.get(), want.y, want.y_tol, "y")
            check_grads(grads, want)
            return
        got = dict({n: o.get() for n, o in grads.items()}, y=y.get())
    finally:
        d.close()
    x_hat = ref.act8(xv)[2] if kept else xv
    at = some(T, 40, (8191, 8192), 3)
    want = ref.Block(xv[at], wgu, bgu, wd, bd, dyv[at], dtype, x_hat[at])
    ref.assert_close(got["y"][at], want.y, want.y_tol, "y")
    ref.assert_close(got["x"][at], want.dx, want.dx_tol, "x")
    # inner columns: the block that holds these alone has their gradients
    cols = some(I, 40, (), 4)
    rows = np.stack((2 * cols, 2 * cols + 1), 1).reshape(-1)
    want = ref.Block(x_hat, wgu[rows], bgu[rows], wd[:, cols], bd, dyv, dtype)
    ref.assert_close(got["gate_up"][rows], want.dwgu, want.dwgu_tol, "gate_up")
    ref.assert_close(got["gate_up_bias"][rows], want.dbgu, want.dbgu_tol, "gate_up_bias")
    ref.assert_close(got["down"][:, cols], want.dwd, want.dwd_tol, "down")
    ref.assert_close(got["down_bias"], want.dbd, want.dbd_tol, "down_bias")
    assert all(np.isfinite(got[n]).all() for n in ("y", *NAMES))


@pytest.mark.parametrize("T,H,V,dtype", sizes.LOSS)
def test_loss(T, H, V, dtype):
    check_loss(T, H, V, dtype)


@pytest.mark.parametrize("T,H,V,dtype", sizes.LOSS_DX)
def test_loss_rows_alone(T, H, V, dtype):
    check_loss(T, H, V, dtype, with_dw=False)


@pytest.mark.parametrize("T,H,I,dtype", sizes.BLOCK)
def test_block(T, H, I, dtype):  # noqa: E741
    check_block(T, H, I, dtype)


@pytest.mark.parametrize("T,H,I,dtype", sizes.KEPT)
def test_block_from_checkpoint(T, H, I, dtype):  # noqa: E741
    check_block(T, H, I, dtype, kept=True)
