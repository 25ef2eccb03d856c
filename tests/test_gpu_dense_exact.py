"""f32 rows of the dense operators to their last bit (tests/dense_exact.py), at every size at which the other tests run f32
rows: with them in every form of launch that f32 rows take."""
import numpy as np
import pytest

from silentotithrandousha_amd import MOE_F32, MOE_MXFP8, DeviceBuffer
from tests import dense_exact as exact
from tests import dense_ref as ref
from tests.test_dense_calls import sizes_run
from tests.test_gpu_dense import BlockOnDevice, context, dev, run_loss, run_loss_backward

pytestmark = pytest.mark.gpu

SIZES = {kind: sorted({s[1:4] for s in sizes_run() if s[0] in of and s[4] == MOE_F32})
         for kind, of in (("loss", ("loss", "dx")), ("block", ("block",)), ("kept", ("kept",)))}


@pytest.mark.parametrize("T,H,V", SIZES["loss"])
def test_loss(T, H, V):
    c = exact.Loss(T, H, V)
    d = context(H, ref.to_bf16(c.w))
    try:
        xd, td, loss, lse = run_loss(d, c.x, MOE_F32, c.targets, V)
        given = dev(c.lse.astype(np.float32))
        dx, dw = run_loss_backward(d, xd, MOE_F32, td, given, c.dloss, T, H, V)
        c.check(dict(loss=loss.get(), lse=lse.get(), dx=dx.get(), dw=dw.get()))
        alone, _ = run_loss_backward(d, xd, MOE_F32, td, given, c.dloss, T, H, V, dw=False)
        assert np.array_equal(alone.get(), c.dx)
    finally:
        d.close()


def run_block(T, H, I, kept):  # noqa: E741
    c = exact.Block(T, H, I, kept=kept)
    case = dict(x=(c.x, None), dy=(c.dy, None), wgu=(ref.to_bf16(c.wgu), None), wd=(ref.to_bf16(c.wd), None),
                bgu=np.zeros(2 * I, np.float32), bd=np.zeros(H, np.float32))
    d = context(H)
    try:
        b = BlockOnDevice(case, bias=False)
        x8 = DeviceBuffer(d.act8_bytes(T, H)) if kept else None
        y = b.forward(d, MOE_F32, x8=x8)
        g = b.backward(d, MOE_F32, x=x8, x_type=MOE_MXFP8) if kept else b.backward(d, MOE_F32)
        d.synchronize()
        c.check(dict({n: o.get() for n, o in g.items()}, y=y.get()))
    finally:
        d.close()


@pytest.mark.parametrize("T,H,I", SIZES["block"])
def test_block(T, H, I):  # noqa: E741
    run_block(T, H, I, kept=False)


@pytest.mark.parametrize("T,H,I", SIZES["kept"])
def test_block_from_checkpoint(T, H, I):  # noqa: E741
    run_block(T, H, I, kept=True)
