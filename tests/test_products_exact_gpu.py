"""The gated feed-forward block on an MI355X on small whole numbers, to the last bit: through every tile, and with 1 to 64
tokens through every form of the kernel for few.  test_products_exact.py counts the forms and shows that a lost K step of
any product is told."""

import numpy as np
import pytest

from mlir_roller_amd import hip
from mlir_roller_amd.products import GatedFfn
from oracle.products_exact import ExactFeedForward
from test_products_gpu import EVERY_TILE, EVERY_TILE_SAMPLED, Matrix, room

pytestmark = pytest.mark.gpu


def run(b, pad=0, shift=0, backward=True):
    """{name: result} of a block whose matrices have `pad` elements behind each row and start `shift` into their buffers."""
    mat = lambda v: Matrix(v, b.dtype, v.shape[1] + pad, shift)
    x, dy, wg, wu, wd = mat(b.x), mat(b.dy), mat(b.wg), mat(b.wu), mat(b.wd)
    like = lambda m: Matrix(None, b.dtype, m.ld, shift, (m.rows, m.cols))
    y, dx, dwg, dwu, dwd = like(x), like(x), like(wg), like(wu), like(wd)
    op = GatedFfn(b.D, b.F, b.dtype, "silu")
    saved = room(op.saved_bytes(b.T)) if backward else None
    ws = room(op.workspace_bytes(b.T, backward=backward, unaligned=bool(pad or shift)))
    lds = dict(ldx=x.ld, ld_gate=wg.ld, ld_up=wu.ld, ld_down=wd.ld)
    op.forward(x.ptr, wg.ptr, wu.ptr, wd.ptr, y.ptr, b.T, ldy=y.ld, saved=saved, workspace=ws, **lds)
    if backward:
        op.backward(dy.ptr, x.ptr, wg.ptr, wu.ptr, wd.ptr, saved, dx.ptr, dwg.ptr, dwu.ptr, dwd.ptr, b.T, lddy=dy.ld, lddx=dx.ld, ldd_gate=dwg.ld,
                    ldd_up=dwu.ld, ldd_down=dwd.ld, workspace=ws, **lds)
    hip.synchronize()
    return {"y": y.get(), **({"dx": dx.get(), "dw_gate": dwg.get(), "dw_up": dwu.get(), "dw_down": dwd.get()} if backward else {})}


def compare(b, got, ts=slice(None), fs=slice(None)):
    wanted = b.of_tokens(ts, backward="dx" in got)
    if "dx" in got:
        wanted.update(b.of_features(fs))
    for n, want in wanted.items():
        result = got[n][ts] if n in ("y", "dx") else got[n][:, fs] if n == "dw_down" else got[n][fs]
        wrong = result != want
        assert not wrong.any(), f"{n}: {wrong.sum()} of {wrong.size} wrong, first at {np.argwhere(wrong)[0]}"


@pytest.mark.parametrize("T,D,F,dtype", EVERY_TILE)
def test_every_tile(device, T, D, F, dtype):
    b = ExactFeedForward(T, D, F, dtype)
    compare(b, run(b))


@pytest.mark.parametrize("T,D,F,dtype", EVERY_TILE_SAMPLED)
def test_every_tile_sampled(device, T, D, F, dtype):
    b = ExactFeedForward(T, D, F, dtype)
    compare(b, run(b), np.arange(T)[T % 31::31], np.arange(F)[F % 31::31])


# 1 to 4, 5 to 8 and 9 to 16 tokens, whose loads take 1024, 512 and 256 16-bit elements of K at a time (32 bits: half as
# many) and share K out to up to 16 waves: lengths below, at and above whole loads, one load and several a wave.
FEW = [(1, 1024, 4096, "bf16"), (1, 8300, 333, "bf16"), (1, 4100, 2050, "fp16"), (1, 512, 513, "fp32"), (2, 16400, 70, "fp32"), (3, 1025, 8203, "bf16"), (3, 1023, 40, "fp16"),
       (4, 2050, 1023, "fp32"), (4, 8203, 2047, "fp16"), (4, 70, 20600, "bf16"), (5, 1024, 4096, "fp16"), (5, 513, 1537, "fp32"), (6, 9000, 30, "bf16"), (7, 6200, 90, "fp32"),
       (8, 2050, 4100, "bf16"), (8, 4096, 1030, "fp32"), (8, 511, 12290, "fp16"), (9, 1025, 2050, "bf16"), (11, 5000, 50, "fp16"), (12, 2600, 24, "fp32"),
       (13, 255, 257, "bf16"), (16, 4100, 8203, "fp16"), (16, 520, 1030, "fp32"), (16, 256, 6000, "bf16"), (10, 40, 9000, "fp32"), (2, 100, 8300, "fp32"), (6, 100, 4500, "fp32"), (16, 256, 6016, "fp32")]


@pytest.mark.parametrize("pad,shift", [(0, 0), (3, 1)])
@pytest.mark.parametrize("T,D,F,dtype", FEW)
def test_few_tokens(device, T, D, F, dtype, pad, shift):
    b = ExactFeedForward(T, D, F, dtype)
    compare(b, run(b, pad, shift, backward=False))
    compare(b, run(b, pad, shift))


# 17 to 64 tokens with 16-bit rows at odd elements take the same kernel, 256 or 128 elements at a time
@pytest.mark.parametrize("T,D,F,dtype", [(17, 1025, 2051, "bf16"), (32, 2047, 515, "fp16"), (33, 515, 4101, "fp16"), (50, 1023, 1025, "bf16"), (64, 4097, 333, "bf16"), (64, 129, 127, "fp16")])
def test_more_tokens_at_odd_rows(device, T, D, F, dtype):
    b = ExactFeedForward(T, D, F, dtype)
    compare(b, run(b))
    compare(b, run(b, 2, 1, backward=False))


# ends of the documented ranges
@pytest.mark.parametrize("T,D,F,dtype", [(3, 1 << 20, 2, "bf16"), (3, 2, 1 << 20, "fp32"), (40, 1 << 20, 3, "fp16"), (200, 7, (1 << 20) - 1, "bf16"), (1 << 20, 1, 1, "bf16")])
def test_long_rows_and_many_tokens(device, T, D, F, dtype):
    b = ExactFeedForward(T, D, F, dtype)
    compare(b, run(b), np.arange(T)[::-(-T // 300)], np.arange(F)[::-(-F // 300)])
