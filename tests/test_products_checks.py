"""What the products of a feed-forward block refuse, and what they choose, before a device is touched, beside
test_products.py."""

import pytest

from mlir_roller_amd import hip, products
from mlir_roller_amd.hip import HipError, Ptr
from mlir_roller_amd.products import GatedFfn


class Buffer:
    """Stands for a device array: an address and a size."""

    def __init__(self, nbytes):
        self.nbytes = nbytes

    def __int__(self):
        return 1 << 40


def test_a_saved_buffer_for_fewer_tokens_is_refused(hip_lib):
    op, at = GatedFfn(64, 512, "bf16"), Ptr(1 << 40)
    need = op.saved_bytes(8)
    for saved, how in ((Buffer(need - 1), {}), (Buffer(op.saved_bytes(7)), {}), (at, dict(saved_bytes=need - 1)), (Buffer(need), dict(saved_bytes=0))):
        for call in (lambda: op.forward(at, at, at, at, at, 8, saved=saved, **how),
                     lambda: op.backward(at, at, at, at, at, saved, at, at, at, at, 8, **how)):
            with pytest.raises(HipError, match=f"8 tokens need a buffer of {need} bytes") as err:
                call()
            assert err.value.status == hip.RL_ERR_INVALID_ARG
    assert op._saved(Buffer(need), None, 8) == op._saved(at, None, 8) == op._saved(at, need, 8) == 1 << 40


def test_the_size_of_a_workspace_is_asked_for():
    assert products._room(None, None) == (None, 0) and products._room(Buffer(512), None) == (1 << 40, 512) and products._room(Ptr(256), 512) == (256, 512)
    for address in (Ptr(256), 256):
        with pytest.raises(ValueError, match="needs its size as workspace_bytes"):
            products._room(address, None)


@pytest.mark.parametrize("T,D,F", [(1 << 24, 5, 2024), (1 << 24, 4, 997), (1 << 24, 1986, 6)])
def test_many_tokens_of_a_small_block_fit_one_launch(hip_lib, T, D, F):
    # rows x columns of results in tiles; gate and up columns count both
    for name, columns in (("gate and up", 2 * F), ("down", D)):
        rows, cols, splits, whole = GatedFfn(D, F, "fp32").tiles(T)[name]
        tiles = -(-T // rows) * -(-columns // cols)
        assert whole + (tiles - whole) * splits <= 0xFFFFFF
