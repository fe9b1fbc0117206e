"""The products of a feed-forward block on an MI355X where their other tests do not look: the per-thread stream."""

import threading

import numpy as np
import pytest

from mlir_roller_amd import hip
from mlir_roller_amd.hip import HipError
from test_products_gpu import Block, room

pytestmark = pytest.mark.gpu
PER_THREAD = 2                                     # hipStreamPerThread: one handle, another stream in every thread


def test_the_per_thread_stream_needs_the_callers_workspace(device):
    b = Block(70, 64, 72, "bf16", "silu")
    saved, ws = room(b.op.saved_bytes(70)), room(b.op.workspace_bytes(70, backward=True))
    for call in (lambda: b.forward(saved, workspace=None, stream=PER_THREAD), lambda: b.backward(saved, workspace=None, stream=PER_THREAD)):
        with pytest.raises(HipError, match="per-thread stream") as err:
            call()
        assert err.value.status == hip.RL_ERR_INVALID_ARG
    hip.synchronize()
    for m in (b.y, *b.grads.values()):
        assert (m.buffer.get().view(np.uint8) == 0xFF).all()
    b.forward(saved, workspace=ws, stream=PER_THREAD)
    b.backward(saved, workspace=ws, stream=PER_THREAD)
    b.check_y()
    b.check_grads()


def test_per_thread_streams_of_two_threads(device):
    blocks = [Block(300, 200, 328, "bf16", "silu", seed=s) for s in range(2)]
    rooms = [(room(b.op.saved_bytes(300)), room(b.op.workspace_bytes(300, backward=True))) for b in blocks]
    failures = []

    def work(b, saved, ws):
        try:
            for _ in range(20):
                b.forward(saved, workspace=ws, stream=PER_THREAD)
                b.backward(saved, workspace=ws, stream=PER_THREAD)
        except Exception as e:                                       # (told by the main thread)
            failures.append(e)

    threads = [threading.Thread(target=work, args=(b, *r)) for b, r in zip(blocks, rooms)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not failures
    for b in blocks:
        b.check_y()
        b.check_grads()
