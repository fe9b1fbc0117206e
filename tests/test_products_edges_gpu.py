"""The products of a feed-forward block on an MI355X where their other tests do not look: activations and slopes far
below zero, element by element; fp16 gradients that are subnormal before they are summed; a launch of more than 2^31
threads; captured first calls; large stacks; the per-thread stream."""

import math
import subprocess
import sys
import threading
from pathlib import Path

import numpy as np
import pytest

from mlir_roller_amd import hip
from mlir_roller_amd.hip import DeviceArray, HipError
from mlir_roller_amd.products import GatedFfn, Orthogonalizer
from oracle import products_oracle as po
from test_products_gpu import Block, Graph, Matrix, room

pytestmark = pytest.mark.gpu
HALF = 2.0 ** -24                                  # half a step of fp32, relative


def fill(m, values):
    """Other values for a matrix that is on the device."""
    m.inside(m.host)[:] = po.encode(values, m.dtype)
    m.values = po.decode(m.inside(m.host), m.dtype)
    m.buffer.set(m.host)


def activation_and_slope(kind, g):
    """act(g) and act'(g) in 64 bits without the cancellation of 1 + erf and 1 + tanh below zero."""
    if kind == "gelu":
        phi = 0.5 * np.vectorize(math.erfc, otypes=[float])(-g / math.sqrt(2))
        return g * phi, phi + g * np.exp(-g * g / 2) / math.sqrt(2 * math.pi)
    z, dz = (g, 1.0) if kind == "silu" else (math.sqrt(8 / math.pi) * (g + 0.044715 * g ** 3), math.sqrt(8 / math.pi) * (1 + 0.134145 * g * g))
    s = np.exp(z) / (1 + np.exp(z))
    return g * s, s + g * s * (1 - s) * dz


def gates_alone(device, kind, g):
    """act(g) and act'(g) as the block computes them in fp32: one token of one feature, up and down weights of one.
    Every product then is one number times one, and dw_up is the activation and dw_gate the slope."""
    b = Block(1, 1, len(g), "fp32", kind)
    for m, v in ((b.x, 1.0), (b.dy, 1.0), (b.wu, 1.0), (b.wd, 1.0), (b.wg, g[:, None])):
        fill(m, np.broadcast_to(v, (m.rows, m.cols)))
    saved = room(b.op.saved_bytes(1))
    b.forward(saved)
    b.backward(saved)
    hip.synchronize()
    return b.wg.values[:, 0], b.grads["dw_up"].get()[:, 0], b.grads["dw_gate"].get()[:, 0]


# Relative errors, in half steps.  The exponential's argument carries two half steps of itself (the constant and the
# product), and so the result 2 |z|; the exponential, the reciprocal, the sum before it and what follows are ten more.
# z of gelu_tanh has seven half steps of its own (9 |z| in all), and its slope's factor six.  gelu: the argument of erfc
# has two half steps, which move it by 2 g^2 (its logarithm's slope is twice the argument), and the normal density's
# exponent three, which is 1.5 g^2; erfc itself is right to 16 steps.  Slope and activation are taken where they are sums
# of terms of one sign or nearly: beyond -8 (silu) and -3 (gelu) nothing cancels.  Down to the smallest normal number.
FAR = [("silu", -8.0, -83.0, lambda g, z: 2 * z + 16), ("gelu", -3.0, -12.4, lambda g, z: 4 * g * g + 64),
       ("gelu_tanh", -3.0, -9.0, lambda g, z: 9 * z + 32)]


@pytest.mark.parametrize("kind,near,far,half_steps", FAR)
def test_activation_and_slope_far_below_zero(device, kind, near, far, half_steps):
    g, act, slope = gates_alone(device, kind, np.linspace(far, near, 1023))
    z = np.abs(g) if kind != "gelu_tanh" else math.sqrt(8 / math.pi) * np.abs(g + 0.044715 * g ** 3)
    want, want_slope = activation_and_slope(kind, g)
    allowed = half_steps(g, z) * HALF
    assert (np.abs(slope / want_slope - 1) <= allowed).all(), f"slope off by {np.max(np.abs(slope / want_slope - 1))}"
    assert (np.abs(act / want - 1) <= allowed).all(), f"activation off by {np.max(np.abs(act / want - 1))}"


@pytest.mark.parametrize("kind", ["silu", "gelu", "gelu_tanh"])
def test_ends_of_activation_and_slope(device, kind):
    g, act, slope = gates_alone(device, kind, np.array([-3e38, -1e30, -1e4, -200.0, -129.0, 0.0, 129.0, 200.0, 1e4, 1e30, 3e38]))
    assert np.array_equal(act, np.maximum(g, 0)) and np.array_equal(slope, np.where(g < 0, 0, np.where(g == 0, 0.5, 1)))


# fp16 gradients of the size that an unscaled loss has: dg and du are products of dy, and below 6e-5 a fp16 number has
# fewer than 11 bits.  The sums over 2048 tokens that they go into are 50 times larger and can be told apart.  Allowed in
# the norm: 2^-25 an element, the most that rounding a subnormal output takes, and 2^-10 of it, twice what one rounding of every
# term (2^-11 of each at most, independent of each other) and one of the output come to.
@pytest.mark.parametrize("rms", [1e-6, 1e-5, 1e-3, 1.0])
def test_small_gradients_in_fp16(device, rms):
    b = Block(2048, 64, 96, "fp16", "silu")
    fill(b.dy, rms * np.random.default_rng(7).standard_normal((2048, 64)))
    saved = room(b.op.saved_bytes(2048))
    b.forward(saved)
    b.backward(saved)
    hip.synchronize()
    want = b.want.backward(b.dy.values)
    for n, g in b.grads.items():
        value = want[n][0]
        off = np.linalg.norm(g.get() - value)
        assert off <= math.sqrt(value.size) * 2.0 ** -25 + 2.0 ** -10 * np.linalg.norm(value), f"{n} off by {off / np.linalg.norm(value)}"


def test_small_gradients_beside_a_token_of_nan_and_infinities(device):
    # what is not finite in dy does not decide how the other tokens' gradients are rounded
    b = Block(300, 64, 2048, "fp16", "silu")
    small = 1e-5 * np.random.default_rng(8).standard_normal((300, 64))
    small[5], small[77, 3], small[200] = np.nan, np.inf, 0.0
    fill(b.dy, small)
    saved = room(b.op.saved_bytes(300))
    b.forward(saved)
    b.backward(saved, ("dx",))
    hip.synchronize()
    keep = [t for t in range(300) if t not in (5, 77)]
    few = po.FeedForward(b.x.values[keep], b.wg.values, b.wu.values, b.wd.values, "silu", "fp16").backward(b.dy.values[keep])["dx"][0]
    got = b.grads["dx"].get()
    assert np.isnan(got[5]).all() and not got[200].any()
    assert np.linalg.norm(got[keep] - few) <= math.sqrt(few.size) * 2.0 ** -25 + 2.0 ** -10 * np.linalg.norm(few)


def test_a_captured_backward_pass_scales_by_the_gradients_of_the_replay(device):
    b = Block(200, 136, 264, "fp16", "silu")
    stream, saved, ws = hip.Stream(), room(b.op.saved_bytes(200)), room(b.op.workspace_bytes(200, backward=True))
    b.forward(saved)
    hip.synchronize()
    graph = Graph(stream)
    with graph:
        b.backward(saved, workspace=ws, stream=stream)
    values = np.random.default_rng(9).standard_normal((200, 136))
    for rms in (1e-6, 1.0, 1e-4, 0.0, 1e-5):
        fill(b.dy, rms * values)
        b.backward(saved, workspace=ws, stream=stream)
        hip.synchronize()
        eager = [m.bits() for m in b.grads.values()]
        for m in b.grads.values():
            m.buffer.fill_bytes(0xFF)
        ws.fill_bytes(0xFF)
        hip.synchronize()
        graph.launch(stream)
        hip.synchronize()
        assert all(np.array_equal(p, m.bits()) for p, m in zip(eager, b.grads.values())), f"replay on gradients of {rms}"


def test_more_than_2_to_the_31_threads(device):
    # 16 million tokens through 64 x 64 tiles: 8.65 million workgroups of 256 threads.  The tokens are one stretch of
    # 100003 again and again; what is looked at is the ends, a stretch 2^31 elements before the end of h, and others
    T, D, F, period = 16776704, 283, 1033, 100003
    op, rng = GatedFfn(D, F, "fp32"), np.random.default_rng(11)
    rows, cols, splits, whole = op.tiles(T, device.compute_units)["gate and up"]
    assert (rows, cols, splits) == (64, 64, 1) and whole * 256 > 1 << 31
    stretch = rng.standard_normal((period, D)).astype(np.float32)
    weights = [Matrix(s * rng.standard_normal(shape), "fp32") for shape, s in (((F, D), D ** -0.5), ((F, D), D ** -0.5), ((D, F), F ** -0.5))]
    x, y = DeviceArray((T, D)), DeviceArray((T, D))
    for t in range(0, T, period):
        hip.check(hip.lib().rl_memcpy_h2d(int(x.ptr) + t * D * 4, stretch.ctypes.data, min(period, T - t) * D * 4))
    ws = DeviceArray((op.workspace_bytes(T),), np.uint8)
    op.forward(x, *[w.ptr for w in weights], y, T, workspace=ws)
    hip.synchronize()
    for start in (0, T - 2 ** 31 // 1056 - 4096, T - 2 ** 31 // 1056 + 1000, T - 4096, *rng.integers(0, T - 4096, 4)):
        got = np.empty((4096, D), np.float32)
        hip.check(hip.lib().rl_memcpy_d2h(got.ctypes.data, int(y.ptr) + int(start) * D * 4, got.nbytes))
        want = po.FeedForward(stretch[np.arange(start, start + 4096) % period].astype(np.float64), *[w.values for w in weights], "silu", "fp32")
        assert (np.abs(got - want.y) <= want.y_bound).all(), f"tokens from {start}"
    x.free(), y.free(), ws.free()


FIRST_CALL = """
import sys
sys.path[:0] = sys.argv[1:]
import numpy as np
from mlir_roller_amd import hip
from mlir_roller_amd.products import Orthogonalizer
from test_products_gpu import Block, Graph, Matrix, gradient, room
hip.init(0)
b, stream = Block(200, 136, 264, "fp16", "silu"), hip.Stream()
saved, ws = room(b.op.saved_bytes(200)), room(b.op.workspace_bytes(200, backward=True))
G, O = Matrix(gradient(np.random.default_rng(1), 1, 60, 90)[0], "fp16"), Matrix(None, "fp16", shape=(60, 90))
o = Orthogonalizer(60, 90, dtype="fp16")
ws_o, graph = room(o.workspace_bytes()), Graph(stream)
with graph:
    b.forward(saved, workspace=ws, stream=stream)
    b.backward(saved, workspace=ws, stream=stream)
    o.launch(G.ptr, O.ptr, workspace=ws_o, stream=stream)
for _ in range(3):
    graph.launch(stream)
b.check_y()
b.check_grads()
captured = O.bits()
o.launch(G.ptr, O.ptr, workspace=ws_o, stream=stream)
hip.synchronize()
assert np.array_equal(captured, O.bits())
print("captured and right")
"""


def test_the_first_calls_of_a_process_may_be_captured(device):
    tests = Path(__file__).resolve().parent
    done = subprocess.run([sys.executable, "-c", FIRST_CALL, str(tests), str(tests.parent)], capture_output=True, text=True, timeout=100)
    assert done.returncode == 0 and "captured and right" in done.stdout, done.stderr


# ends of the documented ranges
@pytest.mark.parametrize("rows,cols,dtype", [(8, 5, "fp32"), (3, 9, "bf16")])
def test_a_stack_of_65535_matrices(device, rows, cols, dtype):
    few = po.encode(1e-3 * np.random.default_rng(1).standard_normal((50, rows, cols)), dtype)
    G = DeviceArray.from_host(few[np.arange(65535) % 50])
    op = Orthogonalizer(rows, cols, batch=65535, dtype=dtype)
    ws = DeviceArray((op.workspace_bytes(),), np.uint8)
    op.launch(G, G, workspace=ws)
    hip.synchronize()
    got = po.decode(G.get(), dtype)
    for i in range(50):
        value = po.decode(few[i], dtype)
        want = po.orthogonalise(value)
        assert np.max(np.linalg.norm(got[i::50] - want, axis=(1, 2))) <= po.orthogonalise_tolerance(value, dtype, want)


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
