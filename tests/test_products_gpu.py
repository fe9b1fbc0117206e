"""The products of a feed-forward block on an MI355X against their 64-bit definitions: the gated block
forward and backward, and Newton-Schulz orthogonalisation.  Whatever lies around a matrix (the rest of its
rows, the bytes before and behind it, the workspace) holds NaN before every call."""

import ctypes as C
import threading

import numpy as np
import pytest

from mlir_roller_amd import hip
from mlir_roller_amd.hip import DeviceArray, HipError, Ptr
from mlir_roller_amd.products import GatedFfn, Orthogonalizer
from oracle import products_oracle as po

pytestmark = pytest.mark.gpu
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}


class Matrix:
    """A row-major device matrix with leading dimension `ld`, starting `shift` elements into its buffer."""

    def __init__(self, values, dtype, ld=None, shift=0, shape=None):
        self.dtype = dtype
        rows, cols = shape if values is None else values.shape
        self.rows, self.cols, self.ld, self.shift = rows, cols, cols if ld is None else ld, shift
        self.host = np.full(shift + max(rows, 1) * self.ld + 64, 0xFF, np.uint8).repeat(SIZE[dtype]).view(po.STORAGE[dtype])
        if values is not None:
            self.inside(self.host)[:] = po.encode(values, dtype)
            self.values = po.decode(self.inside(self.host), dtype)
        self.buffer = DeviceArray.from_host(self.host)
        self.ptr = Ptr(int(self.buffer.ptr) + shift * SIZE[dtype])

    def inside(self, flat):
        return flat[self.shift:self.shift + self.rows * self.ld].reshape(self.rows, self.ld)[:, :self.cols]

    def get(self):
        """The values, after a check that nothing around them was written."""
        now = self.buffer.get()
        outside = np.ones(now.shape, bool)
        self.inside(outside)[:] = False
        assert (now.view(np.uint8).reshape(now.size, -1)[outside] == 0xFF).all(), "written outside the matrix"
        return po.decode(self.inside(now), self.dtype)

    def bits(self):
        return self.inside(self.buffer.get()).copy()


def room(nbytes):
    a = DeviceArray((max(int(nbytes), 256),), np.uint8)
    a.fill_bytes(0xFF)
    return a


class Block:
    """One feed-forward block with seeded inputs on the device and its 64-bit definition."""

    def __init__(self, T, D, F, dtype, act, seed=0, pad=0, shift=0, pad_up=None):
        rng = np.random.default_rng([seed, T, D, F])
        mat = lambda r, c, s, p=pad: Matrix(s * rng.standard_normal((r, c)), dtype, c + p, shift)
        self.x, self.dy = mat(T, D, 1.0), mat(T, D, 1.0)
        self.wg, self.wu = mat(F, D, D ** -0.5), mat(F, D, D ** -0.5, pad if pad_up is None else pad_up)
        self.wd = mat(D, F, F ** -0.5)
        self.T, self.dtype, self.pad, self.shift = T, dtype, pad, shift
        self.op = GatedFfn(D, F, dtype, act)
        self.unaligned = bool(pad or shift)
        self.want = po.FeedForward(self.x.values, self.wg.values, self.wu.values, self.wd.values, act, dtype)
        self.y = self.like(self.x)
        self.grads = {"dx": self.like(self.x), "dw_gate": self.like(self.wg), "dw_up": self.like(self.wu), "dw_down": self.like(self.wd)}

    def like(self, m):
        return Matrix(None, self.dtype, m.ld, self.shift, (m.rows, m.cols))

    def inputs(self):
        return [m.ptr for m in (self.x, self.wg, self.wu, self.wd)]

    def lds(self):
        return dict(ldx=self.x.ld, ld_gate=self.wg.ld, ld_up=self.wu.ld, ld_down=self.wd.ld)

    def forward(self, saved=None, **how):
        if "workspace" not in how:
            how["workspace"] = room(self.op.workspace_bytes(self.T, unaligned=self.unaligned))
        self.op.forward(*self.inputs(), self.y.ptr, self.T, ldy=self.y.ld, saved=saved, **self.lds(), **how)

    def backward(self, saved, names=("dx", "dw_gate", "dw_up", "dw_down"), **how):
        if "workspace" not in how:
            how["workspace"] = room(self.op.workspace_bytes(self.T, backward=True, unaligned=self.unaligned))
        g = self.grads
        self.op.backward(self.dy.ptr, *self.inputs(), saved, *[g[n].ptr if n in names else None for n in g], self.T, lddy=self.dy.ld,
                         lddx=g["dx"].ld, ldd_gate=g["dw_gate"].ld, ldd_up=g["dw_up"].ld, ldd_down=g["dw_down"].ld, **self.lds(), **how)

    def check_y(self):
        hip.synchronize()
        off = np.abs(self.y.get() - self.want.y)
        assert (off <= self.want.y_bound).all(), f"y off by {np.max(off / self.want.y_bound)} bounds"

    def check_grads(self, names=("dx", "dw_gate", "dw_up", "dw_down")):
        hip.synchronize()
        want = self.want.backward(self.dy.values)
        for n in names:
            value, bound = want[n]
            off = np.abs(self.grads[n].get() - value)
            assert (off <= bound).all(), f"{n} off by {np.max(off / bound)} bounds"


FORWARD = [(1, 64, 128, "bf16", "silu"), (1, 1, 1, "fp32", "gelu"), (1, 1000, 333, "fp16", "gelu_tanh"), (2, 72, 40, "bf16", "gelu"),
           (15, 130, 70, "fp32", "silu"), (16, 520, 264, "bf16", "silu"), (17, 65, 33, "fp16", "silu"), (32, 256, 512, "fp16", "gelu"),
           (33, 100, 300, "fp32", "gelu_tanh"), (64, 192, 1030, "bf16", "gelu_tanh"), (65, 64, 64, "bf16", "silu"), (65, 63, 65, "fp32", "silu"),
           (100, 257, 129, "fp16", "gelu"), (129, 512, 130, "bf16", "silu"), (300, 200, 700, "fp32", "gelu_tanh"), (513, 320, 264, "bf16", "gelu"),
           (777, 100, 50, "fp16", "silu"), (1100, 72, 600, "fp32", "gelu")]


@pytest.mark.parametrize("T,D,F,dtype,act", FORWARD)
def test_forward(device, T, D, F, dtype, act):
    b = Block(T, D, F, dtype, act)
    b.forward()
    b.check_y()


BACKWARD = [(1, 64, 128, "bf16", "silu"), (1, 1, 1, "fp32", "silu"), (3, 33, 17, "fp16", "gelu_tanh"), (16, 130, 70, "fp32", "gelu"), (40, 72, 40, "bf16", "gelu"),
            (65, 100, 130, "fp16", "silu"), (130, 257, 129, "bf16", "gelu_tanh"), (260, 264, 520, "fp32", "silu"), (300, 512, 768, "bf16", "silu"),
            (1025, 64, 96, "fp16", "gelu")]


@pytest.mark.parametrize("T,D,F,dtype,act", BACKWARD)
def test_forward_and_backward(device, T, D, F, dtype, act):
    b = Block(T, D, F, dtype, act)
    saved = room(b.op.saved_bytes(T))
    b.forward(saved)
    b.check_y()
    kept = saved.get()
    b.backward(saved)
    b.check_grads()
    assert np.array_equal(kept, saved.get())                    # the backward pass only reads it


# Sizes that between them take every product through every tile, whole and split (test_products.py counts).
EVERY_TILE = [(34, 66, 79, "bf16"), (625, 1732, 3374, "fp16"), (33, 568, 3752, "bf16"), (2162, 72, 110, "fp16"), (257, 1802, 64, "bf16"), (1325, 1546, 80, "fp16"),
              (2140, 67, 2055, "bf16"), (2421, 2066, 85, "fp16"), (35, 323, 2866, "bf16"), (386, 65, 2729, "bf16"), (1174, 71, 3259, "fp16"), (96, 2398, 3940, "bf16"),
              (2422, 106, 3708, "bf16"), (1023, 1920, 1000, "fp16"), (1000, 640, 3000, "bf16"),
              (46, 69, 64, "fp32"), (32, 1710, 1660, "fp32"), (1963, 72, 1583, "fp32"), (2412, 1372, 68, "fp32"), (38, 1586, 4035, "fp32"), (2186, 81, 3130, "fp32"),
              (67, 70, 2774, "fp32"), (2451, 214, 66, "fp32"), (37, 324, 3112, "fp32"), (443, 64, 2813, "fp32")]


@pytest.mark.parametrize("T,D,F,dtype", EVERY_TILE)
def test_every_tile(device, T, D, F, dtype):
    b = Block(T, D, F, dtype, "silu")
    saved = room(b.op.saved_bytes(T))
    b.forward(saved)
    b.check_y()
    b.backward(saved)
    b.check_grads()


# The same where it takes more work: every 31st token and feature is worked out in 64 bits, which is some of every tile.
EVERY_TILE_SAMPLED = [(6906, 4148, 113, "bf16"), (11211, 377, 5573, "fp16"), (650, 8708, 332, "fp16"), (3006, 9557, 668, "bf16"),
                      (2780, 11071, 148, "fp32"), (1508, 6138, 367, "fp32"), (3062, 749, 5255, "fp32"), (2524, 763, 14052, "fp32"),
                      (2973, 15814, 989, "fp32"), (13809, 1832, 494, "fp32"), (13932, 1560, 1140, "fp32"), (3161, 14511, 608, "fp32"),
                      (1651, 10892, 1021, "bf16"), (32, 1424, 8803, "fp16"), (4667, 79, 1889, "fp32"), (641, 80, 753, "fp32"), (654, 1512, 82, "fp32"),
                      (2315, 88, 641, "fp32"), (549, 897, 9763, "fp32"), (32, 364, 8746, "fp32")]


@pytest.mark.parametrize("T,D,F,dtype", EVERY_TILE_SAMPLED)
def test_every_tile_sampled(device, T, D, F, dtype):
    rng = np.random.default_rng([T, D, F])
    mat = lambda r, c, s: Matrix(s * rng.standard_normal((r, c), np.float32), dtype)
    x, dy, wg, wu, wd = mat(T, D, 1.0), mat(T, D, 1.0), mat(F, D, D ** -0.5), mat(F, D, D ** -0.5), mat(D, F, F ** -0.5)
    op = GatedFfn(D, F, dtype, "silu")
    y, dx, dwg, dwu, dwd = [Matrix(None, dtype, shape=s) for s in ((T, D), (T, D), (F, D), (F, D), (D, F))]
    saved, ws = room(op.saved_bytes(T)), room(op.workspace_bytes(T, backward=True))
    op.forward(x.ptr, wg.ptr, wu.ptr, wd.ptr, y.ptr, T, saved=saved, workspace=ws)
    op.backward(dy.ptr, x.ptr, wg.ptr, wu.ptr, wd.ptr, saved, dx.ptr, dwg.ptr, dwu.ptr, dwd.ptr, T, workspace=ws)
    hip.synchronize()

    def close(name, got, want):
        off = np.abs(got - want[0]) / want[1]
        assert (off <= 1).all(), f"{name} off by {np.max(off)} bounds"

    ts, fs = np.arange(T)[T % 31::31], np.arange(F)[F % 31::31]
    rows = po.FeedForward(x.values[ts], wg.values, wu.values, wd.values, "silu", dtype)
    close("y", y.get()[ts], (rows.y, rows.y_bound))
    close("dx", dx.get()[ts], rows.backward(dy.values[ts])["dx"])
    some = po.FeedForward(x.values, wg.values[fs], wu.values[fs], wd.values[:, fs], "silu", dtype).backward(dy.values)
    close("dw_gate", dwg.get()[fs], some["dw_gate"])
    close("dw_up", dwu.get()[fs], some["dw_up"])
    close("dw_down", dwd.get()[:, fs], some["dw_down"])


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("T", [5, 40, 150])
@pytest.mark.parametrize("pad,shift,pad_up", [(8, 0, 24), (3, 1, 3), (0, 5, 0), (16, 8, 9)])
def test_leading_dimensions_and_alignment(device, dtype, T, pad, shift, pad_up):
    b = Block(T, 96, 136, dtype, "silu", pad=pad, shift=shift, pad_up=pad_up)
    saved = room(b.op.saved_bytes(T))
    b.forward(saved)
    b.check_y()
    b.backward(saved)
    b.check_grads()


@pytest.mark.parametrize("T", [17, 40, 64, 65])
def test_odd_extents_with_even_leading_dimensions(device, T):
    # rows of 65 and 33 elements, 72 and 40 apart: the workspace that a query without leading dimensions asks for does
    b = Block(T, 65, 33, "bf16", "silu", pad=7)
    b.unaligned = False
    saved = room(b.op.saved_bytes(T))
    b.forward()
    b.check_y()
    b.forward(saved)
    b.check_y()
    b.backward(saved)
    b.check_grads()


@pytest.mark.parametrize("names", [("dx",), ("dw_down",), ("dw_gate", "dw_up"), ("dx", "dw_down"), ()])
def test_gradients_left_out_are_not_written(device, names):
    b = Block(70, 64, 72, "bf16", "silu")
    saved = room(b.op.saved_bytes(70))
    b.forward(saved)
    b.backward(saved, names)
    b.check_grads(names)
    for n in b.grads:
        if n not in names:
            assert (b.grads[n].buffer.get().view(np.uint8) == 0xFF).all()


def test_no_tokens(device):
    b = Block(0, 24, 40, "fp16", "silu")
    b.forward(workspace=None)
    b.backward(None if b.op.saved_bytes(0) else Ptr(0), workspace=None)
    hip.synchronize()
    for n in ("dw_gate", "dw_up", "dw_down"):
        assert not b.grads[n].get().any()


@pytest.mark.parametrize("T", [6, 100])
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_a_token_of_nan_or_infinities_stays_alone(device, T, dtype):
    b = Block(T, 96, 80, dtype, "silu")
    b.forward()
    hip.synchronize()
    clean = b.y.get()
    for row, value in ((1, np.nan), (T - 2, np.inf)):
        b.x.inside(b.x.host)[row] = po.encode(np.full(96, value), dtype)
    b.x.buffer.set(b.x.host)
    b.forward()
    hip.synchronize()
    got = b.y.get()
    others = [r for r in range(T) if r not in (1, T - 2)]
    assert np.array_equal(got[others], clean[others]) and np.isnan(got[1]).all()


@pytest.mark.parametrize("T,D,F", [(9, 320, 640), (600, 320, 640), (150, 2048, 512)])
def test_same_bits_every_time_and_with_and_without_what_is_saved(device, T, D, F):
    b = Block(T, D, F, "bf16", "gelu")
    saved = room(b.op.saved_bytes(T))
    b.forward()
    hip.synchronize()
    first = b.y.bits()
    b.forward(saved)
    hip.synchronize()
    assert np.array_equal(first, b.y.bits())
    runs = []
    for _ in range(2):
        b.backward(saved)
        hip.synchronize()
        runs.append([b.grads[n].bits() for n in b.grads])
    assert all(np.array_equal(p, q) for p, q in zip(*runs))


def test_gates_far_out(device):
    # gates of -1e4 .. 1e4: the ends of the activations, without a NaN from 0 * infinity
    T, D, F = 70, 64, 64
    for act in ("silu", "gelu", "gelu_tanh"):
        b = Block(T, D, F, "fp32", act)
        b.wg.inside(b.wg.host)[:] *= np.float32(3000)
        b.wg.buffer.set(b.wg.host)
        b.want = po.FeedForward(b.x.values, b.wg.inside(b.wg.host).astype(np.float64), b.wu.values, b.wd.values, act, "fp32")
        saved = room(b.op.saved_bytes(T))
        b.forward(saved)
        b.backward(saved)
        hip.synchronize()
        want = b.want.backward(b.dy.values)
        assert np.isfinite(b.y.get()).all()
        for n in b.grads:
            got = b.grads[n].get()
            assert np.isfinite(got).all()
            # slopes near the turn are steep in g, whose error grows with its size: held to the norm only.
            # |dg| / |g| of 2^-23 * (D + 8) moves the slope of |g| ~ 1 gates, 1 in 3000, by as much as 3000 times that
            assert np.linalg.norm(got - want[n][0]) <= 3000 * 2.0 ** -23 * (D + 8) * np.linalg.norm(want[n][0])


@pytest.mark.parametrize("T", [1, 3, 7, 16, 20, 80])
def test_gated_products_beyond_fp16(device, T):
    # one gated product of 300 * 300 and nothing else: an infinity in fp16, and so is what the weights make of it
    b = Block(T, 64, 64, "fp16", "silu")
    for m, value in ((b.x, 1.0), (b.wg, 300.0), (b.wu, 300.0)):
        m.inside(m.host)[:] = 0
        m.inside(m.host)[:T if m is b.x else 1, 0] = value
        m.buffer.set(m.host)
    b.wd.inside(b.wd.host)[:, 1:] = 0                             # (column 0 belongs to that product)
    b.wd.buffer.set(b.wd.host)
    b.forward()
    hip.synchronize()
    assert np.array_equal(b.y.get(), np.tile(np.sign(b.wd.inside(b.wd.host)[:, 0].astype(np.float64)) * np.inf, (T, 1)))


def test_operands_beyond_4_gib(device):
    # rows so far apart that the last ones lie beyond 2^32 bytes (and 2^31 elements) from the first
    T, D, F, ld = 2304, 64, 96, 1 << 20
    rng = np.random.default_rng(9)
    op = GatedFfn(D, F, "bf16")
    x = po.encode(rng.standard_normal((T, D)), "bf16")
    weights = [Matrix(rng.standard_normal(s) / 8, "bf16") for s in ((F, D), (F, D), (D, F))]
    wide = DeviceArray((T * ld,), np.uint16)
    y = DeviceArray((T * ld,), np.uint16)
    for r in range(T):
        hip.check(hip.lib().rl_memcpy_h2d(int(wide.ptr) + 2 * r * ld, x[r].ctypes.data, 2 * D))
    op.forward(wide, *[w.ptr for w in weights], y, T, ldx=ld, ldy=ld)
    hip.synchronize()
    got = np.empty((T, D), np.uint16)
    for r in range(T):
        hip.check(hip.lib().rl_memcpy_d2h(got[r].ctypes.data, int(y.ptr) + 2 * r * ld, 2 * D))
    want = po.FeedForward(po.decode(x, "bf16"), *[w.values for w in weights], "silu", "bf16")
    assert (np.abs(po.decode(got, "bf16") - want.y) <= want.y_bound).all()


# ---- orthogonalisation -------------------------------------------------------------------------------

def ortho(G, dtype, ld=None, shift=0, in_place=False, **how):
    """O for a stack G[batch, rows, cols] laid out with a gap between the matrices; and the rounded G."""
    batch, rows, cols = G.shape
    ld = cols if ld is None else ld
    gap = 1 if batch > 1 else 0
    flat = np.full((batch * (rows + gap), cols), np.nan)
    for i in range(batch):
        flat[i * (rows + gap):i * (rows + gap) + rows] = G[i]
    g = Matrix(flat, dtype, ld, shift)
    o = g if in_place else Matrix(None, dtype, ld, shift, flat.shape)
    op = Orthogonalizer(rows, cols, batch=batch, dtype=dtype, **how)
    op.launch(g.ptr, o.ptr, ldg=ld, ldo=ld, stride_g=(rows + gap) * ld, stride_o=(rows + gap) * ld, workspace=room(op.workspace_bytes()))
    hip.synchronize()
    got = o.get()
    pick = lambda m: np.stack([m[i * (rows + gap):i * (rows + gap) + rows] for i in range(batch)])
    if gap:
        assert np.isnan(got[rows::rows + 1]).all(), "written between the matrices"
    return pick(got), pick(g.values)


def gradient(rng, batch, rows, cols):
    r = max(1, min(rows, cols) // 8)
    return 1e-3 * (np.einsum("bir,brj->bij", rng.standard_normal((batch, rows, r)), rng.standard_normal((batch, r, cols))) + rng.standard_normal((batch, rows, cols)))


ORTHO = [(1, 64, 64), (1, 1, 1), (1, 1, 40), (1, 40, 1), (1, 65, 130), (1, 130, 65), (3, 33, 70), (2, 100, 31), (1, 256, 512), (1, 300, 257), (1, 520, 264)]


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("batch,rows,cols", ORTHO)
def test_orthogonalise(device, dtype, batch, rows, cols):
    rng = np.random.default_rng([batch, rows, cols])
    got, G = ortho(gradient(rng, batch, rows, cols), dtype)
    for i in range(batch):
        want = po.orthogonalise(G[i])
        assert np.linalg.norm(got[i] - want) <= po.orthogonalise_tolerance(G[i], dtype, want)


# As EVERY_TILE; fp16 and fp32 go the same way.  A large stack holds two matrices in turn.
EVERY_ORTHO_TILE = [(1, 32, 35, "bf16"), (40, 392, 482, "bf16"), (40, 259, 268, "bf16"), (40, 590, 647, "bf16"), (1, 32, 996, "bf16"), (40, 410, 71, "bf16"),
                    (40, 67, 779, "bf16"), (16, 331, 4075, "bf16"), (8, 5248, 907, "bf16"), (19, 325, 5164, "bf16"), (26, 888, 206, "bf16"), (52, 782, 637, "bf16"),
                    (1, 1066, 998, "bf16"), (2, 967, 1233, "bf16"), (52, 1712, 899, "bf16"), (10, 1754, 1742, "bf16"),
                    (1, 42, 32, "fp16"), (40, 257, 274, "fp32"), (40, 385, 398, "fp16"), (40, 639, 595, "fp32"), (2, 1003, 983, "fp32"), (1, 340, 33, "fp16"),
                    (1, 996, 1059, "fp16"), (8, 1997, 907, "fp32"), (1, 1708, 2444, "fp16"), (1, 2828, 3029, "fp32"), (26, 888, 206, "fp16"), (52, 782, 637, "fp32"),
                    (59, 558, 456, "fp32")]


@pytest.mark.parametrize("batch,rows,cols,dtype", EVERY_ORTHO_TILE)
def test_orthogonalise_every_tile(device, batch, rows, cols, dtype):
    two = gradient(np.random.default_rng([batch, rows, cols]), min(batch, 2), rows, cols)
    got, G = ortho(two[np.arange(batch) % 2], dtype)
    for i in range(len(two)):
        want = po.orthogonalise(G[i])
        allowed = po.orthogonalise_tolerance(G[i], dtype, want)
        assert np.max(np.linalg.norm(got[i::2] - want, axis=(1, 2))) <= allowed


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("rows,cols,ld,shift,in_place", [(48, 90, 91, 1, False), (48, 90, 104, 0, True), (90, 48, 51, 3, True), (90, 48, 48, 1, False)])
def test_orthogonalise_strides_and_in_place(device, dtype, rows, cols, ld, shift, in_place):
    rng = np.random.default_rng([rows, ld])
    got, G = ortho(gradient(rng, 2, rows, cols), dtype, ld, shift, in_place)
    for i in range(2):
        want = po.orthogonalise(G[i])
        assert np.linalg.norm(got[i] - want) <= po.orthogonalise_tolerance(G[i], dtype, want)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("how", [dict(steps=0), dict(steps=1), dict(steps=2, scale=0.2), dict(steps=3, coefficients=[(4.0, -6.0, 2.6), (3.0, -4.0, 1.8), (1.875, -1.25, 0.375)]),
                                 dict(eps=0.5), dict(steps=0, scale=-3.0)])
@pytest.mark.parametrize("rows,cols", [(70, 40), (40, 70)])
def test_orthogonalise_options(device, dtype, how, rows, cols):
    rng = np.random.default_rng(17)
    got, G = ortho(gradient(rng, 1, rows, cols), dtype, **how)
    want = po.orthogonalise(G[0], **how)
    assert np.linalg.norm(got[0] - want) <= po.orthogonalise_tolerance(G[0], dtype, want, **how)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_orthogonalise_zero_huge_tiny_and_nan(device, dtype):
    rng = np.random.default_rng(23)
    base = gradient(rng, 1, 40, 60)[0]
    stack = np.stack([np.zeros((40, 60)), base * 1e30, base * 1e-20, np.where(rng.random((40, 60)) < 0.01, np.nan, base), base])
    got, G = ortho(stack, dtype)
    assert not got[0].any()
    for i in (1, 2, 4):                  # squares beyond the range of 32 bits; a norm far below eps; an ordinary neighbour of a NaN
        want = po.orthogonalise(G[i])
        # (eps swallows the tiny one: X starts at 1e-12 and grows by 3.4 a step; in 16 bits it is below an operand's
        # smallest step, and a X in 32 bits is all that is left of it, which is right to the rounding)
        assert np.linalg.norm(got[i] - want) <= po.orthogonalise_tolerance(G[i], dtype, want)
    assert np.isnan(got[3]).all()


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_orthogonalise_a_norm_beyond_fp32(device, dtype):
    rng = np.random.default_rng(29)
    base = gradient(rng, 1, 70, 90)[0]
    G = base * (3e38 / np.abs(base).max())                     # entries up to 3e38, a norm of some 2e39
    got, G = ortho(G[None], dtype)
    want = po.orthogonalise(G[0])
    assert np.linalg.norm(got[0] - want) <= po.orthogonalise_tolerance(G[0], dtype, want)


def test_orthogonalise_same_bits(device):
    rng = np.random.default_rng(31)
    G = gradient(rng, 2, 200, 300)
    for dtype in ("bf16", "fp32"):
        a, b = ortho(G, dtype)[0], ortho(G, dtype)[0]
        assert np.array_equal(a, b)
        # a matrix of a stack comes out as it does alone or beside others
        single = ortho(G[:1], dtype)[0]
        want = po.orthogonalise(ortho(G[:1], dtype)[1][0])
        assert np.linalg.norm(single[0] - a[0]) <= 2 * po.orthogonalise_tolerance(G[0], dtype, want)


# ---- refusals, workspaces, streams, graphs ---------------------------------------------------------

def test_refusals(device):
    b = Block(70, 64, 72, "bf16", "silu")
    need = b.op.workspace_bytes(70)
    ws, saved = room(need + 512), room(b.op.saved_bytes(70))
    x, wg, wu, wd = b.inputs()

    def refuse(needle, call):
        with pytest.raises(HipError, match=needle) as err:
            call()
        assert err.value.status == hip.RL_ERR_INVALID_ARG

    f = lambda x=x, wg=wg, wu=wu, wd=wd, y=b.y.ptr, T=70, **k: b.op.forward(x, wg, wu, wd, y, T, **{"workspace": ws, **k})
    refuse("x is NULL", lambda: f(x=Ptr(0)))
    refuse("w_gate is NULL", lambda: f(wg=Ptr(0)))
    refuse("w_up is NULL", lambda: f(wu=Ptr(0)))
    refuse("w_down is NULL", lambda: f(wd=Ptr(0)))
    refuse("y is NULL", lambda: f(y=Ptr(0)))
    refuse("x is not aligned", lambda: f(x=Ptr(x.address + 1)))
    refuse("x: leading dimension 63", lambda: f(ldx=63))
    refuse("w_down: leading dimension 71", lambda: f(ld_down=71))
    refuse("y: leading dimension -1", lambda: f(ldy=-1))
    refuse("too large for 32-bit", lambda: f(ldx=1 << 23))
    refuse("number of tokens", lambda: f(T=-1))
    refuse("saved must be 256-byte aligned", lambda: f(saved=Ptr(int(saved.ptr) + 16)))
    refuse("256-byte aligned", lambda: f(workspace=Ptr(int(ws.ptr) + 16), workspace_bytes=need))
    refuse(f"needs a workspace of {need} bytes", lambda: f(workspace_bytes=need - 1))
    refuse("packed copy", lambda: f(ldx=65, workspace_bytes=need))
    g = lambda names=tuple(b.grads), saved=saved, T=70: b.op.backward(b.dy.ptr, x, wg, wu, wd, saved, *[b.grads[n].ptr if n in names else None for n in b.grads], T)
    refuse("asked for together", lambda: g(("dw_gate",)))
    refuse("saved is NULL", lambda: g(saved=Ptr(0)))
    refuse("number of tokens", lambda: g(T=(1 << 24) + 1))
    hip.synchronize()
    for m in (b.y, *b.grads.values()):
        assert (m.buffer.get().view(np.uint8) == 0xFF).all()          # nothing was enqueued
    G = Matrix(np.ones((20, 30)), "fp32")
    o = Orthogonalizer(20, 30, batch=2, dtype="fp32")
    refuse("G is NULL", lambda: o.launch(Ptr(0), G.ptr))
    refuse("O is NULL", lambda: o.launch(G.ptr, Ptr(0)))
    refuse("overlap", lambda: o.launch(G.ptr, G.ptr, stride_g=599))
    refuse("G: leading dimension 29", lambda: o.launch(G.ptr, G.ptr, ldg=29))
    refuse("not finite", lambda: Orthogonalizer(20, 30, dtype="fp32", coefficients=(1.0, float("nan"), 1.0)).launch(G.ptr, G.ptr))
    refuse("needs a workspace", lambda: o.launch(G.ptr, G.ptr, workspace=ws, workspace_bytes=256))


@pytest.mark.parametrize("T", [8, 300])
def test_library_workspace_on_two_streams_from_two_threads(device, T):
    blocks = [Block(T, 200, 328, "bf16", "silu", seed=s) for s in range(2)]
    streams = [hip.Stream() for _ in blocks]
    saved = [room(b.op.saved_bytes(T)) for b in blocks]
    failures = []

    def work(b, s, k):
        try:
            for _ in range(20):
                b.forward(k, workspace=None, stream=s)
                b.backward(k, workspace=None, stream=s)
        except Exception as e:                                       # (told by the main thread)
            failures.append(e)

    threads = [threading.Thread(target=work, args=a) for a in zip(blocks, streams, saved)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not failures
    for b in blocks:
        b.check_y()
        b.check_grads()


class Graph:
    """A captured stream, through the HIP runtime that the library has loaded."""

    def __init__(self, stream):
        self.rt, self.stream = C.CDLL("libamdhip64.so.7"), C.c_void_p(stream.handle)
        self.graph, self.exec = C.c_void_p(), C.c_void_p()

    def __enter__(self):
        assert self.rt.hipStreamBeginCapture(self.stream, 2) == 0     # relaxed
        return self

    def __exit__(self, *exc):
        status = self.rt.hipStreamEndCapture(self.stream, C.byref(self.graph))
        if exc[0] is None:
            assert status == 0
            assert self.rt.hipGraphInstantiate(C.byref(self.exec), self.graph, None, None, C.c_size_t(0)) == 0
        return False

    def launch(self, stream):
        assert self.rt.hipGraphLaunch(self.exec, C.c_void_p(stream.handle)) == 0

    def __del__(self):
        if self.exec:
            self.rt.hipGraphExecDestroy(self.exec)
        if self.graph:
            self.rt.hipGraphDestroy(self.graph)


@pytest.mark.parametrize("T,dtype", [(4, "bf16"), (200, "bf16"), (200, "fp32")])
def test_captured_calls_replay(device, T, dtype):
    b = Block(T, 136, 264, dtype, "silu")
    stream, saved = hip.Stream(), room(b.op.saved_bytes(T))
    ws = room(b.op.workspace_bytes(T, backward=True))
    G = Matrix(gradient(np.random.default_rng(1), 1, 60, 90)[0], dtype)
    O, o = Matrix(None, dtype, shape=(60, 90)), Orthogonalizer(60, 90, dtype=dtype)
    ws_o = room(o.workspace_bytes())

    def step():
        b.forward(saved, workspace=ws, stream=stream)
        b.backward(saved, workspace=ws, stream=stream)
        o.launch(G.ptr, O.ptr, workspace=ws_o, stream=stream)

    results = lambda: [m.bits() for m in (b.y, *b.grads.values(), O)]
    step()
    hip.synchronize()
    eager = results()
    b.check_y()
    b.check_grads()
    graph = Graph(stream)
    with graph:
        step()
    for k in range(3):
        for m in (b.y, *b.grads.values(), O):
            m.buffer.fill_bytes(0xFF)
        ws.fill_bytes(0xFF)
        ws_o.fill_bytes(0xFF)
        saved.fill_bytes(0xFF)
        hip.synchronize()
        graph.launch(stream)
        hip.synchronize()
        assert all(np.array_equal(p, q) for p, q in zip(eager, results())), f"replay {k}"
        step()                                                       # the program's own calls in between
        hip.synchronize()
    # the library's own workspace is no place for a graph
    with pytest.raises(HipError, match="captured call needs the caller's workspace"):
        with Graph(stream):
            b.forward(workspace=None, stream=stream)


def test_training_steps_lower_nothing_but_run_as_the_definition_does(device):
    """Two steps of a block: forward, backward, the three gradients orthogonalised, weights changed on the
    host, forward again; the second forward pass against the definition on the weights it was given."""
    T, D, F, dtype = 200, 96, 160, "bf16"
    b = Block(T, D, F, dtype, "silu")
    saved = room(b.op.saved_bytes(T))
    updates = {n: Matrix(None, dtype, shape=(b.grads[n].rows, b.grads[n].cols)) for n in ("dw_gate", "dw_up", "dw_down")}
    for _ in range(2):
        b.forward(saved)
        b.backward(saved)
        b.check_y()
        b.check_grads()
        for n, u in updates.items():
            g = b.grads[n]
            Orthogonalizer(g.rows, g.cols, dtype=dtype, scale=max(1.0, g.rows / g.cols) ** 0.5).launch(g.ptr, u.ptr)
        hip.synchronize()
        for n, w in (("dw_gate", b.wg), ("dw_up", b.wu), ("dw_down", b.wd)):
            G, got = b.grads[n].get(), updates[n].get()
            how = dict(scale=max(1.0, G.shape[0] / G.shape[1]) ** 0.5)
            want = po.orthogonalise(G, **how)
            assert np.linalg.norm(got - want) <= po.orthogonalise_tolerance(G, dtype, want, **how)
            w.inside(w.host)[:] = po.encode(w.values - 0.02 * got, dtype)
            w.values = po.decode(w.inside(w.host), dtype)
            w.buffer.set(w.host)
        b.want = po.FeedForward(b.x.values, b.wg.values, b.wu.values, b.wd.values, "silu", dtype)
