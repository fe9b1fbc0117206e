"""The products of a feed-forward block without a device: the 64-bit definitions against finite differences
and closed forms, sizes, and every refusal that needs no GPU."""

import ctypes as C

import numpy as np
import pytest

from mlir_roller_amd import hip, products
from mlir_roller_amd.hip import HipError, Ptr
from mlir_roller_amd.products import GatedFfn, Orthogonalizer
from oracle import products_oracle as po


@pytest.mark.parametrize("kind", ["silu", "gelu", "gelu_tanh"])
def test_definition_gradients_agree_with_differences(kind):
    rng = np.random.default_rng(3)
    T, D, F = 4, 5, 6
    x, wg, wu, wd, dy = (rng.standard_normal(s) for s in ((T, D), (F, D), (F, D), (D, F), (T, D)))
    got = po.FeedForward(x, wg, wu, wd, kind, "fp32").backward(dy)

    def loss(x, wg, wu, wd):
        return (dy * po.FeedForward(x, wg, wu, wd, kind, "fp32").y).sum()

    args = [x, wg, wu, wd]
    for i, name in enumerate(("dx", "dw_gate", "dw_up", "dw_down")):
        for at in np.ndindex(args[i].shape):
            up, down = [a.copy() for a in args], [a.copy() for a in args]
            up[i][at] += 1e-5
            down[i][at] -= 1e-5
            # central differences: error h^2 / 6 of the third derivative, and 1e-16 / h of the values
            assert abs((loss(*up) - loss(*down)) / 2e-5 - got[name][0][at]) < 1e-7 * max(1.0, np.abs(got[name][0]).max())


def test_activations_far_out():
    g = np.array([-1000.0, -50.0, 0.0, 50.0, 1000.0])
    for kind in ("silu", "gelu", "gelu_tanh"):
        a, slope, _ = po.activation(kind, g)
        assert np.allclose(a, np.maximum(g, 0)) and np.allclose(slope, [0, 0, 0.5, 1, 1])


def test_orthogonalise_definition():
    rng = np.random.default_rng(5)
    G = rng.standard_normal((6, 9))
    # each step maps singular values s to a s + b s^3 + c s^5 and keeps the directions
    U, s, V = np.linalg.svd(G, full_matrices=False)
    s = s / (np.linalg.norm(G) + 1e-7)
    for _ in range(5):
        s = 3.4445 * s - 4.7750 * s ** 3 + 2.0315 * s ** 5
    assert np.allclose(po.orthogonalise(G), U * s @ V, atol=1e-12)
    assert np.allclose(po.orthogonalise(G.T), (U * s @ V).T, atol=1e-12)
    # the model without any rounding is the definition
    assert np.allclose(po.orthogonalise(G, operand=lambda X: X), U * s @ V, atol=1e-12)


def test_bf16_rounding():
    v = np.array([1.0, 1.0 + 2.0 ** -8, 1.0 + 3 * 2.0 ** -8, -3.1e38, 0.0, 65536.5], dtype=np.float32)
    assert np.array_equal(po.decode(po.encode(v, "bf16"), "bf16")[:3], [1.0, 1.0, 1.0 + 2.0 ** -6])
    assert np.isnan(po.decode(po.encode(np.array([np.nan]), "bf16"), "bf16"))[0]


def test_saved_bytes(hip_lib):
    # h in the element type, g and u in 32 bits; rows of an odd number of 128-byte lines of the element type,
    # each part a multiple of 256 bytes
    assert GatedFfn(64, 512, "bf16").saved_bytes(8) == 8 * 576 * (2 + 4 + 4)
    assert GatedFfn(64, 510, "fp16").saved_bytes(8) == 8 * 576 * 10
    assert GatedFfn(64, 510, "fp32").saved_bytes(2) == 3 * 4352        # 2 rows of 17 lines, 4352 bytes
    assert GatedFfn(64, 512, "bf16").saved_bytes(0) == 0


@pytest.mark.parametrize("make,needle", [
    (lambda: GatedFfn(0, 8).saved_bytes(1), "d_model and d_ff"),
    (lambda: GatedFfn(8, -3).saved_bytes(1), "d_model and d_ff"),
    (lambda: GatedFfn(8, 1 << 21).saved_bytes(1), "d_model and d_ff"),
    (lambda: GatedFfn(8, 8).saved_bytes(-1), "number of tokens"),
    (lambda: GatedFfn(8, 8).saved_bytes((1 << 24) + 1), "number of tokens"),
])
def test_ffn_refuses_extents(hip_lib, make, needle):
    with pytest.raises(HipError, match=needle) as err:
        make()
    assert err.value.status == hip.RL_ERR_INVALID_ARG


def test_python_refuses_choices():
    with pytest.raises(ValueError, match="dtype is one of"):
        GatedFfn(8, 8, dtype="fp8")
    with pytest.raises(ValueError, match="activation is one of"):
        GatedFfn(8, 8, activation="tanh")
    with pytest.raises(ValueError, match="dtype is one of"):
        Orthogonalizer(8, 8, dtype="fp64")
    with pytest.raises(ValueError, match="three numbers"):
        Orthogonalizer(8, 8, steps=3, coefficients=[(1, 2, 3)] * 2)
    with pytest.raises(ValueError, match="three numbers"):
        Orthogonalizer(8, 8, coefficients=(1, 2))


def test_c_entry_points_refuse_null_and_wrong_configs(hip_lib):
    out = C.c_size_t(7)
    bad = [hip.FfnConfig(3, 0, 8, 8), hip.FfnConfig(-1, 0, 8, 8), hip.FfnConfig(0, 3, 8, 8), hip.FfnConfig(0, -1, 8, 8)]
    for cfg in bad:
        assert hip_lib.rl_ffn_saved_bytes(C.byref(cfg), 1, C.byref(out)) == hip.RL_ERR_INVALID_ARG
    good = hip.FfnConfig(0, 0, 8, 8)
    assert hip_lib.rl_ffn_saved_bytes(None, 1, C.byref(out)) == hip.RL_ERR_INVALID_ARG
    assert hip_lib.rl_ffn_saved_bytes(C.byref(good), 1, None) == hip.RL_ERR_INVALID_ARG
    assert hip_lib.rl_ffn_workspace_bytes(C.byref(good), -1, 0, 0, C.byref(out)) == hip.RL_ERR_INVALID_ARG
    nothing = [None, 8] * 5
    assert hip_lib.rl_ffn_forward(None, *nothing, 1, None, None, 0, None) == hip.RL_ERR_INVALID_ARG
    assert hip_lib.rl_ffn_forward(C.byref(good), *nothing, -1, None, None, 0, None) == hip.RL_ERR_INVALID_ARG
    assert hip_lib.rl_ffn_forward(C.byref(good), *nothing, 0, None, None, 0, None) == 0          # no tokens: nothing to do
    for field, value, needle in (("dtype", 5, b"dtype"), ("rows", 0, b"rows and cols"), ("cols", 1 << 21, b"rows and cols"), ("batch", -1, b"batch"),
                                 ("batch", 65536, b"batch"), ("steps", -1, b"steps"), ("steps", 65, b"steps"),
                                 ("eps", -1.0, b"eps"), ("eps", float("nan"), b"eps"), ("eps", float("inf"), b"eps"), ("scale", float("inf"), b"scale")):
        cfg = hip.OrthoConfig(0, 8, 8, 1, 5, 1e-7, 1.0)
        setattr(cfg, field, value)
        assert hip_lib.rl_orthogonalize(C.byref(cfg), None, None, 8, 64, None, 8, 64, None, 0, None) == hip.RL_ERR_INVALID_ARG
        assert needle in hip_lib.rl_last_error()
    none = hip.OrthoConfig(0, 8, 8, 0, 5, 1e-7, 1.0)
    assert hip_lib.rl_orthogonalize(C.byref(none), None, None, 8, 64, None, 8, 64, None, 0, None) == 0   # an empty stack


def test_dtypes_and_activations_match_the_header():
    import re
    from pathlib import Path
    header = (Path(__file__).resolve().parent.parent / "include" / "roller_hip.h").read_text()
    value = lambda name: int(re.search(rf"#define {name} (\d+)", header).group(1))
    assert products.DTYPES == {"fp32": value("RL_F32"), "fp16": value("RL_F16"), "bf16": value("RL_BF16")}
    assert products.ACTIVATIONS == {"silu": value("RL_ACT_SILU"), "gelu": value("RL_ACT_GELU"), "gelu_tanh": value("RL_ACT_GELU_TANH")}
    assert Ptr(256).address == 256


def kinds(tiles):
    """Of every product in the result of tiles(): (product, tile rows, some are split), and where that is only those after
    the whole ones, (tile rows,)."""
    return {(name, rows, splits > 1) for name, (rows, _, splits, whole) in tiles.items()} | {(rows,) for rows, _, splits, whole in tiles.values() if splits > 1 and whole}


def test_the_sizes_of_the_gpu_tests_take_every_product_through_every_tile(hip_lib):
    import random
    from test_products_gpu import EVERY_ORTHO_TILE, EVERY_TILE, EVERY_TILE_SAMPLED
    pick = random.Random(1)
    between = lambda lo, hi: int(2 ** pick.uniform(lo, hi))
    for dtypes, most in ((("bf16", "fp16"), 1e15), (("fp32",), 4e10)):        # (T D F; in fp32 what lies beyond would take minutes)
        sizes = [(between(5, 14), between(6, 14), between(6, 14)) for _ in range(4000)]
        reached = set().union(*(kinds(GatedFfn(D, F, dtypes[0]).tiles(T)) for T, D, F in sizes if T * D * F <= most))
        tested = set().union(*(kinds(GatedFfn(D, F, dtype).tiles(T)) for T, D, F, dtype in EVERY_TILE + EVERY_TILE_SAMPLED if dtype in dtypes))
        assert len(reached) > 25 and reached <= tested, reached - tested
    for dtypes in (("bf16",), ("fp16", "fp32")):
        reached = set().union(*(kinds(Orthogonalizer(between(5, 13), between(5, 13), between(0, 6), dtypes[0]).tiles()) for _ in range(4000)))
        tested = set().union(*(kinds(Orthogonalizer(m, n, batch, dtype).tiles()) for batch, m, n, dtype in EVERY_ORTHO_TILE if dtype in dtypes))
        assert len(reached) > 12 and reached <= tested, reached - tested


def test_tiles_refuse(hip_lib):
    for make in (lambda: GatedFfn(8, 8).tiles(0), lambda: GatedFfn(8, 8).tiles(4, compute_units=0), lambda: Orthogonalizer(8, 8, batch=0).tiles(),
                 lambda: Orthogonalizer(8, 8).tiles(compute_units=0), lambda: GatedFfn(0, 8).tiles(4), lambda: Orthogonalizer(8, 0).tiles()):
        with pytest.raises(HipError) as err:
            make()
        assert err.value.status == hip.RL_ERR_INVALID_ARG
