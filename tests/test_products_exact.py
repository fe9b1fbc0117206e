"""What the GPU tests on whole numbers would see, and which forms of the kernel for few tokens they take."""

import random

import numpy as np
import pytest

from oracle.products_exact import PRODUCTS, ExactFeedForward
from test_products_exact_gpu import FEW
from test_products_gpu import EVERY_TILE, EVERY_TILE_SAMPLED


@pytest.mark.parametrize("T,D,F,dtype", EVERY_TILE + EVERY_TILE_SAMPLED + FEW)
def test_a_lost_k_step_is_told(T, D, F, dtype):
    b, pick = ExactFeedForward(T, D, F, dtype), random.Random(T + D + F)
    many = 32 if D * F < 4e6 else 6
    ts, fs = np.arange(T)[::-1][::-(-T // many)], np.arange(F)[::-(-F // min(many, 8))]
    whole, step = {**b.of_tokens(ts), **b.of_features(fs)}, 32 if dtype == "fp32" else 64
    depth = dict(zip(PRODUCTS, (D, F, D, 2 * F, T, T)))
    results = dict(zip(PRODUCTS, (("y",), ("y",), ("dx",), ("dx",), ("dw_gate", "dw_up"), ("dw_down",))))
    for name in PRODUCTS:
        first = pick.randrange(-(-depth[name] // step)) * step
        lose = (name, slice(first, first + step))
        got = b.of_tokens(ts, lose) if name in PRODUCTS[:4] else b.of_features(fs, lose)
        assert all((got[n] != whole[n]).any() for n in results[name]), f"{name} without {lose[1]}"


def forms(T, D, F, dtype):
    """How the kernel for up to 16 tokens takes both products: (parts of K in one block, 16 bits, product, waves, a wave has
    several loads, there is a rest below a load, there are whole loads)."""
    size, parts, out = 4 if dtype == "fp32" else 2, 4 if T <= 4 else 2 if T <= 8 else 1, set()
    for product, N, K in (("gate and up", F, D), ("down", D, F)):
        groups, waves, load = -(-N // (16 // parts)), 1, 512 // size * parts
        while waves < 16 and groups * waves < 16 * 256 and K // parts * size >= 512 * waves:
            waves *= 2
        out.add((parts, size == 2, product, waves == 1, K > waves * load, K % load != 0, K >= load))
    return out


def test_the_sizes_of_the_gpu_tests_take_every_form_of_few_tokens():
    pick = random.Random(2)
    between = lambda lo, hi: int(2 ** pick.uniform(lo, hi))
    for dtypes in (("bf16", "fp16"), ("fp32",)):
        reached = set().union(*(forms(pick.randint(1, 16), between(5, 14), between(5, 14), dtypes[0]) for _ in range(4000)))
        reached = {f for f in reached if f[5]}                        # (K a whole number of loads is hit by design only)
        tested = set().union(*(forms(*s) for s in FEW if s[3] in dtypes))
        assert len(reached) > 12 and reached <= tested, reached - tested
        for parts in (1, 2, 4):
            assert any(f[0] == parts and not f[5] for f in tested), f"no K of whole loads with {parts} parts"
