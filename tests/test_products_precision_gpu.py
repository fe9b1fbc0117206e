"""Orthogonalised fp16 and fp32 matrices on an MI355X, held to the error that their two-part products leave (some 1e-6 of
the norm) rather than to the rounding of the output; test_products_precision.py shows what that tells apart."""

import numpy as np
import pytest

from oracle import products_oracle as po
from test_products_gpu import EVERY_ORTHO_TILE, gradient, ortho

pytestmark = pytest.mark.gpu

TWO_PART = [s for s in EVERY_ORTHO_TILE if s[3] != "bf16"] + [(1, 300, 257, "fp16"), (8, 509, 1023, "fp32"), (1, 64, 64, "fp32"), (2, 130, 65, "fp16")]


@pytest.mark.parametrize("batch,rows,cols,dtype", TWO_PART)
def test_two_part_products(device, batch, rows, cols, dtype):
    two = gradient(np.random.default_rng([batch, rows, cols]), min(batch, 2), rows, cols)
    got, G = ortho(two[np.arange(batch) % 2], dtype)
    for i in range(len(two)):
        exact, model = po.orthogonalise(G[i]), po.orthogonalise_two_part(G[i])
        off = [po.two_part_excess(g, exact, model, dtype) for g in got[i::2]]
        assert max(off) <= 1, f"off by {max(off)} times the tolerance"
