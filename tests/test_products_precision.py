"""What the GPU tests of the two-part products would see: a term left out of every product is far outside their
tolerance, at every size that they take but the largest."""

import numpy as np
import pytest

from oracle import products_oracle as po
from test_products_precision_gpu import TWO_PART


@pytest.mark.parametrize("batch,rows,cols,dtype", [s for s in TWO_PART if s[1] * s[2] < 5e6])   # (the largest takes half a minute here)
def test_a_lost_term_is_told(batch, rows, cols, dtype):
    how = dict(steps=5 if rows * cols < 1.2e6 else 2)          # (the largest with two)
    rng, r = np.random.default_rng([batch, rows, cols]), max(1, min(rows, cols) // 8)
    G = 1e-3 * (rng.standard_normal((rows, r)) @ rng.standard_normal((r, cols)) + rng.standard_normal((rows, cols)))
    G = po.decode(po.encode(G, dtype), dtype)
    exact, model = po.orthogonalise(G, **how), po.orthogonalise_two_part(G, **how)
    assert po.two_part_excess(po.decode(po.encode(model, dtype), dtype), exact, model, dtype) < 0.5
    for lose in ("hi lo", "lo hi"):
        got = po.decode(po.encode(po.orthogonalise_two_part(G, lose=(lose,), **how), dtype), dtype)
        assert po.two_part_excess(got, exact, model, dtype) > (10 if dtype == "fp32" else 2.5)
