"""A gated feed-forward block on small whole numbers, where every sum is exact in fp32 whatever its order and the
library's results can be told to the last bit.  numpy only.

The gates are 128 and a little: x starts with an 8 and every gate weight row with a 16, and the other products, of
numbers -1, 0 and 1, add a random walk of standard deviation 8 at most.  From 18 on a sigmoid is 1 in fp32, so
silu(g) = g and its slope 1.  What is left are products of whole numbers far below 2^24 and the roundings to the element
type that the library states: of the gated product (with up to 16 tokens of 16 bits: only where it is kept), of the
gradients before the gate and up weights, of the results.  A product, a K step or a column that is lost, doubled or
taken from elsewhere moves a result by whole numbers.

``lose`` names a product and a range of its summation index to leave out, which is how the tests of the
tests ask whether a lost K step shows."""

from __future__ import annotations

import numpy as np

from .products_oracle import decode, encode

PRODUCTS = ("gate and up", "down", "dh", "dx", "dw_gate and dw_up", "dw_down")


class ExactFeedForward:
    def __init__(self, T: int, D: int, F: int, dtype: str, seed: int = 0):
        rng = np.random.default_rng([seed, T, D, F])
        self.T, self.D, self.F, self.dtype = T, D, F, dtype

        def ternary(shape, density):
            signs = np.where(rng.integers(0, 2, shape, np.int8), np.float32(1), np.float32(-1))
            return signs if density >= 1 else signs * (rng.random(shape, np.float32) < density)

        walk = min(1.0, 8 / D ** 0.5)                          # of x and of the gate and up weights: 64 products of D
        down = min(1.0, 100 / F)                               # of the down weights: 100 a row
        self.x, self.wg, self.wu = ternary((T, D), walk), ternary((F, D), walk), ternary((F, D), walk)
        self.wd, self.dy = ternary((D, F), down), ternary((T, D), min(1.0, 64 / (D * down), 400 / T))
        self.x[:, 0], self.wg[:, 0] = 8, 16
        self.dy[-1, ::16] = 1                                  # (something of the last token in every K step)

    def _round(self, v):
        return decode(encode(v, self.dtype), self.dtype).astype(np.float32)

    def _product(self, name, a, b, lose):
        """a b^T, without the part of the sum that is lost."""
        if lose and lose[0] == name:
            a = a.copy()
            a[:, lose[1]] = 0
        return a @ b.T

    def _gated(self, x, fs, lose):
        g, u = (self._product("gate and up", x, w[fs], lose) for w in (self.wg, self.wu))
        if not (lose and lose[0] == "gate and up"):
            assert g.min() >= 18
        with np.errstate(over="ignore"):
            s = np.where(g >= 18, np.float32(1), 1 / (1 + np.exp(-g)))
        return g, u, s, g * s * u

    def of_tokens(self, ts=slice(None), lose=None, backward=True) -> dict:
        """y and dx of the tokens ts, as the library stores them."""
        g, u, s, h = self._gated(self.x[ts], slice(None), lose)
        if self.T > 16 or self.dtype == "fp32":
            h = self._round(h)
        out = {"y": self._round(self._product("down", h, self.wd, lose))}
        if backward:
            dh = self._product("dh", self.dy[ts], self.wd.T, lose)
            dg, du = self._round(dh * u * (s + g * s * (1 - s))), self._round(dh * g * s)
            out["dx"] = self._round(self._product("dx", np.concatenate([dg, du], 1), np.concatenate([self.wg, self.wu]).T, lose))
        return out

    def of_features(self, fs=slice(None), lose=None) -> dict:
        """dw_gate, dw_up and the columns of dw_down of the features fs, as the library stores them."""
        g, u, s, h = self._gated(self.x, fs, lose)
        dh = self._product("dh", self.dy, self.wd[:, fs].T, lose)
        dg, du = self._round(dh * u * (s + g * s * (1 - s))), self._round(dh * g * s)
        of = lambda a, b, name: self._round(self._product(name, np.ascontiguousarray(a.T), b.T, lose))
        return {"dw_gate": of(dg, self.x, "dw_gate and dw_up"), "dw_up": of(du, self.x, "dw_gate and dw_up"),
                "dw_down": of(self.dy, self._round(h), "dw_down")}
