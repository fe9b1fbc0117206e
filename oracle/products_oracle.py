"""The feed-forward block and Newton-Schulz orthogonalisation in 64 bits, with bounds on how far kernels
that round where the library says may be off.  numpy only; bf16 values travel as their uint16 bit patterns.

Bounds.  u = half a step of the element type relative to the value (bf16 2^-8, fp16 2^-11, fp32 2^-24), and
for fp16 at least half a subnormal step, 2^-25.  A sum of n products in fp32 is off by at most
(n + 8) 2^-23 times the sum of the magnitudes: products of 16-bit values are exact in fp32, a fp32 product
has one rounding, n additions have one each, and a full step instead of half of one covers a matrix unit
that truncates.  Everything else is first-order error propagation, multiplied by 1.1 for the higher orders.
"""

from __future__ import annotations

import numpy as np
from math import erf, pi, sqrt

HALF_STEP = {"bf16": 2.0 ** -8, "fp16": 2.0 ** -11, "fp32": 2.0 ** -24}
SMALLEST = {"bf16": 0.0, "fp16": 2.0 ** -25, "fp32": 0.0}
STORAGE = {"bf16": np.uint16, "fp16": np.float16, "fp32": np.float32}
STANDARD = (3.4445, -4.7750, 2.0315)


def encode(values: np.ndarray, dtype: str) -> np.ndarray:
    """Values rounded to nearest even, in the storage the device sees."""
    if dtype == "bf16":
        bits = np.ascontiguousarray(values, dtype=np.float32).view(np.uint32)
        rounded = ((bits + (0x7FFF + ((bits >> 16) & 1))) >> 16).astype(np.uint16)
        return np.where(np.isnan(values), np.uint16(0x7FC0), rounded)
    with np.errstate(over="ignore"):
        return np.asarray(values).astype(STORAGE[dtype])


def decode(stored: np.ndarray, dtype: str) -> np.ndarray:
    if dtype == "bf16":
        return (stored.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    return stored.astype(np.float64)


def sum_error(n: int) -> float:
    return (n + 8) * 2.0 ** -23


def activation(kind: str, g: np.ndarray):
    """(act(g), act'(g), argument of the sigmoid or 0, in magnitude)"""
    if kind == "gelu":
        phi = 0.5 * (1 + np.vectorize(erf, otypes=[float])(g / sqrt(2)))
        return g * phi, phi + g * np.exp(-g * g / 2) / sqrt(2 * pi), np.zeros_like(g)
    if kind == "silu":
        z, dz = g, 1.0
    else:
        z, dz = 2 * sqrt(2 / pi) * (g + 0.044715 * g ** 3), 2 * sqrt(2 / pi) * (1 + 3 * 0.044715 * g * g)
    s = np.where(z >= 0, 1 / (1 + np.exp(-np.abs(z))), np.exp(-np.abs(z)) / (1 + np.exp(-np.abs(z))))
    return g * s, s + g * s * (1 - s) * dz, np.abs(z)


def round_error(values: np.ndarray, dtype: str) -> np.ndarray:
    return np.maximum(HALF_STEP[dtype] * np.abs(values), SMALLEST[dtype])


class FeedForward:
    """The block on the (already rounded) inputs, in 64 bits, with a bound for every result."""

    def __init__(self, x, w_gate, w_up, w_down, kind: str, dtype: str):
        self.x, self.wg, self.wu, self.wd, self.kind, self.dtype = x, w_gate, w_up, w_down, kind, dtype
        D, F = x.shape[1], w_gate.shape[0]
        A = np.abs
        self.g, self.u = x @ w_gate.T, x @ w_up.T
        self.a, self.slope, z = activation(kind, self.g)
        self.h = self.a * self.u
        # errors of g and u (sums of D products), of the activation in fp32 (exponential, reciprocal and a
        # few roundings: 8 half steps of |g|, and the rounding of the exponent's argument, |z| half steps of
        # the value), and of h before and after its rounding
        self.eg, self.eu = sum_error(D) * (A(x) @ A(w_gate).T), sum_error(D) * (A(x) @ A(w_up).T)
        self.ea = 1.13 * self.eg + 2.0 ** -24 * (8 * A(self.g) + 2 * z * A(self.a))
        eh = 1.1 * (A(self.u) * self.ea + A(self.a) * self.eu) + 2.0 ** -24 * A(self.h)
        self.eh = eh + round_error(A(self.h) + eh, dtype)
        self.y = self.h @ w_down.T
        ey = 1.1 * (self.eh @ A(w_down).T) + sum_error(F) * ((A(self.h) + self.eh) @ A(w_down).T)
        self.y_bound = ey + round_error(A(self.y) + ey, dtype)
        # slope: |act''| <= 1.13, and in fp32 a dozen roundings of terms up to 1 + |g| (gelu_tanh: the cubic's
        # derivative, up to 1 + 3.2 |g|^2 |act'| near the turn, is covered by |z|)
        self.es = 1.13 * self.eg + 2.0 ** -24 * 16 * (1 + A(self.g) + z)

    def backward(self, dy) -> dict:
        """{name: (value, bound)} of the gradients of sum(dy * y)."""
        A, dtype = np.abs, self.dtype
        T, D = dy.shape
        F = self.wg.shape[0]
        dh = dy @ self.wd
        e_dh = sum_error(D) * (A(dy) @ A(self.wd))
        dg, du = dh * self.u * self.slope, dh * self.a
        e_dg = 1.1 * (A(self.u * self.slope) * e_dh + A(dh * self.slope) * self.eu + A(dh * self.u) * self.es) + 2.0 ** -23 * A(dg)
        e_du = 1.1 * (A(self.a) * e_dh + A(dh) * self.ea) + 2.0 ** -24 * A(du)
        e_dg = e_dg + round_error(A(dg) + e_dg, dtype)
        e_du = e_du + round_error(A(du) + e_du, dtype)

        def product(pairs, n):
            """sum of a @ b over pairs of (a, error of a, b, error of b), n products to a result"""
            value = sum(a @ b for a, _, b, _ in pairs)
            err = sum(1.1 * (ea @ A(b) + A(a) @ eb) + sum_error(n) * ((A(a) + ea) @ (A(b) + eb)) for a, ea, b, eb in pairs)
            return value, err + round_error(A(value) + err, dtype)

        zero = np.zeros_like
        return {"dx": product([(dg, e_dg, self.wg, zero(self.wg)), (du, e_du, self.wu, zero(self.wu))], 2 * F),
                "dw_gate": product([(dg.T, e_dg.T, self.x, zero(self.x))], T),
                "dw_up": product([(du.T, e_du.T, self.x, zero(self.x))], T),
                "dw_down": product([(dy.T, zero(dy.T), self.h, self.eh)], T)}


def orthogonalise(G: np.ndarray, steps: int = 5, coefficients=STANDARD, eps: float = 1e-7, scale: float = 1.0,
                  keep=lambda X: X, operand=None) -> np.ndarray:
    """Newton-Schulz in 64 bits.  With ``keep`` (rounding of what is kept between products) and ``operand``
    (rounding of what the products read) it is a model of an implementation: the operands then are X, and A
    and B without their diagonals."""
    tall = G.shape[0] > G.shape[1]
    X = G.T if tall else G
    X = keep(X / (np.sqrt((X * X).sum()) + eps))
    per_step = coefficients if steps and np.ndim(coefficients) == 2 else [coefficients] * steps
    for a, b, c in per_step:
        if operand is None:
            A = X @ X.T
            X = a * X + (b * A + c * (A @ A)) @ X
            continue
        x = operand(X)
        A = keep(x @ x.T)
        D = np.diag(A).copy()
        Ao = operand(A - np.diag(D))
        B = keep(b * (Ao + np.diag(D)) + c * (Ao @ Ao + (D[:, None] + D[None, :]) * Ao + np.diag(D * D)))
        E = np.diag(B).copy()
        X = keep((a + E)[:, None] * X + operand(B - np.diag(E)) @ x)
    return scale * (X.T if tall else X)


def orthogonalise_tolerance(G: np.ndarray, dtype: str, exact: np.ndarray, **how) -> float:
    """How far the library's result may be from ``exact``, in the Frobenius norm.

    The iteration multiplies errors by up to 3.4 in every step, so a worst-case bound says nothing; but the
    roundings are many and independent, and their sum over a matrix has a sharp norm.  A model with the
    library's roundings in 64-bit arithmetic (fp16 operands scaled by 2^9 and fp32 for the rest where the
    matrices are bf16; where they are fp16 or fp32, operands of 21 bits: the high and the low part of a
    two-part fp16 number, or more) gives that norm for the matrix at hand; sums of n products in
    fp32 add a random walk of n half steps, at most sqrt(n) 2^-24 of the sum's terms, amplified alike.
    Allowed: three times the model's error, the walk times the largest amplification of five standard
    steps (3.4445^5 = 485, of errors that start at the size of the small singular directions: 64 in the
    norm), and half a step of the output."""
    f32 = lambda X: X.astype(np.float32).astype(np.float64)
    if dtype == "bf16":
        operand = lambda X: (X * 512).astype(np.float16).astype(np.float64) / 512
    else:
        operand = lambda X: np.round(X * 2.0 ** 21 / 2.0 ** np.ceil(np.log2(np.abs(X) + 1e-300))) / 2.0 ** 21 * 2.0 ** np.ceil(np.log2(np.abs(X) + 1e-300))
    model = orthogonalise(G, keep=f32, operand=operand, **how)
    norm = np.linalg.norm(exact)
    n = max(G.shape)
    return 3 * np.linalg.norm(model - exact) + (64 * sqrt(n) * 2.0 ** -24 + HALF_STEP[dtype]) * norm + SMALLEST[dtype] * sqrt(exact.size)


def orthogonalise_two_part(G: np.ndarray, steps: int = 5, coefficients=STANDARD, eps: float = 1e-7, scale: float = 1.0, lose=()) -> np.ndarray:
    """Newton-Schulz as fp16 and fp32 matrices take it, in fp32 on the host: operands are two fp16 numbers, scaled by 2^9,
    and a product is hi hi + hi lo + lo hi.  ``lose`` leaves terms out: "hi lo", "lo hi"."""
    f = np.float32
    tall = G.shape[0] > G.shape[1]
    X = G.T if tall else G
    X = np.ascontiguousarray((X / (np.sqrt((X * X).sum()) + eps)).astype(f))

    def parts(M):
        M = M * f(512)
        hi = M.astype(np.float16).astype(f)
        return hi, (M - hi).astype(np.float16).astype(f)

    def product(a, b):
        p = a[0] @ b[0]
        if "hi lo" not in lose:
            p += a[0] @ b[1]
        if "lo hi" not in lose:
            p += a[1] @ b[0]
        return p * f(2.0 ** -18)

    per_step = coefficients if steps and np.ndim(coefficients) == 2 else [coefficients] * steps
    for a, b, c in ([f(v) for v in step] for step in per_step):
        x = parts(X)
        A = product(x, [np.ascontiguousarray(p.T) for p in x])
        D = np.diag(A).copy()
        ao = parts(A - np.diag(D))
        Ao, square = (ao[0] + ao[1]) * f(1 / 512), product(ao, ao)
        B = b * Ao + c * (square + (D[:, None] + D[None, :]) * Ao)
        E = b * D + c * (np.diag(square) + D * D)
        np.fill_diagonal(B, 0)
        X = (a + E)[:, None] * X + product(parts(B), x)
    X = scale * X.astype(np.float64)
    return X.T if tall else X


def two_part_excess(got: np.ndarray, exact: np.ndarray, model: np.ndarray, dtype: str) -> float:
    """How far fp16 or fp32 results are off, in the norm, as a multiple of what they may be; for sides of 30 and more,
    whose many roundings make one sample of an error's norm tell the next one.

    ``model`` (orthogonalise_two_part) has the library's roundings and sums of fp32 in another order, one rounding per
    product where a matrix unit has one per 16, so its error e stands for the library's; four times it is allowed, and
    half a step of the output.  For fp16 that half step is 500 times e; the result is held to the exact one after its rounding
    instead.  The two differ where an error of e_i takes an element over the border between two numbers, a step s_i apart:
    with probability |e_i| / s_i, which adds s_i^2; so the square of the norm is sum |e_i| s_i, at most |e| |s|, and
    where e_i is more than a step, |e|^2."""
    e = 4 * np.linalg.norm(model - exact)
    if dtype == "fp32":
        return np.linalg.norm(got - exact) / (e + HALF_STEP[dtype] * np.linalg.norm(exact))
    rounded = exact.astype(np.float16)
    steps = np.maximum(np.spacing(np.abs(rounded)).astype(np.float64), 2.0 ** -24)
    return np.linalg.norm(got - rounded.astype(np.float64)) / (np.sqrt(e * np.linalg.norm(steps)) + e)
