"""Products of a language model's feed-forward block on MI355X: the gated block itself, forward and
backward (``GatedFfn``), and the orthogonalisation of an update of its weights (``Orthogonalizer``).

They stand beside ``hip.GemmPlan``: a matrix argument is a ``DeviceArray``, a ``hip.Ptr`` or an ``int``
device address (``hip.Ptr(tensor.data_ptr())`` for a torch tensor), row-major, with an optional leading
dimension in elements; a stream is a ``hip.Stream`` or a raw handle; a workspace is the caller's or, by
default, one that the library keeps per stream.  Calls enqueue work and return; a refused call raises
``HipError`` with the library's text before anything is enqueued.

numpy has no bfloat16: device buffers of that type are made as ``uint16`` (or by another library).

(A process that also uses torch imports torch first, so that both find the same HIP runtime.)
"""

from __future__ import annotations

import ctypes as C
from typing import Optional, Sequence

from . import hip
from .hip import RL_ERR_INVALID_ARG, FfnConfig, HipError, OrthoConfig, ProductTile, Ptr, _stream_handle, check, lib

DTYPES = {"fp32": 0, "fp16": 1, "bf16": 2}
ACTIVATIONS = {"silu": 0, "gelu": 1, "gelu_tanh": 2}


def _choice(what: str, value: str, table: dict) -> int:
    if value not in table:
        raise ValueError(f"{what} is one of {', '.join(table)}, got {value!r}")
    return table[value]


def _address(x) -> int:
    """``hip._address``, for a call that takes a handful of them and may last a few microseconds."""
    return x.address if type(x) is Ptr else hip._address(x)


def _room(workspace, workspace_bytes: Optional[int]) -> tuple[Optional[int], int]:
    if workspace is None:
        return None, 0
    if workspace_bytes is None:
        workspace_bytes = getattr(workspace, "nbytes", None)
        if workspace_bytes is None:
            raise ValueError("workspace: an address needs its size as workspace_bytes")
    return _address(workspace), int(workspace_bytes)


class GatedFfn:
    """``y = (act(x Wg^T) * (x Wu^T)) Wd^T`` with weights stored as ``[outputs, inputs]``:
    ``w_gate[d_ff, d_model]``, ``w_up[d_ff, d_model]``, ``w_down[d_model, d_ff]``.

    ``dtype`` is "bf16", "fp16" or "fp32" (all matrices; sums are fp32), ``activation`` "silu", "gelu"
    (erf) or "gelu_tanh".  The object holds the configuration and nothing of a call."""

    def __init__(self, d_model: int, d_ff: int, dtype: str = "bf16", activation: str = "silu"):
        self.d_model, self.d_ff, self.dtype, self.activation = int(d_model), int(d_ff), dtype, activation
        self._config = FfnConfig(_choice("dtype", dtype, DTYPES), _choice("activation", activation, ACTIVATIONS), self.d_model, self.d_ff)
        self._at = C.byref(self._config)

    def workspace_bytes(self, tokens: int, backward: bool = False, unaligned: bool = False) -> int:
        """Workspace of a forward call (with ``backward``: enough for both passes).  ``unaligned``: for
        16-bit rows that start at odd elements although the extents are even, and for a backward call whose
        gate and up weights have different leading dimensions."""
        hip.init()
        out = C.c_size_t()
        check(lib().rl_ffn_workspace_bytes(self._at, tokens, int(backward), int(unaligned), C.byref(out)))
        return out.value

    def saved_bytes(self, tokens: int) -> int:
        """Size of the buffer in which a forward call keeps what the backward pass reads."""
        out = C.c_size_t()
        check(lib().rl_ffn_saved_bytes(self._at, tokens, C.byref(out)))
        return out.value

    def _saved(self, saved, nbytes: Optional[int], tokens: int) -> int:
        """Address of ``saved``, whose size, where it is known, has to hold ``tokens`` (the library is told none)."""
        if nbytes is None:
            nbytes = getattr(saved, "nbytes", None)
        if nbytes is not None and nbytes < self.saved_bytes(tokens):
            raise HipError(RL_ERR_INVALID_ARG, f"saved: {tokens} tokens need a buffer of {self.saved_bytes(tokens)} bytes, got {nbytes}")
        return _address(saved)

    PRODUCTS = ("gate and up", "down", "dw_down", "dh", "dx", "dw_gate and dw_up")

    def tiles(self, tokens: int, compute_units: int = 256) -> dict:
        """{product: (tile rows, tile columns, splits, tiles not split)}: what a block of so many tokens runs with (host
        arithmetic, no device)."""
        out = (ProductTile * 6)()
        check(lib().rl_ffn_tiles(self._at, tokens, compute_units, out))
        return {name: (t.rows, t.cols, t.splits, t.whole) for name, t in zip(self.PRODUCTS, out)}

    def forward(self, x, w_gate, w_up, w_down, y, tokens: int, *, ldx: Optional[int] = None, ld_gate: Optional[int] = None,
                ld_up: Optional[int] = None, ld_down: Optional[int] = None, ldy: Optional[int] = None, saved=None,
                stream=None, workspace=None, workspace_bytes: Optional[int] = None, saved_bytes: Optional[int] = None) -> None:
        """Enqueues the block for ``tokens`` rows.  ``saved`` keeps what ``backward`` reads and has the size that the
        method ``saved_bytes`` tells: a ``DeviceArray`` is held to it, an address with the argument ``saved_bytes``."""
        at_saved = None if saved is None else self._saved(saved, saved_bytes, tokens)
        hip.init()
        d, f, room = self.d_model, self.d_ff, _room(workspace, workspace_bytes)
        check(lib().rl_ffn_forward(
            self._at, _address(x), d if ldx is None else ldx, _address(w_gate), d if ld_gate is None else ld_gate,
            _address(w_up), d if ld_up is None else ld_up, _address(w_down), f if ld_down is None else ld_down,
            _address(y), d if ldy is None else ldy, tokens, at_saved, *room, _stream_handle(stream)))

    def backward(self, dy, x, w_gate, w_up, w_down, saved, dx, dw_gate, dw_up, dw_down, tokens: int, *,
                 lddy: Optional[int] = None, ldx: Optional[int] = None, ld_gate: Optional[int] = None, ld_up: Optional[int] = None,
                 ld_down: Optional[int] = None, lddx: Optional[int] = None, ldd_gate: Optional[int] = None,
                 ldd_up: Optional[int] = None, ldd_down: Optional[int] = None, stream=None, workspace=None,
                 workspace_bytes: Optional[int] = None, saved_bytes: Optional[int] = None) -> None:
        """Enqueues the gradients of ``sum(dy * y)``.  ``dx``, ``dw_down``, and ``dw_gate`` with ``dw_up``, may be
        None: not computed.  ``saved`` as in ``forward``, for as many tokens."""
        at_saved = self._saved(saved, saved_bytes, tokens)
        hip.init()
        d, f, room = self.d_model, self.d_ff, _room(workspace, workspace_bytes)
        out = [None if g is None else _address(g) for g in (dx, dw_gate, dw_up, dw_down)]
        check(lib().rl_ffn_backward(
            self._at, _address(dy), d if lddy is None else lddy, _address(x), d if ldx is None else ldx,
            _address(w_gate), d if ld_gate is None else ld_gate, _address(w_up), d if ld_up is None else ld_up,
            _address(w_down), f if ld_down is None else ld_down, _address(saved),
            out[0], d if lddx is None else lddx, out[1], d if ldd_gate is None else ldd_gate, out[2], d if ldd_up is None else ldd_up,
            out[3], f if ldd_down is None else ldd_down, tokens, *room, _stream_handle(stream)))


class Orthogonalizer:
    """Newton-Schulz orthogonalisation of ``G[rows, cols]``, or of a stack of ``batch`` of them:
    ``X = G / (||G|| + eps)``, then ``steps`` times ``X <- a X + (b A + c A A) X`` with ``A = X X^T`` of the
    shorter side, and ``O = scale X``.

    ``coefficients`` is one ``(a, b, c)`` for all steps, or one for each; they keep the elements of X, A and
    b A + c A A below 100."""

    STANDARD = (3.4445, -4.7750, 2.0315)

    def __init__(self, rows: int, cols: int, batch: int = 1, dtype: str = "bf16", steps: int = 5,
                 coefficients: Sequence = STANDARD, eps: float = 1e-7, scale: float = 1.0):
        self.rows, self.cols, self.batch, self.dtype, self.steps = int(rows), int(cols), int(batch), dtype, int(steps)
        per_step = [tuple(c) for c in coefficients] if len(coefficients) and hasattr(coefficients[0], "__len__") else [tuple(coefficients)] * max(self.steps, 0)
        if len(per_step) != max(self.steps, 0) or any(len(c) != 3 for c in per_step):
            raise ValueError(f"coefficients are three numbers, or three for each of the {steps} steps")
        self._coefficients = (C.c_float * max(1, 3 * len(per_step)))(*[float(v) for c in per_step for v in c])
        self._config = OrthoConfig(_choice("dtype", dtype, DTYPES), self.rows, self.cols, self.batch, self.steps, float(eps), float(scale))
        self._at = C.byref(self._config)

    def workspace_bytes(self) -> int:
        hip.init()
        out = C.c_size_t()
        check(lib().rl_ortho_workspace_bytes(self._at, C.byref(out)))
        return out.value

    PRODUCTS = ("X X^T", "A A", "B X")

    def tiles(self, compute_units: int = 256) -> dict:
        """{product: (tile rows, tile columns, splits, tiles not split)} of one step (host arithmetic, no device)."""
        out = (ProductTile * 3)()
        check(lib().rl_ortho_tiles(self._at, compute_units, out))
        return {name: (t.rows, t.cols, t.splits, t.whole) for name, t in zip(self.PRODUCTS, out)}

    def launch(self, G, O, *, ldg: Optional[int] = None, ldo: Optional[int] = None, stride_g: Optional[int] = None,
               stride_o: Optional[int] = None, stream=None, workspace=None, workspace_bytes: Optional[int] = None) -> None:
        """Enqueues ``O = orthogonalised G`` (``O`` may be ``G``)."""
        hip.init()
        ldg, ldo = self.cols if ldg is None else ldg, self.cols if ldo is None else ldo
        check(lib().rl_orthogonalize(
            self._at, self._coefficients, _address(G), ldg, self.rows * ldg if stride_g is None else stride_g,
            _address(O), ldo, self.rows * ldo if stride_o is None else stride_o, *_room(workspace, workspace_bytes), _stream_handle(stream)))
