"""The operators of a language model's feed-forward block, as a user's program calls them: what is
measured, in which sizes, and the same operators in plain torch.

Two operators.  ``ffn`` is the gated feed-forward block ``y = (act(x Wg^T) * (x Wu^T)) Wd^T``: its
forward pass for serving (``ffn``) and a training step, forward and backward (``ffn_train``).
``ortho`` orthogonalises an update of such a weight (or of a stack of them) by Newton-Schulz
products, the heart of the Muon optimiser: five steps of ``X <- a X + (b A + c A A) X``,
``A = X X^T``, from ``X = G / ||G||``.
"""

import math

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
STEPS, COEFFICIENTS, EPS = 5, (3.4445, -4.7750, 2.0315), 1e-7


def listed():
    return [
        # one token through a small block: latency
        dict(name="token small bf16", op="ffn", T=1, D=1024, F=4096, type="bf16", act="silu"),
        # one token through a wide block: how fast the weights stream
        dict(name="token bf16", op="ffn", T=1, D=4096, F=12288, type="bf16", act="silu"),
        # a batch of decoding requests
        dict(name="batch 24 fp16", op="ffn", T=24, D=4096, F=8192, type="fp16", act="gelu_tanh"),
        # a large decoding batch, or a short prompt, of a ragged length
        dict(name="batch 200 bf16", op="ffn", T=200, D=2880, F=7680, type="bf16", act="silu"),
        # a prompt
        dict(name="prompt 4096 bf16", op="ffn", T=4096, D=4096, F=12288, type="bf16", act="silu"),
        # nothing aligned, in 32 bits
        dict(name="odd fp32", op="ffn", T=333, D=1001, F=2731, type="fp32", act="gelu"),
        # training steps: a large block, one of ragged sizes in half precision, one in 32 bits
        dict(name="train 8192 bf16", op="ffn_train", T=8192, D=4096, F=12288, type="bf16", act="silu"),
        dict(name="train 1023 fp16", op="ffn_train", T=1023, D=1920, F=5000, type="fp16", act="gelu_tanh"),
        dict(name="train 2048 fp32", op="ffn_train", T=2048, D=2048, F=4096, type="fp32", act="silu"),
        # updates of a square projection, of a tall one, and of a stack of small odd ones
        dict(name="ortho 4096x4096 bf16", op="ortho", batch=1, rows=4096, cols=4096, type="bf16"),
        dict(name="ortho 12288x4096 bf16", op="ortho", batch=1, rows=12288, cols=4096, type="bf16"),
        dict(name="ortho 8x509x1023 fp32", op="ortho", batch=8, rows=509, cols=1023, type="fp32"),
    ]


def _spread(rng, low, high):
    """A size between the two, even over its logarithm; every second one a multiple of 64 where it can be."""
    v = round(math.exp(rng.uniform(math.log(low), math.log(high))))
    return max(64, v // 64 * 64) if v >= 64 and rng.random() < 0.5 else v


def draw(rng):
    op = rng.choice(["ffn", "ffn", "ffn_train", "ortho"])
    kind = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if op == "ortho":
        batch = rng.choice([1, 1, 2, 6])
        top = 4096 if batch == 1 and kind != "fp32" else 1500
        return dict(op=op, batch=batch, rows=_spread(rng, 64, top), cols=_spread(rng, 64, top), type=kind)
    top_t = (4096 if kind != "fp32" else 1024) if op == "ffn" else (4096 if kind != "fp32" else 1024)
    T = _spread(rng, 1 if op == "ffn" else 16, top_t)
    return dict(op=op, T=T, D=_spread(rng, 256, 4096), F=_spread(rng, 512, 12288 if kind != "fp32" else 4096), type=kind,
                act=rng.choice(["silu", "gelu", "gelu_tanh"]))


def _inputs(case, seed):
    """The inputs, from the seed alone, in the case's type."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    t = TYPES[case["type"]]

    def normal(*shape, scale=1.0):
        return torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32).mul_(scale).to(t)

    if case["op"] == "ortho":
        b, m, n = case["batch"], case["rows"], case["cols"]
        # a gradient: a few strong directions above noise
        r = max(1, min(m, n) // 16)
        low = torch.stack([torch.randn(m, r, generator=gen, device="cuda") @ torch.randn(r, n, generator=gen, device="cuda") for _ in range(b)])
        return {"G": (low.mul_(1e-3 / math.sqrt(r)) + torch.randn(b, m, n, generator=gen, device="cuda").mul_(1e-3)).to(t)}
    T, D, F = case["T"], case["D"], case["F"]
    made = {"x": normal(T, D), "w_gate": normal(F, D, scale=D ** -0.5), "w_up": normal(F, D, scale=D ** -0.5),
            "w_down": normal(D, F, scale=F ** -0.5)}
    if case["op"] == "ffn_train":
        made["dy"] = normal(T, D)
    return made


def prepare(case, seed):
    state = _inputs(case, seed)
    state["case"] = case
    if own:
        from mlir_roller_amd import hip, products
        hip.init(torch.cuda.current_device())

        def room(nbytes):
            return torch.empty(max(int(nbytes), 256), dtype=torch.uint8, device="cuda")

        if case["op"] == "ortho":
            op = products.Orthogonalizer(case["rows"], case["cols"], batch=case["batch"], dtype=case["type"], steps=STEPS,
                                         coefficients=COEFFICIENTS, eps=EPS)
            state["out"] = torch.empty_like(state["G"])
            state["workspace"] = room(op.workspace_bytes())
        else:
            op = products.GatedFfn(case["D"], case["F"], dtype=case["type"], activation=case["act"])
            state["y"] = torch.empty_like(state["x"])
            training = case["op"] == "ffn_train"
            state["workspace"] = room(op.workspace_bytes(case["T"], backward=training))
            if training:
                state["saved"] = room(op.saved_bytes(case["T"]))
                for name in ("x", "w_gate", "w_up", "w_down"):
                    state["d" + name] = torch.empty_like(state[name])
        state["op"] = op
    return state


def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(s):
    from mlir_roller_amd.hip import Ptr
    op, case = s["op"], s["case"]
    stream = torch.cuda.current_stream().cuda_stream
    at = {k: Ptr(v.data_ptr()) for k, v in s.items() if isinstance(v, torch.Tensor)}
    room = dict(workspace=at["workspace"], workspace_bytes=s["workspace"].numel(), stream=stream)
    if case["op"] == "ortho":
        op.launch(at["G"], at["out"], **room)
        return s["out"]
    T = case["T"]
    op.forward(at["x"], at["w_gate"], at["w_up"], at["w_down"], at["y"], T, saved=at.get("saved"), **room)
    if case["op"] == "ffn":
        return s["y"]
    op.backward(at["dy"], at["x"], at["w_gate"], at["w_up"], at["w_down"], at["saved"],
                at["dx"], at["dw_gate"], at["dw_up"], at["dw_down"], T, **room)
    return {k: s[k] for k in ("y", "dx", "dw_gate", "dw_up", "dw_down")}


# ---- the operators in plain torch, in 32 bits, rounded once at the end ------------------------------

_C0, _C1 = math.sqrt(2 / math.pi), 0.044715


def _act(kind, g):
    if kind == "silu":
        return g * torch.sigmoid(g)
    if kind == "gelu":
        return 0.5 * g * (1 + torch.erf(g * math.sqrt(0.5)))
    return 0.5 * g * (1 + torch.tanh(_C0 * (g + _C1 * g * g * g)))


def _act_slope(kind, g):
    if kind == "silu":
        s = torch.sigmoid(g)
        return s * (1 + g * (1 - s))
    if kind == "gelu":
        return 0.5 * (1 + torch.erf(g * math.sqrt(0.5))) + g * torch.exp(-0.5 * g * g) / math.sqrt(2 * math.pi)
    t = torch.tanh(_C0 * (g + _C1 * g * g * g))
    return 0.5 * (1 + t) + 0.5 * g * (1 - t * t) * _C0 * (1 + 3 * _C1 * g * g)


def _run_plain(s):
    case = s["case"]
    t = TYPES[case["type"]]
    if case["op"] == "ortho":
        X = s["G"].float()
        X = X / (torch.sqrt((X * X).sum(dim=(1, 2), keepdim=True)) + EPS)
        tall = case["rows"] > case["cols"]
        if tall:
            X = X.transpose(1, 2).contiguous()
        a, b, c = COEFFICIENTS
        for _ in range(STEPS):
            A = torch.bmm(X, X.transpose(1, 2).contiguous())
            X = a * X + torch.bmm(b * A + c * torch.bmm(A, A), X)
        if tall:
            X = X.transpose(1, 2)
        return X.to(t).contiguous()
    x, wg, wu, wd = (s[k].float() for k in ("x", "w_gate", "w_up", "w_down"))
    g, u = x @ wg.t(), x @ wu.t()
    a = _act(case["act"], g)
    h = a * u
    y = (h @ wd.t()).to(t)
    if case["op"] == "ffn":
        return y
    dy = s["dy"].float()
    dh = dy @ wd
    dg, du = dh * u * _act_slope(case["act"], g), dh * a
    return {"y": y, "dx": (dg @ wg + du @ wu).to(t), "dw_gate": (dg.t() @ x).to(t), "dw_up": (du.t() @ x).to(t),
            "dw_down": (dy.t() @ h).to(t)}


# ---- what one pass cannot do without ---------------------------------------------------------------

def work(case):
    size = 4 if case["type"] == "fp32" else 2
    if case["op"] == "ortho":
        s, l = sorted((case["rows"], case["cols"]))
        # per step: the Gram matrix and its square are symmetric (half the products), and the update
        flops = case["batch"] * STEPS * (s * s * l + s * s * s + 2.0 * s * s * l)
        return {"bytes": 2.0 * case["batch"] * s * l * size, "flops": flops}
    T, D, F = case["T"], case["D"], case["F"]
    if case["op"] == "ffn":
        return {"bytes": size * (2.0 * T * D + 3.0 * D * F), "flops": 6.0 * T * D * F}
    return {"bytes": size * (4.0 * T * D + 6.0 * D * F), "flops": 18.0 * T * D * F}


# ---- the definition in 64 bits ---------------------------------------------------------------------

def exact(case, seed):
    made = {k: v.double() for k, v in _inputs(case, seed).items()}
    if case["op"] == "ortho":
        out = []
        a, b, c = COEFFICIENTS
        for G in made["G"]:
            X = G / (G.norm() + EPS)
            wide = X.shape[0] <= X.shape[1]
            for _ in range(STEPS):
                # a X + b (X X^T) X + c (X X^T)^2 X, from the shorter side
                if wide:
                    A = X.mm(X.t())
                    AX = A.mm(X)
                    X = a * X + b * AX + c * A.mm(AX)
                else:
                    A = X.t().mm(X)
                    XA = X.mm(A)
                    X = a * X + b * XA + c * XA.mm(A)
            out.append(X)
        return torch.stack(out)
    from torch import special
    x, wg, wu, wd = made["x"], made["w_gate"], made["w_up"], made["w_down"]
    g, u = x.mm(wg.t()), x.mm(wu.t())
    if case["act"] == "silu":
        gate = special.expit(g)                        # act = g * gate
        slope = gate + g * gate * special.expit(-g)
    elif case["act"] == "gelu":
        gate = special.ndtr(g)
        slope = gate + g * torch.exp(-g.square() / 2) * (2 * math.pi) ** -0.5
    else:
        z = math.sqrt(8 / math.pi) * (g + 0.044715 * g ** 3)
        gate = special.expit(z)                        # (1 + tanh(z / 2)) / 2
        slope = gate + g * gate * special.expit(-z) * math.sqrt(8 / math.pi) * (1 + 0.134145 * g.square())
    h = g * gate * u
    y = h.mm(wd.t())
    if case["op"] == "ffn":
        return y
    dy = made["dy"]
    dh = dy.mm(wd)
    dw_down = dy.t().mm(h)
    dg, du = dh * u * slope, dh * (g * gate)
    return {"y": y, "dx": dg.mm(wg).add_(du.mm(wu)), "dw_gate": dg.t().mm(x), "dw_up": du.t().mm(x), "dw_down": dw_down}
