"""The dense feed-forward operators beside the MegaMoE layer, as a model's program calls them: the gated feed-forward block
in 16 bits with its gradients (a dense layer or a shared expert that is trained or not quantised), and the same block's
products in 8-bit integers (per-token activation scales, per-channel weight scales) with the quantiser in front.

Sizes are those of the layer that this package serves (hidden 5120, intermediate 2304, up to 3840 tokens a call), and for
drawn cases other multiples of 16.
"""

import math

import torch

own = False                     # False: elementary torch operations; True: the package's operators

HIDDEN, INTER = 5120, 2304
MAX_TOKENS = 3840
CLAMP = 10.0
MOST = MAX_TOKENS * HIDDEN * INTER


def _block(name, tokens, hidden=HIDDEN, inter=INTER, dtype="bf16", clamp=CLAMP, train=False):
    return {"name": name, "kind": "block", "tokens": tokens, "hidden": hidden, "inter": inter, "dtype": dtype, "clamp": clamp,
            "train": train}


def _quantize(name, tokens, width, dtype="bf16"):
    return {"name": name, "kind": "quantize", "tokens": tokens, "width": width, "dtype": dtype}


def _gated(name, tokens, hidden=HIDDEN, inter=INTER, dtype="bf16", clamp=CLAMP):
    return {"name": name, "kind": "int8-gated", "tokens": tokens, "hidden": hidden, "inter": inter, "dtype": dtype, "clamp": clamp}


def _project(name, tokens, width, channels, dtype="bf16", bias=False):
    return {"name": name, "kind": "int8-project", "tokens": tokens, "width": width, "channels": channels, "dtype": dtype, "bias": bias}


def listed():
    return [
        # one sequence being generated through an unquantised block: latency, and the weights' bytes
        _block("block-decode-1", 1),
        # a decode batch
        _block("block-batch-64", 64),
        # a mixed prefill and decode step of no round size
        _block("block-mixed-1021", 1021),
        # a training step of a shared expert: output and all gradients, a full batch
        _block("train-3840", 3840, train=True),
        # ... and of a small block in FP16, an odd number of tokens, no clamp
        _block("train-333-fp16", 333, 1024, 688, dtype="fp16", clamp=0.0, train=True),
        # activations of a decode step, hidden width
        _quantize("quantize-7", 7, HIDDEN),
        # activations of a full prefill step, between the block's two products
        _quantize("quantize-3840", 3840, INTER, dtype="fp16"),
        # first products of the 8-bit block: one sequence, a full prefill step
        _gated("int8-gated-1", 1),
        _gated("int8-gated-3840", 3840),
        # second product, a decode batch
        _project("int8-project-16", 16, INTER, HIDDEN),
        # a square projection with bias, FP32 result, no round size
        _project("int8-project-bias-777", 777, HIDDEN, HIDDEN, dtype="fp32", bias=True),
        # second product, a full prefill step
        _project("int8-project-3840", 3840, INTER, HIDDEN),
    ]


def _spread(rng, low, high, step=1):
    return max(low, min(high, int(math.exp(rng.uniform(math.log(low), math.log(high + 1))) // step * step)))


def draw(rng):
    kind = rng.choice(("block", "block", "train", "quantize", "int8-gated", "int8-project"))
    tokens = _spread(rng, 1, MAX_TOKENS)
    hidden = HIDDEN if rng.random() < 0.3 else _spread(rng, 256, 8192, 16)
    inter = INTER if rng.random() < 0.3 else _spread(rng, 128, 8192, 16)
    clamp = rng.choice((0.0, CLAMP, 2.5))
    tokens = max(1, min(tokens, MOST // (hidden * inter)))
    if kind == "quantize":
        case = _quantize("", tokens, rng.choice((hidden, inter)), rng.choice(("bf16", "fp16")))
    elif kind == "int8-gated":
        case = _gated("", tokens, hidden, inter, rng.choice(("bf16", "bf16", "fp16", "fp32")), clamp)
    elif kind == "int8-project":
        sizes = rng.choice(((hidden, inter), (inter, hidden), (hidden, hidden), (hidden, inter + rng.randint(1, 15))))
        tokens = max(1, min(tokens, MOST // (sizes[0] * sizes[1])))
        case = _project("", tokens, *sizes, dtype=rng.choice(("bf16", "bf16", "fp16", "fp32")), bias=rng.random() < 0.4)
    else:
        case = _block("", tokens, hidden, inter, rng.choice(("bf16", "bf16", "fp16")), clamp, kind == "train")
    del case["name"]
    return case


_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def prepare(case, seed):
    device = torch.device("cuda", torch.cuda.current_device())
    gen = torch.Generator(device=device).manual_seed(seed)

    def normal(*shape, std=1.0):
        return torch.randn(shape, generator=gen, device=device) * std

    def eight_bit(t):
        """Rows of whole numbers in [-127, 127] and a scale for each."""
        scale = t.abs().amax(dim=1) / 127
        return torch.round(t / scale[:, None]).to(torch.int8), scale

    state = {"kind": case["kind"], "dtype": _TYPES[case["dtype"]], "clamp": case.get("clamp") or None}
    tokens = case["tokens"]
    if case["kind"] == "block":
        hidden, inter = case["hidden"], case["inter"]
        state["x"] = normal(tokens, hidden).to(state["dtype"])
        state["w13"] = normal(2 * inter, hidden, std=0.02).to(state["dtype"])
        state["w2"] = normal(hidden, inter, std=0.02).to(state["dtype"])
        state["train"] = case["train"]
        if case["train"]:
            state["dy"] = normal(tokens, hidden).to(state["dtype"])
            for name in ("x", "w13", "w2"):
                state[name].requires_grad_(True)
    elif case["kind"] == "quantize":
        # a few channels are far larger than the others, as in hidden states
        wide = torch.where(torch.rand(case["width"], generator=gen, device=device) < 0.005, 20.0, 1.0)
        state["x"] = (normal(tokens, case["width"]) * wide).to(state["dtype"])
    elif case["kind"] == "int8-gated":
        state["x"], state["sx"] = eight_bit(normal(tokens, case["hidden"]))
        state["w"], state["sw"] = eight_bit(normal(2 * case["inter"], case["hidden"], std=0.02))
    else:
        state["x"], state["sx"] = eight_bit(normal(tokens, case["width"]))
        state["w"], state["sw"] = eight_bit(normal(case["channels"], case["width"], std=0.02))
        state["bias"] = normal(case["channels"], std=0.5) if case["bias"] else None
    return state


def _activation(g, u, clamp):
    """silu(min(g, c)) * clip(u, -c, c)."""
    if clamp is not None:
        g, u = g.clamp(max=clamp), u.clamp(-clamp, clamp)
    return g * torch.sigmoid(g) * u


def _plain_block(state):
    x, w13, w2 = (state[n].detach().float() for n in ("x", "w13", "w2"))
    clamp, dtype = state["clamp"], state["dtype"]
    g, u = (x @ w13.T).chunk(2, dim=1)
    h = _activation(g, u, clamp)
    out = {"y": (h @ w2.T).to(dtype)}
    if not state["train"]:
        return out
    dy = state["dy"].float()
    gc, uc = (g, u) if clamp is None else (g.clamp(max=clamp), u.clamp(-clamp, clamp))
    s = torch.sigmoid(gc)
    dh = dy @ w2
    dg = dh * uc * (s * (1 + gc * (1 - s)))
    du = dh * (gc * s)
    if clamp is not None:
        dg = dg * (g <= clamp)
        du = du * (u.abs() <= clamp)
    d13 = torch.cat((dg, du), dim=1)
    out["dx"] = (d13 @ w13).to(dtype)
    out["dw13"] = (d13.T @ x).to(dtype)
    out["dw2"] = (dy.T @ h).to(dtype)
    return out


def _plain_quantize(state):
    x = state["x"].float()
    amax = x.abs().amax(dim=1)
    scale = torch.where(amax > 0, (amax.double() / 127).float(), torch.ones_like(amax))
    # a quotient next to the border between two whole numbers needs more than 32 bits
    q = torch.round(x.double() / scale[:, None]).float()
    return {"values": q * scale[:, None], "scales": scale}


def _plain_gated(state):
    g, u = ((state["x"].float() @ state["w"].float().T) * state["sx"][:, None] * state["sw"]).chunk(2, dim=1)
    return {"h": _activation(g, u, state["clamp"]).to(state["dtype"])}


def _plain_project(state):
    y = (state["x"].float() @ state["w"].float().T) * state["sx"][:, None] * state["sw"]
    if state["bias"] is not None:
        y = y + state["bias"]
    return {"y": y.to(state["dtype"])}


def run(state):
    kind = state["kind"]
    if not own:
        return {"block": _plain_block, "quantize": _plain_quantize, "int8-gated": _plain_gated, "int8-project": _plain_project}[kind](state)
    from vllm_plugin_b200 import api
    if kind == "block":
        y = api.gated_feed_forward(state["x"], state["w13"], state["w2"], activation_clamp=state["clamp"])
        if not state["train"]:
            return {"y": y}
        dx, dw13, dw2 = torch.autograd.grad(y, (state["x"], state["w13"], state["w2"]), state["dy"])
        return {"y": y.detach(), "dx": dx, "dw13": dw13, "dw2": dw2}
    if kind == "quantize":
        q, scale = api.prepare_int8_inputs(state["x"])
        return {"values": q * scale[:, None], "scales": scale}
    if kind == "int8-gated":
        return {"h": api.int8_gated_projection(state["x"], state["sx"], state["w"], state["sw"], activation_clamp=state["clamp"],
                                               out_dtype=state["dtype"])}
    return {"y": api.int8_projection(state["x"], state["sx"], state["w"], state["sw"], bias=state["bias"], out_dtype=state["dtype"])}


def work(case):
    out = {"bf16": 2, "fp16": 2, "fp32": 4}[case["dtype"]]
    m = case["tokens"]
    if case["kind"] == "block":
        h, i = case["hidden"], case["inter"]
        if not case["train"]:
            return {"bytes": 2 * (2 * m * h + 3 * h * i), "flops": 6 * m * h * i}
        # x, weights and dy in; y, dx and the weights' gradients out
        return {"bytes": 2 * (4 * m * h + 6 * h * i), "flops": 18 * m * h * i}
    if case["kind"] == "quantize":
        # the values that the whole numbers stand for, in 32 bits
        return {"bytes": m * case["width"] * (2 + 4) + 4 * m, "flops": 0}
    if case["kind"] == "int8-gated":
        h, i = case["hidden"], case["inter"]
        return {"bytes": m * h + 2 * i * h + 4 * (m + 2 * i) + out * m * i, "flops": 4 * m * h * i}
    k, n = case["width"], case["channels"]
    return {"bytes": m * k + n * k + 4 * (m + n) + (4 * n if case["bias"] else 0) + out * m * n, "flops": 2 * m * k * n}


def exact(case, seed):
    """The definitions in 64 bits, gradients by differentiation."""
    state = prepare(case, seed)
    c = state["clamp"] if state["clamp"] is not None else math.inf
    if case["kind"] == "quantize":
        x = state["x"].double()
        # the scale is a number of 32 bits, and the whole numbers go by it as it is
        step = x.abs().max(dim=1).values.div(127).float().double()
        step[step == 0] = 1
        return {"values": torch.round(x / step.unsqueeze(1)).mul(step.unsqueeze(1)), "scales": step}

    def swiglu(first, second):
        first, second = first.clamp(max=c), second.clamp(min=-c, max=c)
        return first / (1 + torch.exp(-first)) * second

    if case["kind"] == "block":
        leaves = [state[n].detach().double().requires_grad_(case["train"]) for n in ("x", "w13", "w2")]
        x, w13, w2 = leaves
        i = case["inter"]
        y = torch.matmul(swiglu(torch.matmul(x, w13[:i].t()), torch.matmul(x, w13[i:].t())), w2.t())
        if not case["train"]:
            return {"y": y}
        grads = torch.autograd.grad(y, leaves, state["dy"].double())
        return {"y": y.detach(), **dict(zip(("dx", "dw13", "dw2"), grads))}
    x = state["x"].double() * state["sx"].double().unsqueeze(1)
    w = state["w"].double() * state["sw"].double().unsqueeze(1)
    if case["kind"] == "int8-gated":
        i = case["inter"]
        return {"h": swiglu(x.mm(w[:i].t()), x.mm(w[i:].t()))}
    y = x.mm(w.t())
    return {"y": y if state["bias"] is None else y + state["bias"].double()}
