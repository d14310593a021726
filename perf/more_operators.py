"""The products of a layer's experts beside the MXFP8 x MXFP4 layer, as a model's program calls them: experts in 16 bits over rows
that are grouped by expert, with their gradients (experts that are trained or not quantised), and products in 8-bit floating point with
a scale for each 128 values of a token and each block of 128 x 128 weights, dense or grouped, with the quantiser in front.

Sizes are those of the layer that this package serves (hidden 5120, intermediate 2304, 384 experts on 8 ranks, top-6, up to 3840 tokens a
call), and for drawn cases others in the operators' ranges.
"""

import math
import random

import torch

own = False                     # False: elementary torch operations; True: the package's operators

HIDDEN, INTER = 5120, 2304
LOCAL_EXPERTS = 48              # 384 on 8 ranks
MAX_ROWS = 3840 * 6             # what 8 ranks' tokens leave on one of them on average
MAX_TOKENS = 3840
CLAMP = 10.0
MOST = MAX_ROWS * HIDDEN * INTER
MOST_WEIGHTS = LOCAL_EXPERTS * HIDDEN * INTER


# experts: weights there are; used: experts with rows; rows: those of all experts together; spare: rows behind the last expert's
def _experts(name, rows, experts, used, hidden=HIDDEN, inter=INTER, dtype="bf16", clamp=CLAMP, train=False, spare=0):
    return {"name": name, "kind": "experts", "rows": rows, "experts": experts, "used": used, "spare": spare, "hidden": hidden,
            "inter": inter, "dtype": dtype, "clamp": clamp, "train": train}


def _grouped(name, rows, experts, used, width, channels, dtype="bf16", train=False, spare=0):
    return {"name": name, "kind": "grouped", "rows": rows, "experts": experts, "used": used, "spare": spare, "width": width,
            "channels": channels, "dtype": dtype, "train": train}


def _quantize(name, tokens, width, dtype="bf16"):
    return {"name": name, "kind": "quantize", "rows": tokens, "width": width, "dtype": dtype}


# experts = 0: one weight for all rows
def _project(name, rows, width, channels, dtype="bf16", experts=0, used=0, spare=0):
    return {"name": name, "kind": "fp8-project", "rows": rows, "experts": experts, "used": used, "spare": spare, "width": width,
            "channels": channels, "dtype": dtype}


def _gated(name, rows, hidden=HIDDEN, inter=INTER, dtype="bf16", clamp=CLAMP, experts=0, used=0, spare=0):
    return {"name": name, "kind": "fp8-gated", "rows": rows, "experts": experts, "used": used, "spare": spare, "hidden": hidden,
            "inter": inter, "dtype": dtype, "clamp": clamp}


def listed():
    return [
        # one sequence being generated: the six experts of its token, the weights' bytes
        _experts("experts-decode-6", 6, LOCAL_EXPERTS, 6),
        # a full prefill step of eight ranks on one of them, a few experts without rows
        _experts("experts-prefill-23040", MAX_ROWS, LOCAL_EXPERTS, 46),
        # a training step of 640 tokens with eight experts: outputs and all gradients
        _experts("experts-train-3840", 3840, 8, 7, train=True),
        # small experts, a handful of rows: latency
        _grouped("grouped-7-fp16", 7, 16, 5, 1024, 688, dtype="fp16"),
        # a training step of small experts, ragged, with rows behind the last expert's
        _grouped("grouped-train-1021", 1021, 24, 19, 1024, 688, train=True, spare=27),
        # activations of a decode step, hidden width
        _quantize("fp8-quantize-7", 7, HIDDEN),
        # activations of a full prefill step, between a block's two products
        _quantize("fp8-quantize-3840", 3840, INTER, dtype="fp16"),
        # second product of a shared expert: one sequence, then a full prefill step
        _project("fp8-project-1", 1, INTER, HIDDEN),
        _project("fp8-project-3840", 3840, INTER, HIDDEN),
        # a projection of no round size, FP32 result
        _project("fp8-project-777-fp32", 777, HIDDEN, 5003, dtype="fp32"),
        # first products of a decode batch's experts (64 tokens), most of them with a few rows
        _gated("fp8-gated-experts-384", 384, experts=LOCAL_EXPERTS, used=41, spare=16),
        # first products of a shared expert, a full prefill step
        _gated("fp8-gated-3840", 3840),
    ]


def _spread(rng, low, high, step=1):
    return max(low, min(high, int(math.exp(rng.uniform(math.log(low), math.log(high + 1))) // step * step)))


def draw(rng):
    kind = rng.choice(("experts", "experts-train", "grouped", "grouped-train", "quantize", "fp8-project", "fp8-gated"))
    hidden = HIDDEN if rng.random() < 0.3 else _spread(rng, 256, 8192, 16)
    inter = INTER if rng.random() < 0.3 else _spread(rng, 128, 8192, 16)
    if kind == "quantize":
        case = _quantize("", _spread(rng, 1, MAX_TOKENS), rng.choice((hidden, inter)), rng.choice(("bf16", "fp16")))
    else:
        most, most_weights = MOST, MOST_WEIGHTS
        if kind.endswith("train"):
            most, most_weights = MOST // 3, MOST_WEIGHTS // 3
        experts = max(1, min(_spread(rng, 1, 128), most_weights // (hidden * inter)))
        rows = max(1, min(_spread(rng, 1, MAX_ROWS), most // (hidden * inter)))
        if kind.startswith("fp8") and rng.random() < 0.5:
            experts, rows = 0, min(rows, MAX_TOKENS)
        used = min(rows, rng.randint((experts + 1) // 2, experts))
        spare = rng.choice((0, 0, rng.randint(1, 200))) if experts else 0
        dtype = rng.choice(("bf16", "bf16", "fp16"))
        wide = dtype if rng.random() < 0.7 else "fp32"
        clamp = rng.choice((0.0, CLAMP, 2.5))
        if kind.startswith("experts"):
            case = _experts("", rows, experts, used, hidden, inter, dtype, clamp, kind.endswith("train"), spare)
        elif kind.startswith("grouped"):
            case = _grouped("", rows, experts, used, *rng.choice(((hidden, inter), (inter, hidden))), dtype, kind.endswith("train"), spare)
        elif kind == "fp8-project":
            sizes = rng.choice(((hidden, inter), (inter, hidden), (hidden, inter - rng.randint(1, 15))))
            case = _project("", rows, *sizes, wide, experts, used, spare)
        else:
            case = _gated("", rows, hidden, inter, wide, clamp, experts, used, spare)
    del case["name"]
    return case


_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_BLOCK = 128


def _counts(case, seed):
    """Rows of each expert: some have none, the others unequal shares."""
    rng = random.Random(seed)
    chosen = rng.sample(range(case["experts"]), case["used"])
    share = [math.exp(rng.gauss(0, 0.7)) for _ in chosen]
    left = case["rows"] - len(chosen)
    counts = [0] * case["experts"]
    for e, s in zip(chosen, share):
        counts[e] = 1 + int(left * s / sum(share))
    for i in range(case["rows"] - sum(counts)):
        counts[chosen[i % len(chosen)]] += 1
    return counts


def prepare(case, seed):
    device = torch.device("cuda", torch.cuda.current_device())
    gen = torch.Generator(device=device).manual_seed(seed)
    kind, dtype = case["kind"], _TYPES[case["dtype"]]

    def normal(*shape, std=1.0):
        return torch.randn(shape, generator=gen, device=device) * std

    def matrices(count, rows, cols):
        out = torch.empty((count, rows, cols), dtype=dtype, device=device)
        for e in range(count):
            out[e] = normal(rows, cols, std=0.02)
        return out

    def in_groups(t):
        """E4M3 rows and a scale for each 128 values."""
        rows, cols = t.shape
        groups = torch.nn.functional.pad(t, (0, -cols % _BLOCK)).view(rows, -1, _BLOCK)
        scale = groups.abs().amax(dim=2) / 448
        q = (groups / scale[:, :, None]).to(torch.float8_e4m3fn)
        return q.view(rows, -1)[:, :cols].contiguous(), scale

    def in_blocks(count, parts, rows, cols):
        """E4M3 weights of `parts` matrices each, one below the other, and a scale for each block of 128 x 128 of those."""
        q = torch.empty((count, parts * rows, cols), dtype=torch.float8_e4m3fn, device=device)
        down, along = -(-rows // _BLOCK), -(-cols // _BLOCK)
        scales = torch.empty((count, parts * down, along), device=device)
        for e in range(count):
            for i in range(parts):
                t = torch.nn.functional.pad(normal(rows, cols, std=0.02), (0, along * _BLOCK - cols, 0, down * _BLOCK - rows))
                t = t.view(down, _BLOCK, along, _BLOCK)
                s = t.abs().amax(dim=(1, 3)) / 448
                scales[e, i * down:(i + 1) * down] = s
                q[e, i * rows:(i + 1) * rows] = (t / s[:, None, :, None]).view(down * _BLOCK, -1)[:rows, :cols].to(torch.float8_e4m3fn)
        return q, scales

    state = {"kind": kind, "dtype": dtype, "clamp": case.get("clamp") or None, "train": case.get("train", False), "ends": None}
    rows = case["rows"] + case.get("spare", 0)
    if case.get("experts"):
        state["counts"] = _counts(case, seed)
        state["ends"] = torch.tensor(state["counts"]).cumsum(0).to(torch.int32).to(device)
    if kind == "experts":
        hidden, inter, count = case["hidden"], case["inter"], case["experts"]
        state["x"] = normal(rows, hidden).to(dtype)
        state["w13"], state["w2"] = matrices(count, 2 * inter, hidden), matrices(count, hidden, inter)
        if case["train"]:
            state["dy"] = normal(rows, hidden).to(dtype)
            for name in ("x", "w13", "w2"):
                state[name].requires_grad_(True)
    elif kind == "grouped":
        state["x"] = normal(rows, case["width"]).to(dtype)
        state["w"] = matrices(case["experts"], case["channels"], case["width"])
        if case["train"]:
            state["dy"] = normal(rows, case["channels"]).to(dtype)
            for name in ("x", "w"):
                state[name].requires_grad_(True)
    elif kind == "quantize":
        # a few channels are far larger than the others, as in hidden states
        wide = torch.where(torch.rand(case["width"], generator=gen, device=device) < 0.005, 20.0, 1.0)
        state["x"] = (normal(rows, case["width"]) * wide).to(dtype)
    else:
        gated = kind == "fp8-gated"
        width = case["hidden"] if gated else case["width"]
        state["x"], state["sx"] = in_groups(normal(rows, width))
        state["w"], state["sw"] = in_blocks(case["experts"] or 1, 2 if gated else 1, case["inter"] if gated else case["channels"], width)
        if not case["experts"]:
            state["w"], state["sw"] = state["w"][0], state["sw"][0]
    return state


def _activation(g, u, clamp):
    """silu(min(g, c)) * clip(u, -c, c)."""
    if clamp is not None:
        g, u = g.clamp(max=clamp), u.clamp(-clamp, clamp)
    return g * torch.sigmoid(g) * u


def _pieces(counts):
    """(expert, first row, row behind the last) of the experts that have rows."""
    at = 0
    for e, n in enumerate(counts):
        if n:
            yield e, at, at + n
        at += n


def _plain_experts(state):
    x, w13, w2, dtype, clamp = state["x"].detach(), state["w13"].detach(), state["w2"].detach(), state["dtype"], state["clamp"]
    out = {"y": torch.zeros_like(x)}
    if state["train"]:
        dy = state["dy"]
        out.update(dx=torch.zeros_like(x), dw13=torch.zeros_like(w13), dw2=torch.zeros_like(w2))
    for e, a, b in _pieces(state["counts"]):
        xe, first, second = x[a:b].float(), w13[e].float(), w2[e].float()
        g, u = (xe @ first.T).chunk(2, dim=1)
        h = _activation(g, u, clamp)
        out["y"][a:b] = (h @ second.T).to(dtype)
        if not state["train"]:
            continue
        de = dy[a:b].float()
        gc, uc = (g, u) if clamp is None else (g.clamp(max=clamp), u.clamp(-clamp, clamp))
        s = torch.sigmoid(gc)
        dh = de @ second
        dg = dh * uc * (s * (1 + gc * (1 - s)))
        du = dh * (gc * s)
        if clamp is not None:
            dg = dg * (g <= clamp)
            du = du * (u.abs() <= clamp)
        d13 = torch.cat((dg, du), dim=1)
        out["dx"][a:b] = (d13 @ first).to(dtype)
        out["dw13"][e] = (d13.T @ xe).to(dtype)
        out["dw2"][e] = (de.T @ h).to(dtype)
    return out


def _plain_grouped(state):
    x, w, dtype = state["x"].detach(), state["w"].detach(), state["dtype"]
    out = {"y": torch.zeros((x.shape[0], w.shape[1]), dtype=dtype, device=x.device)}
    if state["train"]:
        out.update(dx=torch.zeros_like(x), dw=torch.zeros_like(w))
    for e, a, b in _pieces(state["counts"]):
        xe, we = x[a:b].float(), w[e].float()
        out["y"][a:b] = (xe @ we.T).to(dtype)
        if state["train"]:
            de = state["dy"][a:b].float()
            out["dx"][a:b] = (de @ we).to(dtype)
            out["dw"][e] = (de.T @ xe).to(dtype)
    return out


def _plain_quantize(state):
    x = state["x"].float()
    rows, cols = x.shape
    groups = torch.nn.functional.pad(x, (0, -cols % _BLOCK)).view(rows, -1, _BLOCK)
    amax = groups.abs().amax(dim=2)
    scale = torch.where(amax > 0, (amax.double() / 448).float(), torch.ones_like(amax))
    # a quotient next to the border between two values of 8 bits needs more than 32 bits: steps of 2^-3 of its binade, 2^-9 at least
    r = groups.double() / scale[:, :, None]
    step = torch.exp2(torch.floor(torch.log2(r.abs().clamp(min=2.0 ** -6))) - 3)
    q = (torch.round(r / step) * step).clamp(-448, 448).float()
    return {"values": (q * scale[:, :, None]).view(rows, -1)[:, :cols].contiguous(), "scales": scale}


def _spread_scales(scales, rows, cols, parts=1):
    """A scale for each value: of groups of 128 columns, and (`parts` > 0) of 128 rows of each part."""
    s = scales.repeat_interleave(_BLOCK, dim=1)[:, :cols]
    if parts:
        s = torch.cat([p.repeat_interleave(_BLOCK, dim=0)[:rows // parts] for p in s.chunk(parts, dim=0)])
    return s


def _plain_fp8(state):
    gated = state["kind"] == "fp8-gated"
    w, sw = (state["w"], state["sw"]) if state["ends"] is not None else (state["w"][None], state["sw"][None])
    x = state["x"].float() * _spread_scales(state["sx"], 0, state["x"].shape[1], 0)
    counts = state["counts"] if state["ends"] is not None else [x.shape[0]]
    channels, cols = w.shape[1:]
    name = "h" if gated else "y"
    out = {name: torch.zeros((x.shape[0], channels // 2 if gated else channels), dtype=state["dtype"], device=x.device)}
    for e, a, b in _pieces(counts):
        y = x[a:b] @ (w[e].float() * _spread_scales(sw[e], channels, cols, 2 if gated else 1)).T
        out[name][a:b] = (_activation(*y.chunk(2, dim=1), state["clamp"]) if gated else y).to(state["dtype"])
    return out


def run(state):
    kind = state["kind"]
    if not own:
        return {"experts": _plain_experts, "grouped": _plain_grouped, "quantize": _plain_quantize}.get(kind, _plain_fp8)(state)
    from vllm_plugin_b200 import api
    if kind == "experts":
        y = api.grouped_feed_forward(state["x"], state["w13"], state["w2"], state["ends"], activation_clamp=state["clamp"])
        if not state["train"]:
            return {"y": y}
        dx, dw13, dw2 = torch.autograd.grad(y, (state["x"], state["w13"], state["w2"]), state["dy"])
        return {"y": y.detach(), "dx": dx, "dw13": dw13, "dw2": dw2}
    if kind == "grouped":
        y = api.grouped_projection(state["x"], state["w"], state["ends"])
        if not state["train"]:
            return {"y": y}
        dx, dw = torch.autograd.grad(y, (state["x"], state["w"]), state["dy"])
        return {"y": y.detach(), "dx": dx, "dw": dw}
    if kind == "quantize":
        q, scales = api.prepare_fp8_inputs(state["x"])
        rows, cols = q.shape
        if cols % _BLOCK == 0:
            return {"values": (q.view(rows, -1, _BLOCK).float() * scales[:, :, None]).view(rows, cols), "scales": scales}
        return {"values": q.float() * scales.repeat_interleave(_BLOCK, dim=1)[:, :cols], "scales": scales}
    if kind == "fp8-gated":
        return {"h": api.fp8_gated_projection(state["x"], state["sx"], state["w"], state["sw"], ends=state["ends"],
                                              activation_clamp=state["clamp"], out_dtype=state["dtype"])}
    return {"y": api.fp8_projection(state["x"], state["sx"], state["w"], state["sw"], ends=state["ends"], out_dtype=state["dtype"])}


def work(case):
    kind, m, spare = case["kind"], case["rows"], case.get("spare", 0)
    out = {"bf16": 2, "fp16": 2, "fp32": 4}[case["dtype"]]
    ends, used = 4 * case.get("experts", 0), case.get("used") or 1
    if kind in ("experts", "grouped"):
        if kind == "experts":
            width = channels = case["hidden"]
            weights = 3 * case["hidden"] * case["inter"]
        else:
            width, channels = case["width"], case["channels"]
            weights = width * channels
        # rows in; the output, zeros behind the last expert's rows among it; weights of experts with rows
        moved = 2 * (m * width + (m + spare) * channels + used * weights) + ends
        if not case["train"]:
            return {"bytes": moved, "flops": 2 * m * weights}
        # dy in, dx and the weights' gradients out, those of experts without rows too
        return {"bytes": moved + 2 * (m * channels + (m + spare) * width + case["experts"] * weights), "flops": 6 * m * weights}
    if kind == "quantize":
        # the values that the 8 bits stand for, in 32 bits
        return {"bytes": m * case["width"] * (2 + 4) + 4 * m * -(-case["width"] // _BLOCK), "flops": 0}
    gated = kind == "fp8-gated"
    k, n = (case["hidden"], 2 * case["inter"]) if gated else (case["width"], case["channels"])
    groups = -(-k // _BLOCK)
    blocks = groups * (2 * -(-case["inter"] // _BLOCK) if gated else -(-n // _BLOCK))
    return {"bytes": m * (k + 4 * groups) + used * (n * k + 4 * blocks) + out * (m + spare) * (n // 2 if gated else n) + ends,
            "flops": 2 * m * n * k}


def exact(case, seed):
    """The definitions in 64 bits, gradients by differentiation."""
    state = prepare(case, seed)
    kind = case["kind"]
    c = state["clamp"] if state["clamp"] is not None else math.inf

    def swiglu(both):
        first, second = both.tensor_split(2, dim=-1)
        first, second = first.clamp(max=c), second.clamp(min=-c, max=c)
        return first / (1 + torch.exp(-first)) * second

    if kind == "quantize":
        x = state["x"].double()
        values, scales = torch.empty_like(x), []
        codes = torch.arange(127, dtype=torch.uint8, device=x.device).view(torch.float8_e4m3fn).double()
        borders = (codes[1:] + codes[:-1]) / 2
        for at in range(0, case["width"], _BLOCK):
            piece = x[:, at:at + _BLOCK]
            # the scale is a number of 32 bits, and the values of 8 bits go by it as it is
            step = piece.abs().max(dim=1, keepdim=True).values.div(448).float().double()
            step[step == 0] = 1
            ratio = (piece / step).abs()
            # on a border the code whose last bit is 0
            low, high = torch.bucketize(ratio, borders), torch.bucketize(ratio, borders, right=True)
            code = torch.where(low % 2 == 0, low, high)
            values[:, at:at + _BLOCK] = codes[code] * piece.sign() * step
            scales.append(step)
        return {"values": values, "scales": torch.cat(scales, dim=1)}

    rows = case["rows"] + case["spare"]
    if kind.startswith("fp8"):
        def values(t, s, down):
            t = t.double().clone()
            for i in range(s.shape[0] if down else 1):
                for j in range(s.shape[1]):
                    cols = slice(j * _BLOCK, (j + 1) * _BLOCK)
                    if down:
                        per = s.shape[0] // parts
                        first = i // per * (t.shape[0] // parts) + i % per * _BLOCK
                        last = min(first + _BLOCK, (i // per + 1) * (t.shape[0] // parts))
                        t[first:last, cols] *= s[i, j].double()
                    else:
                        t[:, cols] *= s[:, j:j + 1].double()
            return t

        parts = 2 if kind == "fp8-gated" else 1
        grouped = state["ends"] is not None
        ends = state["ends"].tolist() if grouped else [rows]
        x = values(state["x"], state["sx"], False)
        name, channels = ("h", case["inter"]) if parts == 2 else ("y", case["channels"])
        result = torch.zeros((rows, channels), dtype=torch.float64, device=x.device)
        for e, end in enumerate(ends):
            first = ends[e - 1] if e else 0
            if end > first:
                w = values(state["w"][e] if grouped else state["w"], (state["sw"][e] if grouped else state["sw"]).cpu(), True)
                y = torch.matmul(x[first:end], w.t())
                result[first:end] = swiglu(y) if parts == 2 else y
        return {name: result}

    ends = state["ends"].tolist()
    names = ("w13", "w2") if kind == "experts" else ("w",)
    y = torch.zeros((rows, case["hidden"] if kind == "experts" else case["channels"]), dtype=torch.float64, device=state["x"].device)
    grads = {"d" + n: torch.zeros(state[n].shape, dtype=torch.float64, device=y.device) for n in names}
    grads["dx"] = torch.zeros(state["x"].shape, dtype=torch.float64, device=y.device)
    for e, end in enumerate(ends):
        first = ends[e - 1] if e else 0
        if end == first:
            continue
        leaves = [state["x"][first:end].detach().double()] + [state[n][e].detach().double() for n in names]
        for leaf in leaves:
            leaf.requires_grad_(case["train"])
        inner = torch.matmul(leaves[0], leaves[1].t())
        ye = torch.matmul(swiglu(inner), leaves[2].t()) if kind == "experts" else inner
        y[first:end] = ye.detach()
        if case["train"]:
            gx, *gw = torch.autograd.grad(ye, leaves, state["dy"][first:end].double())
            grads["dx"][first:end] = gx
            for n, g in zip(names, gw):
                grads["d" + n][e] = g
    return {"y": y, **grads} if case["train"] else {"y": y}
