"""The operators between a backward pass and the quantisers, as cases to measure: the global gradient norm over many
tensors, clipping by it, and the AdamW update that applies the clip and writes the low-precision weights.

The tensors of a case are views into flat buffers, as a trainer's gradient and parameter buffers hold them, so the plain
forms work on whole buffers.  Matrices come first in a buffer and take weight decay, vectors follow and take none.
"""

import itertools
import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
_BETAS, _EPS, _LR, _DECAY = (0.9, 0.95), 1e-8, 3e-4, 0.1
_CHUNK = 1 << 26


def _shapes(case):
    """-> (matrices, vectors) of the case's layout, as lists of shapes."""
    h, f, n = case["hidden"], case["ffn"], case["count"]
    if case["layout"] == "layer":          # dense transformer layers: attention and MLP projections, norm vectors
        layer = [(case["q"], h), (case["kv"], h), (case["kv"], h), (h, case["q"]), (f, h), (f, h), (h, f)]
        return layer * n, [(h,), (h,), (128,), (128,)] * n
    if case["layout"] == "experts":        # gate, up and down of n experts, all of one size
        return [(f, h), (f, h), (h, f)] * n, []
    if case["layout"] == "router":         # what stays unquantised in a mixture layer: router, its bias, norm vectors
        return [(f, h)] * n, [(f,), (h,), (h,)] * n
    return [(f, h), (7, 2 * h + 1), (4 * f + 1, 129)] * n, [(h + 3,), (1,)] * n      # "ragged": odd sizes


def _offsets(case):
    """-> (shapes, offsets, decayed, total): where each tensor starts in a flat buffer whose tensors start at multiples of
    ``align`` elements; the first ``decayed`` elements of the buffer are the matrices."""
    matrices, vectors = _shapes(case)
    room = [-(-math.prod(s) // case["align"]) * case["align"] for s in matrices + vectors]
    offs = list(itertools.accumulate(room, initial=0))
    return matrices + vectors, offs[:-1], offs[len(matrices)], offs[-1]


def _numel(case):
    return sum(math.prod(s) for part in _shapes(case) for s in part)


def _case(name, op, layout, hidden, ffn, count, grad, align=64, q=0, kv=0, **more):
    return {"name": name, "op": op, "layout": layout, "hidden": hidden, "ffn": ffn, "count": count, "q": q, "kv": kv,
            "grad": grad, "align": align, **more}


def listed():
    dense = {"q": 4096, "kv": 1024}
    return [
        # a mixture layer's router and norm vectors: the per-step check that costs only latency
        _case("norm router fp32 inf", "norm", "router", 2048, 128, 1, "fp32", norm="inf"),
        # one dense layer's bf16 gradients
        _case("norm layer bf16", "norm", "layer", 2560, 9728, 1, "bf16", norm="2", **dense),
        # one mixture layer's experts with the norm of every tensor, as a trainer logs them
        _case("norm experts bf16 each", "norm", "experts", 2048, 768, 128, "bf16", norm="2", each=True),
        # the fp32 main gradients of a whole 36-layer dense model
        _case("norm dense model fp32", "norm", "layer", 2560, 9728, 36, "fp32", norm="2", **dense),
        # the same small list clipped through the parameters
        _case("clip router fp32", "clip", "router", 2048, 128, 1, "fp32", out="", norm="2"),
        # one dense layer, in place
        _case("clip layer bf16", "clip", "layer", 2560, 9728, 1, "bf16", out="", norm="2", **dense),
        # odd matrices packed back to back, scaled gradients cast into fp32 main gradients while they are clipped
        _case("clip ragged bf16 to fp32", "clip", "ragged", 3000, 4100, 6, "bf16", align=1, out="fp32", norm="2"),
        # a mixture layer's fp32 main gradients, in place
        _case("clip experts fp32", "clip", "experts", 2048, 768, 128, "fp32", out="", norm="2"),
        # router and norm vectors: latency
        _case("adamw router fp32", "adamw", "router", 2048, 128, 1, "fp32", weight="", clip=False),
        # odd matrices packed back to back, fp16 gradients under a loss scale
        _case("adamw ragged fp16", "adamw", "ragged", 1001, 1367, 2, "fp16", align=1, weight="fp16", clip=True),
        # a mixture layer's experts with fp32 main gradients
        _case("adamw experts fp32", "adamw", "experts", 2048, 768, 128, "fp32", weight="bf16", clip=True),
        # eight dense layers with bf16 gradients
        _case("adamw layers bf16", "adamw", "layer", 2560, 9728, 8, "bf16", weight="bf16", clip=True, **dense),
    ]


def _between(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "clip", "adamw"])
    layout = rng.choice(["layer", "experts", "router", "ragged"])
    hidden = _between(rng, 256, 5120) if rng.random() < 0.5 else 64 * _between(rng, 4, 80)
    ffn = _between(rng, 64, 512) if layout == "router" else _between(rng, 256, 9728)
    grad = rng.choice(["bf16", "fp16", "fp32"])
    case = {"op": op, "layout": layout, "hidden": hidden, "ffn": ffn, "count": 1, "q": 128 * rng.randint(1, 40),
            "kv": 128 * rng.randint(1, 8), "grad": grad, "align": rng.choice([1, 1, 8, 64])}
    if op == "norm":
        case.update(norm=rng.choice(["2", "2", "inf"]))
        if layout == "experts" and rng.random() < 0.5:
            case["each"] = True
    elif op == "clip":
        case.update(norm=rng.choice(["2", "2", "inf"]), out=rng.choice(["", "", "fp32", grad]))
    else:
        case.update(weight=rng.choice(["", "bf16", "fp16"]), clip=rng.random() < 0.7)
    most = {"norm": 2_000_000_000, "clip": 600_000_000, "adamw": 600_000_000}[op]
    fits = max(1, most // _numel(case))
    case["count"] = min({"layer": 36, "experts": 128, "router": 48, "ragged": 24}[layout], _between(rng, 1, fits + 0.4))
    return case


def _views(case, flat):
    shapes, offs, _, _ = _offsets(case)
    return [flat[o:o + math.prod(s)].view(s) for s, o in zip(shapes, offs)]


def _norm_type(case):
    return math.inf if case.get("norm") == "inf" else 2.0


def _normals(n, dtype, scale, gen, pad):
    """n normal values of the scale in a buffer, zeros where the mask ``pad`` marks the space between tensors."""
    x = torch.randn(n, generator=gen, device="cuda", dtype=dtype).mul_(scale)
    return x if pad is None else x.masked_fill_(pad, 0)


def _padding(case, total):
    shapes, offs, _, _ = _offsets(case)
    if total == _numel(case):
        return None
    lengths = [(math.prod(s), end - o - math.prod(s)) for s, o, end in zip(shapes, offs, offs[1:] + [total])]
    lengths = torch.tensor(lengths, device="cuda").flatten()
    return torch.tensor([False, True], device="cuda").repeat(len(shapes)).repeat_interleave(lengths, output_size=total)


def prepare(case, seed):
    """The buffers, the tensors in them and, for the framework's form, the plan that a trainer builds once."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    _, _, decayed, total = _offsets(case)
    pad = _padding(case, total)
    # gradients whose norm is about 4 before any clip to 1; those of an update and of a cast are sums over tokens
    scaled = case["op"] == "adamw" or bool(case.get("out"))
    tokens = 64.0 if scaled else 1.0
    dtype = _DTYPES[case["grad"]]
    flat = _normals(total, dtype, 4.0 * tokens / math.sqrt(total), gen, pad)
    state = {"case": case, "flat": flat, "scale": 1.0 / tokens, "max_norm": 1.0, "decayed": decayed}
    grads = state["grads"] = _views(case, flat)
    if case["op"] == "norm":
        if own and case["layout"] != "router":
            import slime_amd

            state["plan"] = slime_amd.GradNormPlan(grads, _norm_type(case), per_tensor=bool(case.get("each")))
    elif case["op"] == "clip":
        if case["norm"] == "inf":
            state["max_norm"] = 1.0 / math.sqrt(total)
        if case["out"]:
            state["out"] = torch.zeros(total, dtype=_DTYPES[case["out"]], device="cuda")
        if case["layout"] == "router":
            state["params"] = [torch.nn.Parameter(torch.zeros_like(g)) for g in grads]
            for p, g in zip(state["params"], grads):
                p.grad = g
        if own:
            import slime_amd

            outs = _views(case, state["out"]) if case["out"] else None
            if case["layout"] != "router" or outs:
                state["plan"] = slime_amd.GradClipPlan(grads, _norm_type(case), out=outs)
    else:
        state["step"] = 20
        state["param"] = _normals(total, torch.float32, 0.02, gen, pad)
        state["m"] = _normals(total, torch.float32, 1.0 / math.sqrt(total), gen, pad)
        state["v"] = _normals(total, torch.float32, 2.0 / math.sqrt(total), gen, pad).square_()
        if case["weight"]:
            state["weight"] = state["param"].to(_DTYPES[case["weight"]])
        if own:
            import slime_amd

            matrices = len(_shapes(case)[0])
            state["plan"] = slime_amd.AdamWPlan(
                _views(case, state["param"]), grads, weights=_views(case, state["weight"]) if case["weight"] else None,
                exp_avgs=_views(case, state["m"]), exp_avg_sqs=_views(case, state["v"]), betas=_BETAS, eps=_EPS,
                weight_decay=[_DECAY if i < matrices else 0.0 for i in range(len(grads))], step=state["step"])
    return state


def _plain_norm(case, flat, scale):
    if case.get("norm") == "inf":
        return flat.float().abs().amax() * scale
    return (flat.float().square().sum(dtype=torch.float64).sqrt() * scale).float()


def _plain_coefficient(norm, max_norm):
    return torch.clamp(max_norm / (norm + 1e-6), max=1.0)


def run(state):
    case = state["case"]
    return {"norm": _run_norm, "clip": _run_clip, "adamw": _run_adamw}[case["op"]](state, case)


def _run_norm(state, case):
    if own:
        if "plan" in state:
            return state["plan"].run()
        import slime_amd

        return slime_amd.get_total_norm(state["grads"], _norm_type(case))
    total = _plain_norm(case, state["flat"], 1.0)
    if not case.get("each"):
        return total
    x = state["flat"].view(3 * case["count"], -1).float()
    return total, x.abs().amax(1) if case["norm"] == "inf" else x.square().sum(1, dtype=torch.float64).sqrt().float()


def _run_clip(state, case):
    max_norm, scale = state["max_norm"], state["scale"]
    if not case["out"]:
        state["max_norm"] *= 0.999      # gradients clipped in place are clipped further by the next pass, never left alone
    if own:
        if "plan" in state:
            norm = state["plan"].run(max_norm, grad_scale=scale)
        else:
            import slime_amd

            norm = slime_amd.clip_grad_norm_(state["params"], max_norm, _norm_type(case))
    else:
        norm = _plain_norm(case, state["flat"], scale)
        scaled = state["flat"].float() * (_plain_coefficient(norm, max_norm) * scale)
        (state["out"] if case["out"] else state["flat"]).copy_(scaled)
    return norm, state["out"] if case["out"] else state["flat"]


def _run_adamw(state, case):
    max_norm = state["max_norm"] if case["clip"] else None
    state["step"] += 1
    if own:
        norm = state["plan"].run(_LR, max_norm=max_norm, grad_scale=state["scale"])
    else:
        norm = None
        grad = state["flat"].float() * state["scale"]
        if case["clip"]:
            norm = _plain_norm(case, state["flat"], state["scale"])
            grad = grad * _plain_coefficient(norm, max_norm)
        param, m, v, t = state["param"], state["m"], state["v"], state["step"]
        m.mul_(_BETAS[0]).add_(grad * (1 - _BETAS[0]))
        v.mul_(_BETAS[1]).add_(grad.square() * (1 - _BETAS[1]))
        param[:state["decayed"]].mul_(1 - _LR * _DECAY)
        denom = v.sqrt() / math.sqrt(1 - _BETAS[1] ** t) + _EPS
        param.sub_(m / denom * (_LR / (1 - _BETAS[0] ** t)))
        if case["weight"]:
            state["weight"].copy_(param)
    out = {"param": state["param"], "m": state["m"], "v": state["v"]}
    if case["weight"]:
        out["weight"] = state["weight"]
    if case["clip"]:
        out["norm"] = norm
    return out


def work(case):
    n, e = _numel(case), _BYTES[case["grad"]]
    if case["op"] == "norm":
        return {"bytes": n * e + 4, "flops": 2 * n}
    if case["op"] == "clip":
        return {"bytes": n * (e + (_BYTES[case["out"]] if case["out"] else e)) + 4, "flops": 3 * n}
    return {"bytes": n * (e + 24 + (_BYTES[case["weight"]] if case["weight"] else 0)), "flops": (18 if case["clip"] else 16) * n}


def exact(case, seed):
    """The definitions in 64 bits, a piece of the buffer at a time."""
    state = prepare(case, seed)
    flat = state["flat"]
    pieces = [slice(i, min(i + _CHUNK, flat.numel())) for i in range(0, flat.numel(), _CHUNK)]
    inf = case.get("norm") == "inf"
    total = 0.0
    for s in pieces:
        x = flat[s].double()
        total = max(total, x.abs().max().item()) if inf else total + torch.dot(x, x).item()
    norm = (total if inf else math.sqrt(total)) * state["scale"]
    told = torch.tensor(norm, dtype=torch.float64)
    if case["op"] == "norm":
        if not case.get("each"):
            return told
        each = [g.double().abs().max() if inf else torch.linalg.vector_norm(g.double()) for g in state["grads"]]
        return told, torch.stack(each)
    c = state["scale"]
    if case["op"] == "clip" or case["clip"]:
        c *= min(1.0, state["max_norm"] / (norm + 1e-6))
    if case["op"] == "clip":
        y = torch.empty(flat.numel(), dtype=torch.float64, device="cuda")
        for s in pieces:
            y[s] = flat[s].double() * c
        return told, y
    t, (b1, b2) = state["step"] + 1, _BETAS
    out = {k: torch.empty(flat.numel(), dtype=torch.float64, device="cuda") for k in ("param", "m", "v")}
    where = torch.arange(_CHUNK, device="cuda")
    for s in pieces:
        g = flat[s].double() * c
        m = b1 * state["m"][s].double() + (1 - b1) * g
        v = b2 * state["v"][s].double() + (1 - b2) * g * g
        decay = torch.where(where[:g.numel()] + s.start < state["decayed"], _DECAY, 0.0).double()
        p = state["param"][s].double() * (1 - _LR * decay)
        out["m"][s], out["v"][s] = m, v
        out["param"][s] = p - _LR * (m / (1 - b1 ** t)) / (torch.sqrt(v / (1 - b2 ** t)) + _EPS)
    if case["weight"]:
        out["weight"] = out["param"]
    if case["clip"]:
        out["norm"] = told
    return out
