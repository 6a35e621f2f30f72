"""The int8 linear operators of language models, as measurable cases.

Kinds of case:

* ``linear``  - activations (bf16, fp16, fp32, or int8 with their row scales)
  times int8 weights: rows quantized on the fly, then
  ``act((sum q w) * row scale * channel scale + bias) + residual``; gated layers
  multiply the activated half by the other one;
* ``experts`` - the same with one weight matrix per expert, over rows sorted by
  expert (groups of any size, empty ones among them), gathered from the tokens
  or taken as they are;
* ``route``   - the stable sort of the tokens' expert choices;
* ``combine`` - each token's weighted sum of its experts' rows;
* ``block``   - a feed-forward layer of experts from its tokens to its output:
  route, gated product, product back, combine.

``own`` chooses between the plain form in elementary torch operations (32 bits,
rounded once) and the calls of the library.
"""
from __future__ import annotations

import math

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32, "int8": torch.int8}
SIZES = {"bf16": 2, "fp16": 2, "fp32": 4, "int8": 1}
TINY = 2.0 ** -100  # rows whose largest magnitude is below it quantize to zeros

# The largest listed case (prompt_16384): no drawn one costs more.
MOST_FLOPS = 2 * 16384 * 8192 * 8192
MOST_BYTES = 600e6


def _linear(name, rows, inputs, outputs, x="bf16", y="bf16", act="none", gated=False, bias=False,
            residual=False):
    return {"name": name, "kind": "linear", "rows": rows, "inputs": inputs, "outputs": outputs,
            "x": x, "y": y, "act": act, "gated": gated, "bias": bias, "residual": residual}


def _experts(name, tokens, choices, experts, inputs, outputs, x="bf16", y="bf16", act="none",
             gated=False, bias=False, gather=True):
    return {"name": name, "kind": "experts", "tokens": tokens, "choices": choices,
            "experts": experts, "inputs": inputs, "outputs": outputs, "x": x, "y": y, "act": act,
            "gated": gated, "bias": bias, "gather": gather}


def _block(name, tokens, choices, experts, inputs, hidden, x="bf16", padding=0):
    return {"name": name, "kind": "block", "tokens": tokens, "choices": choices,
            "experts": experts, "inputs": inputs, "hidden": hidden, "x": x, "padding": padding}


def listed():
    return [
        # One new token through a projection with bias and residual: the
        # smallest linear call, where launches and the weights' bytes count.
        _linear("token_4096x4096", 1, 4096, 4096, bias=True, residual=True),
        # Sixteen sequences decoded together, the gated half of a feed-forward
        # layer: the weights' bytes are everything.
        _linear("batch16_gated", 16, 4096, 12288, act="silu", gated=True),
        # A short prompt through layers of no round size, fp16.
        _linear("prompt_777_odd", 777, 2000, 1003, x="fp16", y="fp16", act="gelu", bias=True),
        # A prompt whose rows another layer has quantized already, fp32 result
        # (scores, or the input of a norm).
        _linear("prompt_2048_int8", 2048, 4096, 4096, x="int8", y="fp32"),
        # The largest: a batch of prompts, throughput.
        _linear("prompt_16384", 16384, 8192, 8192, residual=True),
        # One token through a whole layer of experts: latency of the chain.
        _block("token_experts", 1, 8, 64, 2048, 1024),
        # A decode batch of which some sequences have ended (their choices are
        # dropped), odd sizes, fp16.
        _block("batch37_experts", 37, 4, 60, 1040, 720, x="fp16", padding=5),
        # A small batch through few experts, relu, biases, ragged groups.
        _experts("batch300_ragged", 300, 2, 10, 1008, 523, y="fp32", act="relu", bias=True),
        # A prompt's gated product, rows gathered from the tokens.
        _experts("prompt_experts_up", 4096, 8, 64, 2048, 1024, act="silu", gated=True),
        # ... and the product back, rows as they lie.
        _experts("prompt_experts_down", 4096, 8, 64, 1024, 2048, gather=False),
        # The choices of a batch of prompts sorted by expert.
        {"name": "route_16384", "kind": "route", "tokens": 16384, "choices": 8, "experts": 128},
        # The expert rows of a prompt summed back into its tokens.
        {"name": "combine_4096", "kind": "combine", "tokens": 4096, "choices": 8, "outputs": 2048,
         "x": "bf16", "y": "bf16", "residual": True},
    ]


# ---- drawn cases -------------------------------------------------------------

def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, unit, lo, hi):
    """A layer's width: mostly an odd multiple of 128, else of `unit`."""
    step = 128 if rng.random() < 0.6 else unit
    return step * (2 * int(_log(rng, lo, hi) / step / 2) + 1)


def _draw_once(rng):
    kind = rng.choice(("linear", "linear", "linear", "experts", "experts", "block", "route",
                       "combine"))
    floats = ("bf16", "bf16", "fp16", "fp32")
    x, y = rng.choice(floats), rng.choice(floats)
    act = rng.choice(("none", "relu", "gelu", "gelu_tanh", "silu"))
    gated = rng.random() < 0.35
    inputs, outputs = _width(rng, 16, 256, 8192), _width(rng, 1, 200, 12288)
    experts = _log(rng, 4, 128)
    choices = rng.randint(1, min(8, experts))
    if kind == "linear":
        case = _linear("", _log(rng, 1, 16384), inputs, outputs, rng.choice((x, x, "int8")), y, act,
                       gated, rng.random() < 0.5, rng.random() < 0.4)
    elif kind == "experts":
        case = _experts("", _log(rng, 1, 8192), choices, experts, _width(rng, 16, 256, 4096),
                        _width(rng, 1, 64, 4096), x, y, act, gated, rng.random() < 0.3,
                        rng.random() < 0.6)
    elif kind == "block":
        tokens = _log(rng, 1, 2048)
        case = _block("", tokens, choices, experts, _width(rng, 16, 256, 3000),
                      _width(rng, 16, 256, 2000), rng.choice(("bf16", "fp16")),
                      rng.choice((0, 0, tokens // 7)))
    elif kind == "route":
        case = {"kind": "route", "tokens": _log(rng, 1, 32768), "choices": choices,
                "experts": experts}
    else:
        case = {"kind": "combine", "tokens": _log(rng, 1, 8192), "choices": choices,
                "outputs": outputs, "x": x, "y": y, "residual": rng.random() < 0.5}
    case.pop("name", None)
    return case


def draw(rng):
    while True:
        case = _draw_once(rng)
        total = work(case)
        # the weights of every expert are in memory, with and without rows
        stored = case.get("experts", 0) * case.get("inputs", 0) * max(
            3 * case.get("hidden", 0), (2 if case.get("gated") else 1) * case.get("outputs", 0))
        if total["bytes"] <= MOST_BYTES and total["flops"] <= MOST_FLOPS / 4 and stored <= 600e6 \
                and 3072 not in case.values():
            return case


# ---- inputs ------------------------------------------------------------------

class _Make:
    """Tensors from one seed, on the GPU."""

    def __init__(self, seed):
        self.g = torch.Generator(device="cuda")
        self.g.manual_seed(seed)

    def normal(self, *shape):
        return torch.randn(shape, generator=self.g, device="cuda")

    def activations(self, rows, width, kind):
        """Normal values with a spread of scales over channels and a few
        channels far above the rest, as a network's hidden states have."""
        channel = torch.exp(0.5 * self.normal(width))
        channel = torch.where(torch.rand(width, generator=self.g, device="cuda") < 0.005,
                              10.0 * channel, channel)
        return (self.normal(rows, width) * channel).to(TYPES[kind])

    def weights(self, *shape):
        """Normal values scaled so that the largest of a row fill int8."""
        return (self.normal(*shape) * 33.0).round_().clamp_(-127, 127).to(torch.int8)

    def scales(self, *shape):
        """Weight scales that bring a product of a few thousand terms near 1."""
        return torch.exp(0.2 * self.normal(*shape)) * 5e-4

    def bias(self, *shape):
        return 0.5 * self.normal(*shape)

    def choices(self, tokens, choices, experts, padding=0):
        """Distinct experts for each token, some experts preferred, the most
        likely first, and their weights; the last `padding` tokens choose none."""
        logits = self.normal(tokens, experts) + 0.7 * self.normal(experts)
        top, ids = torch.topk(logits, choices, dim=1)
        ids = ids.to(torch.int32)
        if padding:
            ids[tokens - padding:] = -1
        return ids.contiguous(), torch.softmax(top, dim=1).contiguous()


def _sorted(ids, experts):
    """offsets, sources and places of the choices (see ``route``)."""
    flat = ids.reshape(-1).long()
    key = torch.where((flat >= 0) & (flat < experts), flat, experts)
    order = torch.argsort(key, stable=True)
    counts = torch.bincount(key, minlength=experts + 1)
    offsets = torch.zeros(experts + 1, dtype=torch.int64, device=ids.device)
    offsets[1:] = torch.cumsum(counts[:experts], 0)
    index = torch.arange(flat.numel(), device=ids.device)
    kept = index < offsets[experts]
    sources = torch.where(kept, order // ids.shape[1], -1)
    places = torch.empty_like(index)
    places[order] = torch.where(kept, index, -1)
    return offsets.to(torch.int32), sources.to(torch.int32), places.to(torch.int32).reshape(ids.shape)


def _weights(m, case, outputs, inputs, gated, bias, *lead):
    n = 2 * outputs if gated else outputs
    return {"w": m.weights(*lead, n, inputs), "ws": m.scales(*lead, n),
            "b": m.bias(*lead, n) if bias else None}


def prepare(case, seed):
    m = _Make(seed)
    kind = case["kind"]
    state = {"case": case, "kind": kind}
    if kind == "linear":
        rows, inputs, outputs = case["rows"], case["inputs"], case["outputs"]
        if case["x"] == "int8":
            state["x"] = m.weights(rows, inputs)
            state["xs"] = torch.exp(0.3 * m.normal(rows)) * 0.02
        else:
            state["x"], state["xs"] = m.activations(rows, inputs, case["x"]), None
        state.update(_weights(m, case, outputs, inputs, case["gated"], case["bias"]))
        state["r"] = m.normal(rows, outputs).to(TYPES[case["y"]]) if case["residual"] else None
        state["y"] = torch.empty((rows, outputs), device="cuda", dtype=TYPES[case["y"]])
        return state
    tokens, choices = case["tokens"], case["choices"]
    if kind == "combine":
        # places as a sort over a few experts would leave them
        ids, weights = m.choices(tokens, choices, max(8, choices))
        _, _, places = _sorted(ids, max(8, choices))
        state.update(x=m.normal(tokens * choices, case["outputs"]).to(TYPES[case["x"]]),
                     places=places.contiguous(), weights=weights,
                     r=m.normal(tokens, case["outputs"]).to(TYPES[case["y"]])
                     if case["residual"] else None,
                     y=torch.empty((tokens, case["outputs"]), device="cuda", dtype=TYPES[case["y"]]))
        return state
    experts = case["experts"]
    ids, weights = m.choices(tokens, choices, experts, case.get("padding", 0))
    state["ids"], state["weights"] = ids, weights
    state["offsets"] = torch.zeros(experts + 1, device="cuda", dtype=torch.int32)
    state["sources"] = torch.zeros(tokens * choices, device="cuda", dtype=torch.int32)
    state["places"] = torch.zeros((tokens, choices), device="cuda", dtype=torch.int32)
    if kind == "route":
        return state
    offsets, sources, places = _sorted(ids, experts)
    # the plain form walks the experts on the host
    state["bounds"] = offsets.tolist()
    if kind == "experts":
        state["offsets"], state["sources"] = offsets, sources
        inputs, outputs = case["inputs"], case["outputs"]
        state["x"] = m.activations(tokens if case["gather"] else tokens * choices, inputs, case["x"])
        state.update(_weights(m, case, outputs, inputs, case["gated"], case["bias"], experts))
        state["y"] = torch.zeros((tokens * choices, outputs), device="cuda",
                                 dtype=TYPES[case["y"]])
        return state
    inputs, hidden = case["inputs"], case["hidden"]
    state["x"] = m.activations(tokens, inputs, case["x"])
    state["up"] = _weights(m, case, hidden, inputs, True, False, experts)
    state["down"] = _weights(m, case, inputs, hidden, False, False, experts)
    kind_ = TYPES[case["x"]]
    state["h"] = torch.zeros((tokens * choices, hidden), device="cuda", dtype=kind_)
    state["z"] = torch.zeros((tokens * choices, inputs), device="cuda", dtype=kind_)
    state["y"] = torch.empty((tokens, inputs), device="cuda", dtype=kind_)
    return state


# ---- the plain form: 32 bits, rounded once -----------------------------------

def _quantized(x, scale=None):
    """(codes, row scales) in the arithmetic type of `x`."""
    if scale is not None:
        return x, scale[:, None]
    top = x.abs().amax(dim=1, keepdim=True)
    live = top >= TINY
    codes = torch.round(x * 127 / torch.where(live, top, torch.ones_like(top)))
    sound = torch.isfinite(top)
    codes = torch.where(live & sound, codes, torch.zeros_like(codes))
    scale = top / torch.full_like(top, 127)
    return codes, torch.where(sound, torch.where(live, scale, torch.zeros_like(scale)),
                              torch.full_like(scale, float("nan")))


def _activated(v, act):
    if act == "relu":
        return torch.where(v < 0, torch.zeros_like(v), v)
    if act == "gelu":
        return 0.5 * v * (1 + torch.erf(v * math.sqrt(0.5)))
    if act == "gelu_tanh":
        return 0.5 * v * (1 + torch.tanh(math.sqrt(2 / math.pi) * (v + 0.044715 * v * v * v)))
    if act == "silu":
        return v / (1 + torch.exp(-v))
    return v


def _product(codes, scale, p, act, gated, e=None):
    """act(codes w^T * scales + bias) of one weight matrix, in codes' type."""
    w, ws, b = (p[k] if e is None or p[k] is None else p[k][e] for k in ("w", "ws", "b"))
    v = codes @ w.to(codes.dtype).t()
    v = v * scale * ws.to(v.dtype)
    if b is not None:
        v = v + b.to(v.dtype)
    if not gated:
        return _activated(v, act)
    half = v.shape[1] // 2
    return _activated(v[:, :half], act) * v[:, half:]


def _by_expert(x, p, bounds, sources, act, gated, out):
    """One product per expert that has rows (the groups differ in size, so this
    is the plain way to write them: a batch of padded groups would do more)."""
    codes, scale = _quantized(x)
    for e, (lo, hi) in enumerate(zip(bounds, bounds[1:])):
        if lo == hi:
            continue
        rows = slice(lo, hi) if sources is None else sources[lo:hi].long()
        out[lo:hi] = _product(codes[rows], scale[rows], p, act, gated, e).to(out.dtype)
    return out


def _combined(x, places, weights, residual):
    picked = x[places.clamp(min=0).long()]
    live = (places >= 0)[..., None]
    total = (torch.where(live, picked, torch.zeros_like(picked)) * weights[..., None]).sum(1)
    return total if residual is None else total + residual


def _plain(state):
    case, kind = state["case"], state["kind"]
    if kind == "linear":
        x = state["x"].float()
        codes, scale = _quantized(x, state["xs"])
        v = _product(codes, scale, state, case["act"], case["gated"])
        if state["r"] is not None:
            v = v + state["r"].float()
        return v.to(state["y"].dtype)
    if kind == "route":
        return _sorted(state["ids"], case["experts"])
    if kind == "combine":
        r = None if state["r"] is None else state["r"].float()
        return _combined(state["x"].float(), state["places"], state["weights"], r).to(state["y"].dtype)
    if kind == "experts":
        return _by_expert(state["x"].float(), state, state["bounds"],
                          state["sources"] if case["gather"] else None, case["act"], case["gated"],
                          state["y"])
    _, sources, places = _sorted(state["ids"], case["experts"])
    h = _by_expert(state["x"].float(), state["up"], state["bounds"], sources, "silu", True, state["h"])
    z = _by_expert(h.float(), state["down"], state["bounds"], None, "none", False, state["z"])
    return _combined(z.float(), places, state["weights"], None).to(state["y"].dtype)


# ---- the library's calls -------------------------------------------------------

def _plan(state):
    """What a program sets up once: the shapes and the workspace they need."""
    import int8_kernel_lab_amd as lab

    case, kind = state["case"], state["kind"]
    plan = {"lab": lab, "need": 0}
    if kind == "linear":
        plan["shape"] = lab.LinearShape(
            case["rows"], case["inputs"], case["outputs"], input_type=case["x"],
            output_type=case["y"], activation=case["act"], gated=case["gated"])
        plan["need"] = lab.linear_workspace_bytes(plan["shape"])
    elif kind == "experts":
        routed = case["tokens"] * case["choices"]
        plan["shape"] = lab.LinearShape(
            case["tokens"] if case["gather"] else routed, case["inputs"], case["outputs"],
            input_type=case["x"], output_type=case["y"], activation=case["act"],
            gated=case["gated"], experts=case["experts"], routed=routed)
        plan["need"] = lab.linear_workspace_bytes(plan["shape"])
    elif kind == "block":
        routed = case["tokens"] * case["choices"]
        x, experts = case["x"], case["experts"]
        plan["up"] = lab.LinearShape(case["tokens"], case["inputs"], case["hidden"], input_type=x,
                                     output_type=x, activation="silu", gated=True,
                                     experts=experts, routed=routed)
        plan["down"] = lab.LinearShape(routed, case["hidden"], case["inputs"], input_type=x,
                                       output_type=x, experts=experts, routed=routed)
        plan["need"] = max(lab.linear_workspace_bytes(plan["up"]),
                           lab.linear_workspace_bytes(plan["down"]))
    if kind in ("route", "block"):
        plan["route"] = lab.RouteShape(case["tokens"], case["choices"], case["experts"])
        plan["need"] = max(plan["need"], lab.route_workspace_bytes(plan["route"]))
    if kind == "combine":
        plan["combine"] = lab.CombineShape(case["tokens"], case["choices"], case["outputs"],
                                           input_type=case["x"], output_type=case["y"])
    elif kind == "block":
        plan["combine"] = lab.CombineShape(case["tokens"], case["choices"], case["inputs"],
                                           input_type=case["x"], output_type=case["x"])
    plan["ws"] = torch.empty(max(plan["need"], 1), device="cuda", dtype=torch.uint8)
    return plan


def _at(tensor):
    return None if tensor is None else tensor.data_ptr()


def _own(state):
    plan = state.get("plan")
    if plan is None:
        plan = state["plan"] = _plan(state)
    lab, kind = plan["lab"], state["kind"]
    stream = torch.cuda.current_stream().cuda_stream
    ws, need = _at(plan["ws"]), plan["need"]
    if kind == "linear":
        lab.launch_linear(plan["shape"], _at(state["x"]), _at(state["xs"]), _at(state["w"]),
                          _at(state["ws"]), _at(state["b"]), _at(state["r"]), _at(state["y"]), ws,
                          need, stream)
        return state["y"]
    if kind == "experts":
        lab.launch_expert_linear(plan["shape"], _at(state["x"]), None, _at(state["w"]),
                                 _at(state["ws"]), _at(state["b"]), _at(state["offsets"]),
                                 _at(state["sources"]) if state["case"]["gather"] else None,
                                 _at(state["y"]), ws, need, stream)
        return state["y"]
    if kind == "combine":
        lab.launch_combine(plan["combine"], _at(state["x"]), _at(state["places"]),
                           _at(state["weights"]), _at(state["r"]), _at(state["y"]), stream)
        return state["y"]
    offsets, sources, places = _at(state["offsets"]), _at(state["sources"]), _at(state["places"])
    lab.launch_route(plan["route"], _at(state["ids"]), offsets, sources, places, ws, need, stream)
    if kind == "route":
        return state["offsets"], state["sources"], state["places"]
    up, down = state["up"], state["down"]
    lab.launch_expert_linear(plan["up"], _at(state["x"]), None, _at(up["w"]), _at(up["ws"]), None,
                             offsets, sources, _at(state["h"]), ws, need, stream)
    lab.launch_expert_linear(plan["down"], _at(state["h"]), None, _at(down["w"]), _at(down["ws"]),
                             None, offsets, None, _at(state["z"]), ws, need, stream)
    lab.launch_combine(plan["combine"], _at(state["z"]), places, _at(state["weights"]), None,
                       _at(state["y"]), stream)
    return state["y"]


def run(state):
    return _own(state) if own else _plain(state)


# ---- work, and the same in 64 bits ---------------------------------------------

def _used_experts(case):
    """Experts that have rows, in the mean, were all equally likely."""
    tokens = case["tokens"] - case.get("padding", 0)
    return case["experts"] * (1 - (1 - case["choices"] / case["experts"]) ** tokens)


def work(case):
    kind = case["kind"]
    if kind == "linear":
        rows, inputs, outputs = case["rows"], case["inputs"], case["outputs"]
        n = outputs * (2 if case["gated"] else 1)
        nbytes = rows * inputs * SIZES[case["x"]] + (4 * rows if case["x"] == "int8" else 0)
        nbytes += n * inputs + (8 if case["bias"] else 4) * n
        nbytes += rows * outputs * SIZES[case["y"]] * (2 if case["residual"] else 1)
        return {"bytes": nbytes, "flops": 2 * rows * n * inputs}
    tokens, choices = case["tokens"], case["choices"]
    routed = tokens * choices
    if kind == "route":
        return {"bytes": 12 * routed + 4 * (case["experts"] + 1), "flops": 0}
    if kind == "combine":
        outputs = case["outputs"]
        nbytes = routed * (outputs * SIZES[case["x"]] + 8)
        nbytes += tokens * outputs * SIZES[case["y"]] * (2 if case["residual"] else 1)
        return {"bytes": nbytes, "flops": 2 * routed * outputs}
    used = _used_experts(case)
    if kind == "experts":
        inputs, outputs = case["inputs"], case["outputs"]
        n = outputs * (2 if case["gated"] else 1)
        nbytes = (tokens if case["gather"] else routed) * inputs * SIZES[case["x"]]
        nbytes += used * n * (inputs + (8 if case["bias"] else 4)) + 4 * (case["experts"] + 1)
        nbytes += routed * (outputs * SIZES[case["y"]] + (4 if case["gather"] else 0))
        return {"bytes": nbytes, "flops": 2 * routed * n * inputs}
    inputs, hidden = case["inputs"], case["hidden"]
    live = (tokens - case["padding"]) * choices
    # tokens in, choices and weights, the experts' matrices, tokens out
    nbytes = 2 * tokens * inputs * SIZES[case["x"]] + 8 * routed
    nbytes += used * (3 * hidden * inputs + 8 * hidden + 4 * inputs)
    return {"bytes": nbytes, "flops": 2 * live * 3 * hidden * inputs}


def _exact_codes(x):
    """The nearest of 255 even steps to each value of a row, in 64 bits."""
    x = x.double()
    top = x.abs().max(dim=1, keepdim=True).values
    step = top / 127
    zero = top < TINY
    codes = torch.round(x * 127 / torch.where(zero, torch.ones_like(top), top))
    return codes * ~zero, step * ~zero


def _exact_layer(codes, step, w, ws, b, act, gated):
    v = torch.matmul(codes, w.double().t()) * step * ws.double()
    if b is not None:
        v += b.double()
    u = None
    if gated:
        v, u = v.chunk(2, dim=1)
    if act == "relu":
        v = v.clamp(min=0)
    elif act == "gelu":
        v = v * 0.5 * torch.special.erfc(-v / math.sqrt(2.0))
    elif act == "gelu_tanh":
        v = v * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3))
    elif act == "silu":
        v = v * torch.sigmoid(v)
    return v if u is None else v * u


def _exact_experts(x, p, ids, act, gated, rows, gather):
    """Rows in the order of a stable sort of `ids`; x's rows in that order
    where `gather` is false."""
    flat = ids.reshape(-1).cpu().tolist()
    n = p["w"].shape[1] // (2 if gated else 1)
    out = torch.zeros((rows, n), device="cuda", dtype=torch.float64)
    codes, step = _exact_codes(x)
    at = 0
    for e in range(p["w"].shape[0]):
        mine = [i for i, v in enumerate(flat) if v == e] if len(flat) < 4096 else \
            torch.nonzero(ids.reshape(-1) == e).flatten().tolist()
        if not mine:
            continue
        index = torch.tensor([i // ids.shape[1] for i in mine], device="cuda") if gather else \
            torch.arange(at, at + len(mine), device="cuda")
        b = None if p["b"] is None else p["b"][e]
        out[at:at + len(mine)] = _exact_layer(codes[index], step[index], p["w"][e], p["ws"][e], b,
                                              act, gated)
        at += len(mine)
    return out


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "route":
        return None  # whole numbers: the plain form's have no rounding
    if kind == "linear":
        codes, step = (s["x"].double(), s["xs"].double()[:, None]) if case["x"] == "int8" else \
            _exact_codes(s["x"])
        v = _exact_layer(codes, step, s["w"], s["ws"], s["b"], case["act"], case["gated"])
        return v if s["r"] is None else v + s["r"].double()
    if kind == "combine":
        v = torch.zeros(s["y"].shape, device="cuda", dtype=torch.float64)
        if s["r"] is not None:
            v += s["r"]
        for c in range(case["choices"]):
            v += s["x"][s["places"][:, c].long()].double() * s["weights"][:, c, None].double()
        return v
    routed = case["tokens"] * case["choices"]
    if kind == "experts":
        return _exact_experts(s["x"], s, s["ids"], case["act"], case["gated"], routed,
                              case["gather"])
    h = _exact_experts(s["x"], s["up"], s["ids"], "silu", True, routed, True)
    z = _exact_experts(h, s["down"], s["ids"], "none", False, routed, False)
    v = torch.zeros(s["y"].shape, device="cuda", dtype=torch.float64)
    at, ids = 0, s["ids"].cpu()
    for e in range(case["experts"]):
        for t, c in torch.nonzero(ids == e).tolist():
            v[t] += z[at] * s["weights"][t, c].double()
            at += 1
    return v
