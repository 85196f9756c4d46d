"""The operators of quantised and differential transformers, as cases that can be timed and checked.

Four operators, each a node of the framework in a graph of its own:

``norm``       SkipRMSNormalization: x + skip, its root-mean-square norm, and that in eight bits with a scale to each row
``linear``     QuantizedLinear: int8 rows times int8 weights, scaled, with bias, activation and residual
``rotary``     RotaryPositions: queries and keys turned by the angles of their positions along several axes
``attention``  DifferentialAttention: the difference of two softmax maps, applied to the values

``own`` chooses between their plain form in elementary torch operations and the framework's nodes. A program keeps one
compiled model for each set of sizes; weights, caches and tokens are inputs of its calls.
"""
import functools
import math

import torch

own = False

TYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
ELEMENTS = {"float32": 1, "float16": 10, "bfloat16": 16}   # ONNX element types
BYTES = {"float32": 4, "float16": 2, "bfloat16": 2}
ACTIVATIONS = ("none", "relu", "gelu", "silu")


def listed():
    return [
        # the norm before a projection while one token is generated for each of four requests
        {"name": "norm_token", "kind": "norm", "rows": 4, "columns": 2048, "type": "bfloat16", "skip": True, "plain": False, "eight": True},
        # the same in a batch of long prompts: the largest norm of a step
        {"name": "norm_prompts", "kind": "norm", "rows": 16384, "columns": 4096, "type": "bfloat16", "skip": True, "plain": False, "eight": True},
        # an fp32 graph of odd width that goes on in floating point
        {"name": "norm_odd", "kind": "norm", "rows": 1777, "columns": 1001, "type": "float32", "skip": True, "plain": True, "eight": False},
        # a projection with its residual for a few generated tokens: the weights are read once and that is the work
        {"name": "linear_token", "kind": "linear", "rows": 4, "inner": 4096, "columns": 4096, "type": "bfloat16", "activation": "none",
         "bias": False, "residual": True},
        # the wide layer of a feed-forward block over a batch of prompts
        {"name": "linear_prompts", "kind": "linear", "rows": 8192, "inner": 4096, "columns": 8192, "type": "bfloat16", "activation": "silu",
         "bias": True, "residual": False},
        # one sentence through a layer of odd extents, results for an fp32 graph
        {"name": "linear_odd", "kind": "linear", "rows": 197, "inner": 1001, "columns": 2049, "type": "float32", "activation": "gelu",
         "bias": True, "residual": True},
        # queries and keys of one generated token to a request, far into their contexts
        {"name": "rotary_token", "kind": "rotary", "batch": 8, "tokens": 1, "heads": 32, "kv_heads": 8, "size": 128, "rotated": 128, "axes": 3,
         "interleaved": False, "type": "bfloat16"},
        # a video of 16 frames of 32 x 32 patches with time, height and width
        {"name": "rotary_video", "kind": "rotary", "batch": 2, "tokens": 16384, "heads": 16, "kv_heads": 4, "size": 128, "rotated": 128, "axes": 3,
         "interleaved": False, "type": "bfloat16"},
        # images of an odd number of patches in an fp32 graph, part of each head turned, neighbours as pairs
        {"name": "rotary_images", "kind": "rotary", "batch": 8, "tokens": 577, "heads": 12, "kv_heads": 0, "size": 64, "rotated": 48, "axes": 2,
         "interleaved": True, "type": "float32"},
        # one generated token for each of eight requests over caches of unequal length
        {"name": "attention_token", "kind": "attention", "batch": 8, "queries": 1, "keys": 8192, "heads": 16, "kv_heads": 4, "size": 64,
         "causal": True, "ragged": True, "type": "bfloat16"},
        # a long prompt, every token attending to those before it
        {"name": "attention_prompt", "kind": "attention", "batch": 1, "queries": 8192, "keys": 8192, "heads": 8, "kv_heads": 8, "size": 64,
         "causal": True, "ragged": False, "type": "bfloat16"},
        # a padded batch of odd length through an fp32 encoder
        {"name": "attention_padded", "kind": "attention", "batch": 3, "queries": 333, "keys": 333, "heads": 6, "kv_heads": 6, "size": 64,
         "causal": False, "ragged": True, "type": "float32"},
    ]


def _spread(rng, low, high):
    """A whole number of [low, high], spread over its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def _cost(case):
    w = work(case)
    return max(w["bytes"], w["flops"] / 50)


def draw(rng):
    most = max(_cost(c) for c in listed())
    while True:
        kind = rng.choice(["norm", "linear", "rotary", "attention"])
        case = {"kind": kind, "type": rng.choice(list(TYPES))}
        if kind == "norm":
            case.update(rows=_spread(rng, 1, 16384), columns=_spread(rng, 64, 16384), skip=rng.random() < 0.7, plain=rng.random() < 0.5)
            case["eight"] = not case["plain"] or rng.random() < 0.3
            if rng.random() < 0.5:
                case["columns"] = max(64, case["columns"] // 64 * 64)
        elif kind == "linear":
            case.update(rows=_spread(rng, 1, 8192), inner=_spread(rng, 64, 8192), columns=_spread(rng, 64, 16384),
                        activation=rng.choice(ACTIVATIONS), bias=rng.random() < 0.5, residual=rng.random() < 0.5)
            if rng.random() < 0.6:   # layers of networks have round extents more often than not
                case["inner"], case["columns"] = max(64, case["inner"] // 64 * 64), max(64, case["columns"] // 64 * 64)
        elif kind == "rotary":
            case.update(batch=_spread(rng, 1, 32), tokens=_spread(rng, 1, 32768), heads=rng.randint(1, 32), kv_heads=rng.choice([0, 1, 2, 4, 8]),
                        size=rng.choice([32, 64, 80, 128, 256]), axes=rng.randint(1, 4), interleaved=rng.random() < 0.5)
            case["rotated"] = case["size"] if rng.random() < 0.6 else 2 * rng.randint(case["axes"], case["size"] // 2)
        else:
            case.update(batch=_spread(rng, 1, 16), queries=_spread(rng, 1, 8192) if rng.random() < 0.6 else 1, kv_heads=rng.choice([1, 2, 3, 4, 8]),
                        size=rng.choice([32, 64, 128]), causal=rng.random() < 0.5, ragged=rng.random() < 0.5)
            case["heads"] = case["kv_heads"] * rng.choice([1, 1, 2, 4])
            case["keys"] = case["queries"] if rng.random() < 0.5 and case["queries"] > 1 else _spread(rng, case["queries"], 16384)
            if 8 * case["batch"] * case["heads"] * case["queries"] * case["keys"] > 5 << 30:   # the plain form's two maps
                continue
        if _cost(case) <= most:
            return case


# ------------------------------------------------------------------------------------------------ inputs


def _device():
    return "cuda" if torch.cuda.is_available() else "cpu"


class _Normal:
    """Normal numbers on the device, from one seed."""

    def __init__(self, seed):
        self.generator = torch.Generator(_device()).manual_seed(seed)

    def __call__(self, *shape, scale=1.0, mean=0.0, dtype=torch.float32):
        return torch.randn(*shape, generator=self.generator, device=_device()).mul_(scale).add_(mean).to(dtype)

    def integers(self, low, high, *shape, dtype=torch.int64):
        return torch.randint(low, high, shape, generator=self.generator, device=_device()).to(dtype)


def _sections(case):
    """Pairs of a head that each axis turns: equal shares, the first axes have what is left over."""
    pairs, axes = case["rotated"] // 2, case["axes"]
    return [pairs // axes + (i < pairs % axes) for i in range(axes)]


LAMBDA_INIT = 0.5   # that of the first layers; learned vectors move it
EPSILON = 1e-5


def _lengths(case, normal):
    """Keys that each batch entry has."""
    if not case["ragged"]:
        return None
    low = max(case["queries"] if case["causal"] else 1, case["keys"] // 3)
    return normal.integers(low, case["keys"] + 1, case["batch"], dtype=torch.int32)


def prepare(case, seed):
    normal, dtype, kind = _Normal(seed), TYPES[case["type"]], case["kind"]
    state = {"case": dict(case)}
    if kind == "norm":
        rows, columns = case["rows"], case["columns"]
        # a residual stream: some channels are much larger than the others
        channels = torch.exp(normal(columns, scale=0.5))
        state["x"] = (normal(rows, columns) * channels).to(dtype)
        state["skip"] = normal(rows, columns, scale=0.7, dtype=dtype) if case["skip"] else None
        state["gain"] = normal(columns, scale=0.2, mean=1.0, dtype=dtype)
        state["wide"] = torch.empty(rows, columns, dtype=torch.float16 if dtype == torch.float32 else dtype, device=_device()) if case["eight"] else None
    elif kind == "linear":
        rows, inner, columns = case["rows"], case["inner"], case["columns"]
        state["x"] = normal(rows, inner, scale=38.0).round_().clamp_(-127, 127).to(torch.int8)
        state["w"] = normal(columns, inner, scale=38.0).round_().clamp_(-127, 127).to(torch.int8)
        state["x_scale"] = torch.exp(normal(rows, scale=0.3)) / 38
        state["w_scale"] = torch.exp(normal(columns, scale=0.3)) / (38 * math.sqrt(inner))
        state["bias"] = normal(columns, scale=0.2, dtype=dtype) if case["bias"] else None
        state["residual"] = normal(rows, columns, dtype=dtype) if case["residual"] else None
    elif kind == "rotary":
        batch, tokens, size = case["batch"], case["tokens"], case["size"]
        state["q"] = normal(batch, tokens, case["heads"], size, dtype=dtype)
        state["k"] = normal(batch, tokens, case["kv_heads"], size, dtype=dtype) if case["kv_heads"] else None
        # tokens in order along the last axis, rows of 32, frames of 1024, behind a context of any length
        at = torch.arange(tokens, device=_device())
        place = torch.stack([at // 32 ** (case["axes"] - 1 - axis) % (32 if axis else 1 << 62) for axis in range(case["axes"])])
        state["positions"] = (place[:, None, :] + normal.integers(0, 100000, 1, batch, 1)).contiguous()
        pairs = torch.arange(case["rotated"] // 2, dtype=torch.float64, device=_device())
        state["frequencies"] = torch.pow(10000.0, -2.0 * pairs / case["rotated"]).to(torch.float32)
    else:
        batch, size, heads, kv_heads = case["batch"], case["size"], case["heads"], case["kv_heads"]
        state["q"] = normal(batch, case["queries"], 2 * heads, size, scale=2.0, dtype=dtype)
        state["k"] = normal(batch, case["keys"], 2 * kv_heads, size, dtype=dtype)
        # values differ from channel to channel by more than their mean over the tokens does
        state["v"] = (normal(batch, case["keys"], kv_heads, 2 * size) + normal(2 * size, scale=0.5)).to(dtype)
        state["weights"] = [normal(size, scale=0.1) for _ in range(4)]
        state["lengths"] = _lengths(case, normal)
    return state


# ------------------------------------------------------------------------------------------------ plain forms


def _plain_norm(state):
    case, x = state["case"], state["x"].to(torch.float32)
    total = x + state["skip"].to(torch.float32) if case["skip"] else x
    y = total * (1.0 / torch.sqrt((total * total).mean(dim=-1, keepdim=True) + EPSILON)) * state["gain"].to(torch.float32)
    out = [y.to(state["x"].dtype)] if case["plain"] else []
    if case["skip"]:
        out.append(total.to(state["x"].dtype))
    if case["eight"]:
        scale = y.abs().amax(dim=-1, keepdim=True) / 127.0
        whole = torch.round(y / torch.where(scale > 0, scale, 1.0)).to(torch.int8)
        out += [(whole * scale).to(state["wide"].dtype), scale.reshape(-1)]
    return out


def _activated(v, activation):
    if activation == "relu":
        return torch.relu(v)
    if activation == "gelu":
        return 0.5 * v * (1.0 + torch.erf(v * math.sqrt(0.5)))
    return v / (1.0 + torch.exp(-v)) if activation == "silu" else v


def _plain_linear(state):
    case = state["case"]
    y = torch.matmul(state["x"].to(torch.float32), state["w"].to(torch.float32).t())
    y = y * state["x_scale"][:, None] * state["w_scale"]
    if case["bias"]:
        y = y + state["bias"].to(torch.float32)
    y = _activated(y, case["activation"])
    if case["residual"]:
        y = y + state["residual"].to(torch.float32)
    return y.to(TYPES[case["type"]])


def _turned(x, cos, sin, rotated, interleaved):
    part = x[..., :rotated].to(torch.float32)
    if interleaved:
        a, b = part[..., 0::2], part[..., 1::2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2)
    else:
        a, b = part[..., :rotated // 2], part[..., rotated // 2:]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)
    return torch.cat([turned.to(x.dtype), x[..., rotated:]], dim=-1)


def _plain_rotary(state):
    case = state["case"]
    sections = torch.tensor(_sections(case), device=state["positions"].device)
    axis = torch.repeat_interleave(torch.arange(case["axes"], device=sections.device), sections, output_size=case["rotated"] // 2)
    angles = state["positions"][axis].permute(1, 2, 0).to(torch.float64) * state["frequencies"].to(torch.float64)
    cos, sin = (f(angles).to(torch.float32)[:, :, None, :] for f in (torch.cos, torch.sin))
    out = [_turned(state["q"], cos, sin, case["rotated"], case["interleaved"])]
    if case["kv_heads"]:
        out.append(_turned(state["k"], cos, sin, case["rotated"], case["interleaved"]))
    return out


def _plain_attention(state):
    case = state["case"]
    batch, queries, keys, kv_heads, size = case["batch"], case["queries"], case["keys"], case["kv_heads"], case["size"]
    group = case["heads"] // kv_heads
    q = state["q"].to(torch.float32).reshape(batch, queries, kv_heads, group, 2, size).permute(0, 2, 4, 3, 1, 5).reshape(batch, kv_heads, 2, group * queries, size)
    k = state["k"].to(torch.float32).reshape(batch, keys, kv_heads, 2, size).permute(0, 2, 3, 4, 1).contiguous()
    scores = torch.matmul(q, k).mul_(1.0 / math.sqrt(size)).reshape(batch, kv_heads, 2, group, queries, keys)
    if case["causal"] or case["ragged"]:
        last = state["lengths"].to(torch.int64) if case["ragged"] else torch.full((batch,), keys, device=scores.device)
        at = torch.arange(keys, device=scores.device)
        hidden = at >= last[:, None, None]
        if case["causal"]:
            hidden = hidden | (at > torch.arange(queries, device=scores.device)[:, None] + last[:, None, None] - queries)
        scores.masked_fill_(hidden[:, None, None, None], -math.inf)
    # (every row of these cases has a key)
    maps = torch.exp(scores.sub_(scores.amax(dim=-1, keepdim=True)))
    maps = maps / maps.sum(dim=-1, keepdim=True)
    a, b, c, d = state["weights"]
    weight = torch.exp((a * b).sum()) - torch.exp((c * d).sum()) + LAMBDA_INIT
    difference = (maps[:, :, 0] - weight * maps[:, :, 1]).reshape(batch, kv_heads, group * queries, keys)
    v = state["v"].to(torch.float32).permute(0, 2, 1, 3).contiguous()
    out = torch.matmul(difference, v).reshape(batch, kv_heads, group, queries, 2 * size).permute(0, 3, 1, 2, 4)
    return out.reshape(batch, queries, case["heads"], 2 * size).to(state["q"].dtype)


# ------------------------------------------------------------------------------------------------ the framework's nodes


@functools.lru_cache(maxsize=64)
def _model(op, inputs, outputs, attributes):
    """A compiled graph of one node; inputs and outputs as (name, element type, shape), None for one that is left out."""
    import dace_onnx_amd.onnx as donnx
    from dace_onnx_amd.onnx.proto import helper
    info = lambda values: [helper.make_tensor_value_info(name, element, list(shape)) for name, element, shape in filter(None, values)]  # noqa: E731
    names = lambda values: [v[0] if v else "" for v in values]  # noqa: E731
    node = helper.make_node(op, names(inputs), names(outputs), name=op.lower(), **{k: list(v) if isinstance(v, tuple) else v for k, v in attributes})
    return donnx.ONNXModel(op.lower(), helper.make_model(helper.make_graph([node], op.lower(), info(inputs), info(outputs))))


def _built(state):
    """The node's model and the tensors of a call."""
    case, kind, t = state["case"], state["case"]["kind"], ELEMENTS[state["case"]["type"]]
    given = lambda name, tensor, element: None if tensor is None else (name, element, tuple(tensor.shape))  # noqa: E731
    if kind == "norm":
        shape = (case["rows"], case["columns"])
        model = _model("SkipRMSNormalization", (given("x", state["x"], t), given("gain", state["gain"], t), given("skip", state["skip"], t)),
                       (("y", t, shape) if case["plain"] else None, ("sum", t, shape) if case["skip"] else None,
                        ("q", 3, shape) if case["eight"] else None, ("q_scale", 1, shape[:1]) if case["eight"] else None), (("epsilon", EPSILON),))
        tensors = (state["x"], state["gain"], state["skip"])
    elif kind == "linear":
        model = _model("QuantizedLinear", (given("x", state["x"], 3), given("w", state["w"], 3), given("x_scale", state["x_scale"], 1),
                                           given("w_scale", state["w_scale"], 1), given("bias", state["bias"], t), given("residual", state["residual"], t)),
                       (("y", t, (case["rows"], case["columns"])),), (("activation", case["activation"]), ("to", t)))
        tensors = tuple(state[k] for k in ("x", "w", "x_scale", "w_scale", "bias", "residual"))
    elif kind == "rotary":
        model = _model("RotaryPositions", (given("q", state["q"], t), given("positions", state["positions"], 7), given("frequencies", state["frequencies"], 1),
                                           given("k", state["k"], t)),
                       (("q_turned", t, tuple(state["q"].shape)), given("k_turned", state["k"], t)),
                       (("sections", tuple(_sections(case))), ("interleaved", int(case["interleaved"]))))
        tensors = (state["q"], state["positions"], state["frequencies"], state["k"])
    else:
        vectors = tuple(given("lambda_" + n, w, 1) for n, w in zip(("q1", "k1", "q2", "k2"), state["weights"]))
        model = _model("DifferentialAttention", (given("q", state["q"], t), given("k", state["k"], t), given("v", state["v"], t)) + vectors
                       + (given("lengths", state["lengths"], 6),),
                       (("o", t, (case["batch"], case["queries"], case["heads"], 2 * case["size"])),),
                       (("lambda_init", LAMBDA_INIT), ("causal", int(case["causal"]))))
        tensors = (state["q"], state["k"], state["v"], *state["weights"], state["lengths"])
    return model, tuple(v for v in tensors if v is not None)


def run(state):
    if not own:
        return {"norm": _plain_norm, "linear": _plain_linear, "rotary": _plain_rotary, "attention": _plain_attention}[state["case"]["kind"]](state)
    if "model" not in state:
        state["model"] = _built(state)
    model, tensors = state["model"]
    out = model(*tensors)
    if state["case"]["kind"] in ("norm", "rotary"):
        out = list(out) if isinstance(out, tuple) else [out]
        if state["case"].get("eight"):   # the values that the eight bits stand for
            out[-2] = torch.mul(out[-2], out[-1][:, None], out=state["wide"])
    return out


# ------------------------------------------------------------------------------------------------ floors


def work(case):
    kind, item = case["kind"], BYTES[case["type"]]
    if kind == "norm":
        count = case["rows"] * case["columns"]
        wide = 1 + 2 * case["skip"] + case["plain"]
        return {"bytes": float(item * (wide * count + case["columns"]) + case["eight"] * (count + 4 * case["rows"])), "flops": 5.0 * count}
    if kind == "linear":
        rows, inner, columns = case["rows"], case["inner"], case["columns"]
        floats = rows * columns * (1 + case["residual"]) + columns * case["bias"]
        return {"bytes": float(rows * inner + inner * columns + 4 * (rows + columns) + item * floats), "flops": 2.0 * rows * inner * columns}
    if kind == "rotary":
        tokens = case["batch"] * case["tokens"]
        values = tokens * (case["heads"] + case["kv_heads"]) * case["size"]
        return {"bytes": float(2 * item * values + 8 * case["axes"] * tokens + 2 * case["rotated"]), "flops": 3.0 * values}
    batch, queries, keys, heads, kv_heads, size = (case[k] for k in ("batch", "queries", "keys", "heads", "kv_heads", "size"))
    seen = keys * 2 / 3 if case["ragged"] else keys   # keys of a row, on average: lengths lie between a third and all of them
    pairs = queries * max(seen - (queries - 1) / 2, seen / 2) if case["causal"] else queries * seen
    values = 4 * batch * size * (heads * queries + kv_heads * seen)
    return {"bytes": float(item * values), "flops": 8.0 * batch * heads * size * pairs}   # two products of scores, one with the values


# ------------------------------------------------------------------------------------------------ the definitions in 64 bits


def _exact_norm(case, state):
    s = state["x"].double() + (state["skip"].double() if case["skip"] else 0.0)
    y = s / (s.pow(2).sum(-1, keepdim=True) / case["columns"] + EPSILON).sqrt() * state["gain"].double()
    scale = y.abs().max(-1, keepdim=True).values / 127
    return [y] * case["plain"] + [s] * case["skip"] + [(y / scale).round() * scale, scale[:, 0]] * case["eight"]


def _exact_linear(case, state):
    blocks = []
    for x, scale, *residual in zip(*(t.split(1024) for t in (state["x"], state["x_scale"], *([state["residual"]] if case["residual"] else [])))):
        y = (x.double() @ state["w"].double().T) * torch.outer(scale.double(), state["w_scale"].double())
        y += state["bias"].double() if case["bias"] else 0.0
        f = {"none": lambda v: v, "relu": lambda v: v.clamp(min=0), "gelu": lambda v: v * torch.special.ndtr(v), "silu": lambda v: v * torch.sigmoid(v)}
        y = f[case["activation"]](y)
        blocks.append(y + residual[0].double() if residual else y)
    return torch.cat(blocks)


def _exact_rotary(case, state):
    out = []
    for x in filter(lambda t: t is not None, (state["q"], state["k"])):
        y, pair = x.double(), 0
        for axis, count in enumerate(_sections(case)):
            for _ in range(count):
                i, j = (2 * pair, 2 * pair + 1) if case["interleaved"] else (pair, pair + case["rotated"] // 2)
                turn = torch.polar(torch.ones((), dtype=torch.float64, device=x.device),
                                   state["positions"][axis].double() * state["frequencies"][pair].double())[..., None]
                z = torch.complex(x[..., i].double(), x[..., j].double()) * turn
                y[..., i], y[..., j] = z.real, z.imag
                pair += 1
        out.append(y)
    return out


def _exact_attention(case, state):
    group, size = case["heads"] // case["kv_heads"], case["size"]
    lq1, lk1, lq2, lk2 = (w.double() for w in state["weights"])
    weight = (lq1 @ lk1).exp() - (lq2 @ lk2).exp() + LAMBDA_INIT
    out = torch.zeros(case["batch"], case["queries"], case["heads"], 2 * size, dtype=torch.float64, device=state["q"].device)
    for b in range(case["batch"]):
        length = int(state["lengths"][b]) if case["ragged"] else case["keys"]
        for h in range(case["heads"]):
            kv = h // group
            v = state["v"][b, :length, kv].double()
            for start in range(0, case["queries"], 2048):
                rows = slice(start, min(start + 2048, case["queries"]))
                maps = []
                for m in range(2):
                    s = state["q"][b, rows, 2 * h + m].double() @ state["k"][b, :length, 2 * kv + m].double().T / math.sqrt(size)
                    if case["causal"]:
                        place = torch.arange(rows.start, rows.stop, device=s.device)[:, None] + (length - case["queries"])
                        s = s.where(torch.arange(length, device=s.device) <= place, -math.inf)
                    maps.append(torch.softmax(s, -1))
                out[b, rows, h] = (maps[0] - weight * maps[1]) @ v
    return out


def exact(case, seed):
    state = prepare(case, seed)
    return {"norm": _exact_norm, "linear": _exact_linear, "rotary": _exact_rotary, "attention": _exact_attention}[case["kind"]](case, state)
