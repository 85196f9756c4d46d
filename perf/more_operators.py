"""The operators that verify drafted tokens over a paged cache, as cases that can be timed and checked.

Three operators, each a node of the framework in a graph of its own:

``append``      PagedCacheAppend: keys and values into the pages of a cache, keys and queries turned by their positions on the way
``attention``   TreeAttention: the tokens of a call, a tree or a chain, attend to the cache before them and to their ancestors
``acceptance``  DraftAcceptance: the path of a tree that the model itself would have taken, and the token after it

``own`` chooses between their plain form in elementary torch operations and the framework's nodes. A program keeps one
compiled model for each set of sizes; caches, tables and tokens are inputs of its calls, and a cache is updated where it lies.
"""
import functools
import math

import torch

own = False

TYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
ELEMENTS = {torch.float32: 1, torch.int32: 6, torch.int64: 7, torch.float16: 10, torch.bfloat16: 16}   # ONNX element types
BYTES = {"float32": 4, "float16": 2, "bfloat16": 2}


def listed():
    return [
        # one generated token for each of sixteen requests: queries and keys turned, keys and values to their pages
        {"name": "append_token", "kind": "append", "batch": 16, "tokens": 1, "heads": 32, "kv_heads": 8, "size": 128, "rotated": 128, "axes": 1,
         "interleaved": False, "page": 16, "context": 4096, "order": False, "type": "bfloat16"},
        # four long prompts at once: the largest append of a step
        {"name": "append_prompts", "kind": "append", "batch": 4, "tokens": 4096, "heads": 32, "kv_heads": 8, "size": 128, "rotated": 128, "axes": 1,
         "interleaved": False, "page": 16, "context": 2048, "order": False, "type": "bfloat16"},
        # the accepted ones among the drafted tokens of an fp32 graph, part of each head turned, pages of an odd number of tokens
        {"name": "append_accepted", "kind": "append", "batch": 5, "tokens": 45, "heads": 0, "kv_heads": 6, "size": 64, "rotated": 48, "axes": 2,
         "interleaved": True, "page": 23, "context": 777, "order": True, "type": "float32"},
        # one generated token for each of sixteen requests over caches of unequal length
        {"name": "attention_token", "kind": "attention", "batch": 16, "tokens": 1, "heads": 32, "kv_heads": 8, "size": 128, "page": 16, "context": 8192,
         "ragged": True, "tree": False, "type": "bfloat16"},
        # one token far into one long document
        {"name": "attention_document", "kind": "attention", "batch": 1, "tokens": 1, "heads": 16, "kv_heads": 4, "size": 128, "page": 64, "context": 131072,
         "ragged": False, "tree": False, "type": "float16"},
        # trees of drafted tokens for a few requests
        {"name": "attention_drafts", "kind": "attention", "batch": 4, "tokens": 32, "heads": 32, "kv_heads": 8, "size": 128, "page": 32, "context": 4096,
         "ragged": True, "tree": True, "type": "bfloat16"},
        # a part of a long prompt, every token attending to those before it, in the cache too
        {"name": "attention_prompt", "kind": "attention", "batch": 1, "tokens": 4096, "heads": 16, "kv_heads": 4, "size": 128, "page": 64, "context": 4096,
         "ragged": False, "tree": False, "type": "bfloat16"},
        # an fp32 graph of odd sizes: small trees over short caches
        {"name": "attention_odd", "kind": "attention", "batch": 3, "tokens": 13, "heads": 6, "kv_heads": 3, "size": 64, "page": 23, "context": 777,
         "ragged": True, "tree": True, "type": "float32"},
        # the drafts of one request
        {"name": "acceptance_one", "kind": "acceptance", "batch": 1, "tokens": 8, "vocabulary": 32000, "tree": False, "type": "bfloat16"},
        # trees of a batch over a large vocabulary
        {"name": "acceptance_batch", "kind": "acceptance", "batch": 16, "tokens": 32, "vocabulary": 131072, "tree": True, "type": "bfloat16"},
        # fp32 logits of an odd vocabulary
        {"name": "acceptance_odd", "kind": "acceptance", "batch": 5, "tokens": 13, "vocabulary": 49999, "tree": True, "type": "float32"},
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
        kind = rng.choice(["append", "attention", "attention", "acceptance"])
        case = {"kind": kind, "type": rng.choice(list(TYPES))}
        if kind == "acceptance":
            case.update(batch=_spread(rng, 1, 32), tokens=_spread(rng, 1, 64), vocabulary=_spread(rng, 1000, 262144), tree=rng.random() < 0.7)
            if rng.random() < 0.5:
                case["vocabulary"] = max(1024, case["vocabulary"] // 1024 * 1024)
        else:
            case.update(batch=_spread(rng, 1, 32), kv_heads=rng.choice([1, 2, 3, 4, 8]), page=rng.choice([8, 16, 16, 23, 32, 64, 128, 256]))
            case["context"] = _spread(rng, 1, 8192)
            if kind == "append":
                case.update(size=rng.choice([32, 64, 80, 128, 256]), axes=rng.randint(1, 3), interleaved=rng.random() < 0.5, order=rng.random() < 0.3)
                case["rotated"] = case["size"] if rng.random() < 0.6 else 2 * rng.randint(0, case["size"] // 2)
                case["tokens"] = _spread(rng, 1, 64) if case["order"] else _spread(rng, 1, 4096)
                case["heads"] = 0 if case["order"] or case["rotated"] == 0 else case["kv_heads"] * rng.choice([0, 1, 2, 4, 8])
            else:
                case.update(size=rng.choice([64, 64, 128, 128, 256]), ragged=rng.random() < 0.6, tree=rng.random() < 0.4)
                case["heads"] = case["kv_heads"] * rng.choice([1, 1, 2, 4, 8])
                case["tokens"] = _spread(rng, 1, 256) if case["tree"] else 1 if rng.random() < 0.4 else _spread(rng, 1, 4096)
                if rng.random() < 0.3 and case["tokens"] < 64:
                    case["batch"], case["context"] = _spread(rng, 1, 4), _spread(rng, 4096, 131072)
                if 12 * case["batch"] * case["heads"] * case["tokens"] * (case["context"] + case["tokens"]) > 8 << 30:   # the plain form's scores
                    continue
            if 4 * case["batch"] * (case["context"] + case["tokens"]) * case["kv_heads"] * case["size"] > 2 << 30:   # its keys, or values
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

    def uniform(self, *shape):
        return torch.rand(*shape, generator=self.generator, device=_device())

    def integers(self, low, high, *shape, dtype=torch.int64):
        return torch.randint(low, high, shape, generator=self.generator, device=_device()).to(dtype)


def _sections(case):
    """Pairs of a head that each axis turns: equal shares, the first axes have what is left over."""
    pairs, axes = case["rotated"] // 2, case["axes"]
    return [pairs // axes + (i < pairs % axes) for i in range(axes)]


def _parents(case, normal):
    """Trees whose root is the last token that is known; drafts branch most near it."""
    batch, tokens = case["batch"], case["tokens"]
    at = torch.arange(tokens, device=_device())
    parents = (normal.uniform(batch, tokens) * at).to(torch.int64).clamp(max=at - 1)   # (of the root: -1)
    return parents.to(torch.int32)


def _cache(case, normal, state):
    """Pages in the order in which they were handed out, long ago; lengths of the entries before the call."""
    batch, tokens, page = case["batch"], case["tokens"], case["page"]
    ragged = case.get("ragged", True) and case["context"] > 1
    state["lengths"] = normal.integers(case["context"] // 3, case["context"] + 1, batch, dtype=torch.int32) if ragged else \
        torch.full((batch,), case["context"], dtype=torch.int32, device=_device())
    columns = -(-(case["context"] + tokens) // page)
    pages = batch * columns + 3
    state["table"] = torch.randperm(pages, generator=normal.generator, device=_device())[:batch * columns].reshape(batch, columns).to(torch.int32)
    shape, dtype = (pages, case["kv_heads"], page, case["size"]), TYPES[case["type"]]
    state["k_pages"] = normal(*shape, dtype=dtype)
    # values differ from channel to channel by more than their mean over the tokens does
    state["v_pages"] = (normal(*shape) + normal(case["size"], scale=0.5)).to(dtype)


def prepare(case, seed):
    normal, dtype, kind = _Normal(seed), TYPES[case["type"]], case["kind"]
    state = {"case": dict(case)}
    batch, tokens = case["batch"], case["tokens"]
    if kind == "append":
        _cache(case, normal, state)
        size = case["size"]
        state["k"] = normal(batch, tokens, case["kv_heads"], size, dtype=dtype)
        state["v"] = normal(batch, tokens, case["kv_heads"], size, dtype=dtype)
        state["q"] = normal(batch, tokens, case["heads"], size, dtype=dtype) if case["heads"] else None
        pairs = torch.arange(case["rotated"] // 2, dtype=torch.float64, device=_device())
        state["frequencies"] = torch.pow(10000.0, -2.0 * pairs / max(case["rotated"], 1)).to(torch.float32) if case["rotated"] else None
        state["positions"] = state["order"] = None
        if case["axes"] > 1 and case["rotated"]:   # rows of 32, frames of 1024, behind a context of any length
            at = torch.arange(tokens, device=_device())
            place = torch.stack([at // 32 ** (case["axes"] - 1 - axis) % (32 if axis else 1 << 62) for axis in range(case["axes"])])
            state["positions"] = (place[:, None, :] + normal.integers(0, 100000, 1, batch, 1)).contiguous()
        if case["order"]:   # paths of unequal length through trees: tokens in rising order, then nothing
            taken = (normal.uniform(batch, tokens) < 0.3).to(torch.int64)
            taken[:, 0] = 1
            at = torch.arange(tokens, device=_device())
            order = torch.where(taken > 0, at, tokens).sort(dim=1).values
            state["order"] = torch.where(order < tokens, order, -1).to(torch.int32)
    elif kind == "attention":
        _cache(case, normal, state)
        state["q"] = normal(batch, tokens, case["heads"], case["size"], scale=2.0, dtype=dtype)
        state["parents"] = _parents(case, normal) if case["tree"] else None
    else:
        vocabulary = case["vocabulary"]
        state["logits"] = normal(batch, tokens, vocabulary, scale=2.5, dtype=dtype)
        state["parents"] = _parents(case, normal) if case["tree"] else None
        parents = state["parents"].to(torch.int64) if case["tree"] else torch.arange(-1, tokens - 1, device=_device()).expand(batch, tokens)
        # a good draft: two thirds of the tokens are what the model says after their parents, the first of equal ones
        said = _first_largest(state["logits"])
        follow = torch.gather(said, 1, parents.clamp(min=0))
        other = normal.integers(0, vocabulary, batch, tokens)
        state["tokens"] = torch.where(normal.uniform(batch, tokens) < 0.67, follow, other).to(torch.int32)
    return state


# ------------------------------------------------------------------------------------------------ plain forms


def _slots(state, count):
    """Page and row of the positions behind each entry's length."""
    page = state["case"]["page"]
    at = state["lengths"].to(torch.int64)[:, None] + torch.arange(count, device=_device())
    return torch.gather(state["table"].to(torch.int64), 1, at // page), at % page, at


def _turned(x, cos, sin, rotated, interleaved):
    part = x[..., :rotated].to(torch.float32)
    if interleaved:
        a, b = part[..., 0::2], part[..., 1::2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2)
    else:
        a, b = part[..., :rotated // 2], part[..., rotated // 2:]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)
    return torch.cat([turned.to(x.dtype), x[..., rotated:]], dim=-1)


def _plain_append(state):
    case = state["case"]
    tokens, rotated = case["tokens"], case["rotated"]
    pages, rows, at = _slots(state, tokens)
    k, v, order = state["k"], state["v"], state["order"]
    place = state["positions"]
    place = at[None] if place is None else place
    if order is not None:
        # what is not taken goes where the first token of the path goes, again
        first = torch.zeros_like(at)
        taken = order >= 0
        target = torch.where(taken, torch.arange(tokens, device=at.device), first)
        source = torch.gather(order.to(torch.int64), 1, target)
        pages, rows, at = (torch.gather(t, 1, target) for t in (pages, rows, at))
        place = at[None] if state["positions"] is None else torch.gather(place, 2, source[None].expand(place.shape))
        pick = source[:, :, None, None].expand(k.shape)
        k, v = torch.gather(k, 1, pick), torch.gather(v, 1, pick)
    out = []
    if rotated:
        axis = torch.repeat_interleave(torch.arange(case["axes"], device=at.device) if place.shape[0] > 1 else torch.zeros(case["axes"], dtype=torch.int64, device=at.device),
                                       torch.tensor(_sections(case), device=at.device), output_size=rotated // 2)
        angles = place[axis].permute(1, 2, 0).to(torch.float64) * state["frequencies"].to(torch.float64)
        cos, sin = (f(angles).to(torch.float32)[:, :, None, :] for f in (torch.cos, torch.sin))
        k = _turned(k, cos, sin, rotated, case["interleaved"])
        if state["q"] is not None:
            out.append(_turned(state["q"], cos, sin, rotated, case["interleaved"]))
    state["k_pages"][pages, :, rows] = k
    state["v_pages"][pages, :, rows] = v
    return [state["k_pages"], state["v_pages"], *out]


def _seen(state, keys):
    """Which of the keys each row sees: [batch, tokens, keys]."""
    case = state["case"]
    batch, tokens = case["batch"], case["tokens"]
    device = state["lengths"].device
    own_tokens = torch.eye(tokens, dtype=torch.bool, device=device).expand(batch, tokens, tokens)
    if state["parents"] is None:
        own_tokens = torch.ones(tokens, tokens, dtype=torch.bool, device=device).tril().expand(batch, tokens, tokens)
    else:
        # ancestors twice as far with each step
        lines, up = own_tokens, state["parents"].to(torch.int64)
        for _ in range(max(tokens - 1, 1).bit_length()):
            more = torch.gather(lines, 1, up.clamp(min=0)[:, :, None].expand(lines.shape)) & (up >= 0)[:, :, None]
            lines = lines | more
            up = torch.where(up >= 0, torch.gather(up, 1, up.clamp(min=0)), up)
        own_tokens = lines
    at = torch.arange(keys, device=device) - state["lengths"].to(torch.int64)[:, None]   # counted from the call's first token
    inside = (at >= 0) & (at < tokens)
    picked = torch.gather(own_tokens, 2, at.clamp(0, tokens - 1)[:, None, :].expand(batch, tokens, keys))
    return (at < 0)[:, None, :] | (picked & inside[:, None, :])


def _plain_attention(state):
    case = state["case"]
    batch, tokens, kv_heads, size = case["batch"], case["tokens"], case["kv_heads"], case["size"]
    group = case["heads"] // kv_heads
    table = state["table"].to(torch.int64)
    keys = table.shape[1] * case["page"]
    k = state["k_pages"][table].to(torch.float32).permute(0, 2, 4, 1, 3).reshape(batch, kv_heads, size, keys)
    q = state["q"].to(torch.float32).reshape(batch, tokens, kv_heads, group, size).permute(0, 2, 3, 1, 4).reshape(batch, kv_heads, group * tokens, size)
    scores = torch.matmul(q, k).mul_(1.0 / math.sqrt(size)).reshape(batch, kv_heads, group, tokens, keys)
    del k
    scores.masked_fill_(~_seen(state, keys)[:, None, None], -math.inf)
    # (every row sees itself)
    maps = torch.exp(scores.sub_(scores.amax(dim=-1, keepdim=True)))
    maps /= maps.sum(dim=-1, keepdim=True)
    v = state["v_pages"][table].to(torch.float32).permute(0, 2, 1, 3, 4).reshape(batch, kv_heads, keys, size)
    out = torch.matmul(maps.reshape(batch, kv_heads, group * tokens, keys), v).reshape(batch, kv_heads, group, tokens, size)
    return out.permute(0, 3, 1, 2, 4).reshape(batch, tokens, case["heads"], size).to(state["q"].dtype)


def _first_largest(x):
    """The place of the largest value along the last axis, the first of equal ones."""
    places = torch.arange(x.shape[-1], device=x.device)
    return torch.where(x == x.amax(dim=-1, keepdim=True), places, x.shape[-1]).amin(dim=-1)


def _plain_acceptance(state):
    case, tokens = state["case"], state["tokens"].to(torch.int64)
    batch, count = tokens.shape
    said = _first_largest(state["logits"])
    places = torch.arange(count, device=tokens.device)
    parents = state["parents"].to(torch.int64) if case["tree"] else (places - 1).expand(batch, count)
    node = torch.zeros(batch, 1, dtype=torch.int64, device=tokens.device)
    path, going = [node], torch.ones_like(node, dtype=torch.bool)
    for _ in range(count - 1):
        fits = (parents == node) & (tokens == torch.gather(said, 1, node))
        child = torch.where(fits, places, count).amin(dim=1, keepdim=True)
        going = going & (child < count)
        node = torch.where(going, child, node)
        path.append(torch.where(going, child, -1))
    path = torch.cat(path, dim=1).to(torch.int32)
    return [path, (path >= 0).sum(dim=1).to(torch.int32), torch.gather(said, 1, node)[:, 0].to(torch.int32)]


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


NODES = {"append": ("PagedCacheAppend", ("k", "v", "k_pages", "v_pages", "table", "lengths", "frequencies", "positions", "order", "q")),
         "attention": ("TreeAttention", ("q", "k_pages", "v_pages", "table", "lengths", "parents")),
         "acceptance": ("DraftAcceptance", ("logits", "tokens", "parents"))}


def _built(state):
    """The node's model and the tensors of a call."""
    case, kind = state["case"], state["case"]["kind"]
    op, names = NODES[kind]
    like = lambda name, tensor: None if tensor is None else (name, ELEMENTS[tensor.dtype], tuple(tensor.shape))  # noqa: E731
    attributes = ()
    if kind == "append":
        outputs = (like("k_pages_out", state["k_pages"]), like("v_pages_out", state["v_pages"]), like("q_out", state["q"]))
        if case["rotated"]:
            sections = _sections(case) if state["positions"] is not None else [case["rotated"] // 2]
            attributes = (("sections", tuple(sections)), ("interleaved", int(case["interleaved"])))
    elif kind == "attention":
        outputs = (like("o", state["q"]),)
    else:
        outputs = (like("path", state["tokens"]), ("count", 6, (case["batch"],)), ("next", 6, (case["batch"],)))
    model = _model(op, tuple(like(n, state[n]) for n in names), outputs, attributes)
    return model, tuple(state[n] for n in names if state[n] is not None)


def run(state):
    if not own:
        return {"append": _plain_append, "attention": _plain_attention, "acceptance": _plain_acceptance}[state["case"]["kind"]](state)
    if "model" not in state:
        state["model"] = _built(state)
    model, tensors = state["model"]
    out = model(*tensors)
    return list(out) if isinstance(out, tuple) else out


# ------------------------------------------------------------------------------------------------ floors


def work(case):
    kind, item, batch, tokens = case["kind"], BYTES[case["type"]], case["batch"], case["tokens"]
    if kind == "acceptance":
        count = batch * tokens * case["vocabulary"]
        return {"bytes": float(item * count + 4 * batch * (3 * tokens + 2)), "flops": float(count)}
    if kind == "append":
        taken = batch * (1 + 0.3 * (tokens - 1) if case["order"] else tokens)
        values = taken * (case["heads"] + 2 * case["kv_heads"]) * case["size"]
        turned = taken * (case["heads"] + case["kv_heads"]) * case["rotated"]
        small = 4 * taken + 8 * case["axes"] * taken * (case["axes"] > 1) + 2 * case["rotated"]
        return {"bytes": float(2 * item * values + small), "flops": 3.0 * turned}
    heads, kv_heads, size = case["heads"], case["kv_heads"], case["size"]
    context = case["context"] * 2 / 3 if case["ragged"] else case["context"]   # lengths lie between a third and all of it
    line = math.log(tokens) + 1 if case["tree"] else (tokens + 1) / 2          # tokens of the call that a row sees, on average
    values = 2 * batch * size * (heads * tokens + kv_heads * (context + tokens))
    return {"bytes": float(item * values + 4 * batch * context / case["page"]), "flops": 4.0 * batch * heads * size * tokens * (context + line)}


# ------------------------------------------------------------------------------------------------ the definitions in 64 bits


def _exact_append(case, state):
    k_pages, v_pages = state["k_pages"].double(), state["v_pages"].double()
    table, page = state["table"].long(), case["page"]
    pairs = case["rotated"] // 2

    def turned(x, position):   # x: [..., tokens, heads, size], position(pair) -> [..., tokens]
        y, axis_end, axis = x.double(), 0, -1
        ends = [sum(_sections(case)[:i + 1]) for i in range(case["axes"])]
        for pair in range(pairs):
            axis = next(a for a, end in enumerate(ends) if pair < end)
            i, j = (2 * pair, 2 * pair + 1) if case["interleaved"] else (pair, pair + pairs)
            turn = torch.polar(torch.ones((), dtype=torch.float64, device=x.device), position(axis).double() * state["frequencies"][pair].double())[..., None]
            z = torch.complex(x[..., i].double(), x[..., j].double()) * turn
            y[..., i], y[..., j] = z.real, z.imag
        return y

    for b in range(case["batch"]):
        source = torch.arange(case["tokens"], device=table.device)
        if state["order"] is not None:
            source = state["order"][b][state["order"][b] >= 0].long()
        at = int(state["lengths"][b]) + torch.arange(len(source), device=table.device)
        k = state["k"][b, source]
        if pairs:
            k = turned(k, lambda axis: at if state["positions"] is None else state["positions"][axis, b, source])
        k_pages[table[b, at // page], :, at % page] = k.double()
        v_pages[table[b, at // page], :, at % page] = state["v"][b, source].double()
    out = [k_pages, v_pages]
    if state["q"] is not None:
        at = state["lengths"].long()[:, None] + torch.arange(case["tokens"], device=table.device)
        out.append(turned(state["q"], lambda axis: at if state["positions"] is None else state["positions"][axis]))
    return out


def _exact_attention(case, state):
    heads, group, size, tokens = case["heads"], case["heads"] // case["kv_heads"], case["size"], case["tokens"]
    out = torch.zeros(case["batch"], tokens, heads, size, dtype=torch.float64, device=state["q"].device)
    for b in range(case["batch"]):
        length = int(state["lengths"][b])
        pages = state["table"][b, :-(-(length + tokens) // case["page"])].long()
        lines = torch.ones(tokens, tokens, dtype=torch.bool).tril()
        if case["tree"]:
            lines.zero_()
            for i, parent in enumerate(state["parents"][b].tolist()):
                if parent >= 0:
                    lines[i] = lines[parent]
                lines[i, i] = True
        lines = lines.to(out.device)
        for kv in range(case["kv_heads"]):
            k, v = (state[n][pages, kv].reshape(-1, size)[:length + tokens].double() for n in ("k_pages", "v_pages"))
            for h in range(kv * group, (kv + 1) * group):
                for rows in torch.arange(tokens, device=out.device).split(1024):
                    s = state["q"][b, rows, h].double() @ k.T / math.sqrt(size)
                    s[:, length:] = s[:, length:].where(lines[rows], -math.inf)
                    out[b, rows, h] = torch.softmax(s, -1) @ v
    return out


def _exact_acceptance(case, state):
    said = [[int((row == row.max()).nonzero()[0, 0]) for row in entry] for entry in state["logits"]]
    drafted = state["tokens"].tolist()
    parents = state["parents"].tolist() if case["tree"] else [list(range(-1, case["tokens"] - 1))] * case["batch"]
    paths, after = [], []
    for b in range(case["batch"]):
        path = [0]
        while True:
            children = [i for i in range(1, case["tokens"]) if parents[b][i] == path[-1] and drafted[b][i] == said[b][path[-1]]]
            if not children:
                break
            path.append(children[0])
        paths.append(path)
        after.append(said[b][path[-1]])
    whole = lambda values: torch.tensor(values, dtype=torch.int32, device=state["tokens"].device)  # noqa: E731
    return [whole([p + [-1] * (case["tokens"] - len(p)) for p in paths]), whole([len(p) for p in paths]), whole(after)]


def exact(case, seed):
    state = prepare(case, seed)
    return {"append": _exact_append, "attention": _exact_attention, "acceptance": _exact_acceptance}[case["kind"]](case, state)
