"""Definitions in float64 of the operators that verify drafted tokens over a paged cache, and a small transformer that uses them, as graphs and as sums."""
import numpy as np
import torch

import dace_onnx_amd.onnx as donnx
from dace_onnx_amd.onnx.proto import helper, numpy_helper
import llm_operators as R


def append_model(k, v, k_pages, v_pages, table, lengths, frequencies=None, positions=None, order=None, q=None, **attributes):
    inputs = [("k", k), ("v", v), ("k_pages", k_pages), ("v_pages", v_pages), ("table", table), ("lengths", lengths), ("frequencies", frequencies),
              ("positions", positions), ("order", order), ("q", q)]
    outputs = [("k_pages_out", k_pages.dtype, tuple(k_pages.shape)), ("v_pages_out", v_pages.dtype, tuple(v_pages.shape)),
               None if q is None else ("q_out", q.dtype, tuple(q.shape))]
    return R.model("PagedCacheAppend", inputs, outputs, **attributes), [t for _, t in inputs if t is not None]


def attention_model(q, k_pages, v_pages, table, lengths, parents=None, **attributes):
    inputs = [("q", q), ("k_pages", k_pages), ("v_pages", v_pages), ("table", table), ("lengths", lengths), ("parents", parents)]
    return R.model("TreeAttention", inputs, [("o", q.dtype, tuple(q.shape))], **attributes), [t for _, t in inputs if t is not None]


def acceptance_model(logits, tokens, parents=None):
    inputs = [("logits", logits), ("tokens", tokens), ("parents", parents)]
    batch = logits.shape[0]
    return R.model("DraftAcceptance", inputs, [("path", torch.int32, tuple(logits.shape[:2])), ("count", torch.int32, (batch,)), ("next", torch.int32, (batch,))]), \
        [t for _, t in inputs if t is not None]


# ---------------------------------------------------------------------------------------------- definitions


def append(k, v, k_pages, v_pages, table, lengths, frequencies=None, positions=None, order=None, q=None, sections=None, interleaved=0):
    """The pages afterwards (in float64), which rows [pages, row] of them were written, the turned queries, and each turned value's pair as |a| + |b| (0 for the others)."""
    (B, S, G, D), (P, _, page, _) = k.shape, k_pages.shape
    k_after, v_after = k_pages.double(), v_pages.double()
    written = torch.zeros(P, page, dtype=torch.bool)
    pairs = 0 if frequencies is None else len(frequencies)
    sections = sections or [pairs] + [0] * ((1 if positions is None else positions.shape[0]) - 1)
    q_after = None if q is None else q.double()
    k_size, q_size = torch.zeros_like(k_after), None if q is None else torch.zeros_like(q_after)

    def turn(x, places):   # x [heads, D], places: a number for each axis
        y, size, pair = x.double(), torch.zeros(x.shape, dtype=torch.float64, device=x.device), 0
        for axis, count in enumerate(sections):
            for _ in range(count):
                i, j = (2 * pair, 2 * pair + 1) if interleaved else (pair, pair + pairs)
                angle = torch.tensor(float(places[axis]), dtype=torch.float64) * frequencies[pair].double().cpu()
                a, b = x[:, i].double(), x[:, j].double()
                y[:, i], y[:, j] = a * angle.cos().item() - b * angle.sin().item(), b * angle.cos().item() + a * angle.sin().item()
                size[:, i] = size[:, j] = a.abs() + b.abs()
                pair += 1
        return y, size

    for b in range(B):
        start = max(int(lengths[b]), 0)
        for i in range(S if q is not None else 0):
            q_after[b, i], q_size[b, i] = turn(q[b, i], [start + i] if positions is None else positions[:, b, i].tolist())
        for j in range(S if order is None else order.shape[1]):
            i, number = (j if order is None else int(order[b, j])), start + j
            if not 0 <= i < S or number // page >= table.shape[1] or not 0 <= int(table[b, number // page]) < P:
                continue
            to, row = int(table[b, number // page]), number % page
            k_after[to, :, row], k_size[to, :, row] = turn(k[b, i], [number] if positions is None else positions[:, b, i].tolist())
            v_after[to, :, row] = v[b, i].double()
            written[to, row] = True
    return k_after, v_after, written, q_after, k_size, q_size


def lines(parents):
    """Which tokens [S, S] each of one entry's tokens sees."""
    S = len(parents)
    seen = torch.eye(S, dtype=torch.bool)
    for i, parent in enumerate(parents):
        if 0 <= parent < i:
            seen[i] |= seen[parent]
    return seen


def attention(q, k_pages, v_pages, table, lengths, parents=None, scale=None):
    """The result, and sum_j P |V|: what an error relative to the probabilities or the values goes by. Nothing that a row does not see is looked at."""
    (B, S, H, D), (P, G, page, _) = q.shape, k_pages.shape
    scale = D ** -0.5 if scale is None else scale
    capacity = page * table.shape[1]
    out = torch.zeros(B, S, H, D, dtype=torch.float64, device=q.device)
    size = torch.zeros_like(out)
    for b in range(B):
        length = min(max(int(lengths[b]), 0), capacity)
        keys = min(length + S, capacity)
        numbers = torch.arange(keys, device=q.device)
        pages = table[b].long().clamp(0, P - 1)[numbers // page] if keys else numbers
        seen = torch.ones(S, keys, dtype=torch.bool, device=q.device)
        own = lines(list(range(-1, S - 1)) if parents is None else parents[b].tolist()).to(q.device)
        seen[:, length:] = own[:, :keys - length]
        for h in range(H):
            g = h // (H // G)
            s = scale * q[b, :, h].double() @ k_pages[pages, g, numbers % page].double().t()
            s = torch.where(seen, s, -torch.inf)
            value = v_pages[pages, g, numbers % page].double()
            top = s.amax(-1, keepdim=True) if keys else s.new_zeros(S, 1)
            e = torch.exp(s - torch.where(top == -torch.inf, 0.0, top))
            e = torch.where(seen, e, 0.0)
            total = e.sum(-1, keepdim=True)
            e = e / torch.where(total == 0, 1.0, total)
            odd = (~torch.isfinite(value)).any(-1)
            out[b, :, h], size[b, :, h] = e @ torch.where(odd[:, None], 0.0, value), e @ torch.where(odd[:, None], 0.0, value).abs()
            for n in odd.nonzero()[:, 0].tolist():
                for i in seen[:, n].nonzero()[:, 0].tolist():
                    out[b, i, h] += e[i, n] * value[n]
    return out, size


def acceptance(logits, tokens, parents=None):
    paths, counts, after = [], [], []
    for b in range(len(logits)):
        row = logits[b].double().cpu().numpy()
        said = [int(np.argmax(np.where(np.isnan(r), -np.inf, r))) if not np.isnan(r).all() else 0 for r in row]
        for i, r in enumerate(row):   # of minus infinity and NaN the first number, whichever it is
            if not np.isnan(r).all() and np.isnan(r[said[i]]):
                said[i] = int(np.flatnonzero(~np.isnan(r))[0])
        up = list(range(-1, tokens.shape[1] - 1)) if parents is None else [p if 0 <= p < i else -1 for i, p in enumerate(parents[b].tolist())]
        path = [0]
        while True:
            child = [i for i in range(1, len(up)) if up[i] == path[-1] and int(tokens[b, i]) == said[path[-1]]]
            if not child:
                break
            path.append(child[0])
        paths.append(path + [-1] * (len(up) - len(path)))
        counts.append(len(path))
        after.append(said[path[-1]])
    return [torch.tensor(x, dtype=torch.int32) for x in (paths, counts, after)]


# ---------------------------------------------------------------------------------------------- a small transformer

LAYERS, HEADS, GROUPS, SIZE, HIDDEN, VOCABULARY = 2, 4, 2, 64, 96, 211


def transformer_weights(seed):
    rng = np.random.default_rng(seed)
    n = lambda *shape, scale: rng.normal(size=shape, scale=scale).astype(np.float32)   # noqa: E731
    weights = {"embedding": n(VOCABULARY, HIDDEN, scale=1.0), "out": n(HIDDEN, VOCABULARY, scale=HIDDEN ** -0.5), "gain": np.ones(HIDDEN, dtype=np.float32),
               "frequencies": (10000.0 ** (-np.arange(SIZE // 2) / (SIZE // 2))).astype(np.float32)}
    for i in range(LAYERS):
        weights[f"wq{i}"] = n(HIDDEN, HEADS * SIZE, scale=2 * HIDDEN ** -0.5)
        weights[f"wk{i}"], weights[f"wv{i}"] = (n(HIDDEN, GROUPS * SIZE, scale=HIDDEN ** -0.5) for _ in range(2))
        weights[f"wo{i}"] = n(HEADS * SIZE, HIDDEN, scale=2 * (HEADS * SIZE) ** -0.5)
    return weights


def _graph(nodes, inputs, outputs, initializers):
    infos = lambda values: [helper.make_tensor_value_info(n, R.ELEMENT[t], list(s)) for n, t, s in values]   # noqa: E731
    return helper.make_model(helper.make_graph(nodes, "graph", infos(inputs), infos(outputs), initializer=[numpy_helper.from_array(v, name=k) for k, v in initializers.items()]))


def verifying_graph(weights, batch, tokens, cache, columns):
    """Tokens of a tree through the layers, whose caches it updates: the path that the model takes, and the keys and values as they were before they were turned."""
    F32, I32 = torch.float32, torch.int32
    nodes = []
    node = lambda op, ins, outs, **a: nodes.append(helper.make_node(op, ins, outs, name=f"{op.lower()}{len(nodes)}", **a))   # noqa: E731
    inputs = [("x", F32, (batch, tokens, HIDDEN)), ("drafted", I32, (batch, tokens)), ("parents", I32, (batch, tokens)), ("positions", I32, (1, batch, tokens)),
              ("table", I32, (batch, columns)), ("lengths", I32, (batch,))]
    outputs = [("path", I32, (batch, tokens)), ("count", I32, (batch,)), ("next", I32, (batch,))]
    constants = {k: w for k, w in weights.items() if k != "embedding"}
    for name, heads in (("q", HEADS), ("kv", GROUPS)):
        constants[name + "_shape"] = np.array([batch, tokens, heads, SIZE], dtype=np.int64)
    constants["o_shape"] = np.array([batch, tokens, HEADS * SIZE], dtype=np.int64)
    stream = "x"
    for i in range(LAYERS):
        node("SkipRMSNormalization", [stream, "gain"], [f"n{i}"])
        for c, shape in (("q", "q_shape"), ("k", "kv_shape"), ("v", "kv_shape")):
            node("MatMul", [f"n{i}", f"w{c}{i}"], [f"{c}_flat{i}"])
            node("Reshape", [f"{c}_flat{i}", shape], [f"{c}{i}"])
        node("PagedCacheAppend", [f"k{i}", f"v{i}", f"k_pages{i}", f"v_pages{i}", "table", "lengths", "frequencies", "positions", "", f"q{i}"],
             [f"k_after{i}", f"v_after{i}", f"q_turned{i}"])
        node("TreeAttention", [f"q_turned{i}", f"k_after{i}", f"v_after{i}", "table", "lengths", "parents"], [f"o{i}"])
        node("Reshape", [f"o{i}", "o_shape"], [f"o_flat{i}"])
        node("MatMul", [f"o_flat{i}", f"wo{i}"], [f"p{i}"])
        node("Add", [stream, f"p{i}"], [f"x{i}"])
        stream = f"x{i}"
        inputs += [(f"{c}_pages{i}", F32, cache) for c in "kv"]
        outputs += [(f"{c}{i}", F32, (batch, tokens, GROUPS, SIZE)) for c in "kv"]
    node("SkipRMSNormalization", [stream, "gain"], ["last"])
    node("MatMul", ["last", "out"], ["logits"])
    node("DraftAcceptance", ["logits", "drafted", "parents"], ["path", "count", "next"])
    return _graph(nodes, inputs, outputs, constants)


def keeping_graph(weights, batch, tokens, cache, columns):
    """The tokens on the path to where they belong, in the caches of all layers."""
    F32, I32 = torch.float32, torch.int32
    inputs = [("path", I32, (batch, tokens)), ("table", I32, (batch, columns)), ("lengths", I32, (batch,))]
    nodes, outputs = [], []
    for i in range(LAYERS):
        inputs += [(f"{c}{i}", F32, (batch, tokens, GROUPS, SIZE)) for c in "kv"] + [(f"{c}_pages{i}", F32, cache) for c in "kv"]
        nodes.append(helper.make_node("PagedCacheAppend", [f"k{i}", f"v{i}", f"k_pages{i}", f"v_pages{i}", "table", "lengths", "frequencies", "", "path"],
                                      [f"k_after{i}", f"v_after{i}"], name=f"keep{i}"))
        outputs += [(f"{c}_after{i}", F32, cache) for c in "kv"]
    return _graph(nodes, inputs, outputs, {"frequencies": weights["frequencies"]})


def greedy(weights, prompt, count):
    """`count` tokens behind `prompt` by whole passes in float64, and the least distance between the two largest logits on the way."""
    w = {k: torch.from_numpy(v).double() for k, v in weights.items()}
    tokens, least = list(prompt), float("inf")
    norm = lambda x: x / (x.pow(2).mean(-1, keepdim=True) + 1e-5).sqrt()   # noqa: E731
    for _ in range(count):
        S = len(tokens)
        x = w["embedding"][tokens]
        angle = torch.arange(S, dtype=torch.float64)[:, None] * w["frequencies"]
        cos, sin = angle.cos()[:, None], angle.sin()[:, None]

        def turned(t):
            a, b = t[..., :SIZE // 2], t[..., SIZE // 2:]
            return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)

        for i in range(LAYERS):
            q = turned((norm(x) @ w[f"wq{i}"]).reshape(S, HEADS, SIZE))
            k = turned((norm(x) @ w[f"wk{i}"]).reshape(S, GROUPS, SIZE)).repeat_interleave(HEADS // GROUPS, 1)
            v = (norm(x) @ w[f"wv{i}"]).reshape(S, GROUPS, SIZE).repeat_interleave(HEADS // GROUPS, 1)
            s = torch.einsum("ihd,jhd->hij", q, k) / SIZE ** 0.5
            s = s.masked_fill(torch.ones(S, S, dtype=torch.bool).triu(1), -torch.inf)
            x = x + torch.einsum("hij,jhd->ihd", torch.softmax(s, -1), v).reshape(S, -1) @ w[f"wo{i}"]
        top = (norm(x[-1]) @ w["out"]).topk(2)
        least = min(least, float(top.values[0] - top.values[1]))
        tokens.append(int(top.indices[0]))
    return tokens[len(prompt):], least


# ---------------------------------------------------------------------------------------------- attention, row by row
# Each row of D values has a bound of its own on its error's 2-norm, of what its own scores and weights are. U = 2^-24, P the row's weights, s its scores, w = scale sqrt(sum q^2 k^2), the size
# of a random walk of a score's products.
# Scores: n products of 16 terms go to one sum (D / 16, six times that in float32), each may lose up to 2^-23 of the sum so far, towards zero: U of it on average. A sum that walks from 0 to s is
#   |s| / 2 + 0.4 w on the way. What float32 leaves out of a product is 2^-24.5 of it (one U more). The power's argument is rounded by U of itself, and the scale by 2 U: 3 U |s - largest|; the
#   power by 2 U. A weight is off by A U of itself, A = n (|s| / 2 + 0.4 w) + |s| + 3 |s - largest| + 2. Such errors are of either sign for one key and another once the sum of the weights is
#   divided by: sqrt(sum P^2 A^2 |v|^2) U, and sqrt(sum P^2 A^2) U of the result.
# Values: 12 products for 32 keys, U of their sum each, and 2^-23.5 left out; the sums of N / 32 blocks are added at random; scaling, joining and dividing are a rounding each: (16 + sqrt(N / 32)) U
#   of the result or of sqrt(sum P^2 |v|^2), whichever is larger (random values' results are as large as that).
# 16 bits: weights and results are rounded, uniformly within half a step of their binade: sqrt(1 / 3) of it, of numbers of 1 to 2 in it whose root mean square is 1.47 to 1.53 (of even logarithms,
#   of even values), so 0.4 of half a step relative to them as a mean over many, up to one half step for few: 0.4 (1 + 3 / sqrt(count)), count = D results, or as many keys as the weights are
#   spread over. The two are independent.


def attention_rows(q, k_pages, v_pages, table, lengths, parents=None, without=None, scores=None, weights=None):
    """The result, and the bound of every row [B, S, H]. Every row sees a key, and what rows see is finite. ``without``: (entry, key) that is left out; ``scores`` and ``weights`` compute the two
    products in another way."""
    (B, S, H, D), (P, G, page, _) = q.shape, k_pages.shape
    U, half, scale = 2.0 ** -24, R.HALF[q.dtype], D ** -0.5
    products = D / 16 * (6 if q.dtype == torch.float32 else 1)
    scores = scores or (lambda a, b: a @ b.t())
    weights = weights or (lambda a, b: a @ b)
    out = torch.zeros(B, S, H, D, dtype=torch.float64, device=q.device)
    bound = torch.zeros(B, S, H, dtype=torch.float64, device=q.device)
    spread = lambda count: (0.4 * (1 + 3 / count.sqrt())).clamp(max=1.0)   # noqa: E731
    for b in range(B):
        length = int(lengths[b])
        numbers = torch.arange(min(length + S, page * table.shape[1]), device=q.device)
        pages = table[b].long()[numbers // page]
        seen = torch.ones(S, len(numbers), dtype=torch.bool, device=q.device)
        own = lines(list(range(-1, S - 1)) if parents is None else parents[b].tolist()).to(q.device)
        seen[:, length:] = own[:, :len(numbers) - length]
        if without is not None and without[0] == b:
            seen[:, without[1]] = False
        for h in range(H):
            x, k, v = q[b, :, h], k_pages[pages, h // (H // G), numbers % page], v_pages[pages, h // (H // G), numbers % page]
            s = torch.where(seen, scale * scores(x.double(), k.double()), -torch.inf)
            top = s.amax(-1, keepdim=True)
            p = torch.exp(s - top)
            total = p.sum(-1, keepdim=True)
            out[b, :, h] = weights(p, v.double()) / total
            p, s = p / total, torch.where(seen, s, 0.0)
            walk = scale * (x.double().square() @ k.double().square().t()).sqrt()
            off = torch.where(seen, products * (s.abs() / 2 + 0.4 * walk) + s.abs() + 3 * (top - s) + 2, 0.0)
            values, size = v.double().square().sum(-1), out[b, :, h].norm(dim=-1)
            each = (p.square() @ values).sqrt()
            bound[b, :, h] = U * (((p * off).square() @ values).sqrt() + (p * off).norm(dim=-1) * size + (16 + (len(numbers) / 32) ** 0.5) * torch.maximum(each, size))
            if q.dtype != torch.float32:
                keys = (p.square() @ values).square() / (p.square().square() @ values.square())
                bound[b, :, h] += half * ((spread(torch.tensor(float(D))) * size).square() + spread(keys).square() * (each.square() + p.square().sum(-1) * size.square())).sqrt()
                bound[b, :, h] += D ** 0.5 * 2.0 ** -25 * (q.dtype == torch.float16)
    return out, bound


def attention_case(seed, batch, tokens, heads, groups, d, page, context, dtype, tree=False, device="cpu"):
    """Entries of unequal lengths, pages in no order, what belongs to no token not a number."""
    g = torch.Generator().manual_seed(seed)
    normal = lambda *shape, scale=1.0: (torch.randn(*shape, generator=g) * scale).to(dtype)   # noqa: E731
    lengths = [max(context - (7 * b + 1) * context // (4 * batch), 0) if b else context for b in range(batch)]
    columns = -(-(context + tokens) // page)
    pages = batch * columns + 2
    table = torch.randperm(pages, generator=g)[:batch * columns].reshape(batch, columns).to(torch.int32)
    q, k, v = normal(batch, tokens, heads, d, scale=2.0), normal(pages, groups, page, d), normal(pages, groups, page, d)
    used = torch.zeros(pages, page, dtype=torch.bool)
    for b in range(batch):
        numbers = torch.arange(lengths[b] + tokens)
        used[table[b].long()[numbers // page], numbers % page] = True
    hidden = ~used[:, None, :, None].expand(k.shape)
    k[hidden] = v[hidden] = float("nan")
    parents = (torch.rand(batch, tokens, generator=g) * torch.arange(tokens)).to(torch.int32).clamp(max=torch.arange(tokens, dtype=torch.int32) - 1) if tree else None
    return [None if t is None else t.to(device) for t in (q, k, v, table, torch.tensor(lengths, dtype=torch.int32), parents)]


def parts_of(x, count):
    """x as `count` bfloat16 numbers, cut off one after the other, and what is left over dropped."""
    x, result = x.float(), []
    for _ in range(count):
        part = (x.view(torch.int32) & -65536).view(torch.float32)
        result.append(part.double())
        x = x - part
    return result


def by_parts(count, least):
    """A product of matrices by the partial products of `count` parts of each operand, the i-th with the j-th where i + j <= least."""
    def product(a, b):
        a, b = parts_of(a, count), parts_of(b, count)
        return sum(a[i] @ b[j] for i in range(count) for j in range(count) if i + j <= least)
    return {"scores": lambda x, k: product(x, k.t().contiguous()), "weights": product}
