"""Inputs of float32 attention whose results only the low-order parts of its operands decide, and the arithmetic of its products on the CPU.

The kernel splits a float32 in three bfloat16 numbers, its first, middle and last eight bits, and takes six of the nine products of two such sums. U = 2^-24 is half a
step of float32."""
import numpy as np
import torch

import llm_operators as R

U = 2.0 ** -24
ALL = ((0, 2), (1, 1), (2, 0), (0, 1), (1, 0), (0, 0))   # smallest first: what the kernel adds up
WEIGHT = 0.5   # l: there are no learned vectors, and lambda_init is exact


def parts(x):
    """The three parts of float32 values: what is left has no bits after the third."""
    x, found = np.asarray(x, dtype=np.float32), []
    for _ in range(3):
        found.append((x.view(np.uint32) & np.uint32(0xffff0000)).view(np.float32))
        x = x - found[-1]
    return found


def product(a, b, taken=ALL):
    """a [m, n] b [n, p] in float32: the sums of 16 products of parts at a time, one pair of parts after the other."""
    pa, pb = parts(a), parts(b)
    acc = np.zeros((a.shape[0], b.shape[1]), dtype=np.float32)
    for n in range(0, a.shape[1], 16):
        for i, j in taken:
            acc = (acc + (pa[i][:, n:n + 16].astype(np.float64) @ pb[j][n:n + 16].astype(np.float64)).astype(np.float32)).astype(np.float32)
    return acc


def emulated(case, scores=ALL, values=ALL):
    """The results of one head as the kernel computes them, with the products of parts that are named."""
    q, k, v = (case[n].numpy() for n in "qkv")
    out = []
    for m in range(2):
        s = product(q[0, :, m], np.ascontiguousarray(k[0, :, m].T), scores) * np.float32(case["scale"])
        p = np.exp(s - s.max(-1, keepdims=True)).astype(np.float32)
        out.append(product(p, v[0, :, 0], values) / p.sum(-1, dtype=np.float32, keepdims=True))
    return torch.from_numpy(out[0] - np.float32(WEIGHT) * out[1])[None, :, None]


def expected(case):
    none = [torch.zeros(0, dtype=torch.float32, device=case["q"].device)] * 4
    return R.differential_attention(case["q"], case["k"], case["v"], none, WEIGHT, case["scale"])


def _random(rng, *shape, bits=24):
    """Numbers of [128, 256) with so many bits."""
    return ((1 << (bits - 1)) + rng.integers(0, 1 << (bits - 1), shape)) * 2.0 ** (8 - bits)


def cancelling_scores(kind, rows, d, keys, seed=0):
    """One head. Two of the keys matter: one whose score is 0, and one whose score is a sum of two or four products of up to 2^16 that cancel but for what the parts named by
    `kind` give: at most a few units. Of the first map the result is the logistic function of that score, of the second 1/2.

    All partial products that the kernel leaves out are 0 here, those that it takes are exact, and four terms of up to `largest` and one sum are added where they meet:
    with a rounding or a truncation each, 2 U, the score is off by less than 16 U largest, and the result, whose slope is at most 1/4, by 4 U largest; the exponentials,
    sums and the quotient give less than 32 U more."""
    rng = np.random.default_rng(seed)
    q, k, v = np.zeros((1, rows, 2, d)), np.zeros((1, keys, 2, d)), np.zeros((1, keys, 1, 2 * d))
    blocks = d // 16 - 1                                                 # the last one holds what hides the other keys
    zero, one = rng.choice(keys, 2, replace=False)
    q[0, :, :, -1], k[0, :, :, -1] = 64.0, -64.0
    k[0, [zero, one], :, -1] = 0.0
    v[0, one, 0] = rng.choice([-1.0, 1.0], 2 * d)
    largest = np.zeros(rows)
    places = [16 * b + rng.choice(16, 4, replace=False) for b in range(blocks)]
    if kind == "middle":   # (h + m) (h' + m') - h h' - h m' - m h'
        h, m = _random(rng, blocks, bits=8), _random(rng, blocks, bits=8) * 2.0 ** -8 * rng.choice([-1, 1], blocks)
        h, m = np.where(m < 0, h - 1, h), np.where(m < 0, m + 1, m)       # parts have the value's sign
        for b in range(blocks):
            k[0, one, 0, places[b]] = h[b] + m[b], h[b], m[b], h[b]
        for r in range(rows):
            a, c = _random(rng, bits=8), _random(rng, bits=8) * 2.0 ** -8
            q[0, r, 0, places[r % blocks]] = a + c, -a, -a, -c
            largest[r] = (a + c) * (h + m)[r % blocks]
    else:   # a (b - b'), b and b' alike in their first 16 bits
        first = np.floor(_random(rng, blocks if kind == "keys" else rows, bits=16) * 2.0 ** 8) * 2.0 ** -8
        pair = first[:, None] + rng.integers(0, 256, (len(first), 2)) * 2.0 ** -16
        other = _random(rng, rows if kind == "keys" else blocks, bits=8)
        for b in range(blocks):
            k[0, one, 0, places[b][:2]] = pair[b] if kind == "keys" else [other[b], -other[b]]
        for r in range(rows):
            q[0, r, 0, places[r % blocks][:2]] = [other[r], -other[r]] if kind == "keys" else pair[r]
            largest[r] = 256 * (other[r] if kind == "keys" else other[r % blocks])
    case = {n: torch.from_numpy(t.astype(np.float32)) for n, t in zip("qkv", (q, k, v))}
    assert all(np.array_equal(case[n].numpy(), t) for n, t in zip("qkv", (q, k, v)))   # nothing was rounded
    return {**case, "scale": 1.0, "bound": (4 * U * torch.from_numpy(largest) + 32 * U)[None, :, None, None]}


def few_keys(rows, d, keys, seed=0):
    """One head; a few keys of nearly equal weight, values of 24 bits. Scores are one product, exact (seven bits and one) and below 2: the base of two and the difference from
    the largest move a power by 4 U, the power itself is off by 2 U, and both numerator and sum take part, 12 U. `keys` terms are added twice, truncated 2 U or rounded
    U each; the last addition of the six passes 2 U; the products that are left out are below 2^-21, 8 U; quotient, product and difference 3 U: together
    (3 keys + 25) U of sum (P1 + l P2) |V|."""
    rng = np.random.default_rng(seed)
    q, k = np.zeros((1, rows, 2, d)), np.zeros((1, keys, 2, d))
    q[0, :, :, 5], k[0, :, :, 5] = rng.integers(64, 128, (rows, 2)) / 64, rng.choice([-1.0, -0.5, 0.5, 1.0], (keys, 2))
    v = rng.uniform(0.5, 2, (1, keys, 1, 2 * d))
    return {**{n: torch.from_numpy(t.astype(np.float32)) for n, t in zip("qkv", (q, k, v))}, "scale": 1.0, "relative": (3 * keys + 25) * U}


def one_key(rows, d, seed=0):
    """One key, whose weight is exactly 1: the result is half of its value, whose three parts are added (a rounding or a truncation each, 2 U)."""
    rng = np.random.default_rng(seed)
    q, k, v = rng.normal(size=(1, rows, 2, d)), np.zeros((1, 1, 2, d)), rng.uniform(0.5, 2, (1, 1, 1, 2 * d))
    return {**{n: torch.from_numpy(t.astype(np.float32)) for n, t in zip("qkv", (q, k, v))}, "scale": 1.0, "relative": 6 * U}


def error(case, got):
    """The largest error of `got` as a multiple of the bound."""
    want, size = expected(case)
    bound = case["bound"].to(size.device) if "bound" in case else case["relative"] * size
    return float(((got.double() - want).abs() / bound).max())


def normal_case(b, sq, sk, h, g, d, seed=0):
    """Heads of normal numbers, and a bound for the 2-norm of the error: roundings of products of this kind are as good as independent. A score of standard deviation 2 is
    rounded 6 d / 16 times (48 at most), U / sqrt(3) of it each and U 2^-0.5 of it by the products that are left out on average: 10 U in all; its power as much, numerator
    and sum both, 14 U relative to each map. Two maps with l = 1/2 are less than 1.2 of their difference, as they are independent: 17 U, and about 5 U for the powers, sums
    and quotients: 2^-19.4 is 24 U."""
    rng = np.random.default_rng(seed)
    made = {n: torch.from_numpy(rng.normal(size=s).astype(np.float32)) for n, s in zip("qkv", ((b, sq, 2 * h, d), (b, sk, 2 * g, d), (b, sk, g, 2 * d)))}
    made["q"] *= 2
    return {**made, "scale": d ** -0.5}


NORM = 24 * U


def norm_error(case, got):
    want, _ = expected(case)
    return float((got.double() - want).norm() / want.norm())
