"""The operators that verify drafted tokens over a paged cache on the GPU, against their definitions in float64.

Tolerances count roundings. U = 2^-24 is half a step of float32, HALF[T] half a step of the arrays' type; results of float16 below its normal range are
off by up to 2^-25 on top."""
import numpy as np
import pytest
import torch

import dace_onnx_amd.onnx as donnx
from dace_onnx_amd import _lib
import cache_operators as C
import llm_operators as R

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
F32, F16, BF = R.TYPES
I32 = torch.int32
TINY = {F32: 2.0 ** -149, F16: 2.0 ** -25, BF: 2.0 ** -134}


def normal(seed, *shape, scale=1.0, dtype=F32):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype).cuda()


def whole(values, dtype=I32):
    return torch.tensor(values, dtype=dtype).cuda()


def within(got, expected, bound):
    """|got - expected| <= bound, element by element."""
    assert got.shape == expected.shape
    error = (got.double() - expected).abs()
    worst = (error / bound).max().item() if got.numel() else 0.0
    assert worst <= 1, f"{worst:.3g} of the bound; largest error {error.max().item():.3g}"


def shuffled_table(seed, batch, columns, spare=2):
    """Every column a page of its own, in no order; the number of pages."""
    pages = batch * columns + spare
    return torch.randperm(pages, generator=torch.Generator().manual_seed(seed))[:batch * columns].reshape(batch, columns).to(I32).cuda(), pages


# ---------------------------------------------------------------------------------------------- PagedCacheAppend
# An angle is off by 2^-51 of its turns, 2 pi 2^-24 / 2 by its rounding and what cosine and sine are off by: at most 3 U of their values, which are 1 at most. Two products
# and a sum are a rounding each. A value is at most |a| + |b|.


def append_bound(size, expected, dtype, farthest):
    angle = 2 * np.pi * 2.0 ** -51 * farthest + np.pi * U + 3 * U
    return (angle + 3 * U) * size + R.HALF[dtype] * expected.abs() * (1 + 2.0 ** -7) + TINY[dtype]


def check_append(batch, tokens, groups, size, page, dtype, pairs=0, axes=0, taken=None, heads=0, interleaved=0, lengths=None, order=None, seed=0, change_table=None, wide=True):
    lengths = [7 * b + 3 for b in range(batch)] if lengths is None else lengths
    columns = max(1, -(-(max(max(lengths), 0) + max(tokens, taken or 0)) // page))
    table, pages = shuffled_table(seed, batch, columns)
    if change_table:
        change_table(table)
    k, v = normal(seed + 1, batch, tokens, groups, size, dtype=dtype), normal(seed + 2, batch, tokens, groups, size, dtype=dtype)
    kp, vp = normal(seed + 3, pages, groups, page, size, dtype=dtype), normal(seed + 4, pages, groups, page, size, dtype=dtype)
    q = normal(seed + 5, batch, tokens, heads, size, dtype=dtype) if heads else None
    f = (10000.0 ** (-torch.arange(pairs) / max(pairs, 1))).float().cuda() if pairs or heads else None
    positions = sections = None
    if axes:
        positions = torch.randint(0, 50000, (axes, batch, tokens), generator=torch.Generator().manual_seed(seed)).to(torch.int64 if wide else I32).cuda()
        sections = [pairs // axes] * (axes - 1) + [pairs - pairs // axes * (axes - 1)]
    if taken is not None and order is None:
        order = torch.randint(-2, tokens + 2, (batch, taken), generator=torch.Generator().manual_seed(seed + 6)).tolist()
    order = None if order is None else whole(order)
    lengths = whole(lengths)
    before = kp.clone(), vp.clone()
    ek, ev, written, eq, k_size, q_size = C.append(k, v, kp, vp, table, lengths, f, positions, order, q, sections, interleaved)
    attributes = {"interleaved": interleaved, **({"sections": sections} if axes else {})}
    m, inputs = C.append_model(k, v, kp, vp, table, lengths, f, positions, order, q, **(attributes if f is not None else {}))
    for _ in range(3):   # the general way, then the short one
        got = m(*inputs)
        assert got[0] is kp and got[1] is vp
        written = written.cuda()
        farthest = 50000 if axes else float(lengths.max().clamp(min=0)) + max(tokens, taken or 0)
        assert torch.equal(vp, ev.to(dtype))                                                                    # bit by bit
        untouched = ~written[:, None, :, None].expand(kp.shape)
        assert torch.equal(kp[untouched].view(torch.uint8), before[0][untouched].view(torch.uint8))
        turned = k_size > 0
        assert torch.equal(kp[~turned], ek.to(dtype)[~turned])
        within(kp[turned], ek[turned], append_bound(k_size, ek, dtype, farthest)[turned])
        if q is not None:
            within(got[2], eq, append_bound(q_size, eq, dtype, farthest))
        kp.copy_(before[0])
        vp.copy_(before[1])


@pytest.mark.parametrize("dtype", R.TYPES)
@pytest.mark.parametrize("batch, tokens, groups, size, page", [(1, 1, 1, 64, 16), (3, 1, 2, 128, 16), (2, 5, 3, 80, 1), (2, 33, 2, 64, 23), (5, 7, 1, 7, 4), (1, 300, 2, 64, 128), (2, 9, 1, 256, 8)])
def test_append_as_it_is(dtype, batch, tokens, groups, size, page):
    check_append(batch, tokens, groups, size, page, dtype)


@pytest.mark.parametrize("dtype", R.TYPES)
@pytest.mark.parametrize("interleaved", [0, 1])
@pytest.mark.parametrize("size, pairs, axes", [(64, 32, 0), (64, 24, 2), (128, 64, 3), (80, 5, 1), (80, 18, 0), (6, 2, 2), (256, 128, 0)])
def test_append_turned(dtype, interleaved, size, pairs, axes):
    check_append(2, 6, 2, size, 5, dtype, pairs, axes, heads=6, interleaved=interleaved, wide=axes != 2)


@pytest.mark.parametrize("dtype", R.TYPES)
@pytest.mark.parametrize("taken, axes", [(1, 0), (4, 0), (9, 2), (40, 0)])
def test_append_in_an_order(dtype, taken, axes):
    """Any of the tokens, some of them twice, some of them none of the call's; with more places than tokens."""
    check_append(3, 9, 2, 64, 7, dtype, 16, axes, taken=taken)


def test_append_where_there_is_no_place():
    """Lengths below zero and past the table, table values that are no page."""
    def change(table):
        table[0, 0], table[1, 0], table[1, 1] = -1, 1 << 30, -(1 << 31)
    check_append(4, 6, 2, 64, 5, F32, 32, heads=4, lengths=[-9, 2, 0, 11], change_table=change)
    check_append(2, 4, 1, 64, 4, BF, order=[[5, -1, 4, -(1 << 31)], [3, 0, (1 << 31) - 1, 1]])
    check_append(2, 4, 1, 64, 4, BF, taken=0)
    # numbers that 32 bits do not hold
    k, kp = normal(1, 1, 2, 1, 64), normal(2, 3, 1, 4, 64)
    before = kp.clone()
    m, inputs = C.append_model(k, k, kp, kp.clone(), whole([[0, 1]]), whole([(1 << 31) - 1]))
    m(*inputs)
    assert torch.equal(kp, before)


def test_append_into_pages_of_more_than_two_gibibytes():
    """Rows whose offsets do not fit 32 bits."""
    size, groups, page = 256, 8, 256
    pages = (5 << 30) // (2 * groups * page * size)
    kp, vp = (torch.zeros(pages, groups, page, size, dtype=BF, device="cuda") for _ in range(2))
    k, v = normal(1, 2, 3, groups, size, dtype=BF), normal(2, 2, 3, groups, size, dtype=BF)
    m, inputs = C.append_model(k, v, kp, vp, whole([[pages - 1], [pages // 2 + 1]]), whole([page - 3, 9]))
    m(*inputs)
    for b, (to, row) in enumerate([(pages - 1, page - 3), (pages // 2 + 1, 9)]):
        assert torch.equal(kp[to, :, row:row + 3], k[b].transpose(0, 1)) and torch.equal(vp[to, :, row:row + 3], v[b].transpose(0, 1))
    assert int((kp != 0).any(-1).sum()) == int((vp != 0).any(-1).sum()) == 2 * 3 * groups


def test_append_at_any_address():
    """Arrays that begin between 16-byte boundaries: tokens and pages."""
    for dtype in R.TYPES:
        k, v, q = (normal(i, 2 * 3 * 2 * 64 + 1, dtype=dtype)[1:].reshape(2, 3, 2, 64) for i in range(3))
        kp, vp = (normal(3 + i, 6 * 2 * 4 * 64 + 1, dtype=dtype)[1:].reshape(6, 2, 4, 64) for i in range(2))
        table, lengths, f = whole([[5, 1], [0, 2]]), whole([3, 0]), normal(6, 33)[1:].abs()
        ek, ev, _, eq, k_size, q_size = C.append(k, v, kp, vp, table, lengths, f, None, None, q)
        m, inputs = C.append_model(k, v, kp, vp, table, lengths, f, q=q)
        got = m(*inputs)
        assert torch.equal(vp, ev.to(dtype))
        within(kp, ek, append_bound(k_size, ek, dtype, 6))
        within(got[2], eq, append_bound(q_size, eq, dtype, 6))


def test_queries_may_be_turned_where_they_lie():
    q, k, v, kp, vp = normal(1, 1, 3, 4, 64), normal(2, 1, 3, 2, 64), normal(3, 1, 3, 2, 64), normal(4, 3, 2, 4, 64), normal(5, 3, 2, 4, 64)
    table, lengths, f = whole([[2, 0]]), whole([3]), normal(6, 32).abs()
    expected = C.append_model(k, v, kp.clone(), vp.clone(), table, lengths, f, q=q)
    expected = expected[0](*expected[1])
    lib, sections = _lib.library(), _lib.i64_array([32])
    _lib.check(lib.mi355x_paged_cache_append(k.data_ptr(), v.data_ptr(), q.data_ptr(), kp.data_ptr(), vp.data_ptr(), q.data_ptr(), table.data_ptr(), lengths.data_ptr(), f.data_ptr(),
                                             None, None, 1, 3, 4, 2, 64, 3, 4, 2, 3, 64, 1, sections, 0, 8, 1, _lib.current_stream()), "append")
    assert torch.equal(q, expected[2]) and torch.equal(kp, expected[0]) and torch.equal(vp, expected[1])


# ---------------------------------------------------------------------------------------------- TreeAttention
# size = sum_j P |V|. A score is a sum of D products in float32: off by (D + 2) U sum |q k| scale, and by 3 U of its largest magnitude in the base of two; P is off by
# twice that relatively (numerator and sum). The sums over the keys are off by up to U for each key, and by as much again where parts are joined; P is rounded to 16
# bits where the arrays have them.


def attention_bound(q, k_pages, keys, size, expected, scale):
    dtype, d = q.dtype, q.shape[-1]
    k = torch.nan_to_num(k_pages.double(), 0.0, 0.0, 0.0)
    magnitude = scale * float((q.double().abs().reshape(-1, d).amax(0) * k.abs().reshape(-1, d).amax(0)).sum())
    relative = 2 * ((d + 2) * U * magnitude + 5 * U * magnitude) + (3 * keys + 32) * U + (R.HALF[dtype] if dtype != F32 else 0.0)
    return relative * size * (1 + 2.0 ** -7) + R.HALF[dtype] * expected.abs() + TINY[dtype]


def trees(seed, batch, tokens):
    g = torch.Generator().manual_seed(seed)
    return (torch.rand(batch, tokens, generator=g) * torch.arange(tokens)).to(I32).clamp(max=torch.arange(tokens, dtype=I32) - 1).cuda()


def check_attention(batch, tokens, heads, groups, d, page, context, dtype, tree=False, lengths=None, seed=0, spread=2.0, scale=None, parents=None, change=None, table=None, columns=None,
                    outside=float("nan")):
    lengths = [max(context - 5 * b, 0) for b in range(batch)] if lengths is None else lengths
    columns = -(-(context + tokens) // page) if columns is None else columns
    pages = batch * columns + 2
    if table is None:
        table, pages = shuffled_table(seed, batch, columns)
    q = normal(seed + 1, batch, tokens, heads, d, scale=spread, dtype=dtype)
    kp, vp = normal(seed + 2, pages, groups, page, d, dtype=dtype), normal(seed + 3, pages, groups, page, d, dtype=dtype)
    if outside is not None:   # what belongs to no token
        used = torch.zeros(pages, page, dtype=torch.bool)
        for b in range(batch):
            for n in range(min(max(lengths[b], 0) + tokens, columns * page)):
                used[min(max(int(table[b, n // page]), 0), pages - 1), n % page] = True
        hidden = ~used[:, None, :, None].expand(kp.shape).cuda()
        kp[hidden], vp[hidden] = outside, outside
    parents = trees(seed, batch, tokens) if tree else parents
    lengths = whole(lengths)
    if change:
        change(kp, vp, table)
    expected, size = C.attention(q, kp, vp, table, lengths, parents, scale)
    m, inputs = C.attention_model(q, kp, vp, table, lengths, parents, **({} if scale is None else {"scale": scale}))
    o = m(*inputs)
    assert o.dtype == dtype
    bound = attention_bound(q, kp, min(context + tokens, columns * page), size, expected, scale or d ** -0.5)
    finite = torch.isfinite(expected)
    within(o[finite], expected[finite], bound[finite])
    if dtype == F32:   # an infinite value is split in three parts
        assert not torch.isfinite(o[~finite]).any()
    else:
        assert torch.equal(torch.nan_to_num(o[~finite].float(), -1.5), torch.nan_to_num(expected[~finite].float(), -1.5))
    assert torch.equal(o.view(torch.uint8), m(*inputs).view(torch.uint8))   # whatever order workgroups run in
    return o


SMALL = [(1, 1, 1, 1, 16, 0), (1, 2, 1, 1, 16, 1), (2, 31, 2, 1, 5, 2), (1, 65, 2, 2, 16, 0), (2, 40, 3, 3, 23, 100), (1, 5, 4, 2, 64, 700), (3, 9, 12, 2, 1, 33), (1, 130, 4, 1, 32, 70)]


@pytest.mark.parametrize("dtype", R.TYPES)
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("batch, tokens, heads, groups, page, context", SMALL)
def test_attention(dtype, d, tree, batch, tokens, heads, groups, page, context):
    check_attention(batch, tokens, heads, groups, d, page, context, dtype, tree)


@pytest.mark.parametrize("dtype", R.TYPES)
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("batch, tokens, heads, groups, page, context", [(1, 1, 8, 2, 16, 5000), (3, 1, 4, 4, 64, 1000), (2, 1, 12, 2, 23, 2049), (9, 1, 40, 1, 8, 96), (2, 4, 4, 1, 256, 3001),
                                                                           (1, 17, 4, 2, 16, 4500)])
def test_attention_of_few_rows(dtype, d, batch, tokens, heads, groups, page, context):
    check_attention(batch, tokens, heads, groups, d, page, context, dtype, tokens > 4)


@pytest.mark.parametrize("dtype", R.TYPES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("tokens, heads, groups, page, context", [(700, 4, 2, 16, 0), (513, 2, 2, 64, 300), (333, 8, 1, 23, 1000), (300, 8, 8, 128, 77)])
def test_attention_of_prompts(dtype, d, tokens, heads, groups, page, context):
    check_attention(2, tokens, heads, groups, d, page, context, dtype)


@pytest.mark.parametrize("form", range(3))
@pytest.mark.parametrize("dealt", [0, 5, 64, 512])
@pytest.mark.parametrize("dtype", R.TYPES)
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("batch, tokens, heads, groups, page, context, tree", [(1, 3, 2, 1, 16, 300, True), (2, 150, 2, 2, 4, 129, False), (3, 70, 4, 1, 7, 260, True), (1, 300, 1, 1, 64, 0, False)])
def test_attention_by_every_kernel(form, dealt, dtype, d, batch, tokens, heads, groups, page, context, tree, tuning):
    """One workgroup to a block of rows, and its keys in parts: fewer workgroups than blocks (which have one each then), about as many, and more than there are stages."""
    tuning(MI355X_TREE_FORM=form, MI355X_TREE_DEAL=dealt)
    check_attention(batch, tokens, heads, groups, d, page, context, dtype, tree)


@pytest.mark.parametrize("dealt", [0, 300, 512])
@pytest.mark.parametrize("batch", [63, 64, 65, 130, 256, 257])
def test_attention_of_many_entries(batch, dealt, tuning):
    """Entries of all lengths, more of them than a wave has lanes, and than parts are dealt for."""
    tuning(MI355X_TREE_DEAL=dealt)
    lengths = [(37 * b * b) % 700 if b % 5 else 0 for b in range(batch)]
    check_attention(batch, 2, 2, 1, 64, 16, 700, BF, lengths=lengths)


def test_attention_of_one_long_entry_among_short_ones(tuning):
    for dealt in (-1, 64, 256):
        tuning(MI355X_TREE_DEAL=dealt)
        check_attention(8, 1, 4, 2, 128, 16, 20000, BF, lengths=[0, 3, 20000, 1, 0, 64, 127, 128])


@pytest.mark.parametrize("dtype", R.TYPES)
def test_attention_of_large_trees(dtype):
    check_attention(1, 1024, 2, 1, 64, 16, 50, dtype, True)
    # a chain as a tree, and every token a child of the cache
    check_attention(1, 300, 2, 1, 64, 16, 50, dtype, parents=torch.arange(-1, 299, dtype=I32)[None].cuda())
    check_attention(2, 70, 2, 2, 128, 16, 50, dtype, parents=torch.full((2, 70), -1, dtype=I32).cuda())


@pytest.mark.parametrize("dtype", R.TYPES)
def test_attention_of_parents_that_are_none(dtype):
    """A parent that does not stand before its child: a later one, itself, one past the call's tokens."""
    parents = whole([[0, 0, 5, 3, 1 << 30, -(1 << 31), 2, 7], [-1, 0, 1, 2, 3, 4, 5, 6]])
    check_attention(2, 8, 4, 2, 64, 5, 30, dtype, parents=parents)


@pytest.mark.parametrize("dtype", R.TYPES)
@pytest.mark.parametrize("tokens", [1, 40])
def test_attention_lengths(dtype, tokens):
    """No key before the call, one, all that the table has room for, more, fewer than none; rows for which there is no key."""
    capacity, page = 300, 12
    o = check_attention(7, tokens, 4, 2, 64, page, capacity - tokens, dtype, lengths=[0, 1, capacity - tokens, capacity, capacity + 5, -3, (1 << 31) - 1], columns=25)
    assert (o[3] != 0).any()
    table = torch.zeros(2, 0, dtype=I32).cuda()
    o = check_attention(2, tokens, 4, 2, 64, page, 0, dtype, lengths=[0, 7], table=table, columns=0)
    assert (o == 0).all()


def test_attention_of_table_values_that_are_no_page():
    table = whole([[0, -1, 1 << 30], [-(1 << 31), 3, (1 << 31) - 1]])
    check_attention(2, 4, 4, 2, 64, 8, 20, BF, lengths=[20, 13], table=table, columns=3, outside=None)


@pytest.mark.parametrize("dtype", R.TYPES)
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_attention_of_values_that_some_rows_do_not_see(dtype, d, bad):
    """A key or a value of a drafted token that is not finite reaches that token and its descendants, nobody else."""
    tokens, context, page = 20, 50, 8

    def change_values(kp, vp, table):
        for n in (3, 11):
            at = context + n
            vp[int(table[0, at // page]), :, at % page, n] = bad
    parents = whole([[-1, 0, 1, 1, 2, 3, 0, 6, 3, 8, 9, 0, 11, 11, 4, 14, 14, 5, 7, 18]])
    o = check_attention(1, tokens, 4, 2, d, page, context, dtype, parents=parents, change=change_values)
    below = C.lines(parents[0].tolist())
    for i in range(tokens):
        assert bool(torch.isfinite(o[0, i]).all()) == (not (below[i, 3] or below[i, 11]))

    def change_keys(kp, vp, table):
        at = context + 3
        kp[int(table[0, at // page]), :, at % page, 5] = float("nan")
    o = check_attention(1, tokens, 4, 2, d, page, context, dtype, parents=parents, change=change_keys)
    for i in range(tokens):
        assert bool(torch.isfinite(o[0, i]).all()) == (not below[i, 3])


@pytest.mark.parametrize("form", range(3))
@pytest.mark.parametrize("dealt", [0, 40])
@pytest.mark.parametrize("dtype", R.TYPES)
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("page", [16, 11])
def test_attention_of_values_that_some_rows_do_not_see_by_every_kernel(form, dealt, dtype, d, page, tuning):
    """Of a chain: what later tokens hold, in several columns and of both halves of a wave, behind and across the ends of stages."""
    tuning(MI355X_TREE_FORM=form, MI355X_TREE_DEAL=dealt)
    tokens, context = 150, 100
    bad = {30: (0, float("inf")), 61: (d - 1, float("nan")), 62: (d // 2 + 5, float("-inf")), 149: (7, float("inf"))}

    def change(kp, vp, table):
        for n, (column, value) in bad.items():
            vp[int(table[0, (context + n) // page]), :, (context + n) % page, column] = value
    o = check_attention(1, tokens, 4, 2, d, page, context, dtype, change=change)
    for n, (column, value) in bad.items():
        assert torch.isfinite(o[0, :n, :, column]).all() and not torch.isfinite(o[0, n:, :, column]).any()


@pytest.mark.parametrize("dtype", R.TYPES)
def test_attention_of_a_padded_prompt(dtype):
    """The tokens behind a prompt's end hold anything: those before them do not see it."""
    def change(kp, vp, table):
        for n in range(20 + 150, 20 + 200):
            kp[int(table[0, n // 16]), :, n % 16], vp[int(table[0, n // 16]), :, n % 16] = float("nan"), float("inf")
    o = check_attention(1, 200, 4, 2, 64, 16, 20, dtype, change=change)
    assert torch.isfinite(o[0, :150]).all()


@pytest.mark.parametrize("dtype", R.TYPES)
def test_attention_of_infinite_context(dtype):
    """What every row sees reaches every row."""
    def change(kp, vp, table):
        vp[int(table[0, 1]), 0, 3, 7] = float("inf")
    o = check_attention(1, 3, 4, 2, 64, 8, 30, dtype, change=change)
    assert not torch.isfinite(o[0, :, :2, 7]).any() and torch.isfinite(o[0, :, 2:]).all()


@pytest.mark.parametrize("dtype", R.TYPES)
def test_attention_of_far_scores(dtype):
    """Scores of hundreds, rising and falling along the cache: the running maximum moves a long way."""
    for flip in (False, True):
        def change(kp, vp, table):
            weight = torch.linspace(0.01, 2, 8 * 40).cuda().flip(0 if flip else ())
            order = table[0].long()
            kp[order] = (kp[order].float() * weight.reshape(40, 1, 8, 1)).to(kp.dtype)
        check_attention(1, 10, 4, 2, 64, 8, 310, dtype, spread=20.0, change=change, outside=0.0)


def test_attention_scale_and_addresses():
    for dtype in R.TYPES:
        check_attention(2, 3, 4, 2, 64, 8, 30, dtype, scale=0.5)
        q = normal(1, 2 * 3 * 4 * 64 + 1, dtype=dtype)[1:].reshape(2, 3, 4, 64)   # between 16-byte boundaries
        kp, vp = normal(2, 9, 2, 8, 64, dtype=dtype), normal(3, 9, 2, 8, 64, dtype=dtype)
        table, lengths = whole([[5, 1], [0, 2]]), whole([3, 0])
        expected, size = C.attention(q, kp, vp, table, lengths)
        m, inputs = C.attention_model(q, kp, vp, table, lengths)
        within(m(*inputs), expected, attention_bound(q, kp, 6, size, expected, 0.125))
        odd = normal(2, 9 * 2 * 8 * 64 + 1, dtype=dtype)[1:].reshape(9, 2, 8, 64)
        with pytest.raises(_lib.MI355XError, match="16-byte"):
            m(q, odd, vp, table, lengths)


def test_attention_over_pages_of_more_than_four_gibibytes():
    page, groups, d = 64, 2, 128
    pages = (9 << 30) // (2 * groups * page * d)
    kp, vp = (torch.zeros(pages, groups, page, d, dtype=BF, device="cuda") for _ in range(2))
    table = whole([[pages - 1, 3, pages // 2 + 1], [pages - 7, pages // 2 - 9, 0]])
    for t in table.flatten().tolist():
        kp[t], vp[t] = normal(t % 1000, groups, page, d, dtype=BF), normal(t % 1000 + 1, groups, page, d, dtype=BF)
    q, lengths = normal(1, 2, 2, 4, d, scale=2.0, dtype=BF), whole([150, 99])
    small = torch.unique(table)
    place = torch.zeros(pages, dtype=I32, device="cuda")
    place[small.long()] = torch.arange(len(small), dtype=I32, device="cuda")
    expected, size = C.attention(q, kp[small.long()], vp[small.long()], place[table.long()], lengths)
    m, inputs = C.attention_model(q, kp, vp, table, lengths)
    within(m(*inputs), expected, attention_bound(q, kp[small.long()], 152, size, expected, d ** -0.5))


# ---------------------------------------------------------------------------------------------- DraftAcceptance


def check_acceptance(logits, tokens, parents=None):
    expected = C.acceptance(logits, tokens, parents)
    m, inputs = C.acceptance_model(logits, tokens, parents)
    for _ in range(2):
        for got, want in zip(m(*inputs), expected):
            assert got.dtype == I32 and torch.equal(got.cpu(), want)
    return expected


def drafts(seed, logits, parents, hit):
    """Tokens of which a share is what the logits say after their parents."""
    g = torch.Generator().manual_seed(seed)
    said = logits.double().cpu().argmax(-1)
    up = torch.arange(-1, logits.shape[1] - 1).expand(said.shape) if parents is None else parents.cpu().long()
    follow = torch.gather(said, 1, up.clamp(0, logits.shape[1] - 1))
    other = torch.randint(0, logits.shape[2], said.shape, generator=g)
    return torch.where(torch.rand(said.shape, generator=g) < hit, follow, other).to(I32).cuda()


@pytest.mark.parametrize("dtype", R.TYPES)
@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("batch, tokens, vocabulary", [(1, 1, 1), (1, 1, 50), (2, 3, 7), (3, 8, 1000), (5, 13, 4999), (2, 33, 32000), (1, 2, 131073), (40, 5, 65), (1, 1024, 40)])
def test_acceptance(dtype, tree, batch, tokens, vocabulary):
    logits = normal(1, batch, tokens, vocabulary, scale=2.0, dtype=dtype)
    parents = trees(2, batch, tokens) if tree else None
    for hit in (0.0, 0.7, 1.0):
        check_acceptance(logits, drafts(3, logits, parents, hit), parents)


@pytest.mark.parametrize("parts", [1, 2, 7, 64])
@pytest.mark.parametrize("dtype", R.TYPES)
@pytest.mark.parametrize("vocabulary", [1, 5, 63, 1025, 40001])
def test_acceptance_in_any_number_of_parts(parts, dtype, vocabulary, tuning):
    tuning(MI355X_ACCEPT_PARTS=parts)
    logits = normal(1, 2, 5, vocabulary, scale=2.0, dtype=dtype)
    check_acceptance(logits, drafts(3, logits, None, 0.8))


@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("tokens", [32, 63, 64, 65, 128, 129])
def test_acceptance_of_trees_that_a_wave_has_lanes_for_and_larger_ones(tokens, tree):
    logits = normal(1, 3, tokens, 200, scale=2.0)
    parents = trees(2, 3, tokens) if tree else None
    for hit in (0.0, 0.9, 1.0):
        check_acceptance(logits, drafts(3, logits, parents, hit), parents)


@pytest.mark.parametrize("parts", [None, 5])
@pytest.mark.parametrize("dtype", R.TYPES)
def test_acceptance_of_equal_logits_and_of_none(dtype, parts, tuning):
    """The first of equal ones wherever they stand, 0 and -0 alike; rows of infinities and of NaN; a NaN next to numbers."""
    tuning(MI355X_ACCEPT_PARTS=parts)
    inf, nan, V = float("inf"), float("nan"), 3001
    rows = torch.full((1, 12, V), -1.0)
    rows[0, 0, [17, 16, 2999]] = 5.0
    rows[0, 1, [8, 9]] = torch.tensor([-0.0, 0.0])
    rows[0, 2, [9, 8]] = torch.tensor([-0.0, 0.0])
    rows[0, 3], rows[0, 4], rows[0, 5] = -inf, nan, inf
    rows[0, 6, [5, 700]] = torch.tensor([nan, 3.0])
    rows[0, 7] = nan
    rows[0, 7, 2047] = -inf
    rows[0, 8] = -inf
    rows[0, 8, :600] = nan
    rows[0, 9, 2500] = inf
    rows[0, 10, -1] = -0.5
    said = [16, 8, 8, 0, 0, 0, 700, 2047, 600, 2500, V - 1, 0]
    assert C.acceptance(rows, torch.tensor([[0] + said[:-1]], dtype=I32))[0].tolist() == [list(range(12))]
    check_acceptance(rows.to(dtype).cuda(), whole([[0] + said[:-1]]))
    for i in range(12):   # each row's answer by itself
        assert check_acceptance(rows[:, i:i + 1].to(dtype).contiguous().cuda(), whole([[0]]))[2].tolist() == [said[i]]


def test_acceptance_of_odd_trees():
    logits = normal(1, 2, 9, 40)
    said = logits.argmax(-1)
    parents = whole([[0, 0, 0, 1, 2, 9, 1 << 30, 7, 3], [3, 0, 5, 1, -7, 4, 2, 6, 3]])
    tokens = torch.gather(said, 1, parents.long().clamp(0, 8)).to(I32)
    path, _, _ = check_acceptance(logits, tokens, parents)
    assert path[0, :4].tolist() == [0, 1, 3, 8]   # of children with the same token the first


# ---------------------------------------------------------------------------------------------- together


def _prompt_and_model(weights, graph_calls):
    """One entry's cache for each layer, and a way to run the two graphs of any number of tokens."""
    page, columns, pages = 7, 9, 14
    shape = (pages, C.GROUPS, page, C.SIZE)
    caches = [torch.full(shape, float("nan"), device="cuda") for _ in range(2 * C.LAYERS)]
    table = whole([[3, 11, 0, 7, 5, 13, 2, 9, 1]])
    models = {}

    def step(tokens, parents, depth, length):
        S = len(tokens)
        if S not in models:
            models[S] = [donnx.ONNXModel(f.__name__, f(weights, 1, S, shape, columns), use_hip_graph=graph_calls) for f in (C.verifying_graph, C.keeping_graph)]
        verify, keep = models[S]
        x = torch.from_numpy(weights["embedding"]).cuda()[torch.tensor(tokens).cuda()][None]
        lengths = whole([length])
        out = verify(x, whole([tokens]), whole([parents]), whole([[[length + d for d in depth]]]), table, lengths, *caches)
        path, count, after, *kv = out
        keep(path, table, lengths, *[t for i in range(C.LAYERS) for t in (*kv[2 * i:2 * i + 2], *caches[2 * i:2 * i + 2])])
        return path[0].tolist(), int(count), int(after)
    return step


@pytest.mark.parametrize("graph_calls", [False, True])
@pytest.mark.parametrize("prompt", [[5, 17, 3, 200, 44, 9, 101], [77, 8]])
def test_drafted_tokens_of_a_small_transformer(graph_calls, prompt):
    """A prompt, then trees whose drafts are right now and then: the tokens are those of whole passes in float64."""
    weights = C.transformer_weights(7)
    expected, _ = C.greedy(weights, prompt, 24)
    step = _prompt_and_model(weights, graph_calls)
    length = 0
    for token in prompt:
        path, count, after = step([token], [-1], [0], length)
        assert path == [0] and count == 1
        length += 1
    said, rng, accepted = [after], np.random.default_rng(1), []
    while len(said) < 20:
        true = expected[len(said):len(said) + 3] + [0] * 3
        wrong = [int(t) for t in rng.integers(0, C.VOCABULARY, 6)]
        hits = rng.random(3) < 0.7
        # 0 - 1 - 3 - 5, 0 - 2 - 4; the true continuation, where it is drafted at all, goes by 2 or by 1
        by = 1 + int(rng.integers(0, 2))
        tokens = [said[-1]] + wrong[:5]
        parents, depth = [-1, 0, 0, 1, 2, 3], [0, 1, 1, 2, 2, 3]
        for node, level in ((by, 0), (by + 2, 1), (5, 2)):
            if hits[level]:
                tokens[node] = true[level]
        path, count, after = step(tokens, parents, depth, length)
        taken = [tokens[i] for i in path[:count]]
        assert path[count:] == [-1] * (6 - count)
        said += taken[1:] + [after]
        length += count
        accepted.append(count)
    assert said[:20] == expected[:20]
    assert max(accepted) > 2 and min(accepted) == 1


def test_a_prompt_and_the_tokens_behind_it():
    """A prompt of a padded batch in one call, one token at a time behind it, keys and values of both by their pages: the attention of the whole."""
    B, S, H, G, D, page = 2, 37, 4, 2, 64, 8
    ends = [37, 20]
    table, pages = shuffled_table(1, B, 6)
    kp, vp = (torch.full((pages, G, page, D), float("nan"), dtype=BF, device="cuda") for _ in range(2))
    k, v, q = normal(2, B, S + 3, G, D, dtype=BF), normal(3, B, S + 3, G, D, dtype=BF), normal(4, B, S + 3, H, D, scale=2.0, dtype=BF)
    f = (10000.0 ** (-torch.arange(D // 2) / (D // 2))).float().cuda()
    got = {}

    def call(at, lengths):   # at[b]: which of the entry's tokens
        pick = lambda t: torch.stack([t[b, at[b]] for b in range(B)]).contiguous()   # noqa: E731
        m, inputs = C.append_model(pick(k), pick(v), kp, vp, table, lengths, f, q=pick(q))
        _, _, turned = m(*inputs)
        m, inputs = C.attention_model(turned, kp, vp, table, lengths)
        o = m(*inputs)
        for b in range(B):
            for j, i in enumerate(at[b].tolist()):
                got[b, i] = o[b, j]
    call([torch.arange(S)] * B, whole([0, 0]))
    for step in range(3):
        call([torch.tensor([e + step]) for e in ends], whole([e + step for e in ends]))
    for b, end in enumerate(ends):
        tokens = end + 3
        angle = torch.arange(tokens, dtype=torch.float64, device="cuda")[:, None, None] * f.double()

        def turned(t):
            a, c = t[b, :tokens, :, :D // 2].double(), t[b, :tokens, :, D // 2:].double()
            return torch.cat([a * angle.cos() - c * angle.sin(), c * angle.cos() + a * angle.sin()], -1).to(BF)   # as they are stored
        expected, size = C.attention(turned(q)[None], turned(k).transpose(0, 1)[None].contiguous(), v[b, :tokens].transpose(0, 1)[None].contiguous(), whole([[0]]), whole([0]))
        o = torch.stack([got[b, i] for i in range(tokens)])[None]
        # a turned value next to a border may be rounded the other way: a whole step of queries and keys, 2 HALF of a score's magnitude each
        magnitude = D ** -0.5 * float((turned(q).abs().reshape(-1, D).amax(0) * turned(k).abs().reshape(-1, D).amax(0)).sum())
        relative = 2 * (4 * R.HALF[BF] * magnitude) + R.HALF[BF] + 1e-4
        within(o, expected, relative * size * (1 + 2.0 ** -7) + R.HALF[BF] * expected.abs())


def test_another_cache_in_a_recorded_graph_and_tensors_that_cannot_be_updated():
    k, v, table, lengths = normal(1, 2, 3, 2, 64), normal(2, 2, 3, 2, 64), whole([[4, 1], [0, 2]]), whole([3, 0])
    caches = [(normal(3 + i, 5, 2, 4, 64), normal(9 + i, 5, 2, 4, 64)) for i in range(2)]
    for recorded in (True, False):
        m = donnx.ONNXModel("m", _append_proto(k, caches[0][0], table), use_hip_graph=recorded)
        for turn in range(6):
            kp, vp = (t.clone() for t in caches[turn // 3])
            new = normal(20 + turn, 2, 3, 2, 64)
            ek, ev, *_ = C.append(new, v, kp, vp, table, lengths)
            got = m(new, v, kp, vp, table, lengths)
            assert got[0] is kp and got[1] is vp
            torch.cuda.synchronize()
            assert torch.equal(kp.double(), ek) and torch.equal(vp.double(), ev)
            got = m(k, v, kp, vp, table, lengths)   # the same cache again: a replay
            ek, ev, *_ = C.append(k, v, kp, vp, table, lengths)
            assert torch.equal(kp.double(), ek) and torch.equal(vp.double(), ev)
        kp, vp = caches[0]
        for bad in (kp.cpu(), kp.cpu().numpy(), kp.transpose(0, 1).contiguous().transpose(0, 1), kp[:4].contiguous(), kp.to(BF)):
            with pytest.raises(TypeError, match="updated where it lies"):
                m(k, v, bad, vp, table, lengths)


def test_keys_and_values_side_by_side_and_in_one_array():
    """Pages of one allocation, one half behind the other; the same half twice is refused, on the first call and on those by the plan."""
    k, v, table, lengths = normal(1, 2, 3, 2, 64), normal(2, 2, 3, 2, 64), whole([[4, 1], [0, 2]]), whole([3, 0])
    cache = normal(3, 2, 5, 2, 4, 64)
    m = donnx.ONNXModel("m", _append_proto(k, cache[0], table))
    for turn in range(3):
        ek, ev, *_ = C.append(k, v, cache[0].clone(), cache[1].clone(), table, lengths)
        m(k, v, cache[0], cache[1], table, lengths)
        assert torch.equal(cache[0].double(), ek) and torch.equal(cache[1].double(), ev)
        before = cache.clone()
        with pytest.raises(Exception, match="share pages"):
            m(k, v, cache[0], cache[0], table, lengths)
        assert torch.equal(cache, before)


def _append_proto(k, kp, table):
    from dace_onnx_amd.onnx.proto import helper
    info = lambda n, t, s: helper.make_tensor_value_info(n, t, list(s))   # noqa: E731
    inputs = [info("k", 1, k.shape), info("v", 1, k.shape), info("kp", 1, kp.shape), info("vp", 1, kp.shape), info("table", 6, table.shape), info("lengths", 6, table.shape[:1])]
    node = helper.make_node("PagedCacheAppend", [i.name for i in inputs], ["ko", "vo"], name="append")
    return helper.make_model(helper.make_graph([node], "g", inputs, [info("ko", 1, kp.shape), info("vo", 1, kp.shape)]))


def test_the_call_form():
    """Tensors and numpy arrays that the caller passes are updated."""
    k, v, table, lengths = normal(1, 2, 3, 2, 64), normal(2, 2, 3, 2, 64), whole([[4, 1], [0, 2]]), whole([3, 0])
    kp, vp = normal(3, 5, 2, 4, 64), normal(4, 5, 2, 4, 64)
    ek, ev, *_ = C.append(k, v, kp, vp, table, lengths)
    on_host = [t.cpu().numpy().copy() for t in (k, v, kp, vp, table, lengths)]
    donnx.ONNXPagedCacheAppend(K=k, V=v, k_pages=kp, v_pages=vp, table=table, lengths=lengths, k_pages_out=kp, v_pages_out=vp)
    assert torch.equal(kp.double(), ek) and torch.equal(vp.double(), ev)
    a, b, c, d, e, f = on_host
    donnx.ONNXPagedCacheAppend(K=a, V=b, k_pages=c, v_pages=d, table=e, lengths=f, k_pages_out=c, v_pages_out=d)
    assert np.array_equal(c, kp.cpu().numpy()) and np.array_equal(d, vp.cpu().numpy())
    q, o = normal(5, 2, 3, 4, 64), torch.empty(2, 3, 4, 64, device="cuda")
    donnx.ONNXTreeAttention(Q=q, k_pages=kp, v_pages=vp, table=table, lengths=lengths, O=o)
    expected, size = C.attention(q, kp, vp, table, lengths)
    within(o, expected, attention_bound(q, kp, 6, size, expected, 0.125))


def test_another_stream_and_recordings_of_the_caller():
    """All three nodes on a side stream, and captured by the caller: replays follow what is written between them."""
    B, S, H, G, D, page, V = 2, 5, 4, 2, 64, 8, 3000
    table, pages = shuffled_table(1, B, 100)
    lengths = whole([700, 300])
    k, v, q = normal(2, B, S, G, D, dtype=BF), normal(3, B, S, G, D, dtype=BF), normal(4, B, S, H, D, dtype=BF)
    kp, vp = normal(5, pages, G, page, D, dtype=BF), normal(6, pages, G, page, D, dtype=BF)
    parents, logits = trees(7, B, S), normal(8, B, S, V, dtype=BF)
    tokens = drafts(9, logits, parents, 0.8)
    append, attend, accept = C.append_model(k, v, kp, vp, table, lengths), C.attention_model(q, kp, vp, table, lengths, parents), C.acceptance_model(logits, tokens, parents)

    def run():
        append[0](*append[1])
        return attend[0](*attend[1]), *accept[0](*accept[1])

    def check(outputs):
        expected, size = C.attention(q, kp, vp, table, lengths, parents)
        within(outputs[0], expected, attention_bound(q, kp, 705, size, expected, 0.125))
        for got, want in zip(outputs[1:], C.acceptance(logits, tokens, parents)):
            assert torch.equal(got.cpu(), want)
    check(run())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        outputs = run()
    torch.cuda.current_stream().wait_stream(side)
    check(outputs)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outputs = run()
    for turn in range(3):
        k.copy_(normal(30 + turn, B, S, G, D, dtype=BF))
        q.copy_(normal(40 + turn, B, S, H, D, dtype=BF))
        logits.copy_(normal(50 + turn, B, S, V, dtype=BF))
        tokens.copy_(drafts(60 + turn, logits, parents, 0.8))
        lengths.copy_(whole([700 - 99 * turn, 300 + 7 * turn]))
        graph.replay()
        check(outputs)
        check(run())   # and the program's own calls in between


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("form, dealt", [(0, 0), (1, 0), (2, 0), (0, 512)])
def test_attention_in_float32_over_many_keys(form, dealt, d, tuning):
    """Sums of 20000 products in float32, which one sum for all of them would not keep (7e-6). Each 32 keys have sums of their own, of twelve products that may lose half of 2^-23 of the sum so
    far each, towards zero: 12 2^-24 / 2 = 3.6e-7 of weights that add up to one, and products left out 4e-8: 5e-7 on average. The additions of 625 such sums are off by 2^-24 of the sum so
    far, at random: 2^-24 sqrt(625) / 3 = 5e-7 where it grows evenly, three times that for the farthest of 4096 outputs: 2e-6. Outputs of random values are 1 / sqrt(N) of their weights' sum of
    magnitudes, as are what they lose at random: 1e-6 in 2-norm with scores off by 1.4e-7 of 8."""
    tuning(MI355X_TREE_FORM=form, MI355X_TREE_DEAL=dealt)
    table, pages = shuffled_table(1, 1, 1252)
    q, kp, vp = normal(2, 1, 8, 4, d), normal(3, pages, 1, 16, d), normal(4, pages, 1, 16, d)
    lengths = whole([20000])
    m, inputs = C.attention_model(q, kp, vp, table, lengths, None)
    o = m(*inputs).double()
    expected, _ = C.attention(q, kp, vp, table, lengths, None, None)
    assert (o - expected).norm() <= 1e-6 * expected.norm()
    inputs = [torch.ones_like(t) if t is vp else t for t in inputs]   # weights add up to one: a loss of all products shows whole
    o = m(*inputs).double()
    assert (o - 1).abs().max() <= 2e-6 and abs(float((o - 1).mean())) <= 5e-7


@pytest.mark.parametrize("form, dealt", [(0, 0), (1, 0), (2, 0), (0, 40), (2, 40)])
@pytest.mark.parametrize("dtype", [F16, BF])
@pytest.mark.parametrize("tree", [False, True])
def test_attention_of_rows_whose_scores_are_all_minus_infinity(form, dealt, dtype, tree, tuning):
    """Softmax of such a row is not a number: 0 is the result of a row without keys alone. A key whose score is minus infinity next to others has no weight."""
    tuning(MI355X_TREE_FORM=form, MI355X_TREE_DEAL=dealt)
    tokens, heads, d, page, columns = 70, 4, 64, 8, 30
    table, pages = shuffled_table(1, 4, columns)
    q, kp, vp = normal(2, 4, tokens, heads, d, dtype=dtype), normal(3, pages, 2, page, d, dtype=dtype), normal(4, pages, 2, page, d, dtype=dtype)
    kp[..., 0] = kp[..., 0].abs() + 0.25
    kp[int(table[0, 0]), :, 0, 1] = float("-inf")   # a key in front of the first entry's call
    q[..., 1] = q[..., 1].abs() + 0.25
    none = torch.zeros(4, tokens, heads, dtype=torch.bool, device="cuda")
    none[0, 5, 1] = none[0, 69, 3] = none[1, 0, 0] = none[1, 40, 2] = none[2, 3, 3] = none[3, 1, 1] = True
    q[..., 0] = torch.where(none, float("-inf"), q[..., 0].abs())
    parents = trees(5, 4, tokens) if tree else None
    capacity = columns * page
    lengths = whole([100, 0, 17, capacity])   # rows of the last see keys, but not their own
    finite = q.clone()
    finite[..., 0] = torch.where(none, 0.0, q[..., 0])
    expected, size = C.attention(finite, kp, vp, table, lengths, parents)
    bound = attention_bound(finite, torch.nan_to_num(kp, neginf=0.0), capacity, size, expected, d ** -0.5)
    m, inputs = C.attention_model(q, kp, vp, table, lengths, parents)
    o = m(*inputs)
    assert torch.isnan(o[none]).all()
    within(o[~none], expected[~none], bound[~none])
    # no column, and no key: a row of minus infinity among them as well
    m, inputs = C.attention_model(q, kp, vp, table[:, :0].contiguous(), lengths, parents)
    assert (m(*inputs) == 0).all()


@pytest.mark.parametrize("form, dealt", [(0, 0), (2, 0), (0, 40)])
@pytest.mark.parametrize("tree", [False, True])
def test_attention_of_empty_entries_that_the_table_has_little_room_for(form, dealt, tree, tuning):
    """No key before the call and a table of one page: a token whose line begins behind it sees nothing, the others of it what the page has."""
    tuning(MI355X_TREE_FORM=form, MI355X_TREE_DEAL=dealt)
    tokens, d, page = 9, 64, 4
    q, kp, vp = normal(2, 1, tokens, 2, d, dtype=BF), normal(3, 3, 1, page, d, dtype=BF).abs(), normal(4, 3, 1, page, d, dtype=BF)
    q[0, :, 1, 0] = float("-inf")
    kp[..., 0] += 0.25
    parents = whole([[-1, 0, 1, -1, 2, -1, 5, 3, -1]]) if tree else None
    m, inputs = C.attention_model(q, kp, vp, whole([[2]]), whole([0]), parents)
    o = m(*inputs)
    sees = [True] * 5 + [False, False, True, False] if tree else [True] * tokens
    for i in range(tokens):
        assert torch.isnan(o[0, i, 1]).all() if sees[i] else (o[0, i] == 0).all()
        assert not sees[i] or (o[0, i, 0] != 0).any()


INFINITE = [float("inf"), float("-inf"), float("nan")]


@pytest.mark.parametrize("form, dealt", [(0, 0), (1, 0), (2, 0), (0, 40), (2, 40)])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_attention_in_float32_of_infinite_values_is_not_a_number_whatever_the_form(form, dealt, d, tuning):
    """Of a context that all rows see, and of tokens that only later ones see, wherever the blocks of a form end."""
    tuning(MI355X_TREE_FORM=form, MI355X_TREE_DEAL=dealt)
    tokens, context, page = 150, 90, 6 if d == 64 else 16
    columns = -(-(context + tokens) // page)
    table, pages = shuffled_table(1, 1, columns)
    q, kp, vp = normal(2, 1, tokens, 2, d, scale=0.1), normal(3, pages, 1, page, d), normal(4, pages, 1, page, d)
    bad = {-7: 3, 0: d - 1, 31: 5, 63: d // 2, 64: 9, 100: 40, 127: 17, 128: 33, 149: 62}   # number after the context -> column
    for i, (n, column) in enumerate(bad.items()):
        vp[int(table[0, (context + n) // page]), :, (context + n) % page, column] = INFINITE[i % 3]
    m, inputs = C.attention_model(q, kp, vp, table, whole([context]))
    o = m(*inputs)
    expected = torch.zeros_like(o, dtype=torch.bool)
    for n, column in bad.items():
        expected[0, max(n, 0):, :, column] = True
    assert torch.equal(torch.isnan(o), expected) and torch.isfinite(o[~expected]).all()


# ---------------------------------------------------------------------------------------------- row by row


def check_rows(*sizes, **more):
    """Every row's error within a bound of its own scores and weights (``cache_operators.attention_rows``)."""
    case = C.attention_case(11, *sizes, **more, device="cuda")
    m, inputs = C.attention_model(*case)
    expected, bound = C.attention_rows(*case)
    for _ in range(2):   # the general way, then the short one
        error = (m(*inputs).double() - expected).norm(dim=-1)
        worst = float((error / bound).max())
        assert worst <= 1, f"{worst:.3g} of the bound in row {tuple(((error / bound) == worst).nonzero()[0].tolist())}"


@pytest.mark.parametrize("form, dealt", [(0, 0), (1, 0), (2, 0), (0, 60), (1, 60), (2, 60)])
@pytest.mark.parametrize("dtype", R.TYPES)
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("batch, tokens, heads, groups, page, context, tree", [(3, 40, 4, 2, 23, 500, True), (2, 150, 2, 2, 16, 300, False)])
def test_rows_of_every_form(form, dealt, dtype, d, batch, tokens, heads, groups, page, context, tree, tuning):
    tuning(MI355X_TREE_FORM=form, MI355X_TREE_DEAL=dealt)
    check_rows(batch, tokens, heads, groups, d, page, context, dtype, tree)


@pytest.mark.parametrize("dtype", R.TYPES)
@pytest.mark.parametrize("page", [1, 5, 7, 8, 11, 32, 64, 256])
@pytest.mark.parametrize("tokens, tree", [(1, False), (9, True)])
def test_rows_over_pages_of_any_size(dtype, page, tokens, tree):
    check_rows(3, tokens, 6, 3, 64, page, 900, dtype, tree)


@pytest.mark.parametrize("dtype", R.TYPES)
@pytest.mark.parametrize("batch, tokens, heads, groups, d, page, context, tree", [
    (1, 1, 8, 2, 128, 16, 9000, False), (70, 1, 2, 1, 64, 16, 700, False), (300, 1, 1, 1, 64, 8, 90, False), (1, 600, 2, 1, 64, 16, 0, False), (1, 200, 2, 1, 128, 16, 700, True), (4, 3, 40, 1, 64, 16, 2000, True)])
def test_rows_of_calls_as_they_are(dtype, batch, tokens, heads, groups, d, page, context, tree):
    """By the form that the sizes choose: few rows behind many keys, more entries than parts are dealt for, prompts, trees, many heads to a group."""
    check_rows(batch, tokens, heads, groups, d, page, context, dtype, tree)


@pytest.mark.parametrize("form, dealt", [(0, 0), (1, 0), (2, 0), (0, 40)])
@pytest.mark.parametrize("dtype", R.TYPES)
def test_attention_of_scores_up_to_2_to_the_23rd(form, dealt, dtype, tuning):
    """Scores that float32 holds, 2^13 or more apart but where they are equal: the mean of the values of a row's largest. Equal weights are rounded alike: what is left are sums of float32 and the
    result's rounding."""
    tuning(MI355X_TREE_FORM=form, MI355X_TREE_DEAL=dealt)
    tokens, page, columns = 20, 8, 40
    table, pages = shuffled_table(1, 2, columns)
    q, kp, vp = torch.zeros(2, tokens, 4, 64, dtype=dtype, device="cuda"), torch.zeros(pages, 2, page, 64, dtype=dtype, device="cuda"), normal(4, pages, 2, page, 64, dtype=dtype)
    q[..., 3] = torch.where(torch.arange(tokens, device="cuda") % 3 > 0, 8192.0, -8192.0)[None, :, None].to(dtype)
    kp[..., 3] = (8192 - 64 * torch.randint(0, 60, (pages, 2, page), generator=torch.Generator().manual_seed(5))).to(dtype).cuda()   # (64 is a step of bfloat16 from 4096 on)
    lengths = whole([290, 37])
    expected, size = C.attention(q, kp, vp, table, lengths)
    m, inputs = C.attention_model(q, kp, vp, table, lengths)
    within(m(*inputs), expected, 64 * U * size + R.HALF[dtype] * expected.abs() * (1 + 2.0 ** -7) + TINY[dtype])


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("form, dealt", [(0, 0), (1, 0), (2, 0), (0, 40)])
def test_attention_of_large_values(form, dealt, dtype, tuning):
    """Of 2^103: 2^8 of them for each of 500 keys are below 2^128."""
    tuning(MI355X_TREE_FORM=form, MI355X_TREE_DEAL=dealt)
    q, kp, vp, *rest = C.attention_case(5, 2, 30, 4, 2, 64, 16, 450, dtype, True, device="cuda")
    vp *= 2.0 ** 101
    m, inputs = C.attention_model(q, kp, vp, *rest)
    expected, bound = C.attention_rows(q, kp, vp, *rest)
    assert ((m(*inputs).double() - expected).norm(dim=-1) <= bound).all()


@pytest.mark.parametrize("form, dealt", [(0, 0), (1, 0), (2, 0), (0, 512), (1, 256), (2, 256)])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("page", [11, 16])
def test_rows_in_float32_of_long_contexts(form, dealt, d, page, tuning):
    """Trees behind 9000 keys, in every form, pages that go through registers and that do not."""
    tuning(MI355X_TREE_FORM=form, MI355X_TREE_DEAL=dealt)
    check_rows(2, 12, 4, 2, d, page, 9000, F32, True)
