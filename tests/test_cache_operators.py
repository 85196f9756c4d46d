"""The nodes of drafted tokens over a paged cache without a GPU: shapes, refusals of nodes and of the C interface, arrays that a node updates, and the definitions in
``cache_operators`` against each other."""
import ctypes

import numpy as np
import pytest
import torch

import dace_onnx_amd.onnx as donnx
from dace_onnx_amd import _lib, sdfg as dace
from dace_onnx_amd.onnx.proto import helper, numpy_helper
from dace_onnx_amd.onnx.shape_inference import ShapeInferenceError
import cache_operators as C
import llm_operators as R

BF, F32, I32, I64 = torch.bfloat16, torch.float32, torch.int32, torch.int64


def _z(*shape, dtype=F32):
    return torch.zeros(shape, dtype=dtype)


def _append(k=None, v=None, k_pages=None, v_pages=None, table=_z(2, 4, dtype=I32), lengths=_z(2, dtype=I32), dtype=F32, **rest):
    given = lambda t, *shape: _z(*shape, dtype=dtype) if t is None else t   # noqa: E731
    return C.append_model(given(k, 2, 3, 2, 8), given(v, 2, 3, 2, 8), given(k_pages, 9, 2, 5, 8), given(v_pages, 9, 2, 5, 8), table, lengths, **rest)[0]


def _attention(q=None, k_pages=None, v_pages=None, table=_z(2, 4, dtype=I32), lengths=_z(2, dtype=I32), dtype=F32, **rest):
    given = lambda t, *shape: _z(*shape, dtype=dtype) if t is None else t   # noqa: E731
    return C.attention_model(given(q, 2, 3, 4, 64), given(k_pages, 9, 2, 5, 64), given(v_pages, 9, 2, 5, 64), table, lengths, **rest)[0]


def _acceptance(logits=_z(2, 3, 50), tokens=_z(2, 3, dtype=I32), parents=None):
    return C.acceptance_model(logits, tokens, parents)[0]


def _calls(m):
    return [n for state in m.expand().nodes() for n in state.nodes() if isinstance(n, dace.KernelCall)]


@pytest.mark.parametrize("make, function", [
    (lambda: _append(), "mi355x_paged_cache_append"), (lambda: _append(dtype=BF, frequencies=_z(4), q=_z(2, 3, 6, 8, dtype=BF)), "mi355x_paged_cache_append"),
    (lambda: _append(frequencies=_z(3), positions=_z(2, 2, 3, dtype=I64), sections=[1, 2], interleaved=1), "mi355x_paged_cache_append"),
    (lambda: _append(order=_z(2, 7, dtype=I32), frequencies=_z(0)), "mi355x_paged_cache_append"),
    (lambda: _attention(), "mi355x_tree_attention"), (lambda: _attention(dtype=BF, parents=_z(2, 3, dtype=I32), scale=0.5), "mi355x_tree_attention"),
    (lambda: _acceptance(), "mi355x_draft_acceptance"), (lambda: _acceptance(_z(2, 3, 50, dtype=BF), parents=_z(2, 3, dtype=I32)), "mi355x_draft_acceptance")])
def test_nodes_expand_to_one_call(make, function):
    calls = _calls(make())
    assert [c.function for c in calls] == [function]
    assert f"{function}(" in calls[0].as_cpp()


@pytest.mark.parametrize("make", [
    lambda: _append(v=_z(2, 3, 2, 4)), lambda: _append(k_pages=_z(9, 3, 5, 8)), lambda: _append(v_pages=_z(8, 2, 5, 8)), lambda: _append(k_pages=_z(9, 2, 0, 8), v_pages=_z(9, 2, 0, 8)),
    lambda: _append(table=_z(3, 4, dtype=I32)), lambda: _append(lengths=_z(3, dtype=I32)), lambda: _append(q=_z(2, 3, 6, 8)),
    lambda: _append(frequencies=_z(4), q=_z(2, 3, 6, 4)), lambda: _append(frequencies=_z(4), q=_z(2, 3, 6, 8), order=_z(2, 3, dtype=I32)), lambda: _append(frequencies=_z(5)),
    lambda: _append(positions=_z(1, 2, 3, dtype=I32)), lambda: _append(frequencies=_z(4), positions=_z(1, 3, 2, dtype=I32)), lambda: _append(frequencies=_z(4), sections=[2, 2]),
    lambda: _append(frequencies=_z(4), sections=[3]), lambda: _append(sections=[0]), lambda: _append(order=_z(3, 3, dtype=I32)),
    lambda: _append(frequencies=_z(4), positions=_z(9, 2, 3, dtype=I32)),
    lambda: _attention(q=_z(2, 3, 4, 32), k_pages=_z(9, 2, 5, 32), v_pages=_z(9, 2, 5, 32)), lambda: _attention(q=_z(2, 3, 3, 64)), lambda: _attention(k_pages=_z(9, 2, 5, 128)),
    lambda: _attention(v_pages=_z(9, 2, 6, 64)), lambda: _attention(k_pages=_z(0, 2, 5, 64), v_pages=_z(0, 2, 5, 64)), lambda: _attention(table=_z(1, 4, dtype=I32)),
    lambda: _attention(lengths=_z(1, dtype=I32)), lambda: _attention(parents=_z(2, 4, dtype=I32)), lambda: _attention(scale=0.0), lambda: _attention(scale=float("inf")),
    lambda: _attention(q=_z(2, 1025, 4, 64), parents=_z(2, 1025, dtype=I32)), lambda: _acceptance(tokens=_z(2, 4, dtype=I32)), lambda: _acceptance(parents=_z(2, 2, dtype=I32)),
    lambda: _acceptance(_z(2, 3, 0)), lambda: _acceptance(_z(2, 0, 50), _z(2, 0, dtype=I32)), lambda: _acceptance(_z(1, 1025, 2), _z(1, 1025, dtype=I32))])
def test_nodes_that_are_refused(make):
    with pytest.raises(donnx.ExpansionRefused):
        make().expand()


@pytest.mark.parametrize("make, error", [
    (lambda: _append(v=_z(2, 3, 2, 8, dtype=BF)), "type constraints"), (lambda: _append(lengths=_z(2, dtype=I64)), "type constraints"), (lambda: _append(table=_z(2, 4, dtype=I64)), "Expected type"),
    (lambda: _append(k_pages=_z(9, 2, 5, 8, dtype=torch.int8), v_pages=_z(9, 2, 5, 8, dtype=torch.int8)), "type constraints"), (lambda: _append(order=_z(2, 3, dtype=I64)), "type constraints"),
    (lambda: _append(frequencies=_z(4, dtype=BF)), "Expected type"), (lambda: _attention(q=_z(2, 3, 4, 64, dtype=BF)), "type constraints"),
    (lambda: _attention(parents=_z(2, 3, dtype=I64)), "type constraints"), (lambda: _acceptance(_z(2, 3, 50, dtype=I32)), "Expected type"), (lambda: _acceptance(tokens=_z(2, 3, dtype=I64)), "Expected type")])
def test_types_that_are_refused(make, error):
    with pytest.raises(ValueError, match=error):
        make().expand()


def test_shapes_that_contradict_the_declared_ones():
    with pytest.raises(ShapeInferenceError):
        R.model("TreeAttention", [("q", _z(2, 3, 4, 64)), ("k", _z(9, 2, 5, 64)), ("v", _z(9, 2, 5, 64)), ("t", _z(2, 4, dtype=I32)), ("n", _z(2, dtype=I32))], [("o", F32, (2, 3, 4, 32))])
    with pytest.raises(ShapeInferenceError):
        R.model("DraftAcceptance", [("l", _z(2, 50)), ("t", _z(2, 3, dtype=I32))], [("p", I32, (2, 3)), ("c", I32, (2,)), ("n", I32, (2,))])


# ---------------------------------------------------------------------------------------------- arrays that a node updates

SHAPES = {"k": (2, 3, 2, 64), "v": (2, 3, 2, 64), "kp": (9, 2, 5, 64), "vp": (9, 2, 5, 64), "table": (2, 4), "lengths": (2,), "q": (2, 3, 4, 64)}


def _graph(nodes, inputs, outputs, initializers=()):
    info = lambda n, shape: helper.make_tensor_value_info(n, 6 if n in ("table", "lengths") else 1, list(shape))   # noqa: E731
    return helper.make_model(helper.make_graph(nodes, "g", [info(n, SHAPES[n]) for n in inputs], [info(n, s) for n, s in outputs],
                                               initializer=[numpy_helper.from_array(np.zeros(SHAPES[n], dtype=np.float32), name=n) for n in initializers]))


def _append_node(outs=("ko", "vo"), caches=("kp", "vp"), name="append"):
    return helper.make_node("PagedCacheAppend", ["k", "v", *caches, "table", "lengths"], list(outs), name=name)


def _attend(k, v, out="o"):
    return helper.make_node("TreeAttention", ["q", k, v, "table", "lengths"], [out], name="attend_" + out)


ALL = ("k", "v", "kp", "vp", "table", "lengths", "q")


def test_an_updated_input_and_what_reads_it_are_one_array():
    m = donnx.ONNXModel("g", _graph([_append_node(), _attend("ko", "vo")], ALL, [("o", SHAPES["q"]), ("vo", SHAPES["vp"])]))
    sdfg = m.expand()
    assert {n for n, d in sdfg.arrays.items() if not d.transient} == {*ALL, "o"} and m.outputs == ["o", "vo"]
    compiled = dace.CompiledSDFG(sdfg)
    assert [n.function for _, n, *_ in compiled._plan] == ["mi355x_paged_cache_append", "mi355x_tree_attention"]   # whatever order the nodes are listed in
    (_, first, keys), (_, second, later) = compiled._plan
    assert keys["k_pages"] == keys["k_pages_out"] == later["k_pages"] == "kp" and keys["v_pages_out"] == later["v_pages"] == "vp"


def test_reads_come_after_the_update_in_any_order_of_the_nodes():
    m = donnx.ONNXModel("g", _graph([_attend("ko", "vo"), _append_node()], ALL, [("o", SHAPES["q"])]), infer_shapes=False)
    assert [n.function for _, n, *_ in dace.CompiledSDFG(m.expand())._plan] == ["mi355x_paged_cache_append", "mi355x_tree_attention"]


@pytest.mark.parametrize("nodes, inputs, outputs, initializers, error", [
    ([_append_node(), _attend("kp", "vo")], ALL, [("o", SHAPES["q"])], (), "other readers"),                                        # the cache before, next to the one after
    ([_append_node(), helper.make_node("Identity", ["kp"], ["x"], name="i")], ALL, [("x", SHAPES["kp"])], (), "other readers"),
    ([_append_node()], ALL, [("kp", SHAPES["kp"])], (), "other readers"),
    ([_append_node(caches=("kp", "kp"))], ALL, [("ko", SHAPES["kp"])], (), "other readers"),                                         # keys and values in one array
    ([_append_node(), _append_node(("k2", "v2"), ("ko", "vo"), "again")], ALL, [("k2", SHAPES["kp"])], (), "input of the graph"),    # an update of an update
    ([_append_node()], tuple(n for n in ALL if n != "kp"), [("ko", SHAPES["kp"])], ("kp",), "input of the graph"),
    ([_append_node()], ALL, [("ko", SHAPES["kp"])], ("kp",), "input of the graph")])
def test_updates_that_are_refused(nodes, inputs, outputs, initializers, error):
    with pytest.raises(ValueError, match=error):
        donnx.ONNXModel("g", _graph(nodes, inputs, outputs, initializers))


def test_a_node_whose_output_is_another_array_is_refused():
    sdfg = dace.SDFG("s")
    state = sdfg.add_state()
    node = donnx.ONNXPagedCacheAppend("append")
    state.add_node(node)
    shapes = {"K": SHAPES["k"], "V": SHAPES["v"], "k_pages": SHAPES["kp"], "v_pages": SHAPES["vp"], "table": (2, 4), "lengths": (2,)}
    for name, shape in shapes.items():
        sdfg.add_array(name, shape, dace.int32 if name in ("table", "lengths") else dace.float32)
        node.add_in_connector(name)
        state.add_edge(state.add_read(name), None, node, name, sdfg.make_array_memlet(name))
    sdfg.add_array("other", SHAPES["kp"], dace.float32)
    for conn, data in (("k_pages_out", "other"), ("v_pages_out", "v_pages")):
        node.add_out_connector(conn)
        state.add_edge(node, conn, state.add_write(data), None, sdfg.make_array_memlet(data))
    with pytest.raises(donnx.ExpansionRefused):
        node.expand(sdfg, state)


@pytest.mark.parametrize("shared", [True, False])
def test_a_state_in_which_another_node_reads_what_the_array_was(shared):
    """Nothing says which of the two comes first where both read one access node. A reader with a node of its own comes after the update."""
    sdfg = dace.SDFG("s")
    state = sdfg.add_state()
    append, attend = donnx.ONNXPagedCacheAppend("append"), donnx.ONNXTreeAttention("attend")
    shapes = {"K": SHAPES["k"], "V": SHAPES["v"], "k_pages": SHAPES["kp"], "v_pages": SHAPES["vp"], "table": (2, 4), "lengths": (2,), "Q": SHAPES["q"], "O": SHAPES["q"]}
    for name, shape in shapes.items():
        sdfg.add_array(name, shape, dace.int32 if name in ("table", "lengths") else dace.float32)
    access = {}

    def connect(node, reads, writes):
        state.add_node(node)
        for name in reads:
            if name not in access or (name.endswith("_pages") and not shared):
                access[name] = state.add_read(name)
            node.add_in_connector(name)
            state.add_edge(access[name], None, node, name, sdfg.make_array_memlet(name))
        for conn, name in writes.items():
            node.add_out_connector(conn)
            state.add_edge(node, conn, state.add_write(name), None, sdfg.make_array_memlet(name))
    connect(attend, ["Q", "k_pages", "v_pages", "table", "lengths"], {"O": "O"})
    connect(append, ["K", "V", "k_pages", "v_pages", "table", "lengths"], {"k_pages_out": "k_pages", "v_pages_out": "v_pages"})
    if shared:
        with pytest.raises(donnx.ExpansionRefused):
            sdfg.expand_library_nodes()
    else:
        sdfg.expand_library_nodes()
        assert [n.function for _, n, *_ in dace.CompiledSDFG(sdfg)._plan] == ["mi355x_paged_cache_append", "mi355x_tree_attention"]


def test_the_call_form_takes_one_array_for_both():
    values = {"K": _z(*SHAPES["k"]), "V": _z(*SHAPES["v"]), "table": _z(2, 4, dtype=I32), "lengths": _z(2, dtype=I32)}
    kp, vp = _z(*SHAPES["kp"]), _z(*SHAPES["vp"])
    with pytest.raises(ValueError, match="the same array"):
        donnx.ONNXPagedCacheAppend(**values, k_pages=kp, v_pages=vp, k_pages_out=_z(*SHAPES["kp"]), v_pages_out=vp)


# ---------------------------------------------------------------------------------------------- the C interface


def _refused(function, *args):
    lib = _lib.library()
    assert getattr(lib, function)(*args) != 0
    return lib.mi355x_last_error().decode()


APPEND = dict(K=16, V=16, Q=None, kp=16, vp=16, Qo=None, table=16, lengths=16, f=16, pos=None, order=None, batch=2, tokens=3, heads=0, kv=2, size=8, pages=9, page=5, columns=4, taken=3,
              rotated=8, axes=1, sections=[4], interleaved=0, bytes=8, type=1)


@pytest.mark.parametrize("change, error", [
    (dict(batch=-1), "negative"), (dict(columns=-1), "negative"), (dict(taken=-1), "negative"), (dict(type=7), "element type"), (dict(page=0), "pages of 0"), (dict(bytes=2), "positions of 2"),
    (dict(rotated=7), "of 8 values"), (dict(rotated=10), "of 8 values"), (dict(axes=0, sections=[]), "axes"), (dict(axes=9, sections=[4] + [0] * 8, pos=16), "axes"),
    (dict(axes=2, sections=[2, 2]), "own number"), (dict(heads=4, Q=16, Qo=16, order=16), "own order"), (dict(taken=2), "without an order"), (dict(sections=[3]), "sections of 3"),
    (dict(sections=[-1]), "section of -1"), (dict(size=1 << 17), "head too large"), (dict(heads=1 << 13, Q=16, Qo=16), "head too large"), (dict(tokens=1 << 31, taken=1 << 31), "too large"),
    (dict(pages=1 << 31), "too large"), (dict(K=None), "null pointer"), (dict(vp=None), "null pointer"), (dict(table=None), "null pointer"), (dict(lengths=None), "null pointer"),
    (dict(f=None), "null pointer"), (dict(heads=4, Q=16), "null pointer"), (dict(batch=(1 << 31) - 1, tokens=1 << 20, taken=1 << 20), "too many")])
def test_append_refusals(change, error):
    a = {**APPEND, **change}
    a["sections"] = (ctypes.c_int64 * max(len(a["sections"]), 1))(*a["sections"])
    assert error in _refused("mi355x_paged_cache_append", *a.values(), None)


ATTENTION = dict(Q=16, kp=16, vp=16, table=16, lengths=16, parents=None, O=16, scratch=None, floats=0, batch=1, tokens=3, heads=4, kv=2, size=64, pages=9, page=5, columns=4, scale=0.125, type=1)


@pytest.mark.parametrize("change, error", [
    (dict(type=3), "element type"), (dict(size=32), "head size 32"), (dict(heads=3), "3 heads"), (dict(kv=0), "heads share"), (dict(scale=0.0), "scale"), (dict(scale=float("nan")), "scale"),
    (dict(parents=16, tokens=1025), "tree of 1025"), (dict(pages=0), "extent"), (dict(page=0), "extent"), (dict(batch=-1), "extent"), (dict(columns=1 << 29, page=4), "extent"),
    (dict(Q=None), "null pointer"), (dict(table=None), "null pointer"), (dict(O=None), "null pointer"), (dict(vp=24), "16-byte")])
def test_attention_refusals(change, error):
    assert error in _refused("mi355x_tree_attention", *{**ATTENTION, **change}.values(), None)


ACCEPTANCE = dict(logits=16, tokens=16, parents=None, path=16, count=16, next=16, scratch=16, words=1 << 20, batch=2, token_count=3, vocabulary=50, type=1)


@pytest.mark.parametrize("change, error", [
    (dict(type=6), "element type"), (dict(token_count=0), "trees of 0"), (dict(token_count=1025), "trees of 1025"), (dict(vocabulary=0), "vocabulary of 0"), (dict(batch=-1), "-1 trees"),
    (dict(vocabulary=1 << 31), "vocabulary"), (dict(logits=None), "null pointer"), (dict(next=None), "null pointer"), (dict(scratch=None), "scratch"), (dict(scratch=20), "scratch"), (dict(words=5), "scratch")])
def test_acceptance_refusals(change, error):
    assert error in _refused("mi355x_draft_acceptance", *{**ACCEPTANCE, **change}.values(), None)


def test_calls_without_tokens_launch_nothing():
    lib = _lib.library()
    one = (ctypes.c_int64 * 1)(4)
    for change in (dict(batch=0), dict(tokens=0, taken=0), dict(kv=0)):
        assert lib.mi355x_paged_cache_append(*{**APPEND, **change, "sections": one}.values(), None) == 0
    for change in (dict(batch=0), dict(tokens=0), dict(heads=0)):
        assert lib.mi355x_tree_attention(*{**ATTENTION, **change}.values(), None) == 0
    assert lib.mi355x_draft_acceptance(*{**ACCEPTANCE, "batch": 0}.values(), None) == 0


# ---------------------------------------------------------------------------------------------- the definitions


def test_attention_of_the_definitions_is_softmax_over_the_gathered_cache():
    g = torch.Generator().manual_seed(1)
    q, kp, vp = (torch.randn(*s, generator=g) for s in ((2, 3, 4, 8), (9, 2, 5, 8), (9, 2, 5, 8)))
    table, lengths = torch.tensor([[3, 1, 7], [0, 8, 2]], dtype=I32), torch.tensor([6, 0], dtype=I32)
    out, _ = C.attention(q, kp, vp, table, lengths)
    for b in range(2):
        n = int(lengths[b]) + 3
        k, v = (t[table[b].long()].permute(1, 0, 2, 3).reshape(2, 15, 8)[:, :n].repeat_interleave(2, 0).double() for t in (kp, vp))
        mask = torch.ones(3, n, dtype=torch.bool).tril(n - 3)
        expected = torch.nn.functional.scaled_dot_product_attention(q[b].transpose(0, 1).double(), k, v, attn_mask=mask)
        assert torch.allclose(out[b].transpose(0, 1), expected)
    chain = torch.arange(-1, 2, dtype=I32).expand(2, 3)
    assert torch.equal(C.attention(q, kp, vp, table, lengths, chain)[0], out)


def test_append_and_acceptance_of_the_definitions():
    g = torch.Generator().manual_seed(2)
    k, v, kp, vp = (torch.randn(*s, generator=g) for s in ((1, 4, 2, 8), (1, 4, 2, 8), (5, 2, 3, 8), (5, 2, 3, 8)))
    table, lengths = torch.tensor([[4, 0, 2]], dtype=I32), torch.tensor([2], dtype=I32)
    after, values, written, *_ = C.append(k, v, kp, vp, table, lengths, order=torch.tensor([[0, 3, -1, 4]], dtype=I32))
    assert written.nonzero().tolist() == [[0, 0], [4, 2]]
    assert torch.equal(after[4, :, 2], k[0, 0].double()) and torch.equal(values[0, :, 0], v[0, 3].double())
    logits = torch.zeros(1, 5, 7)
    logits[0, range(5), [3, 5, 2, 6, 1]] = 1.0
    path, count, after = C.acceptance(logits, torch.tensor([[0, 3, 3, 5, 6]], dtype=I32), torch.tensor([[-1, 0, 0, 1, 3]], dtype=I32))
    assert path.tolist() == [[0, 1, 3, 4, -1]] and count.tolist() == [4] and after.tolist() == [1]


def test_the_small_transformer_has_clear_largest_logits():
    """What the test of a run on the GPU compares are tokens: float32 cannot change which logit is the largest."""
    weights = C.transformer_weights(7)
    for prompt in ([5, 17, 3, 200, 44, 9, 101], [77, 8]):
        _, least = C.greedy(weights, prompt, 24)
        assert least > 2e-3


@pytest.mark.parametrize("apart", [0, 16, 4 * 9 * 2 * 5 * 8 - 16])
def test_keys_and_values_in_the_same_pages(apart):
    first = (ctypes.c_int64 * 1)(4)
    for k, v in ((1 << 20, (1 << 20) + apart), ((1 << 20) + apart, 1 << 20)):
        assert "share pages" in _refused("mi355x_paged_cache_append", *{**APPEND, "kp": k, "vp": v, "sections": first}.values(), None)


def test_a_scale_that_leaves_float32():
    assert "scale" in _refused("mi355x_tree_attention", *{**ATTENTION, "scale": 3e38}.values(), None)


# ---------------------------------------------------------------------------------------------- the bound of a row


@pytest.mark.parametrize("d", [64, 128, 256])
def test_the_bound_of_a_row_takes_three_parts_and_no_two(d):
    """What float32's operands become, in sums without an error of their own: of three parts the six largest products stay within the bound, of two parts the three largest do not."""
    case = C.attention_case(1, 2, 5, 4, 2, d, 7, 300, F32, True)
    expected, bound = C.attention_rows(*case)
    three, two = (C.attention_rows(*case, **C.by_parts(count, least))[0] for count, least in ((3, 2), (2, 1)))
    assert ((three - expected).norm(dim=-1) < bound / 3).all()
    assert ((two - expected).norm(dim=-1) > bound).double().mean() > 0.5


@pytest.mark.parametrize("dtype, share", [(F32, 0.99), (torch.float16, 0.9), (BF, 0.4)])
@pytest.mark.parametrize("d", [64, 256])
def test_the_bound_of_a_row_sees_a_key_that_is_missing(dtype, share, d):
    """One of 5000 keys with scores of a deviation of 2 is worth e^(s - 4) / sqrt(5000) of a row's result. The bound is 2.8e-5 of that, 4.9e-4, 3.9e-3: s above -2.2, 0.6, 2.7, which 86, 38 and 9 % of keys
    have for a row, and 100, 98 and 52 % for one of eight."""
    case = C.attention_case(2, 1, 1, 8, 1, d, 16, 5000, dtype)
    expected, bound = C.attention_rows(*case)
    found = [bool(((C.attention_rows(*case, without=(0, n))[0] - expected).norm(dim=-1) > bound).any()) for n in range(1, 5000, 173)]
    assert np.mean(found) >= share


def test_the_bounds_of_rows_are_near_what_rounding_does():
    """Results and weights rounded to 16 bits, nothing else: within the bound, and above a quarter of it on average."""
    for dtype in (torch.float16, BF):
        case = C.attention_case(3, 2, 9, 4, 2, 64, 16, 700, dtype)
        expected, bound = C.attention_rows(*case)

        def rounded(p, v):
            r = p.to(dtype).double()
            return r @ v * (p.sum(-1, keepdim=True) / r.sum(-1, keepdim=True))
        got = C.attention_rows(*case, weights=rounded)[0].to(dtype)
        error = (got.double() - expected).norm(dim=-1) / bound
        assert error.max() < 1 and error.mean() > 0.25
    out, _ = C.attention(*C.attention_case(4, 2, 9, 4, 2, 64, 16, 70, F32, True))
    assert torch.allclose(out, C.attention_rows(*C.attention_case(4, 2, 9, 4, 2, 64, 16, 70, F32, True))[0], rtol=1e-12, atol=1e-12)
