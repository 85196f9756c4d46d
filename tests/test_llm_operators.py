"""The nodes of quantised and differential transformers without a GPU: shapes, refusals of nodes and of the C interface, bfloat16 on the host,
and the definitions in ``llm_operators`` against elementary sums."""
import glob
import os
import re

import numpy as np
import pytest
import torch

import dace_onnx_amd.onnx as donnx
from dace_onnx_amd import _lib, sdfg as dace
from dace_onnx_amd.onnx import proto
from dace_onnx_amd.onnx.shape_inference import ShapeInferenceError
import llm_operators as R

BF, F32 = torch.bfloat16, torch.float32


def _z(*shape, dtype=F32):
    return torch.zeros(shape, dtype=dtype)


def _functions(m):
    m.expand()
    found = []

    def walk(graph):
        for state in graph.nodes():
            for n in state.nodes():
                if isinstance(n, dace.KernelCall):
                    found.append(n)
                elif isinstance(n, dace.NestedSDFG):
                    walk(n.sdfg)
    walk(m.sdfg)
    return found


def _norm(x=_z(3, 8), gain=_z(8), skip=None, outs="Y", dtype=F32, q_shape=None, **attributes):
    shape = tuple(x.shape)
    made = {"Y": ("y", dtype, shape), "S": ("s", dtype, shape), "Q": ("q", torch.int8, shape), "q": ("qs", F32, q_shape or shape[:attributes.get("axis", -1)])}
    return R.model("SkipRMSNormalization", [("x", x), ("g", gain), ("skip", skip)], [made[k] if k in outs else None for k in "YSQq"], **attributes)


def _linear(x=_z(3, 8, dtype=torch.int8), w=_z(5, 8, dtype=torch.int8), xs=_z(3), ws=_z(5), bias=None, residual=None, dtype=F32, shape=None, **attributes):
    attributes.setdefault("to", R.ELEMENT[dtype])
    return R.model("QuantizedLinear", [("x", x), ("w", w), ("xs", xs), ("ws", ws), ("b", bias), ("r", residual)],
                   [("y", dtype, shape or tuple(x.shape[:-1]) + (w.shape[0],))], **attributes)


def _rotary(q=_z(2, 3, 4, 8), positions=_z(2, 2, 3, dtype=torch.int64), frequencies=_z(4), k=None, **attributes):
    attributes.setdefault("sections", [2, 2])
    return R.model("RotaryPositions", [("q", q), ("p", positions), ("f", frequencies), ("k", k)],
                   [("qo", q.dtype, tuple(q.shape)), None if k is None else ("ko", k.dtype, tuple(k.shape))], **attributes)


def _attention(q=_z(2, 3, 8, 32), k=_z(2, 5, 4, 32), v=_z(2, 5, 2, 64), vectors=(_z(32),) * 4, lengths=None, shape=None, **attributes):
    return R.model("DifferentialAttention", [("q", q), ("k", k), ("v", v)] + [(f"l{i}", w) for i, w in enumerate(vectors)] + [("n", lengths)],
                   [("o", q.dtype, shape or (q.shape[0], q.shape[1], q.shape[2] // 2, v.shape[3]))], **attributes)


@pytest.mark.parametrize("make, function", [
    (lambda: _norm(outs="YSQq", skip=_z(3, 8)), "mi355x_skip_rms_norm"), (lambda: _norm(_z(2, 3, 8, dtype=BF), _z(24, dtype=BF), outs="Qq", dtype=BF, axis=1, q_shape=(2,)), "mi355x_skip_rms_norm"),
    (lambda: _linear(bias=_z(5), residual=_z(3, 5), activation="silu"), "mi355x_quantized_linear"),
    (lambda: _linear(x=_z(2, 3, 8, dtype=torch.int8), xs=_z(2, 3, 1), ws=_z(1), dtype=BF), "mi355x_quantized_linear"),
    (lambda: _rotary(k=_z(2, 3, 1, 8)), "mi355x_rotary_positions"), (lambda: _rotary(positions=_z(1, 2, 3, dtype=torch.int32), sections=None), "mi355x_rotary_positions"),
    (lambda: _attention(lengths=_z(2, dtype=torch.int32), causal=1), "mi355x_differential_attention")])
def test_nodes_expand_to_one_call(make, function):
    calls = _functions(make())
    assert [c.function for c in calls] == [function]
    assert f"{function}(" in calls[0].as_cpp()


def test_sums_of_splits_are_a_transient_of_the_graph():
    """Where keys are dealt to several workgroups the graph has an array for their sums, and one to a node."""
    q, k, v = _z(1, 1, 4, 64, dtype=BF), _z(1, 4096, 4, 64, dtype=BF), _z(1, 4096, 2, 128, dtype=BF)
    vectors = tuple(_z(8) for _ in range(4))
    m = _attention(q, k, v, vectors)
    call, = _functions(m)
    splits = _lib.library().mi355x_differential_attention_splits(1, 1, 4096, 2, 2, 64, 16)
    transients = [d for d in m.sdfg.arrays.values() if d.transient]
    assert splits > 1 and call.args[-4] == 0 and call.args[-3] == splits
    assert [tuple(d.shape) for d in transients] == [(splits * 2 * (4 * 64 + 4),)] and transients[0].dtype == dace.float32
    assert not any(d.transient for d in _attention().expand().arrays.values())


@pytest.mark.parametrize("make", [
    lambda: _norm(outs="Q"), lambda: _norm(outs="q"), lambda: _norm(gain=_z(3)), lambda: _norm(skip=_z(1, 8)), lambda: _norm(epsilon=-1.0),
    lambda: _norm(epsilon=float("nan")), lambda: _norm(_z(3, 0), _z(0)),
    lambda: _linear(xs=_z(2)), lambda: _linear(ws=_z(3)), lambda: _linear(bias=_z(3)), lambda: _linear(residual=_z(1, 5)), lambda: _linear(activation="tanh"),
    lambda: _linear(x=_z(1, 1 << 17, dtype=torch.int8), w=_z(1, 1 << 17, dtype=torch.int8), xs=_z(1), ws=_z(1)), lambda: _linear(xs=_z(1, 3)),
    lambda: _rotary(sections=[1, 2]), lambda: _rotary(sections=[4]), lambda: _rotary(sections=[5, -1]), lambda: _rotary(frequencies=_z(5), sections=[2, 3]),
    lambda: _rotary(positions=_z(2, 3, 2, dtype=torch.int64)), lambda: _rotary(k=_z(2, 3, 1, 6)), lambda: _rotary(sections=None, positions=_z(9, 2, 3, dtype=torch.int64)),
    lambda: _attention(q=_z(2, 3, 8, 48), k=_z(2, 5, 4, 48), v=_z(2, 5, 2, 96)), lambda: _attention(q=_z(2, 3, 6, 32)), lambda: _attention(v=_z(2, 4, 2, 64)),
    lambda: _attention(vectors=(_z(32), _z(31), _z(32), _z(32))), lambda: _attention(lengths=_z(3, dtype=torch.int32)), lambda: _attention(scale=0.0),
    lambda: _attention(scale=-1.0), lambda: _attention(k=_z(2, 5, 3, 32)), lambda: _attention(vectors=(_z(2, 16),) * 4)])
def test_nodes_that_are_refused(make):
    with pytest.raises(donnx.ExpansionRefused):
        make().expand()


@pytest.mark.parametrize("make, error", [
    (lambda: _norm(gain=_z(8, dtype=BF)), "type constraints"), (lambda: _norm(_z(3, 8, dtype=torch.int32), _z(8, dtype=torch.int32), dtype=torch.int32), "Expected type"),
    (lambda: _linear(bias=_z(5, dtype=BF)), "type constraints"), (lambda: _linear(xs=_z(3, dtype=BF)), "Expected type"),
    (lambda: _attention(lengths=_z(2, dtype=torch.int64)), "Expected type"), (lambda: _attention(k=_z(2, 5, 4, 32, dtype=BF)), "type constraints"),
    (lambda: _rotary(frequencies=_z(4, dtype=BF)), "Expected type")])
def test_types_that_are_refused(make, error):
    with pytest.raises(ValueError, match=error):
        make().expand()


@pytest.mark.parametrize("make", [lambda: _linear(w=_z(5, 7, dtype=torch.int8)), lambda: _attention(q=_z(3, 8, 32), shape=(3, 4, 64)), lambda: _norm(axis=2),
                                  lambda: _norm(outs="Qq", q_shape=(4,)), lambda: _linear(shape=(3, 6)), lambda: _attention(shape=(2, 3, 4, 32))])
def test_shapes_that_do_not_fit(make):
    with pytest.raises(ShapeInferenceError):
        make()


def _status(name, *args):
    args = [_lib.i64_array(a) if isinstance(a, list) else a for a in args]
    status = getattr(_lib.library(), name)(*args, None)
    return status, _lib.library().mi355x_last_error().decode()


P = 4096   # an address that no refused call reads
NORM = dict(X=P, skip=P, gain=P, Y=P + 64, Sum=P + 128, Q=P, q_scale=P, rows=4, cols=8, type=1, epsilon=1e-5)
LINEAR = dict(X=P, W=P, xs=P, ws=P, bias=P, residual=P, Y=P, M=4, N=6, K=8, xc=4, wc=6, activation=0, type=1)
ROTARY = dict(Q=P, K=P, positions=P, frequencies=P, Qo=P, Ko=P, tokens=4, heads=2, kv=1, size=8, rotated=8, axes=2, sections=[2, 2], interleaved=0, bytes=8, type=1)
ATTENTION = dict(Q=P, K=P, V=P, q1=P, k1=P, q2=P, k2=P, lengths=P, O=P, scratch=P, batch=2, Sq=3, Sk=4, heads=4, groups=2, size=64, vector=8, init=0.5, scale=1.0,
                 causal=0, splits=1, type=1)


@pytest.mark.parametrize("name, base, change, message", [
    ("mi355x_skip_rms_norm", NORM, dict(rows=-1), "negative"), ("mi355x_skip_rms_norm", NORM, dict(type=11), "element type"),
    ("mi355x_skip_rms_norm", NORM, dict(X=None), "null"), ("mi355x_skip_rms_norm", NORM, dict(Q=None), "together"), ("mi355x_skip_rms_norm", NORM, dict(cols=0), "without columns"),
    ("mi355x_skip_rms_norm", NORM, dict(Y=None, Sum=None, Q=None, q_scale=None), "no output"), ("mi355x_skip_rms_norm", NORM, dict(epsilon=float("inf")), "epsilon"),
    ("mi355x_skip_rms_norm", NORM, dict(rows=1 << 40), "too many"), ("mi355x_skip_rms_norm", NORM, dict(cols=1 << 31), "too many"),
    ("mi355x_skip_rms_norm", NORM, dict(Sum=P, cols=20000), "over the input"), ("mi355x_skip_rms_norm", NORM, dict(Sum=P + 64), "one array"),
    ("mi355x_quantized_linear", LINEAR, dict(K=1 << 17), "2\\^17"), ("mi355x_quantized_linear", LINEAR, dict(xc=3), "x_scale"), ("mi355x_quantized_linear", LINEAR, dict(wc=4), "w_scale"),
    ("mi355x_quantized_linear", LINEAR, dict(activation=4), "activation"), ("mi355x_quantized_linear", LINEAR, dict(type=3), "element type"),
    ("mi355x_quantized_linear", LINEAR, dict(M=-4, xc=1), "negative"), ("mi355x_quantized_linear", LINEAR, dict(W=None), "null"),
    ("mi355x_quantized_linear", LINEAR, dict(M=1 << 31, xc=1), "too large"),
    ("mi355x_quantized_linear", LINEAR, dict(M=(1 << 31) - 1, N=(1 << 31) - 1, xc=1, wc=1), "too large"), ("mi355x_skip_rms_norm", NORM, dict(rows=1 << 26), "too many"),
    ("mi355x_rotary_positions", ROTARY, dict(tokens=1 << 27), "too many"),
    ("mi355x_rotary_positions", ROTARY, dict(rotated=7), "values"), ("mi355x_rotary_positions", ROTARY, dict(rotated=10), "values"), ("mi355x_rotary_positions", ROTARY, dict(axes=9), "axes"),
    ("mi355x_rotary_positions", ROTARY, dict(sections=[2, 1]), "sections"), ("mi355x_rotary_positions", ROTARY, dict(sections=[5, -1]), "section"),
    ("mi355x_rotary_positions", ROTARY, dict(bytes=2), "positions of 2"), ("mi355x_rotary_positions", ROTARY, dict(K=None), "null"), ("mi355x_rotary_positions", ROTARY, dict(type=6), "element type"),
    ("mi355x_rotary_positions", ROTARY, dict(tokens=1 << 40), "too many"), ("mi355x_rotary_positions", ROTARY, dict(heads=-1), "negative"),
    ("mi355x_differential_attention", ATTENTION, dict(size=48), "head size"), ("mi355x_differential_attention", ATTENTION, dict(groups=3), "share"),
    ("mi355x_differential_attention", ATTENTION, dict(groups=0), "share"), ("mi355x_differential_attention", ATTENTION, dict(scale=0.0), "scale"),
    ("mi355x_differential_attention", ATTENTION, dict(scale=float("nan")), "scale"), ("mi355x_differential_attention", ATTENTION, dict(splits=0), "splits"),
    ("mi355x_differential_attention", ATTENTION, dict(splits=2, scratch=None), "scratch"), ("mi355x_differential_attention", ATTENTION, dict(splits=2, scratch=P + 4), "scratch"),
    ("mi355x_differential_attention", ATTENTION, dict(V=None), "null"), ("mi355x_differential_attention", ATTENTION, dict(q1=None), "null"),
    ("mi355x_differential_attention", ATTENTION, dict(Sk=1 << 31), "too large"),
    ("mi355x_differential_attention", ATTENTION, dict(Sk=(1 << 31) - 1), "too large"), ("mi355x_differential_attention", ATTENTION, dict(batch=1 << 30, Sq=1 << 30, heads=16, groups=16), "too large"),
    ("mi355x_differential_attention", ATTENTION, dict(batch=1 << 26, splits=256), "too large"), ("mi355x_differential_attention", ATTENTION, dict(batch=1 << 20, Sq=1 << 16), "too large"),
    ("mi355x_differential_attention", ATTENTION, dict(type=2), "element type"), ("mi355x_differential_attention", ATTENTION, dict(batch=-1), "negative")])
def test_calls_that_are_refused(name, base, change, message):
    status, error = _status(name, *{**base, **change}.values())
    assert status == 1
    assert re.search(message, error), error


@pytest.mark.parametrize("name, base, change", [
    ("mi355x_skip_rms_norm", NORM, dict(rows=0)), ("mi355x_skip_rms_norm", NORM, dict(rows=0, cols=0)), ("mi355x_quantized_linear", LINEAR, dict(M=0, xc=0)),
    ("mi355x_quantized_linear", LINEAR, dict(N=0, wc=1)), ("mi355x_rotary_positions", ROTARY, dict(tokens=0)), ("mi355x_rotary_positions", ROTARY, dict(heads=0, kv=0)),
    ("mi355x_differential_attention", ATTENTION, dict(batch=0)), ("mi355x_differential_attention", ATTENTION, dict(Sq=0)), ("mi355x_differential_attention", ATTENTION, dict(heads=0))])
def test_empty_calls_launch_nothing(name, base, change):
    assert _status(name, *{**base, **change}.values())[0] == 0


def test_parts_of_sizes_that_do_not_exist():
    splits = _lib.library().mi355x_differential_attention_splits
    assert splits(1, 1, 8192, 16, 4, 64, 16) > 1
    for sizes in [(1 << 31, 1 << 31, 1 << 31, 4, 4), (1 << 30, 1 << 30, 1 << 30, 16, 16), (0, 1, 1, 1, 1), (1, 1, 1 << 40, 1, 1), (-1, 1, 1, 1, 1), (1, 1, 1, 3, 2), (1, 1, 1, 1, 0)]:
        assert splits(*sizes, 64, 1) == 1


# ---------------------------------------------------------------------------------------------- bfloat16 on the host


def test_bfloat16_tensors_in_files():
    values = np.array([0.0, -0.0, 1.0, 1.00390625, 1.01171875, -3.14159, 1e-40, 3.4e38, np.inf, -np.inf, np.nan], dtype=np.float32)
    made = proto.helper.make_tensor("w", proto.TensorProto.BFLOAT16, [11], values)
    expected = torch.from_numpy(values).to(BF).float().numpy()   # to the nearest, ties to even
    assert np.array_equal(made.array, expected, equal_nan=True)
    again = proto._parse_tensor(proto._ser_tensor(made))
    assert again.data_type == 16 and np.array_equal(again.array, expected, equal_nan=True) and np.signbit(again.array[1])
    assert proto.np_dtype_to_tensor_dtype(np.float32) == proto.TensorProto.FLOAT


def test_bfloat16_weights_and_descriptors():
    helper, T = proto.helper, proto.TensorProto
    weight = helper.make_tensor("g", T.BFLOAT16, [8], np.arange(8) / 7)
    node = helper.make_node("SkipRMSNormalization", ["x", "g"], ["y"])
    reshape = helper.make_node("Reshape", ["y", "shape"], ["z"])
    shape = proto.numpy_helper.from_array(np.array([8, 3], np.int64), "shape")
    graph = helper.make_graph([node, reshape], "g", [helper.make_tensor_value_info("x", T.BFLOAT16, [3, 8])], [helper.make_tensor_value_info("z", T.BFLOAT16, [8, 3])],
                              initializer=[weight, shape])
    m = donnx.ONNXModel("with_weights", helper.make_model(graph))
    assert m.weights["g"].dtype == BF and torch.equal(m.weights["g"].cpu(), (torch.arange(8) / 7).to(BF))
    assert m.sdfg.arrays["x"].dtype == dace.bfloat16 and dace.bfloat16.bytes == 2 and dace.bfloat16.as_torch() is BF
    assert dace.typeclass_of(BF) == dace.bfloat16 and dace.typeclass_of(np.float32) == dace.float32
    m.expand()
    assert np.array_equal(dace.to_numpy(torch.tensor([1.5, 2.0], dtype=BF)), np.array([1.5, 2.0], np.float32))
    assert dace.from_numpy(np.float32(1.5), dace.bfloat16).shape == ()


def test_constants_of_bfloat16_are_not_computed_with():
    helper, T = proto.helper, proto.TensorProto
    graph = helper.make_graph([helper.make_node("Reshape", ["w", "shape"], ["g"]), helper.make_node("SkipRMSNormalization", ["x", "g"], ["y"])], "g",
                              [helper.make_tensor_value_info("x", T.BFLOAT16, [3, 8])], [helper.make_tensor_value_info("y", T.BFLOAT16, [3, 8])],
                              initializer=[helper.make_tensor("w", T.BFLOAT16, [2, 4], np.ones(8)), proto.numpy_helper.from_array(np.array([8], np.int64), "shape")])
    m = donnx.ONNXModel("constant", helper.make_model(graph))
    m.expand()
    assert m.sdfg.arrays["g"].dtype == dace.bfloat16


# ---------------------------------------------------------------------------------------------- the definitions themselves


def test_definitions_by_elementary_sums():
    g = torch.Generator().manual_seed(5)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    x = r(2, 4)
    y, s, q, scale = R.rms_norm(x, torch.ones(4), epsilon=0.0)
    assert torch.allclose((y * y).mean(-1), torch.ones(2, dtype=torch.float64)) and q.abs().max() == 127 and torch.allclose(scale * 127, y.abs().amax(-1))
    v = torch.tensor([[3, -2]], dtype=torch.int8), torch.tensor([[4, 5], [1, -1]], dtype=torch.int8)
    assert R.quantized_linear(*v, torch.tensor([0.5]), torch.tensor([2.0, 1.0]), bias=torch.tensor([1.0, 0.0]), residual=torch.tensor([[0.0, 1.0]]))[0].tolist() == [[3.0, 3.5]]
    p = torch.tensor([[[2]], [[5]]])
    for interleaved in (False, True):   # a pair is a complex number times exp(i angle); the last value stays
        x = r(1, 1, 1, 5)
        y = R.rotary(x, p, torch.tensor([0.3, 0.7]), [1, 1], interleaved)[0, 0, 0]
        x = x[0, 0, 0]
        pairs = [(0, 1, 0.3 * 2), (2, 3, 0.7 * 5)] if interleaved else [(0, 2, 0.3 * 2), (1, 3, 0.7 * 5)]
        for a, b, angle in pairs:
            z = complex(x[a], x[b]) * complex(np.cos(angle), np.sin(angle))
            assert abs(complex(y[a], y[b]) - z) < 1e-6   # (the frequencies are float32)
        assert y[4] == x[4]
    q, k, v = r(1, 2, 4, 3), r(1, 3, 2, 3), r(1, 3, 1, 6)   # two heads that share keys, three keys, causal: query 0 sees two
    vectors = [0.3 * r(3) for _ in range(4)]
    out, _ = R.differential_attention(q, k, v, vectors, 0.2, scale=0.7, lengths=torch.tensor([3]), causal=True)
    weight = np.exp(float(vectors[0] @ vectors[1])) - np.exp(float(vectors[2] @ vectors[3])) + 0.2
    for i in range(2):
        for h in range(2):
            p1, p2 = ([np.exp(0.7 * float(q[0, i, 2 * h + m] @ k[0, j, m])) for j in range(2 + i)] for m in range(2))
            expected = sum((p1[j] / sum(p1) - weight * p2[j] / sum(p2)) * v[0, j, 0] for j in range(2 + i))
            assert torch.allclose(out[0, i, h], expected)
    assert R.differential_attention(q, k, v, vectors, 0.2, lengths=torch.tensor([1]), causal=True)[0][0, 0].abs().max() == 0


# ---------------------------------------------------------------------------------------------- the documented layer


def test_the_documented_layer_can_be_built():
    """The nodes that the documentation lists for a layer are a graph: every name is an input of the layer, one of its weights or another node's result."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    texts = [open(path).read() for path in glob.glob(os.path.join(root, "*.md"))]
    block, = [b for text in texts for b in re.findall(r"```python\n(.*?)```", text, re.S) if 'node("DifferentialAttention"' in b]
    nodes = []
    exec(block, {"node": lambda op, inputs, outputs, **attributes: nodes.append(proto.helper.make_node(op, inputs, outputs, **attributes))})   # noqa: S102
    B, S, H, G, d = 2, 5, 4, 2, 64
    hidden, T, helper = 2 * H * d, proto.TensorProto, proto.helper
    inputs = {"x": (T.BFLOAT16, [B, S, hidden]), "skip": (T.BFLOAT16, [B, S, hidden]), "positions": (T.INT64, [3, B, S]), "lengths": (T.INT32, [B])}
    weights = {"gain": (T.BFLOAT16, [hidden]), "head_gain": (T.BFLOAT16, [2 * d]), "o_gain": (T.BFLOAT16, [hidden]), "frequencies": (T.FLOAT, [d // 2]),
               **{"lambda_" + n: (T.FLOAT, [d]) for n in ("q1", "k1", "q2", "k2")}}
    for name, columns in (("wq", 2 * H * d), ("wk", 2 * G * d), ("wv", 2 * G * d), ("wo", hidden)):
        weights[name], weights[name + "_scale"] = (T.INT8, [columns, hidden]), (T.FLOAT, [columns])
    shapes = {"q_shape": [B, S, 2 * H, d], "k_shape": [B, S, 2 * G, d], "v_shape": [B, S, G, 2 * d], "o_shape": [B, S, hidden]}
    made = {name for n in nodes for name in n.output}
    assert {name for n in nodes for name in n.input if name} - made == {*inputs, *weights, *shapes}
    initializers = [helper.make_tensor(n, t, shape, np.ones(shape)) for n, (t, shape) in weights.items()] + [proto.numpy_helper.from_array(np.array(v), n) for n, v in shapes.items()]
    graph = helper.make_graph(nodes, "layer", [helper.make_tensor_value_info(n, *v) for n, v in inputs.items()],
                              [helper.make_tensor_value_info(n, T.BFLOAT16, [B, S, hidden]) for n in ("out", "stream")], initializer=initializers)
    assert [c.function for c in _functions(donnx.ONNXModel("documented", helper.make_model(graph)))].count("mi355x_quantized_linear") == 4
