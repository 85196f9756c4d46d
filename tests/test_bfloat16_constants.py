"""Constants of bfloat16 on their way into a graph: ``Constant`` nodes, and constant subgraphs that end or begin in bfloat16."""
import numpy as np
import pytest
import torch

import dace_onnx_amd.onnx as donnx
from dace_onnx_amd import sdfg as dace
from dace_onnx_amd.onnx.proto import TensorProto, helper, numpy_helper

BF = torch.bfloat16
#: no value of bfloat16 among the first three: 1 + 2^-8 is a tie, 1.001 and pi lie between two
VALUES = np.array([1.00390625, 1.001, 3.14159, -2.0, 0.0, 1e-40, 60000.0, 7.0], dtype=np.float32)
ROUNDED = torch.from_numpy(VALUES).to(BF)


def _model(nodes, inputs, outputs, initializers=()):
    infos = lambda values: [helper.make_tensor_value_info(n, t, shape) for n, t, shape in values]  # noqa: E731
    return donnx.ONNXModel("constants", helper.make_model(helper.make_graph(nodes, "g", infos(inputs), infos(outputs), initializer=list(initializers))))


def _norm(nodes, initializers=()):
    """A norm in bfloat16 whose gain the nodes make, as ``g``."""
    return _model([*nodes, helper.make_node("SkipRMSNormalization", ["x", "g"], ["y"])], [("x", TensorProto.BFLOAT16, [3, 8])], [("y", TensorProto.BFLOAT16, [3, 8])], initializers)


def test_a_constant_node_of_bfloat16():
    m = _norm([helper.make_node("Constant", [], ["g"], value=helper.make_tensor("value", TensorProto.BFLOAT16, [8], VALUES))])
    assert m.sdfg.arrays["g"].dtype == dace.bfloat16 and torch.equal(m.weights["g"].cpu(), ROUNDED)
    m.expand()


@pytest.mark.parametrize("dims, values", [([], [5.0]), ([2, 2], [1.0, 2.0, 3.0, 4.0]), ([0], [])])
@pytest.mark.parametrize("kind", [TensorProto.FLOAT, TensorProto.INT64, TensorProto.BFLOAT16, TensorProto.BOOL])
def test_constant_nodes_keep_type_and_shape(kind, dims, values):
    m = _model([helper.make_node("Constant", [], ["c"], value=helper.make_tensor("value", kind, dims, values)), helper.make_node("Identity", ["c"], ["y"])],
               [], [("y", kind, dims)])
    weight, = m.weights.values()
    assert tuple(weight.shape) == tuple(dims) and dace.typeclass_of(weight.dtype) == donnx.onnx_importer.onnx_tensor_type_to_typeclass(kind)
    assert weight.reshape(-1).tolist() == [bool(v) if kind == TensorProto.BOOL else v for v in values]


def test_a_constant_that_is_cast_to_bfloat16():
    m = _norm([helper.make_node("Cast", ["w"], ["g"], to=TensorProto.BFLOAT16)], [numpy_helper.from_array(VALUES, "w")])
    assert m.sdfg.arrays["g"].dtype == dace.bfloat16 and torch.equal(m.weights["g"].cpu(), ROUNDED)
    m.expand()


@pytest.mark.parametrize("to, expected", [(TensorProto.FLOAT, ROUNDED.float()), (TensorProto.FLOAT16, ROUNDED.half()), (TensorProto.INT32, ROUNDED.int()), (TensorProto.BOOL, ROUNDED.bool())])
@pytest.mark.parametrize("first", [[], [helper.make_node("Cast", ["w"], ["b"], to=TensorProto.BFLOAT16)]])
def test_a_constant_of_bfloat16_that_is_cast_back(first, to, expected):
    """By itself, and after a cast to bfloat16 whose rounding has to stay."""
    weight = numpy_helper.from_array(VALUES, "w") if first else helper.make_tensor("b", TensorProto.BFLOAT16, [8], VALUES)
    m = _model([*first, helper.make_node("Cast", ["b"], ["c"], to=to), helper.make_node("Identity", ["c"], ["y"])], [], [("y", to, [8])], [weight])
    m.expand()
    made, = m.weights.values()
    assert made.dtype == expected.dtype and torch.equal(made.cpu(), expected)


def test_a_cast_to_bfloat16_is_not_computed_with():
    """Sums of bfloat16 are not folded in float32: the node stays, and says that it does not take the type."""
    with pytest.raises(ValueError, match="bfloat16"):
        _model([helper.make_node("Cast", ["w"], ["b"], to=TensorProto.BFLOAT16), helper.make_node("Add", ["b", "b"], ["y"])],
               [], [("y", TensorProto.BFLOAT16, [8])], [numpy_helper.from_array(VALUES, "w")]).expand()


def test_a_constant_of_shape_of_bfloat16():
    value = helper.make_tensor("value", TensorProto.BFLOAT16, [1], [1.001])
    m = _norm([helper.make_node("ConstantOfShape", ["s"], ["g"], value=value)], [numpy_helper.from_array(np.array([8], np.int64), "s")])
    assert m.sdfg.arrays["g"].dtype == dace.bfloat16 and torch.equal(m.weights["g"].cpu(), torch.full((8,), 1.001, dtype=BF))
    m.expand()


def test_the_shape_of_a_constant_of_bfloat16():
    m = _model([helper.make_node("Shape", ["w"], ["s"]), helper.make_node("Identity", ["s"], ["y"])], [], [("y", TensorProto.INT64, [2])],
               [helper.make_tensor("w", TensorProto.BFLOAT16, [4, 2], VALUES)])
    assert [w.tolist() for w in m.weights.values()] == [[4, 2]]
