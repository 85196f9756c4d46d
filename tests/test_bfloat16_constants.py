"""Constants of bfloat16 on their way into a graph: ``Constant`` nodes, and constant subgraphs that end or begin in bfloat16."""
import numpy as np
import pytest
import torch

import dace_onnx_amd.onnx as donnx
from dace_onnx_amd import sdfg as dace
from dace_onnx_amd.onnx.proto import TensorProto, helper

BF = torch.bfloat16
#: no value of bfloat16 among the first three: 1 + 2^-8 is a tie, 1.001 and pi lie between two
VALUES = np.array([1.00390625, 1.001, 3.14159, -2.0, 0.0, 1e-40, 65504.0, 7.0], dtype=np.float32)
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
