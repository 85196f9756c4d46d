"""Definitions of the operators of quantised and differential transformers in float64, and one-node calls of the framework's."""
import numpy as np
import torch

import dace_onnx_amd.onnx as donnx
from dace_onnx_amd.onnx.proto import TensorProto, helper

TYPES = (torch.float32, torch.float16, torch.bfloat16)
ELEMENT = {torch.float32: 1, torch.int8: 3, torch.int32: 6, torch.int64: 7, torch.float16: 10, torch.bfloat16: 16}
#: half a step of a type, relative to the value
HALF = {t: torch.finfo(t).eps / 2 for t in TYPES}


def model(op, inputs, outputs, **attributes):
    """A graph of one node: inputs as (name, tensor or None), outputs as (name, dtype, shape) or None; call it with the tensors."""
    named = [(n, t) for n, t in inputs if t is not None]
    infos = [helper.make_tensor_value_info(n, ELEMENT[t.dtype], list(t.shape)) for n, t in named]
    outs = [helper.make_tensor_value_info(o[0], ELEMENT[o[1]], list(o[2])) for o in outputs if o]
    node = helper.make_node(op, [n if t is not None else "" for n, t in inputs], [o[0] if o else "" for o in outputs], name="node", **attributes)
    return donnx.ONNXModel("one_" + op.lower(), helper.make_model(helper.make_graph([node], "one", infos, outs)))


def call(op, inputs, outputs, **attributes):
    results = model(op, inputs, outputs, **attributes)(*[t for _, t in inputs if t is not None])
    return list(results) if isinstance(results, tuple) else [results]


# ---------------------------------------------------------------------------------------------- definitions


def rms_norm(x, gain, skip=None, epsilon=1e-5):
    """y, sum, q, scale for rows [..., columns]."""
    s = x.double() + (0.0 if skip is None else skip.double())
    y = s / torch.sqrt((s * s).mean(-1, keepdim=True) + epsilon) * gain.double()
    scale = y.abs().amax(-1) / 127
    q = torch.round(y / torch.where(scale > 0, scale, 1.0)[..., None])
    return y, s, q, scale


def activated(v, activation):
    return {"none": lambda v: v, "relu": torch.relu, "gelu": lambda v: 0.5 * v * (1 + torch.erf(v / 2 ** 0.5)), "silu": lambda v: v / (1 + torch.exp(-v))}[activation](v)


def quantized_linear(x, w, xs, ws, bias=None, residual=None, activation="none"):
    """The result and the sum of the magnitudes that its roundings go by."""
    v = (x.double() @ w.double().t()) * xs.double().reshape(-1, 1) * ws.double().reshape(1, -1)
    size = v.abs()
    if bias is not None:
        v, size = v + bias.double(), size + bias.double().abs()
    v = activated(v, activation)
    if residual is not None:
        v, size = v + residual.double(), size + residual.double().abs()
    return v, size


def rotary(x, positions, frequencies, sections, interleaved):
    pairs = len(frequencies)
    axis = torch.repeat_interleave(torch.arange(len(sections)), torch.tensor(sections)).to(positions.device)
    angle = (positions[axis].double() * frequencies.double()[:, None, None]).permute(1, 2, 0)[:, :, None]   # [B, S, 1, pairs]
    y = x.double().clone()
    first, second = (y[..., 0:2 * pairs:2], y[..., 1:2 * pairs:2]) if interleaved else (y[..., :pairs], y[..., pairs:2 * pairs])
    a, b = first * angle.cos() - second * angle.sin(), second * angle.cos() + first * angle.sin()
    first.copy_(a)
    second.copy_(b)
    return y


def differential_attention(q, k, v, vectors, lambda_init, scale=None, lengths=None, causal=False):
    """The result, and sum_j (P1 + |l| P2) |V|: what an error relative to the probabilities or the values goes by."""
    (B, Sq, H2, D), (Sk, G) = q.shape, (k.shape[1], k.shape[2] // 2)
    H, share = H2 // 2, H2 // 2 // G
    scale = D ** -0.5 if scale is None else scale
    a, b, c, d = (w.double() for w in vectors)
    weight = torch.exp((a * b).sum()) - torch.exp((c * d).sum()) + lambda_init
    out = torch.zeros(B, Sq, H, 2 * D, dtype=torch.float64, device=q.device)
    size = torch.zeros_like(out)
    for i in range(B):
        n = Sk if lengths is None else min(max(int(lengths[i]), 0), Sk)
        for h in range(H):
            maps = []
            for m in range(2):
                s = scale * q[i, :, 2 * h + m].double() @ k[i, :n, 2 * (h // share) + m].double().t()
                hidden = torch.arange(n, device=q.device) > torch.arange(Sq, device=q.device)[:, None] + n - Sq if causal else torch.zeros_like(s, dtype=torch.bool)
                s = s.masked_fill(hidden, -torch.inf)
                top = s.amax(-1, keepdim=True) if n else s.new_zeros(Sq, 1)
                e = torch.exp(s - torch.where(top == -torch.inf, 0.0, top))
                total = e.sum(-1, keepdim=True)
                maps.append(e / torch.where(total == 0, 1.0, total))
            value = v[i, :n, h // share].double()
            out[i, :, h] = (maps[0] - weight * maps[1]) @ value
            size[i, :, h] = (maps[0] + weight.abs() * maps[1]) @ value.abs()
    return out, size
