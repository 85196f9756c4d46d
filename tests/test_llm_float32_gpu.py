"""DifferentialAttention in float32 where the last bits of its operands decide (``llm_float32`` has the inputs and derives the bounds; ``test_llm_float32`` shows what
they tell apart)."""
import pytest
import torch

import llm_float32 as F
import llm_operators as R

pytestmark = pytest.mark.gpu


def run(case, odd=0):
    """The node's result; `odd` values before each array."""
    inputs = []
    for n in "qkv":
        buffer = torch.zeros(case[n].numel() + odd, device="cuda")
        inputs.append((n, buffer[odd:].view(case[n].shape)))
        inputs[-1][1].copy_(case[n])
    none = torch.zeros(0, device="cuda")
    b, sq, h2, d = case["q"].shape
    o, = R.call("DifferentialAttention", inputs + [(f"l{i}", none) for i in range(4)], [("o", torch.float32, (b, sq, h2 // 2, 2 * d))], lambda_init=F.WEIGHT, scale=case["scale"])
    return o


def on_gpu(case):
    return {n: t.cuda() if n in "qkv" else t for n, t in case.items()}


@pytest.mark.parametrize("form", [None, 0, 1, 2, 3])
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("odd", [0, 1])
def test_scores_and_values_that_low_order_parts_decide(form, d, odd, tuning):
    tuning(MI355X_DIFF_FORM=form)
    kinds = ("keys", "queries", "middle")
    for case in [F.cancelling_scores(kind, 150, d, 70) for kind in kinds] + [F.few_keys(150, d, 2), F.one_key(5, d)]:
        assert F.error(on_gpu(case), run(case, odd)) < 1


@pytest.mark.parametrize("splits", [2, 3])
def test_low_order_parts_of_keys_in_parts(splits, tuning):
    tuning(MI355X_DIFF_SPLITS=splits)
    for case in [F.cancelling_scores(kind, 40, 64, 500, seed=1) for kind in ("keys", "queries", "middle")]:
        assert F.error(on_gpu(case), run(case)) < 1


@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("b, sq, sk, h, g", [(1, 1, 1, 1, 1), (1, 2, 3, 1, 1), (2, 31, 33, 2, 1), (1, 65, 65, 2, 2), (2, 129, 200, 3, 3), (1, 5, 700, 4, 2), (1, 1, 3000, 8, 2), (3, 333, 333, 6, 6),
                                             (8, 300, 300, 4, 2)])
def test_norms_of_errors(d, b, sq, sk, h, g):
    case = F.normal_case(b, sq, sk, h, g, d)
    assert F.norm_error(on_gpu(case), run(case)) < F.NORM
