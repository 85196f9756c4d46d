"""The inputs of ``llm_float32`` on the CPU: the kernel's six products stay within the bounds, and fewer or shorter ones do not."""
import numpy as np
import pytest

import llm_float32 as F

WITHOUT = {missing: tuple(p for p in F.ALL if p != missing) for missing in F.ALL}
CASES = {"keys": lambda: F.cancelling_scores("keys", 40, 64, 70), "queries": lambda: F.cancelling_scores("queries", 40, 64, 70),
         "middle": lambda: F.cancelling_scores("middle", 40, 64, 70), "few": lambda: F.few_keys(150, 64, 2), "one": lambda: F.one_key(5, 64)}


def test_parts_of_a_value():
    x = np.random.default_rng(0).normal(size=1000).astype(np.float32)
    a, b, c = F.parts(x)
    assert np.array_equal((a.astype(np.float64) + b) + c, x.astype(np.float64))
    assert (np.abs(b) <= 2.0 ** -7 * np.abs(x)).all() and (np.abs(c) <= 2.0 ** -15 * np.abs(x)).all() and (a * x > 0).all() and (b * x >= 0).all()


@pytest.mark.parametrize("name", CASES)
def test_six_products_stay_within_the_bound(name):
    case = CASES[name]()
    assert F.error(case, F.emulated(case)) < 1


@pytest.mark.parametrize("name, missing", [("keys", (2, 0)), ("keys", (0, 2)), ("queries", (0, 2)), ("queries", (2, 0)), ("middle", (1, 1))])
def test_scores_with_a_product_left_out(name, missing):
    """One of the two orders of (first, last) is the keys' and the other the queries': each is seen by one kind of input, and each kind sees one."""
    case = CASES[name]()
    seen = F.error(case, F.emulated(case, scores=WITHOUT[missing]))
    wanted = {"keys": (0, 2), "queries": (2, 0), "middle": (1, 1)}[name]   # (first operand: queries)
    assert seen > 2 if missing == wanted else seen < 1, seen


@pytest.mark.parametrize("name, missing", [("few", (0, 2)), ("few", (1, 1)), ("few", (2, 0)), ("one", (0, 2))])
def test_values_with_a_product_left_out(name, missing):
    case = CASES[name]()
    assert F.error(case, F.emulated(case, values=WITHOUT[missing])) > 2


@pytest.mark.parametrize("where", ["scores", "values"])
def test_three_products_are_not_enough(where):
    three = F.ALL[3:]
    assert min(F.error(case, F.emulated(case, **{where: three})) for name, case in ((n, c()) for n, c in CASES.items())
               if (name in ("few", "one")) == (where == "values")) > 2


@pytest.mark.parametrize("d, keys", [(32, 3), (64, 65), (128, 200)])
def test_norms_of_errors(d, keys):
    """What the six products are off by in all, and that three are not enough for it in either place."""
    case = F.normal_case(1, 70, keys, 1, 1, d)
    assert F.norm_error(case, F.emulated(case)) < F.NORM
    assert F.norm_error(case, F.emulated(case, scores=F.ALL[3:])) > 3 * F.NORM
    assert F.norm_error(case, F.emulated(case, values=F.ALL[3:])) > 3 * F.NORM
