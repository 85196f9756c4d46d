"""What the kernels' sources have to say to the compiler, where no result of today's compiler would show that they do not."""
import glob
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "dace-onnx_amd", "csrc")
SOURCES = sorted(glob.glob(os.path.join(CSRC, "*.h*")))


def _text(path):
    with open(path) as f:
        return re.sub(r"//[^\n]*", "", f.read())


@pytest.mark.parametrize("path", SOURCES, ids=os.path.basename)
def test_assembly_that_writes_m0_says_so(path):
    """The compiler keeps values of its own in m0: a statement that changes it lists it."""
    for statement in re.findall(r"\basm\b[^;]*?\((?:[^;\"]|\"(?:[^\"\\]|\\.)*\")*\);", _text(path)):
        if re.search(r"s_mov_b32\s+m0\b", statement):
            assert re.search(r":[^:]*\"m0\"[^:]*\)\s*;$", statement), statement


def test_rows_that_a_wave_hands_round_through_lds_are_fenced():
    """QuantizedLinear's results: a lane reads what other lanes of its wave wrote, and the next rows are written where others have read. No barrier of the workgroup
    stands between."""
    text = _text(os.path.join(CSRC, "quantized_linear.hip"))
    body = text[text.index("float* mine ="):text.index("static bool launch_qlin")]
    steps = re.findall(r"f32x4\*>\(mine \+ [^)]*\)+ =|= \*reinterpret_cast<const f32x4\*>\(mine|wave_lds_fence\(\)|for \(int t = 0", body)
    kinds = ["loop" if s.startswith("for") else "fence" if s.startswith("wave") else "read" if s.startswith("=") else "write" for s in steps]
    assert kinds == ["loop", "write", "fence", "read", "fence"]
    fence = text[text.index("void wave_lds_fence()"):]
    assert re.findall(r"__ATOMIC_\w+|wave_barrier", fence[:fence.index("}")]) == ["__ATOMIC_RELEASE", "wave_barrier", "__ATOMIC_ACQUIRE"]
