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
