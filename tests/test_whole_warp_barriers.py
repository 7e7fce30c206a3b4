"""Barriers whose instructions want all lanes of a warp at once bring the lanes together themselves, whatever branch or loop they come
from: read in the sources, as a GPU that lets lanes run apart may wait for good."""

import os
import re

import pytest

from linquant_b200 import build


def sources():
    return [f for f in sorted(os.listdir(build.CSRC)) if f.endswith((".cu", ".cuh"))]


@pytest.mark.parametrize("name", sources())
def test_cluster_barriers(name):
    text = open(os.path.join(build.CSRC, name)).read()
    for m in re.finditer(r"barrier\.cluster\.arrive", text):
        before = text[:m.start()].rstrip().removesuffix('asm volatile("').rstrip()
        assert before.endswith("__syncwarp();"), f"{name}: line {text[:m.start()].count(chr(10)) + 1}"


def test_decisions_of_a_group_of_warps():
    """Linear attention: one lane of each warp has just stored its warp's largest value."""
    text = open(os.path.join(build.CSRC, "lq_linear_attention_tc.cu")).read()
    assert text.count("bar.red.") == 1
    assert "__syncwarp();" in text[text.index("bool group_and(bool ok)"):text.index("bar.red.")]
