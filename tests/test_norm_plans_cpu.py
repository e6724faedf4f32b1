"""The norm's kernels are built for the blocks that they are launched with: not smaller, which no launch would survive, and not
larger, which would tell the compiler of registers that no block takes."""

import os
import re

import pytest

from moe_bench_b200 import build as mb_build


def _source():
    return re.sub(r"//[^\n]*", "", open(os.path.join(mb_build.CSRC, "layer_norm.cu")).read())


def _threads_launched(text, names):
    """Most threads of a block, for each number of vectors per thread, over the shapes of those tables."""
    most = {}
    for name in names:
        table = re.search(r"constexpr Shape %s\[\] = \{(.*)\};" % name, text).group(1)
        for per, threads, _ in re.findall(r"\{(\d+), (\d+), (\d+)\}", table):
            most[int(per)] = max(most.get(int(per), 0), int(threads))
    return most


@pytest.mark.parametrize("kernel,vec,tables", [
    ("norm_kernel", "kV", ("kForwardVec", "kForwardVecFew")), ("norm_kernel", "1", ("kForwardOne", "kForwardOneFew")),
    ("norm_grad_kernel", "kV", ("kBackwardVec", "kBackwardVecFew")), ("norm_grad_kernel", "1", ("kBackwardOne", "kBackwardOneFew"))])
def test_kernels_are_built_for_the_blocks_they_get(kernel, vec, tables):
    text = _source()
    built = {int(per): int(threads) for per, threads in re.findall(r"\b%s<T, %s, (\d+), (\d+)" % (kernel, vec), text)}
    assert built == _threads_launched(text, tables)
