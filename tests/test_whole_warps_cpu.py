"""Instructions that a warp has to reach as one (``.aligned``).

Lanes that took different branches need not have come together by themselves: what an aligned instruction does then is
undefined, a hang of a cluster among it, and no run can be made to show it.  So the sources are checked."""

import glob
import os
import re

from moe_bench_b200 import build as mb_build


def _source(name):
    return re.sub(r"//[^\n]*", "", open(os.path.join(mb_build.CSRC, name)).read())


def _functions(text, word):
    """The bodies of the innermost braces that hold `word`."""
    return [m.group(0) for m in re.finditer(r"\{[^{}]*\}", re.sub(r'"\{|\}"', '"', text)) if word in m.group(0)]


def test_a_warp_is_whole_when_it_arrives_on_a_cluster_barrier():
    """The barriers themselves bring the lanes together, so every call does, whatever stands before it."""
    bodies = _functions(_source("common.cuh"), "barrier.cluster.arrive")
    assert len(bodies) == 2
    for body in bodies:
        assert re.match(r"\{\s*__syncwarp\(\);\s*asm volatile\(\"barrier\.cluster\.arrive[^;]*\.aligned;", body), body
    for path in glob.glob(os.path.join(mb_build.CSRC, "*")):
        if os.path.basename(path) != "common.cuh":
            assert "barrier.cluster" not in _source(os.path.basename(path)), path
