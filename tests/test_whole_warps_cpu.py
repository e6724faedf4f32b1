"""Instructions that a warp has to reach as one (``.aligned``).

Lanes that took different branches need not have come together by themselves: what an aligned instruction does then is
undefined, a hang of a cluster among it, and no run can be made to show it.  So the sources are checked."""

import glob
import os
import re

import pytest

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


# calls that send lanes different ways (or hold a branch per lane), and what brings a warp together again
BRANCH = r"load_residual_column\(|emit_column<|\brequest\(|inside \?|if \(row_of"
WHOLE = r"__syncwarp\(\);|__syncthreads\(\);|\bcluster_sync|\brelease\(\);|turn_chunk\(|\bstore\("
ALIGNED = r"tmem_ld16\(|tmem_ld_frag16\(|tmem_ld_wait16x?2?\(|stmatrix_x4_trans\(|ldmatrix_x4_trans\(|mma_h16\(|\bplace\("


def _block(text, start):
    """The text from the first brace at or after `start` to the brace that closes it."""
    i = text.index("{", start)
    depth, j = 1, i + 1
    while depth:
        depth += {"{": 1, "}": -1}.get(text[j], 0)
        j += 1
    return text[i:j]


def _loops(text):
    for m in re.finditer(r"\bfor \(", text):
        header_end = text.index("\n", m.start())
        if text[m.start() : header_end].rstrip().endswith("{"):
            yield _block(text, text.rindex("{", m.start(), header_end + 1))


def _split_at(body):
    """What stands before the first aligned instruction that a branch of single lanes comes right before, or None."""
    split = None
    for m in re.finditer(f"(?P<branch>{BRANCH})|(?P<whole>{WHOLE})|(?P<aligned>{ALIGNED})", body):
        if m["branch"]:
            split = m.start()
        elif m["whole"]:
            split = None
        elif split is not None:
            return body[split : m.end()]
    return None


def test_the_scan_sees_a_split_warp():
    assert _split_at("tmem_ld16(a, v); emit_column<kFinish>(p); tmem_ld16(a, v);")
    assert not _split_at("tmem_ld16(a, v); emit_column<kFinish>(p); __syncwarp(); tmem_ld16(a, v);")


@pytest.mark.parametrize("name", ["products.cu", "few_rows.cu"])
def test_a_warp_is_whole_at_the_tensor_cores_registers_and_memory(name):
    """In every loop with such an instruction, from any turn to the next."""
    loops = [b for b in _loops(_source(name)) if re.search(ALIGNED, b)]
    assert loops
    for body in loops:
        assert not _split_at(body + body)


def test_a_warp_is_whole_at_a_named_barrier():
    """bar.sync is the aligned form: the statement before each is the one that brings the lanes together."""
    found = 0
    for path in glob.glob(os.path.join(mb_build.CSRC, "*.cu*")):
        text = _source(os.path.basename(path))
        for m in re.finditer(r'asm volatile\("bar\.sync', text):
            found += 1
            assert re.search(r"__syncwarp\(\);\s*$", text[: m.start()]), path
    assert found
