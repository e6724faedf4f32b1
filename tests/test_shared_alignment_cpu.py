"""Shared arrays that inline assembly reads several elements of at once: the compiler, which does not see how, aligns an array
only to its elements unless it is told."""

import os
import re

from moe_bench_b200 import build as mb_build


def _source(name):
    return re.sub(r"//[^\n]*", "", open(os.path.join(mb_build.CSRC, name)).read())


def test_arrays_behind_16_byte_reads_say_so():
    text = _source("few_rows.cu")
    reads = list(re.finditer(r"ld\.shared::cluster\.v4\.f32", text))
    assert reads
    for m in reads:
        array = re.findall(r"smem_u32\(&(\w+)\[", text[: m.start()])[-1]
        assert re.search(r"__shared__ (__align__|alignas)\(16\) float %s\[" % array, text), array


def test_the_products_turn_blocks_say_so():
    assert re.search(r"alignas\(16\) float turn\[", _source("products.cu"))
