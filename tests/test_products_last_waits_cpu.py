"""What a CTA waits for before it leaves: the arithmetic of the source itself, run over sequences of tiles.

A barrier completes one phase per use, and a wait for parity P is over once the phase of that parity is, so it blocks while
(completed phases) % 2 == P.  The wait for the last of ``uses`` phases has P = (uses - 1) % 2; a barrier that was not used is not
waited for."""

import os
import random
import re

import pytest

from moe_bench_b200 import build as mb_build


def _source():
    return re.sub(r"//[^\n]*", "", open(os.path.join(mb_build.CSRC, "products.cu")).read())


def _one(pattern, text):
    found = re.findall(pattern, text)
    assert len(found) == 1, (pattern, found)
    return found[0]


@pytest.fixture(scope="module")
def roles():
    """The source of the loading warp and of the one that issues the products."""
    text = _source()
    first = text.index("int stage = 0, round = 0;")
    second = text.index("int stage = 0, round = 0;", first + 1)
    end = text.index("} else if (warp == 2) {", second)
    return text[first:second], text[second:end]


def _c(expression):
    return compile(expression.replace("/", "//"), "products.cu", "eval")


def _tiles(rng):
    return [rng.choice([0, 1, 2, 3, rng.randint(1, 40), rng.randint(1, 200)]) for _ in range(rng.choice([0, 1, 2, 3, 4, 7, rng.randint(0, 60)]))]


def test_the_loads_last_waits_are_for_the_last_use_of_every_stage(roles):
    loads, _ = roles
    in_loop = _c(_one(r"lap > 0 && !mbar_wait_lane\(smem_u32\(&t->empty\[at\]\), ([^,]+),", loads))
    guard, parity = _one(r"if \((round > \d+)\) ok = mbar_wait\(smem_u32\(&t->empty\[stage\]\), ([^,]+),", loads)
    guard, parity = _c(guard), _c(parity)
    next_round, next_stage = _c(_one(r"round \+= ([^;]+);", loads)), _c(_one(r"stage = (\(stage[^;]+);", loads))
    assert _one(r"for \(int i = 0; ok && i < (\w+); \+\+i\)", loads) == "stages"
    assert _one(r"if \(\+\+stage == stages\) \{([^}]*)\}", loads).split() == ["stage", "=", "0;", "++round;"]
    rng = random.Random(1)
    for _ in range(3000):
        stages, uses = rng.randint(6, 10), [0] * 10
        stage = round = 0
        for steps in _tiles(rng):
            at, lap = stage, round
            for _ in range(steps):
                if lap > 0:  # the stage's use before this one
                    assert eval(in_loop, {"lap": lap}) == (uses[at] - 1) % 2
                else:
                    assert uses[at] == 0
                uses[at] += 1
                at, lap = (0, lap + 1) if at + 1 == stages else (at + 1, lap)
            env = {"stage": stage, "steps": steps, "stages": stages}
            round, stage = round + eval(next_round, env), eval(next_stage, env)
            assert (stage, round) == (at, lap)
        seen = set()
        for _ in range(stages):
            if eval(guard, {"round": round}):
                assert uses[stage] > 0 and eval(parity, {"round": round}) == (uses[stage] - 1) % 2
            else:
                assert uses[stage] == 0
            seen.add(stage)
            stage, round = (0, round + 1) if stage + 1 == stages else (stage + 1, round)
        assert len(seen) == stages


def test_the_products_last_waits_are_for_the_last_use_of_both_accumulators(roles):
    _, products = roles
    buf, use = _one(r"const uint32_t buf = ([^,]+), use = ([^;]+);", products)
    in_loop = _c(_one(r"mbar_wait_cluster_lane\(smem_u32\(&t->acc_empty\[buf\]\), ([^,]+),", products))
    last = _c(_one(r"mbar_wait_cluster_lane\(smem_u32\(&t->acc_empty\[b\]\), ([^,]+),", products))
    assert _one(r"for \(uint32_t b = 0; ([^;]+); \+\+b\)", products) == "b < 2 && b < it"
    buf, use = _c(buf), _c(use)
    for tiles in range(40):
        uses = [0, 0]  # drained accumulators, as many phases of acc_empty
        for it in range(tiles):
            b, parity = eval(buf, {"it": it}), eval(in_loop, {"use": eval(use, {"it": it})})
            # the one before has to be drained; the first use of either waits for the phase ahead of phase 0, which is over
            assert parity == (uses[b] - 1) % 2
            uses[b] += 1
        for b in range(2):
            if b < tiles:
                assert eval(last, {"it": tiles, "b": b}) == (uses[b] - 1) % 2
            else:
                assert uses[b] == 0
