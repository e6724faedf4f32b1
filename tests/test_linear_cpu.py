"""Refusals of the products and norms around the expert FFN: what the entry points turn down before any GPU work, and the
64-bit oracle against autograd and against differences."""

import ctypes

import pytest
import torch

from moe_bench_b200 import build as mb_build
from moe_bench_b200 import capi
from oracle import ffn_oracle as F


@pytest.fixture(scope="module")
def lib():
    mb_build.build()
    return capi.load()


P = 1 << 20  # an aligned address that no refused call touches


def _linear(lib, **kw):
    a = dict(precision=0, x=P, xp=64, rows=4, w=P, wp=64, n=5, k=64, bias=None, b32=0, act=0, res=None, rp=0, y=P, o32=0, slope=None)
    a.update(kw)
    return lib.mb200_linear(a["precision"], a["x"], a["xp"], a["rows"], a["w"], a["wp"], a["n"], a["k"], a["bias"], a["b32"],
                            a["act"], a["res"], a["rp"], a["y"], a["o32"], a["slope"], 0, None)


@pytest.mark.parametrize("change,words", [
    (dict(precision=1), b"precision"), (dict(precision=3), b"precision"), (dict(rows=-1), b"rows"), (dict(n=0), b"n=0"),
    (dict(k=0), b"k=0"), (dict(k=60, xp=64), b"multiple of 8"), (dict(act=5), b"activation"), (dict(act=-1), b"activation"),
    (dict(x=None), b"x is null"), (dict(w=None), b"w is null"), (dict(y=None), b"y is null"), (dict(x=P + 2), b"16-byte"),
    (dict(w=P + 8), b"16-byte"), (dict(xp=60), b"x has 60"), (dict(xp=68), b"x has 68"), (dict(wp=56), b"w has 56"),
    (dict(res=P, rp=4), b"residual pitch"), (dict(rows=1 << 31), b"32-bit"), (dict(n=(1 << 28) + 1), b"n="),
])
def test_linear_refuses(lib, change, words):
    assert _linear(lib, **change) != 0
    assert words in lib.mb200_last_error()


def test_nothing_to_do_is_no_error(lib):
    assert _linear(lib, rows=0, x=None, y=None) == 0
    assert lib.mb200_grouped_linear(0, None, 64, 0, P, 64, 64 * 5, P, 3, 5, 64, None, 0, None) == 0
    assert lib.mb200_layer_norm(0, None, 64, 0, 64, None, None, 0, 1e-5, None, None, None, 0, None) == 0


def _linear_backward(lib, **kw):
    a = dict(precision=0, dy=P, d32=0, dp=8, slope=None, x=P, xp=64, rows=4, w=P, wp=64, n=8, k=64, dx=P, dw=P, w32=0, db=P, ws=P, wsn=1 << 20)
    a.update(kw)
    return lib.mb200_linear_backward(a["precision"], a["dy"], a["d32"], a["dp"], a["slope"], a["x"], a["xp"], a["rows"], a["w"],
                                     a["wp"], a["n"], a["k"], a["dx"], a["dw"], a["w32"], a["db"], a["ws"], a["wsn"], 0, None)


@pytest.mark.parametrize("change,words", [
    (dict(precision=2, d32=1), b"fp16"), (dict(dp=4), b"dy pitch"), (dict(dy=None), b"dy is null"), (dict(x=P + 4), b"x must"),
    (dict(w=None), b"w is null"), (dict(k=12), b"multiple of 8"), (dict(slope=P, ws=None), b"workspace"),
    (dict(slope=P, wsn=16), b"workspace 16"), (dict(slope=P, ws=P + 4), b"workspace"), (dict(precision=7), b"precision"),
])
def test_linear_backward_refuses(lib, change, words):
    assert _linear_backward(lib, **change) != 0
    assert words in lib.mb200_last_error()


def _grouped(lib, **kw):
    a = dict(precision=0, x=P, xp=64, rows=4, w=P, wp=64, ep=64 * 5, off=P, e=3, n=5, k=64, y=P)
    a.update(kw)
    return lib.mb200_grouped_linear(a["precision"], a["x"], a["xp"], a["rows"], a["w"], a["wp"], a["ep"], a["off"], a["e"], a["n"],
                                    a["k"], a["y"], 0, None)


@pytest.mark.parametrize("change,words", [
    (dict(e=0), b"experts"), (dict(e=1025), b"experts"), (dict(off=None), b"offsets"), (dict(ep=64 * 5 + 4), b"expert to expert"),
    (dict(ep=64), b"expert to expert"), (dict(x=P + 2), b"x must"), (dict(y=None), b"y is null"), (dict(k=4), b"multiple of 8"),
])
def test_grouped_refuses(lib, change, words):
    assert _grouped(lib, **change) != 0
    assert words in lib.mb200_last_error()


def test_grouped_backward_refuses(lib):
    def call(dy=P, dp=8, ws=None, wsn=0, n=8):
        return lib.mb200_grouped_linear_backward(0, dy, dp, P, 64, 4, P, 64, 64 * n, P, 3, n, 64, P, P, 0, ws, wsn, 0, None)

    assert call(dy=None) != 0 and b"dy is null" in lib.mb200_last_error()
    assert call(dp=4) != 0 and b"dy pitch" in lib.mb200_last_error()
    assert call(dp=9) != 0 and b"workspace" in lib.mb200_last_error()
    assert call(dy=P + 2, ws=P, wsn=8) != 0 and b"workspace 8" in lib.mb200_last_error()


def test_norm_refuses(lib):
    def call(precision=0, x=P, xp=64, rows=2, h=64, y=P, m=P, r=P):
        return lib.mb200_layer_norm(precision, x, xp, rows, h, None, None, 0, 1e-5, y, m, r, 0, None)

    for kw, words in ((dict(precision=1), b"precision"), (dict(h=0), b"hidden"), (dict(xp=63), b"pitch"), (dict(x=None), b"null"),
                      (dict(y=None), b"null"), (dict(m=None), b"null"), (dict(rows=-3), b"rows")):
        assert call(**kw) != 0 and words in lib.mb200_last_error()
    back = lib.mb200_layer_norm_backward
    assert back(0, P, 63, P, 64, 2, 64, P, P, None, 0, P, P, P, P, 1 << 20, 0, None) != 0 and b"pitches" in lib.mb200_last_error()
    assert back(0, P, 64, P, 64, 2, 64, None, P, None, 0, P, P, P, P, 1 << 20, 0, None) != 0 and b"null" in lib.mb200_last_error()


# x 4 x 64, w 5 x 64, y 4 x 5 and so on, each on a megabyte of its own unless the case says otherwise
MB = 1 << 20


@pytest.mark.parametrize("change,words", [
    (dict(y=MB), b"y and x share"), (dict(y=MB + 4 * 64 * 2 - 2), b"y and x share"), (dict(y=2 * MB + 5 * 64 * 2 - 8), b"y and w share"),
    (dict(y=3 * MB, bias=3 * MB + 16), b"y and bias share"), (dict(y=MB - 4 * 5 * 2 + 2), b"y and x share"),
    (dict(res=3 * MB, rp=8), b"y and residual share"), (dict(res=3 * MB + 2, rp=5), b"y and residual share"),
    (dict(res=3 * MB, rp=5, o32=1), b"y and residual share"), (dict(slope=3 * MB), b"y and slope share"),
    (dict(slope=MB), b"slope and x share"),
])
def test_linear_refuses_to_write_what_it_reads(lib, change, words):
    assert _linear(lib, **{**dict(x=MB, w=2 * MB, y=3 * MB), **change}) != 0
    assert words in lib.mb200_last_error()


@pytest.mark.parametrize("change,words", [
    (dict(dx=MB), b"dx and dy share"), (dict(dx=2 * MB), b"dx and x share"), (dict(dx=3 * MB), b"dx and w share"),
    (dict(dw=2 * MB), b"dw and x share"), (dict(dw=4 * MB), b"dx and dw share"), (dict(db=6 * MB + 8), b"db and workspace share"),
    (dict(db=8 * MB), b"db and slope share"), (dict(ws=8 * MB), b"workspace and slope share"),
])
def test_linear_backward_refuses_to_write_what_it_reads(lib, change, words):
    apart = dict(dy=MB, x=2 * MB, w=3 * MB, dx=4 * MB, dw=5 * MB, ws=6 * MB, db=7 * MB, slope=8 * MB)
    assert _linear_backward(lib, **{**apart, **change}) != 0
    assert words in lib.mb200_last_error()


def test_grouped_refuses_to_write_what_it_reads(lib):
    apart = dict(x=MB, w=2 * MB, off=3 * MB, y=4 * MB)
    for change, words in ((dict(y=MB), b"y and x share"), (dict(y=2 * MB + (2 * 5 + 4) * 64 * 2), b"y and w share"),
                          (dict(off=4 * MB + 32), b"y and offsets share")):
        assert _grouped(lib, **{**apart, **change}) != 0 and words in lib.mb200_last_error()
    back = lib.mb200_grouped_linear_backward
    for dx, dw, words in ((MB, 8 * MB, b"dx and dy share"), (7 * MB, 2 * MB + 64, b"dw and x share"), (3 * MB, 8 * MB, b"dx and w share"),
                          (8 * MB + 2 * 8 * 64 * 2, 8 * MB, b"dx and dw share")):
        assert back(0, MB, 8, 2 * MB, 64, 4, 3 * MB, 64, 64 * 8, 4 * MB, 3, 8, 64, dx, dw, 0, None, 0, 0, None) != 0
        assert words in lib.mb200_last_error()


def test_norm_refuses_to_write_what_it_reads(lib):
    def call(x=MB, xp=64, w=2 * MB, y=3 * MB, m=4 * MB, r=5 * MB):
        return lib.mb200_layer_norm(0, x, xp, 2, 64, w, None, 1, 1e-5, y, m, r, 0, None)

    for kw, words in ((dict(y=MB, xp=72), b"y and x share"), (dict(y=MB + 2), b"y and x share"), (dict(y=2 * MB + 128), b"y and weight share"),
                      (dict(m=5 * MB + 4), b"mean and rstd share"), (dict(r=MB), b"rstd and x share")):
        assert call(**kw) != 0 and words in lib.mb200_last_error()
    back = lib.mb200_layer_norm_backward
    for dx, dwt, words in ((MB, 8 * MB, b"dx and dy share"), (2 * MB, 8 * MB, b"dx and x share"), (7 * MB, 3 * MB, b"dweight and mean share"),
                           (7 * MB, 9 * MB, b"dweight and workspace share")):
        assert back(0, MB, 64, 2 * MB, 64, 2, 64, 3 * MB, 4 * MB, None, 0, dx, dwt, None, 9 * MB, MB, 0, None) != 0
        assert words in lib.mb200_last_error()


def test_workspace_queries_refuse_bad_sizes(lib):
    assert lib.mb200_linear_backward_workspace_bytes(4, 0, 1, 0) == -1
    assert lib.mb200_grouped_linear_backward_workspace_bytes(-1, 8) == -1
    assert lib.mb200_layer_norm_backward_workspace_bytes(4, 0, 0) == -1


def test_cpu_tensors_are_refused():
    x, w = torch.zeros(4, 64, dtype=torch.bfloat16), torch.zeros(8, 64, dtype=torch.bfloat16)
    off = torch.zeros(2, dtype=torch.int32)
    stats = torch.zeros(4)
    for call in (lambda: capi.linear(x, w), lambda: capi.linear_backward(x, x, w), lambda: capi.grouped_linear(x, w[None], off),
                 lambda: capi.grouped_linear_backward(x, x, w[None], off), lambda: capi.layer_norm(x),
                 lambda: capi.layer_norm_backward(x, x, stats, stats)):
        with pytest.raises(capi.MB200Error, match="CUDA"):
            call()


def test_gated_front_end_needs_a_gpu():
    from moe_bench_b200 import gating
    from moe_bench_b200 import problem as P

    cfg = P.MoEBenchConfig(hidden_size=64, intermediate_size=64, num_experts=4, topk=2, world_size=1, device="cpu")
    with pytest.raises(capi.MB200Error, match="CUDA"):
        gating.make_gated_problem(cfg, 4)


# ---- the oracle itself ----
@pytest.mark.parametrize("act", ["none", "relu", "silu", "gelu", "gelu_tanh"])
def test_oracle_linear_gradients_are_autograds_and_differences(act):
    g = torch.Generator().manual_seed(3)
    x, w, b, dy = (torch.randn(*s, dtype=torch.float64, generator=g) for s in ((5, 8), (6, 8), (6,), (5, 6)))
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    z = leaves[0] @ leaves[1].t() + leaves[2]
    fn = {"none": lambda v: v, "relu": torch.relu, "silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu,
          "gelu_tanh": lambda v: torch.nn.functional.gelu(v, approximate="tanh")}[act]
    fn(z).backward(dy)
    y, slope = F.activation(act, z.detach())
    assert torch.allclose(y, fn(z).detach(), rtol=1e-12, atol=1e-13)
    dz = dy * slope
    for got, leaf in zip((dz @ w, dz.t() @ x, dz.sum(0)), leaves):
        assert torch.allclose(got, leaf.grad, rtol=1e-10, atol=1e-12)
    step = 1e-6
    for i in range(4):  # central differences of the loss along single weights
        wp, wm = w.clone(), w.clone()
        wp[i, i] += step
        wm[i, i] -= step
        loss = [(F.activation(act, x @ v.t() + b)[0] * dy).sum() for v in (wp, wm)]
        assert abs((loss[0] - loss[1]) / (2 * step) - (dz.t() @ x)[i, i]) < 1e-6


def test_oracle_norm_gradients_are_autograds():
    g = torch.Generator().manual_seed(4)
    x, dy = torch.randn(5, 7, dtype=torch.float64, generator=g), torch.randn(5, 7, dtype=torch.float64, generator=g)
    w, b = torch.randn(7, dtype=torch.float64, generator=g), torch.randn(7, dtype=torch.float64, generator=g)
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    y = torch.nn.functional.layer_norm(leaves[0], (7,), leaves[1], leaves[2], eps=1e-5)
    y.backward(dy)
    xf = x.float()
    (ref, _), (mean, _), (rstd, _) = F.layer_norm(xf, w, b, 1e-5)
    assert torch.allclose(ref, y.detach(), atol=1e-5)
    mean = x.mean(1)
    rstd = (x.var(1, unbiased=False) + 1e-5) ** -0.5
    (dx, _), (dw, _), (db, _) = F.layer_norm_backward(dy.float(), xf, mean, rstd, w)
    for got, leaf in zip((dx, dw, db), leaves):
        assert torch.allclose(got, leaf.grad, atol=2e-5)


def test_prototypes_match_the_header(lib):
    """As many arguments as the header declares, of the same kinds."""
    import os
    import re

    text = open(os.path.join(mb_build.ROOT, "include", "moe_bench_b200.h")).read()
    text = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
    kinds = {capi.c_i32: "int", capi.c_i64: "int64_t", capi.c_vp: "*", ctypes.c_float: "float"}
    for name in (n for n in capi.SIGNATURES if re.match(r"mb200_(linear|grouped_linear|layer_norm)", n)):
        args = re.search(r"\b%s\s*\(([^)]*)\)" % name, text).group(1).split(",")
        got = ["*" if "*" in a else a.split()[0] for a in args]
        assert got == [kinds[c] for c in capi.SIGNATURES[name][1]], name


# ---- what no run can be made to show: the sources are held to it ----
def _source(name):
    import os
    import re

    return re.sub(r"//[^\n]*", "", open(os.path.join(mb_build.CSRC, name)).read())


def test_products_poll_through_the_bounded_waits_only():
    text = _source("products.cu") + _source("few_rows.cu") + _source("linear.cuh")
    assert "try_wait" not in text and "test_wait" not in text and "while (true)" not in text


def test_no_cta_leaves_before_its_last_remote_arrivals():
    """Arrivals from the pair's other CTA (the products' commits on `empty`, the epilogue's on `acc_empty`) are waited for after the
    loops, ahead of the cluster barrier that ends the kernel."""
    text = _source("products.cu")
    end = text.rindex("cluster_sync_relaxed();")
    loads, products = text.index("int stage = 0, round = 0;"), text.rindex("int stage = 0, round = 0;")
    masks = text.index("} else if (warp == 2) {")
    after_loads = text[text.rindex("stage = (stage + steps) % stages;", loads, products) : products]
    assert "mbar_wait(smem_u32(&t->empty[stage])" in after_loads
    after_products = text[text.rindex("stage = (stage + steps) % stages;", products, masks) : masks]
    assert "mbar_wait_cluster_lane(smem_u32(&t->acc_empty[b])" in after_products
    assert masks < end


def test_tensor_memory_is_used_only_behind_waits_that_name_the_registers():
    text = _source("products.cu")
    assert "tmem_ld_wait();" not in text
    assert text.count("tmem_ld16(") == text.count("tmem_ld_wait16(v)") == 3 and text.count("tmem_ld_wait16x2(v)") == 1
