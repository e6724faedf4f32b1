"""Layer norm and its gradients against 64 bits."""

import pytest
import torch

from moe_bench_b200 import capi
from oracle import ffn_oracle as F

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _good(got, ref_and_bound, what=""):
    wrong = F.inside(got, *ref_and_bound)
    assert wrong is None, f"{what}: {wrong}"


def _check(x, dy, w, b, eps=1e-5):
    y, mean, rstd = capi.layer_norm(x, w, b, eps=eps)
    ref = F.layer_norm(x, w, b, eps)
    for name, got, r in zip(("y", "mean", "rstd"), (y, mean, rstd), ref):
        _good(got, r, name)
    got = capi.layer_norm_backward(dy, x, mean, rstd, w)
    for name, a, r in zip(("dx", "dweight", "dbias"), got, F.layer_norm_backward(dy, x, mean, rstd, w)):
        _good(a, r, name)
    again = capi.layer_norm_backward(dy, x, mean, rstd, w)
    assert all(torch.equal(a, c) for a, c in zip(got, again))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,hidden", [(1, 1), (1, 7), (3, 8), (2, 100), (17, 512), (5, 1031), (700, 64), (1300, 257), (9, 2048),
                                         (1, 7168), (33, 7168), (610, 4096), (4, 16384), (2, 16392), (3, 40000), (2, 70001)])
def test_forward_and_gradients(rows, hidden, dtype):
    g = _gen(rows + hidden)
    x = (torch.randn(rows, hidden, device=DEV, generator=g) * 2 + 0.5).to(dtype)
    dy = torch.randn(rows, hidden, device=DEV, generator=g).to(dtype)
    w, b = torch.randn(hidden, device=DEV, generator=g), torch.randn(hidden, device=DEV, generator=g)
    _check(x, dy, w.to(dtype), b.to(dtype))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,hidden", [(150, 264), (1001, 520), (300, 768), (601, 1024), (2500, 1032), (333, 2048), (1203, 129), (450, 1031)])
def test_rows_side_by_side_in_a_block(rows, hidden, dtype):
    """Rows of a few warps share a block in the backward pass: last blocks that are not full, rows that end inside a warp."""
    g = _gen(rows * hidden)
    x, dy = (torch.randn(rows, hidden, device=DEV, generator=g).to(dtype) for _ in range(2))
    w, b = torch.randn(hidden, device=DEV, generator=g), torch.randn(hidden, device=DEV, generator=g)
    _check(x, dy, w, b)


@pytest.mark.parametrize("dtype", TYPES[:2])
@pytest.mark.parametrize("which", ["both", "weight", "bias", "none"])
@pytest.mark.parametrize("hidden", [96, 1001])
def test_parameters_in_fp32_or_absent(which, hidden, dtype):
    g = _gen(hidden)
    x, dy = torch.randn(40, hidden, device=DEV, generator=g).to(dtype), torch.randn(40, hidden, device=DEV, generator=g).to(dtype)
    w = torch.randn(hidden, device=DEV, generator=g) if which in ("both", "weight") else None
    b = torch.randn(hidden, device=DEV, generator=g) if which in ("both", "bias") else None
    _check(x, dy, w, b)


@pytest.mark.parametrize("pitch,start", [(136, 8), (131, 0), (200, 3)])
def test_rows_apart_and_off_the_boundaries(pitch, start):
    g = _gen(pitch)
    wide = torch.randn(50, pitch, device=DEV, generator=g).bfloat16()
    x, dy = wide[:, start : start + 120], torch.randn(50, pitch, device=DEV, generator=g).bfloat16()[:, start : start + 120]
    w = torch.randn(133, device=DEV, generator=g).bfloat16()
    _check(x, dy, w[start : start + 120], w[:120])


def test_rows_of_equal_and_of_far_values():
    """A constant row has variance 0; a row far from 0 keeps the digits that its spread has."""
    x = torch.full((3, 640), 5.0, device=DEV)
    x[1] = 0
    x[2] = 4096 + torch.arange(640, device=DEV) % 7
    y, mean, rstd = capi.layer_norm(x)
    assert not y[:2].any() and torch.equal(mean[:2], torch.tensor([5.0, 0.0], device=DEV))
    assert torch.allclose(rstd[:2].double(), torch.full((2,), 1e-5, device=DEV).double() ** -0.5, rtol=1e-6)
    _good(y, F.layer_norm(x, None, None, 1e-5)[0])


def test_a_spoilt_row_spoils_no_other():
    g = _gen(1)
    x = torch.randn(20, 300, device=DEV, generator=g)
    clean = capi.layer_norm(x)
    x[7, 5], x[11, 0] = float("nan"), float("inf")
    y, mean, rstd = capi.layer_norm(x)
    rest = [i for i in range(20) if i not in (7, 11)]
    for a, b in zip((y, mean, rstd), clean):
        assert torch.equal(a[rest], b[rest])
    assert torch.isnan(y[7]).all() and torch.isnan(y[11]).all()


@pytest.mark.parametrize("rows,hidden", [(5, 7), (900, 64), (1500, 520), (40, 7168), (700, 7168), (600, 1031), (6, 40000)])
def test_in_place(rows, hidden):
    g = _gen(rows)
    x, w, b = (torch.randn(*s, device=DEV, generator=g).bfloat16() for s in ((rows, hidden), (hidden,), (hidden,)))
    expect = capi.layer_norm(x, w, b)
    assert all(torch.equal(a, c) for a, c in zip(capi.layer_norm(x, w, b, out=x), expect))


def test_single_gradients_and_no_rows():
    g = _gen(2)
    x, dy = torch.randn(30, 200, device=DEV, generator=g).bfloat16(), torch.randn(30, 200, device=DEV, generator=g).bfloat16()
    _, mean, rstd = capi.layer_norm(x)
    whole = capi.layer_norm_backward(dy, x, mean, rstd)
    for want in ((True, False, False), (False, True, False), (False, False, True), (False, False, False)):
        some = capi.layer_norm_backward(dy, x, mean, rstd, want_dx=want[0], want_dweight=want[1], want_dbias=want[2])
        for a, b, asked in zip(whole, some, want):
            assert torch.equal(a, b) if asked else b is None
    y, m, r = capi.layer_norm(x[:0])
    assert y.shape == (0, 200)
    dx, dw, db = capi.layer_norm_backward(dy[:0], x[:0], m, r)
    assert dx.shape == (0, 200) and not dw.any() and not db.any()


def test_refusals():
    x = torch.zeros(4, 64, device=DEV)
    m = torch.zeros(4, device=DEV)
    for bad in (dict(x=x.double()), dict(x=x[0]), dict(weight=m), dict(x=x.t()), dict(x=x[:, :0]), dict(weight=torch.ones(64)),
                dict(weight=torch.ones(64, device=DEV), bias=torch.ones(64, device=DEV).half())):
        with pytest.raises(capi.MB200Error):
            capi.layer_norm(**{"x": x, **bad})
    with pytest.raises(capi.MB200Error):
        capi.layer_norm_backward(x.half(), x, m, m)
    with pytest.raises(capi.MB200Error):
        capi.layer_norm_backward(x, x, m[:3], m)


def test_captured():
    g = _gen(3)
    x, dy, w = (torch.randn(*s, device=DEV, generator=g).bfloat16() for s in ((100, 512), (100, 512), (512,)))
    _, mean, rstd = capi.layer_norm(x, w)
    capi.layer_norm_backward(dy, x, mean, rstd, w)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, mean, rstd = capi.layer_norm(x, w)
        grads = capi.layer_norm_backward(dy, x, mean, rstd, w)
    x.copy_(torch.randn(100, 512, device=DEV, generator=g).bfloat16())
    graph.replay()
    torch.cuda.synchronize()
    expect = capi.layer_norm(x, w)
    assert all(torch.equal(a, b) for a, b in zip((y, mean, rstd), expect))
    assert all(torch.equal(a, b) for a, b in zip(grads, capi.layer_norm_backward(dy, x, mean, rstd, w)))
