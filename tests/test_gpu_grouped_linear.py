"""Products over ragged row segments with one weight per expert, and their gradients, against 64 bits."""

import pytest
import torch

from moe_bench_b200 import capi
from oracle import ffn_oracle as F

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _normal(g, *shape, scale=1.0, dtype=torch.bfloat16):
    return (torch.randn(*shape, device=DEV, generator=g) * scale).to(dtype)


def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _offsets(sizes, begin=0):
    o = [begin]
    for s in sizes:
        o.append(o[-1] + s)
    return torch.tensor(o, device=DEV, dtype=torch.int32)


def _good(got, ref_and_bound, what=""):
    wrong = F.inside(got, *ref_and_bound)
    assert wrong is None, f"{what}: {wrong}"


SEGMENTS = [[1], [0, 0, 1, 0], [5, 0, 17, 64, 65, 1], [0] * 7, [256, 257, 255], [31, 32, 33, 0, 511, 16, 15, 3], [1] * 40,
            [1000], [0, 700, 0, 0, 129], [2, 3, 5, 7, 11, 13, 17, 19, 23, 29, 31, 37, 41, 43, 47, 53, 59, 61, 67, 71]]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("k,n", [(64, 64), (72, 333), (520, 40), (256, 264), (128, 1), (328, 8)])
@pytest.mark.parametrize("sizes", SEGMENTS, ids=lambda s: f"{len(s)}x{max(s)}")
def test_products_and_gradients(sizes, k, n, dtype):
    rows, e = sum(sizes), len(sizes)
    g = _gen(rows + n)
    x, w = _normal(g, rows, k, dtype=dtype), _normal(g, e, n, k, scale=k ** -0.5, dtype=dtype)
    dy, off = _normal(g, rows, n, scale=0.5, dtype=dtype), _offsets(sizes)
    if rows:
        _good(capi.grouped_linear(x, w, off), F.grouped_linear(x, w, sizes), "y")
    dw_dtype = torch.float32 if n % 2 else dtype
    dx, dw = capi.grouped_linear_backward(dy, x, w, off, dw_dtype=dw_dtype)
    (rx, bx), (rw, bw) = F.grouped_linear_backward(dy, x, w, sizes, dw_dtype)
    _good(dx, (rx, bx), "dx")
    _good(dw, (rw, bw), "dw")
    for i, s in enumerate(sizes):
        if s == 0:
            assert not dw[i].any()


@pytest.mark.parametrize("sizes,k,n", [([30, 0, 50, 20], 1024, 512), ([2000], 512, 300), ([0, 640, 1], 256, 1024), ([513, 0, 0, 255], 2048, 40),
                                       ([100] * 16, 512, 256)])
def test_gradients_where_pairs_share_tiles(sizes, k, n):
    rows, e = sum(sizes), len(sizes)
    g = _gen(rows * 7 + n)
    x, w, dy = _normal(g, rows + 5, k), _normal(g, e, n, k, scale=k ** -0.5), _normal(g, rows + 5, n, scale=0.5)
    x[:2], dy[:2], x[-3:], dy[-3:] = (float("nan"),) * 4  # outside the segments
    keep = torch.full_like(x, 7.0)
    dx, dw = capi.grouped_linear_backward(dy, x, w, _offsets(sizes, 2), dw_dtype=torch.float32, dx_out=keep)
    (rx, bx), (rw, bw) = F.grouped_linear_backward(dy[2:-3], x[2:-3], w, sizes, torch.float32)
    _good(dx[2:-3], (rx, bx), "dx")
    _good(dw, (rw, bw), "dw")
    assert (dx[:2] == 7).all() and (dx[-3:] == 7).all()


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_neighbours_and_rows_outside_have_no_part(bad):
    """NaN and inf in the rows of one expert, and in rows before, behind and between what counts, reach nobody else; rows
    outside the segments stay as they were."""
    g = _gen(3)
    sizes, before, after, k, n = [37, 50, 0, 70], 9, 21, 136, 72
    rows = before + sum(sizes) + after
    x, w, dy = _normal(g, rows, k), _normal(g, 4, n, k, scale=0.1), _normal(g, rows, n)
    off = _offsets(sizes, before)
    inner = slice(before, rows - after)
    ref_y = F.grouped_linear(x[inner], w, sizes)
    ref_dx, ref_dw = F.grouped_linear_backward(dy[inner], x[inner], w, sizes, x.dtype)
    spoil = torch.ones(rows, dtype=torch.bool, device=DEV)
    spoil[before : before + 37] = False
    spoil[before + 87 : before + 157] = False  # expert 1's rows and everything outside are spoilt
    x[spoil], dy[spoil] = bad, bad
    keep_y, keep_dx = torch.full((rows, n), 3.0, device=DEV, dtype=x.dtype), torch.full((rows, k), 3.0, device=DEV, dtype=x.dtype)
    y = capi.grouped_linear(x, w, off, out=keep_y)
    dx, dw = capi.grouped_linear_backward(dy, x, w, off, dx_out=keep_dx)
    for t in (y, dx):
        assert (t[:before] == 3).all() and (t[rows - after :] == 3).all()
    fine = ~spoil[inner]
    _good(y[inner][fine], (ref_y[0][fine], ref_y[1][fine]), "y")
    _good(dx[inner][fine], (ref_dx[0][fine], ref_dx[1][fine]), "dx")
    for e in (0, 2, 3):
        _good(dw[e], (ref_dw[0][e], ref_dw[1][e]), f"dw[{e}]")
    assert not torch.isfinite(dw[1]).any()
    # one expert's weights spoilt
    w[0] = bad
    y2 = capi.grouped_linear(x, w, off)
    late = slice(before + 87, before + 157)
    assert torch.equal(y2[late], y[late])


def test_offsets_past_the_rows_are_cut():
    g = _gen(4)
    x, w = _normal(g, 40, 64), _normal(g, 3, 24, 64, scale=0.1)
    off = torch.tensor([0, 30, 20, 1000], device=DEV, dtype=torch.int32)  # the second ends before it begins
    y = capi.grouped_linear(x, w, off, out=torch.zeros(40, 24, device=DEV, dtype=x.dtype))
    assert torch.equal(y[:20], capi.grouped_linear(x, w[:1], _offsets([30]))[:20])
    dx, dw = capi.grouped_linear_backward(y, x, w, off)
    assert not dw[1].any()
    assert torch.equal(dw[2], capi.grouped_linear_backward(y[20:], x[20:], w[2:], _offsets([20]))[1][0])
    low = torch.tensor([-5, 10, 40, 40], device=DEV, dtype=torch.int32)
    assert torch.equal(capi.grouped_linear(x, w, low), capi.grouped_linear(x, w, _offsets([10, 30, 0])))


def test_segments_that_overlap_end_all_the_same():
    """Offsets that do not ascend name more rows than there are; whatever comes out, every wait completes, and calls after it
    are right."""
    g = _gen(31)
    x, w = _normal(g, 4096, 512), _normal(g, 8, 64, 512, scale=0.05)
    dy = _normal(g, 4096, 64)
    bad = torch.tensor([0, 4096, 0, 4096, 0, 4096, 0, 4096, 0], device=DEV, dtype=torch.int32)
    y = capi.grouped_linear(x, w, bad)
    dx, dw = capi.grouped_linear_backward(dy, x, w, bad)
    assert capi.linear_status() == 0 and y.shape == dy.shape and dx.shape == x.shape and dw.shape == w.shape
    sizes = [512] * 8
    _good(capi.grouped_linear(x, w, _offsets(sizes)), F.grouped_linear(x, w, sizes), "y")


def test_half_of_fused_weights_and_pitches():
    g = _gen(5)
    w1, x = _normal(g, 6, 2 * 40, 96, scale=0.1), _normal(g, 90, 200)[:, 8:104]
    sizes = [20, 0, 33, 7, 30, 0]
    up = w1[:, 40:]
    _good(capi.grouped_linear(x, up, _offsets(sizes)), F.grouped_linear(x, up, sizes), "y")
    dy = _normal(g, 90, 51)[:, 5:45]
    dx, dw = capi.grouped_linear_backward(dy, x, up, _offsets(sizes))
    rx, rw = F.grouped_linear_backward(dy, x, up, sizes, x.dtype)
    _good(dx, rx, "dx")
    _good(dw, rw, "dw")


def test_one_gradient_at_a_time_and_no_rows():
    g = _gen(6)
    x, w, dy, off = _normal(g, 50, 64), _normal(g, 3, 16, 64), _normal(g, 50, 16), _offsets([20, 0, 30])
    both = capi.grouped_linear_backward(dy, x, w, off)
    assert torch.equal(capi.grouped_linear_backward(dy, x, w, off, want_dw=False)[0], both[0])
    assert torch.equal(capi.grouped_linear_backward(dy, x, w, off, want_dx=False)[1], both[1])
    empty = capi.grouped_linear_backward(dy[:0], x[:0], w, torch.zeros(4, device=DEV, dtype=torch.int32))
    assert empty[0].shape == (0, 64) and not empty[1].any()


def test_refusals():
    g = _gen(7)
    x, w, off = _normal(g, 8, 64), _normal(g, 2, 8, 64), _offsets([3, 5])
    for bad in (dict(off=off.long()), dict(off=off[:2]), dict(off=off.cpu()), dict(w=w[0]), dict(w=w.half()), dict(x=x[:, ::2]),
                dict(w=w[:1].expand(2, 8, 64)), dict(x=x[:, :32])):
        a = {"x": x, "w": w, "off": off, **bad}
        with pytest.raises(capi.MB200Error):
            capi.grouped_linear(a["x"], a["w"], a["off"])


def test_many_experts_with_the_schedule_of_the_router():
    """1024 experts, offsets from align at pad_rows = 1, every assignment's row gathered by its sorted id."""
    g = _gen(8)
    tokens, topk, e, k, n = 300, 4, 1024, 64, 40
    logits = torch.randn(tokens, e, device=DEV, generator=g)
    ids, _ = capi.route_topk(logits, topk)
    counts, prefix, sorted_ids, _ = capi.align(ids, None, e, pad_rows=1)
    x, w = _normal(g, tokens, k), _normal(g, e, n, k, scale=0.1)
    rows = x[sorted_ids.long() // topk].contiguous()
    y = capi.grouped_linear(rows, w, prefix)
    _good(y, F.grouped_linear(rows, w, counts.tolist()), "y")


def test_captured_replays_follow_new_offsets():
    g = _gen(9)
    x, w, dy = _normal(g, 200, 128), _normal(g, 4, 72, 128, scale=0.1), _normal(g, 200, 72)
    off = _offsets([50, 50, 50, 50])
    y, dx = torch.zeros(200, 72, device=DEV, dtype=x.dtype), torch.zeros(200, 128, device=DEV, dtype=x.dtype)
    capi.grouped_linear(x, w, off, out=y)
    capi.grouped_linear_backward(dy, x, w, off, dx_out=dx)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        capi.grouped_linear(x, w, off, out=y)
        _, dw = capi.grouped_linear_backward(dy, x, w, off, dx_out=dx)
    sizes = [3, 150, 0, 47]
    off.copy_(_offsets(sizes))
    graph.replay()
    torch.cuda.synchronize()
    _good(y, F.grouped_linear(x, w, sizes), "y")
    rx, rw = F.grouped_linear_backward(dy, x, w, sizes, x.dtype)
    _good(dx, rx, "dx")
    _good(dw, rw, "dw")
    assert capi.linear_status(DEV) == 0
