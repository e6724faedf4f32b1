"""Long sums of the products, to the last bit.

Operands are whole numbers of at most ``most`` whose sums stay below 2^24: every partial sum, in whatever order and however a tile's sum
is split and joined, is a whole number that fp32 holds, so the 32-bit sum is the exact one, an fp32 output equals it and a
16-bit output is its one rounding.  A term left out or taken twice, a sum held in fewer bits or rounded on the way shows in
almost every element."""

import pytest
import torch

from moe_bench_b200 import capi

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
# fp16 outputs end at 65504
MOST = {torch.bfloat16: 31, torch.float16: 3}


def _whole(g, *shape, dtype):
    most = MOST[dtype]
    return torch.randint(-most, most + 1, shape, device=DEV, generator=g).to(dtype)


def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _same(got, exact, dtype):
    """One rounding, from a value that fp32 holds."""
    assert exact.abs().max() < (1 << 24)
    return got.dtype == dtype and torch.equal(got, exact.float().to(dtype))


def _bounded(length, dtype):
    return length * MOST[dtype] ** 2 < (1 << 24 if dtype == torch.bfloat16 else 65504)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,k,n", [(1, 7168, 256), (5, 7168, 61), (16, 4096, 2048), (9, 7000, 40), (17, 7168, 256), (40, 7168, 64),
                                      (131, 7168, 2048), (200, 1024, 512), (300, 5000, 333), (600, 7168, 61), (2100, 1032, 520),
                                      (1500, 4096, 1031)])
def test_forward(rows, k, n, dtype):
    assert _bounded(k, dtype)
    g = _gen(rows + k + n)
    x, w = _whole(g, rows, k, dtype=dtype), _whole(g, n, k, dtype=dtype)
    exact = x.double() @ w.double().t()
    assert _same(capi.linear(x, w, out_dtype=torch.float32), exact, torch.float32)
    assert _same(capi.linear(x, w), exact, dtype)
    bias, res = _whole(g, n, dtype=dtype), _whole(g, rows, n, dtype=dtype)
    assert _same(capi.linear(x, w, bias=bias, residual=res, out_dtype=torch.float32), exact + bias.double() + res.double(), torch.float32)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("with_slope", [False, True])
@pytest.mark.parametrize("rows,k,n", [(7000, 256, 72), (40, 512, 7168), (1000, 2048, 1024), (4100, 136, 515), (7168, 64, 1), (333, 1024, 4096),
                                      (6000, 520, 256), (1031, 1024, 2048)])
def test_gradients(rows, k, n, with_slope, dtype):
    """A slope of 0, 1/2, 1 or 2 and fewer values of dy keep every dz a multiple of 1/2 that the operands' type holds; with an even
    x and w all sums are whole numbers again."""
    g = _gen(rows * 3 + n)
    x, w, dy = _whole(g, rows, k, dtype=dtype), _whole(g, n, k, dtype=dtype), _whole(g, rows, n, dtype=dtype)
    slope = None
    if with_slope:
        slope = torch.tensor([0.0, 0.5, 1.0, 2.0], device=DEV)[torch.randint(0, 4, (rows, n), device=DEV, generator=g)].to(dtype)
        x, w, dy = x // 2 * 2, w // 2 * 2, dy.sign()
    dz = dy.double() if slope is None else dy.double() * slope.double()
    assert slope is not None or _bounded(max(rows, n), dtype)
    dx, dw, db = capi.linear_backward(dy, x, w, slope=slope, dw_dtype=torch.float32)
    assert _same(dx, dz @ w.double(), dtype)
    assert _same(dw, dz.t() @ x.double(), torch.float32)
    assert torch.equal(db, dz.sum(0).float())
    dw16 = capi.linear_backward(dy, x, w, slope=slope, want_dx=False, want_db=False)[1]
    assert _same(dw16, dz.t() @ x.double(), dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("sizes,k,n", [([30, 0, 50, 20], 7168, 512), ([2000], 4096, 300), ([0, 3000, 1, 999], 1024, 264), ([100] * 16, 7168, 256),
                                       ([513, 0, 0, 255], 2048, 4096), ([5, 64, 63, 65, 128, 0, 7], 7160, 72)])
def test_ragged_products_and_gradients(sizes, k, n, dtype):
    assert _bounded(max(k, n, *sizes), dtype)
    rows, e = sum(sizes), len(sizes)
    g = _gen(rows * 7 + n)
    x, w, dy = _whole(g, rows, k, dtype=dtype), _whole(g, e, n, k, dtype=dtype), _whole(g, rows, n, dtype=dtype)
    off = torch.tensor([sum(sizes[:i]) for i in range(e + 1)], device=DEV, dtype=torch.int32)
    y = capi.grouped_linear(x, w, off)
    dx, dw = capi.grouped_linear_backward(dy, x, w, off, dw_dtype=torch.float32)
    begin = 0
    for i, size in enumerate(sizes):
        part = slice(begin, begin + size)
        begin += size
        if size:
            assert _same(y[part], x[part].double() @ w[i].double().t(), dtype), i
            assert _same(dx[part], dy[part].double() @ w[i].double(), dtype), i
            assert _same(dw[i], dy[part].double().t() @ x[part].double(), torch.float32), i
        else:
            assert not dw[i].any()
    assert capi.linear_status() == 0
