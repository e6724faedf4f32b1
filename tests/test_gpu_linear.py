"""The dense product with bias, activation and residual, and its gradients, against 64 bits."""

import pytest
import torch

from moe_bench_b200 import capi
from oracle import ffn_oracle as F

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _normal(g, *shape, scale=1.0, dtype=torch.bfloat16):
    return (torch.randn(*shape, device=DEV, generator=g) * scale).to(dtype)


def _good(got, ref_and_bound, what=""):
    wrong = F.inside(got, *ref_and_bound)
    assert wrong is None, f"{what}: {wrong}"


SIZES = [(1, 8, 1), (1, 256, 33), (2, 72, 8), (31, 64, 64), (33, 136, 100), (64, 520, 256), (129, 64, 257), (255, 200, 130),
         (256, 64, 512), (257, 1000, 61), (513, 320, 264), (1000, 128, 1029), (3, 7168, 256), (300, 4096, 64), (40, 2048, 600)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,k,n", SIZES)
def test_plain_product(rows, k, n, dtype):
    g = _gen(rows * 7 + n)
    x, w = _normal(g, rows, k, dtype=dtype), _normal(g, n, k, scale=k ** -0.5, dtype=dtype)
    y, b, _, _ = F.linear(x, w, None, "none", None, dtype)
    _good(capi.linear(x, w), (y, b))
    y, b, _, _ = F.linear(x, w, None, "none", None, torch.float32)
    _good(capi.linear(x, w, out_dtype=torch.float32), (y, b), "fp32")


@pytest.mark.parametrize("act", sorted(capi.ACTIVATIONS))
@pytest.mark.parametrize("rows,k,n", [(5, 64, 37), (70, 136, 64), (300, 512, 520)])
@pytest.mark.parametrize("dtype,out_dtype,bias_dtype", [
    (torch.bfloat16, torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16, torch.float32),
    (torch.bfloat16, torch.float32, torch.float32), (torch.float16, torch.float32, torch.float16)])
def test_epilogue(act, rows, k, n, dtype, out_dtype, bias_dtype):
    g = _gen(rows + n)
    x, w = _normal(g, rows, k, dtype=dtype), _normal(g, n, k, scale=2 * k ** -0.5, dtype=dtype)
    bias, res = _normal(g, n, dtype=bias_dtype), _normal(g, rows, n, dtype=dtype)
    for b, r in ((bias, None), (None, res), (bias, res)):
        y, yb, s, sb = F.linear(x, w, b, act, r, out_dtype)
        got, slope = capi.linear(x, w, bias=b, activation=act, residual=r, out_dtype=out_dtype, want_slope=True)
        _good(got, (y, yb), "y")
        _good(slope, (s, sb), "slope")
        assert torch.equal(capi.linear(x, w, bias=b, activation=act, residual=r, out_dtype=out_dtype), got)


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh", "relu"])
def test_far_arguments_stay_finite_and_nan_stays(act):
    z = torch.tensor([-3e38, -1e30, -1e4, -100.0, -30.0, -12.0, -5.0, 0.0, 5.0, 12.0, 30.0, 100.0, 1e4, 1e30, 3e38], device=DEV)
    x = torch.zeros(2, 8, device=DEV, dtype=torch.bfloat16)
    x[:, 0] = 1
    w = torch.zeros(z.numel(), 8, device=DEV, dtype=torch.bfloat16)
    x[1, 1] = float("nan")
    y, slope = capi.linear(x, w, bias=z, activation=act, out_dtype=torch.float32, want_slope=True)
    ref, ref_slope = F.activation(act, z.double())
    assert torch.isfinite(y[0]).all() and torch.isfinite(slope[0]).all()
    # the values are rounded to fp32 after a few roundings of terms not larger than z
    assert torch.allclose(y[0].double(), ref, rtol=2e-6, atol=1e-6)
    assert torch.allclose(slope[0].double(), ref_slope.clamp(-2, 2), atol=2.0 ** -8)
    assert torch.isnan(y[1]).all()


def test_gelu_keeps_the_digits_of_its_tail():
    """In fp32, relative to the value: the fit is good to 1.8e-7, the exponential's argument z^2 / 2 is rounded twice (z^2 / 2 steps
    of 2^-24 each), and some 32 roundings of terms of the result's size are left."""
    z = torch.cat([torch.linspace(-9, 9, 100001), -torch.logspace(-30, 0, 500)]).cuda()
    w = torch.zeros(z.numel(), 8, device=DEV, dtype=torch.bfloat16)
    for rows in (1, 40):
        y = capi.linear(torch.zeros(rows, 8, device=DEV, dtype=torch.bfloat16), w, bias=z, activation="gelu", out_dtype=torch.float32)
        ref, _ = F.activation("gelu", z.double())
        bound = (1.8e-7 + (z.double() ** 2 + 32) * F.U32) * ref.abs() + 2.0 ** -140
        for row in y:
            _good(row, (ref, bound))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("with_slope", [False, True])
@pytest.mark.parametrize("rows,k,n", SIZES)
def test_gradients(rows, k, n, dtype, with_slope):
    g = _gen(rows * 3 + n)
    x, w = _normal(g, rows, k, dtype=dtype), _normal(g, n, k, scale=k ** -0.5, dtype=dtype)
    dy = _normal(g, rows, n, scale=0.3, dtype=dtype)
    slope = F.activation("gelu", torch.randn(rows, n, device=DEV, generator=g))[1].to(dtype) if with_slope else None
    dw_dtype = torch.float32 if rows % 2 else dtype
    ref = F.linear_backward(dy, x, w, slope, dw_dtype)
    got = capi.linear_backward(dy, x, w, slope=slope, dw_dtype=dw_dtype)
    for name, a, b in zip(("dx", "dw", "db"), got, ref):
        _good(a, b, name)
    again = capi.linear_backward(dy, x, w, slope=slope, dw_dtype=dw_dtype)
    assert all(torch.equal(a, b) for a, b in zip(got, again))


@pytest.mark.parametrize("rows,k,n", [(20, 512, 512), (300, 1024, 1024), (130, 2048, 264), (600, 512, 333), (64, 4096, 64), (2000, 256, 1500),
                                      (1000, 2048, 1024), (5000, 264, 72), (9000, 256, 520), (1500, 2048, 64), (5000, 2048, 72),
                                      (3000, 1032, 2100)])
def test_both_gradients_with_sums_of_different_lengths(rows, k, n):
    """In one launch or in two, split or not: dx sums over n, dw over the rows."""
    g = _gen(rows + k)
    x, w, dy = _normal(g, rows, k), _normal(g, n, k, scale=k ** -0.5), _normal(g, rows, n, scale=0.3)
    ref = F.linear_backward(dy, x, w, None, torch.float32)
    got = capi.linear_backward(dy, x, w, dw_dtype=torch.float32)
    for name, a, b in zip(("dx", "dw", "db"), got, ref):
        _good(a, b, name)
    assert all(torch.equal(a, b) for a, b in zip(got, capi.linear_backward(dy, x, w, dw_dtype=torch.float32)))


def test_fp32_output_gradient():
    g = _gen(5)
    x, w, dy = _normal(g, 65, 128), _normal(g, 48, 128, scale=0.1), torch.randn(65, 48, device=DEV, generator=g) * 1e-6
    for name, a, b in zip(("dx", "dw", "db"), capi.linear_backward(dy, x, w), F.linear_backward(dy, x, w, None, x.dtype)):
        _good(a, b, name)
    with pytest.raises(capi.MB200Error, match="dy"):
        capi.linear_backward(dy, x.half(), w.half())


@pytest.mark.parametrize("want", [(True, False, False), (False, True, False), (False, False, True), (False, False, False)])
def test_single_gradients(want):
    g = _gen(6)
    x, w, dy, slope = _normal(g, 70, 64), _normal(g, 24, 64), _normal(g, 70, 24), _normal(g, 70, 24)
    whole = capi.linear_backward(dy, x, w, slope=slope)
    some = capi.linear_backward(dy, x, w, slope=slope, want_dx=want[0], want_dw=want[1], want_db=want[2])
    for a, b, asked in zip(whole, some, want):
        assert torch.equal(a, b) if asked else b is None


def test_no_rows():
    x, w = torch.empty(0, 64, device=DEV, dtype=torch.bfloat16), torch.ones(8, 64, device=DEV, dtype=torch.bfloat16)
    assert capi.linear(x, w).shape == (0, 8)
    dx, dw, db = capi.linear_backward(torch.empty(0, 8, device=DEV, dtype=torch.bfloat16), x, w)
    assert dx.shape == (0, 64) and not dw.any() and not db.any()


def test_rows_further_apart_than_long_and_slices():
    g = _gen(8)
    wide, both = _normal(g, 50, 192), _normal(g, 2 * 40, 96, scale=0.1)
    x, w = wide[:, 64:160], both[40:]
    res = _normal(g, 50, 99)[:, 7:47]
    y, b, _, _ = F.linear(x, w, None, "none", res, x.dtype)
    _good(capi.linear(x, w, residual=res), (y, b))
    w2 = _normal(g, 40, 160, scale=0.1)[:, 32:128]
    y, b, _, _ = F.linear(x, w2, None, "none", None, x.dtype)
    _good(capi.linear(x, w2), (y, b))
    dy = _normal(g, 50, 83)[:, 3:43]  # starts on no boundary and has an odd distance from row to row
    for name, a, r in zip(("dx", "dw", "db"), capi.linear_backward(dy, x, w2), F.linear_backward(dy, x, w2, None, x.dtype)):
        _good(a, r, name)


def test_output_into_the_residual_and_into_odd_places():
    g = _gen(9)
    x, w, res = _normal(g, 70, 64), _normal(g, 36, 64, scale=0.1), _normal(g, 70, 36)
    expect = capi.linear(x, w, residual=res)
    assert capi.linear(x, w, residual=res, out=res).data_ptr() == res.data_ptr()
    assert torch.equal(res, expect)
    raw = torch.full((70 * 36 + 3,), 7.0, device=DEV, dtype=torch.bfloat16)
    out = raw[1 : 1 + 70 * 36].view(70, 36)  # on no vector boundary; its neighbours stay
    capi.linear(x, w, out=out)
    assert torch.equal(out, capi.linear(x, w))
    assert raw[0] == 7 and (raw[-2:] == 7).all()


def test_refusals():
    x, w = torch.zeros(4, 64, device=DEV, dtype=torch.bfloat16), torch.zeros(8, 64, device=DEV, dtype=torch.bfloat16)
    for bad in (dict(x=x.float()), dict(w=w.half()), dict(w=w[:, :32]), dict(activation="tanh"), dict(bias=torch.zeros(7, device=DEV)),
                dict(residual=torch.zeros(1, 8, device=DEV, dtype=x.dtype)), dict(out_dtype=torch.float16),
                dict(out=torch.zeros(4, 8, device=DEV)), dict(x=x.t()), dict(x=x[:1].expand(4, 64)), dict(w=w.cpu()),
                dict(residual=torch.zeros(8, device=DEV, dtype=x.dtype).expand(4, 8)), dict(x=x[:, 1:57], w=w[:, :56])):
        with pytest.raises(capi.MB200Error):
            capi.linear(**{"x": x, "w": w, **bad})


def test_captured_and_replayed_beside_eager_calls():
    g = _gen(10)
    x, w, b = _normal(g, 300, 256), _normal(g, 200, 256, scale=0.1), _normal(g, 200)
    dy = _normal(g, 300, 200)

    def step():
        y, slope = capi.linear(x, w, bias=b, activation="silu", want_slope=True)
        return (y, slope) + capi.linear_backward(dy, x, w, slope=slope)

    step()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            kept = step()
        graphs.append((graph, kept))
    fresh = _normal(g, 300, 256)
    x.copy_(fresh)
    expect = [t.clone() for t in step()]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for s, (graph, _) in zip(streams, graphs):
        with torch.cuda.stream(s):
            for _ in range(5):
                graph.replay()
    eager = step()
    torch.cuda.synchronize()
    for got in (graphs[0][1], graphs[1][1], eager):
        assert all(torch.equal(a, c) for a, c in zip(got, expect))
    assert capi.linear_status(DEV) == 0


def test_on_another_stream():
    g = _gen(11)
    x, w = _normal(g, 500, 512), _normal(g, 300, 512, scale=0.1)
    expect = capi.linear(x, w)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = capi.linear(x, w)
    s.synchronize()
    assert torch.equal(got, expect)
