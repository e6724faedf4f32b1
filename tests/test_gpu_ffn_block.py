"""The products and the norm together, as an FFN block uses them: norm, gate projection, selection, sort, ragged expert
products, shared expert with the routed output as its residual; the whole backward pass; and the gated front end."""

import os
import subprocess
import sys

import pytest
import torch

from moe_bench_b200 import capi, gating
from moe_bench_b200 import problem as P
from moe_bench_b200.plugin import get_implementation
from oracle import ffn_oracle as F
from oracle import moe_oracle as O

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _block_forward_backward(p, hidden, dout, topk):
    """Every intermediate is rounded to the operands' type, as a program would keep it."""
    dt, tokens = hidden.dtype, hidden.shape[0]
    e = p["w1"].shape[0]
    x, mean, rstd = capi.layer_norm(hidden, p["nw"], p["nb"])
    logits = capi.linear(x, p["gw"], bias=p["gb"], out_dtype=torch.float32)
    ids, wts = capi.route_topk(logits, topk)
    counts, offsets, sorted_ids, inverse = capi.align(ids, None, e, pad_rows=1)
    src = (sorted_ids[: tokens * topk] // topk).long()
    xs = x[src]
    up = capi.grouped_linear(xs, p["w1"], offsets)
    n = up.shape[1] // 2
    g, u = up[:, :n].float(), up[:, n:].float()
    act = (torch.nn.functional.silu(g) * u).to(dt)
    down = capi.grouped_linear(act, p["w2"], offsets)
    per = down[inverse.long()].view(tokens, topk, -1)
    routed = (per.float() * wts[:, :, None]).sum(1).to(dt)
    hs, slope = capi.linear(x, p["s1"], activation="silu", want_slope=True)
    out = capi.linear(hs, p["s2"], residual=routed)

    grads = {}
    dhs, grads["s2"], _ = capi.linear_backward(dout, hs, p["s2"], want_db=False)
    dx_shared, grads["s1"], _ = capi.linear_backward(dhs, x, p["s1"], slope=slope, want_db=False)
    dper = dout.float()[:, None, :] * wts[:, :, None]
    dwts = (dout.float()[:, None, :] * per.float()).sum(2)
    ddown = torch.empty_like(down)
    ddown[inverse.long()] = dper.reshape(-1, dper.shape[2]).to(dt)
    dact, grads["w2"] = capi.grouped_linear_backward(ddown, act, p["w2"], offsets)
    s = torch.sigmoid(g)
    dg = dact.float() * u * s * (1 + g * (1 - s))
    du = dact.float() * g * s
    dxs, grads["w1"] = capi.grouped_linear_backward(torch.cat([dg, du], 1).to(dt), xs, p["w1"], offsets)
    dlogits = torch.zeros_like(logits)
    dlogits.scatter_(1, ids.long(), wts * (dwts - (wts * dwts).sum(1, keepdim=True)))
    dx_gate, grads["gw"], grads["gb"] = capi.linear_backward(dlogits, x, p["gw"])
    dx = dx_shared.float() + dx_gate.float()
    dx.index_add_(0, src, dxs.float())
    dhidden, grads["nw"], grads["nb"] = capi.layer_norm_backward(dx.to(dt), hidden, mean, rstd, p["nw"])
    grads["hidden"] = dhidden
    return out, ids, grads


def _reference(p, hidden, dout, ids, topk):
    """The same block in 64 bits by autograd, with the selection as it was made."""
    q = {k: v.double().requires_grad_() for k, v in p.items()}
    h = hidden.double().requires_grad_()
    x = torch.nn.functional.layer_norm(h, (h.shape[1],), q["nw"], q["nb"], eps=1e-5)
    logits = x @ q["gw"].t() + q["gb"]
    wts = torch.softmax(logits.gather(1, ids.long()), 1)
    rows = []
    n = q["w2"].shape[2]
    for j in range(topk):
        w1, w2 = q["w1"][ids[:, j].long()], q["w2"][ids[:, j].long()]
        up = torch.einsum("tk,tnk->tn", x, w1)
        act = torch.nn.functional.silu(up[:, :n]) * up[:, n:]
        rows.append(torch.einsum("tn,tkn->tk", act, w2) * wts[:, j : j + 1])
    out = torch.nn.functional.silu(x @ q["s1"].t()) @ q["s2"].t() + sum(rows)
    out.backward(dout.double())
    grads = {k: v.grad for k, v in q.items()}
    grads["hidden"] = h.grad
    return out.detach(), grads


def test_block_forward_and_every_gradient():
    tokens, hidden, inter, e, topk = 203, 256, 136, 10, 3
    g = torch.Generator(device=DEV)
    g.manual_seed(2)

    def normal(*s, scale=1.0, shift=0.0, dtype=torch.bfloat16):
        return (torch.randn(*s, device=DEV, generator=g) * scale + shift).to(dtype)

    p = {"nw": normal(hidden, scale=0.1, shift=1.0), "nb": normal(hidden, scale=0.1), "gw": normal(e, hidden, scale=hidden ** -0.5),
         "gb": normal(e, scale=0.1, dtype=torch.float32), "w1": normal(e, 2 * inter, hidden, scale=hidden ** -0.5),
         "w2": normal(e, hidden, inter, scale=inter ** -0.5), "s1": normal(72, hidden, scale=hidden ** -0.5),
         "s2": normal(hidden, 72, scale=72 ** -0.5)}
    x, dout = normal(tokens, hidden, scale=1.5), normal(tokens, hidden)
    out, ids, grads = _block_forward_backward(p, x, dout, topk)
    ref, ref_grads = _reference(p, x, dout, ids, topk)
    # No path through the block passes more than 12 roundings to bf16, each off by at most 2^-8 of its value, in norm
    # at most that; the sums they enter have terms of either sign, whose norm is at least a third of the terms' norm
    # with these random values: 12 * 2^-8 / sqrt(3) (a rounding's mean square) = 2.7 %.
    bound = 12 * 2.0 ** -8 / 3 ** 0.5
    def rel(a, b):
        return ((a.double() - b).norm() / b.norm()).item()

    assert rel(out, ref) < bound
    for k, v in ref_grads.items():
        assert rel(grads[k], v) < bound, k
    assert capi.linear_status(DEV) == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_products_are_adjoint_to_their_gradients(dtype):
    """The products are linear: their difference quotient along d is the product of d itself, and <dy, f(d)> = <f^T(dy), d>."""
    g = torch.Generator(device=DEV)
    g.manual_seed(3)
    sizes = [37, 0, 300, 12]
    rows, k, n = sum(sizes), 136, 200
    off = torch.tensor([0, 37, 37, 337, 349], device=DEV, dtype=torch.int32)
    x, dy = (torch.randn(rows, c, device=DEV, generator=g).to(dtype) for c in (k, n))
    w = torch.randn(4, n, k, device=DEV, generator=g).to(dtype)
    dx, dw = capi.grouped_linear_backward(dy, x, w, off, dw_dtype=torch.float32)
    # each inner product sums roundings of random sign: half a step of a term's type over the square root of 3, times the norms
    half = torch.finfo(dtype).eps / 2
    d = torch.randn(rows, k, device=DEV, generator=g).to(dtype)
    y = capi.grouped_linear(d, w, off)
    a, b = (dy.double() * y.double()).sum(), (dx.double() * d.double()).sum()
    slack = 4 * half * ((dy.double() * y.double()).norm() + (dx.double() * d.double()).norm())
    assert abs(a - b) < slack
    dv = torch.randn(4, n, k, device=DEV, generator=g).to(dtype)
    y = capi.grouped_linear(x, dv, off)
    a, b = (dy.double() * y.double()).sum(), (dw.double() * dv.double()).sum()
    assert abs(a - b) < 4 * half * (dy.double() * y.double()).norm() + 1e-5 * (dw.double() * dv.double()).norm()


def test_norm_gradient_is_the_difference_quotient():
    g = torch.Generator(device=DEV)
    g.manual_seed(4)
    x, w, dy, d = (torch.randn(*s, device=DEV, generator=g) for s in ((5, 400), (400,), (5, 400), (5, 400)))
    _, mean, rstd = capi.layer_norm(x, w)
    dx, _, _ = capi.layer_norm_backward(dy, x, mean, rstd, w)
    step = 2.0 ** -7
    plus, minus = capi.layer_norm(x + step * d, w)[0], capi.layer_norm(x - step * d, w)[0]
    quotient = ((plus.double() - minus.double()) * dy.double()).sum() / (2 * step)
    # third-order term of the quotient: step^2 times about the size of the gradient, and fp32 roundings over 2 step
    assert abs(quotient - (dx.double() * d.double()).sum()) < step ** 2 * 4 * (dx.norm() * d.norm()) + 2.0 ** -22 / step * dy.norm() * 8


def test_gated_front_end_feeds_the_layer():
    cfg = P.MoEBenchConfig(hidden_size=512, intermediate_size=256, num_experts=16, topk=4, world_size=1, precision=P.Precision.BF16,
                           routing=P.RoutingConfig(distribution=P.Distribution.UNIFORM), seed=0, device=DEV)
    gate = gating.make_gate(cfg)
    base = P.make_problem(cfg, 150)
    prob = gating.make_gated_problem(cfg, 150, gate=gate)
    assert torch.equal(prob.w1, base.w1) and prob.hidden_states.shape == base.hidden_states.shape
    x = torch.nn.functional.layer_norm(base.hidden_states.double(), (512,), gate.norm_weight.double(), gate.norm_bias.double(), eps=1e-5)
    assert (prob.hidden_states.double() - x).abs().max() < 2.0 ** -8 * x.abs().max() + 1e-5
    logits = prob.hidden_states.double() @ gate.weight.double().t() + gate.bias.double()
    top = logits.gather(1, prob.topk_ids.long())
    # the selection is the logits' own up to fp32 sums of 512 terms
    assert (top.min(1).values >= logits.topk(cfg.topk, 1).values.min(1).values - 1e-4).all()
    assert torch.allclose(prob.topk_weights.double(), torch.softmax(top, 1), atol=1e-4)
    impl = get_implementation("b200")
    impl.setup(prob)
    res = O.verify_output("bf16", impl.run(prob), O.reference_moe(prob))
    assert res.passed, res.message
    again = gating.make_gated_problem(cfg, 150)
    assert torch.equal(again.topk_ids, prob.topk_ids) and torch.equal(again.hidden_states, prob.hidden_states)


def test_threads_with_streams_of_their_own():
    """Four host threads, each with its stream, tensors and sizes: nothing but the device is shared, and every result is the
    one that the calls give alone."""
    from concurrent.futures import ThreadPoolExecutor

    def operands(i):
        g = torch.Generator(device=DEV)
        g.manual_seed(i)
        rows, k, n = 300 + 137 * i, 1024, 256 + 8 * i
        t = [(torch.randn(*s, device=DEV, generator=g) * 0.1).bfloat16() for s in ((rows, k), (n, k), (rows, n), (3, n, k), (k,))]
        return t + [torch.tensor([0, 100, 100, rows], device=DEV, dtype=torch.int32)]

    def calls(t):
        x, w, dy, experts, gain, off = t
        y, slope = capi.linear(x, w, activation="silu", want_slope=True)
        out = [y, slope, capi.linear(x[:5], w), *capi.linear_backward(dy, x, w, slope=slope), capi.grouped_linear(x, experts, off)]
        out += capi.grouped_linear_backward(dy, x, experts, off)
        h, mean, rstd = capi.layer_norm(x, gain)
        return out + [h, mean, rstd, *capi.layer_norm_backward(x, x, mean, rstd, gain)]

    sets = [operands(i) for i in range(4)]
    alone = [calls(t) for t in sets]
    torch.cuda.synchronize()

    def work(t):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            results = [calls(t) for _ in range(20)]
        stream.synchronize()
        return results

    with ThreadPoolExecutor(4) as pool:
        together = list(pool.map(work, sets))
    for expect, many in zip(alone, together):
        for got in many:
            assert all(torch.equal(a, b) for a, b in zip(got, expect))
    assert capi.linear_status() == 0



FIRST_CALLS = """
import torch
from moe_bench_b200 import capi
d = "cuda:0"
x = torch.randn(300, 256, device=d).bfloat16()
w = torch.randn(200, 256, device=d).bfloat16()
w3 = torch.randn(3, 200, 256, device=d).bfloat16()
dy = torch.randn(300, 200, device=d).bfloat16()
off = torch.tensor([0, 50, 50, 300], device=d, dtype=torch.int32)
stats = torch.ones(300, device=d)
torch.cuda.synchronize()

def calls():
    out = [capi.linear(x, w, activation="gelu"), capi.linear(x[:5], w), capi.linear(x[:40], w)]
    out += capi.linear_backward(dy, x, w) + (capi.grouped_linear(x, w3, off),) + capi.grouped_linear_backward(dy, x, w3, off)
    out += capi.layer_norm(x) + capi.layer_norm_backward(x, x, stats, stats)
    return out

graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    captured = calls()
graph.replay()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(captured, calls()))
print("fine")
"""


def test_first_calls_of_a_process_may_be_captured():
    """Kernels, their attributes and the cluster query are all new to the process when the capture begins."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    res = subprocess.run([sys.executable, "-c", FIRST_CALLS], cwd=root, capture_output=True, text=True, timeout=180)
    assert res.returncode == 0 and "fine" in res.stdout, res.stderr[-2000:]


def test_tensors_of_more_elements_than_32_bits_count():
    """Rows repeat, so that every element of the large results has a known value; gradients come from the last rows alone."""
    rows, n, k, period = 128 * 2064, 16400, 8, 128
    assert rows * n > 1 << 32
    g = torch.Generator(device=DEV)
    g.manual_seed(5)

    def normal(*shape):
        return torch.randn(*shape, device=DEV, generator=g).bfloat16()

    def repeats(t, expect):
        return all(torch.equal(t[i : i + 16 * period].view(-1, period, t.shape[1]), expect.expand(16, *expect.shape))
                   for i in range(0, rows, 16 * period))

    w, few, bias, tail = normal(n, k), normal(period, k), normal(n), normal(100, n)
    x = few.repeat(rows // period, 1)
    y = capi.linear(x, w, bias)
    assert not F.inside(y[:period], *F.linear(few, w, bias, "none", None, y.dtype)[:2]) and repeats(y, y[:period].clone())
    dy = y.zero_()
    dy[-100:] = tail
    slope = torch.ones_like(dy)
    expect = F.linear_backward(tail, x[-100:], w, slope[:100], w.dtype)
    for s in (None, slope):  # with a slope the products read a copy of dy
        dx, dw, db = capi.linear_backward(dy, x, w, slope=s)
        assert not dx[:-100].any()
        for got, ref in zip((dx[-100:], dw, db), expect):
            assert not F.inside(got, *ref)
    del slope
    experts = torch.stack([w, w.flip(0), -w])
    off = torch.tensor([0, rows - 50, rows - 50, rows], device=DEV, dtype=torch.int32)
    out = capi.grouped_linear(x, experts, off, out=dy)
    front = capi.linear(few, w)
    assert torch.equal(out[-50:], -front[-50:])
    out[-50:] = front[-50:]
    assert repeats(out, front)
    h = out[:, : n - 16]  # rows apart
    few_h = h[:period]
    h, (one, mean, rstd) = capi.layer_norm(h), capi.layer_norm(few_h)
    assert repeats(h[0], one) and torch.equal(h[1].view(-1, period), mean.expand(rows // period, period))
    dh = torch.zeros_like(h[0])
    dh[-100:] = tail[:, : n - 16]
    got = capi.layer_norm_backward(dh, out[:, : n - 16], h[1], h[2])
    assert not got[0][:-100].any()
    alone = F.layer_norm_backward(dh[-100:], few_h[-100:], mean[-100:], rstd[-100:], None)
    for a, r in zip((got[0][-100:], *got[1:]), alone):
        assert not F.inside(a, *r)
    assert capi.linear_status() == 0
