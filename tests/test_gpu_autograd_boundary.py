"""The products stand outside autograd, and a Function around them, as the documents show it, is how they enter it."""

import os
import re

import pytest
import torch

from moe_bench_b200 import capi

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _documented_function():
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    text = open(os.path.join(root, "INTEGRATION.md")).read()
    scope = {"torch": torch, "capi": capi}
    exec(re.search(r"```python\n(class Linear\(.*?)```", text, re.S).group(1), scope)
    return scope["Linear"]


def test_results_carry_no_graph():
    x = torch.randn(5, 64, device=DEV).bfloat16().requires_grad_()
    w = torch.randn(24, 64, device=DEV).bfloat16().requires_grad_()
    off = torch.tensor([0, 5], device=DEV, dtype=torch.int32)
    y, mean, rstd = capi.layer_norm(x)
    for t in (capi.linear(x, w), capi.grouped_linear(x, w[None].detach(), off), y, mean, rstd, *capi.linear_backward(x.new_ones(5, 24), x, w)):
        assert not t.requires_grad and t.grad_fn is None


def test_the_documented_function_gives_the_gradients():
    g = torch.Generator(device=DEV)
    g.manual_seed(1)
    x, w, dy = ((torch.randn(*s, device=DEV, generator=g)).bfloat16() for s in ((70, 64), (24, 64), (70, 24)))
    leaves = [t.clone().requires_grad_() for t in (x, w)]
    fn = _documented_function()
    y = fn.apply(*leaves)
    assert torch.equal(y, capi.linear(x, w))
    y.backward(dy)
    dx, dw, _ = capi.linear_backward(dy, x, w)
    assert torch.equal(leaves[0].grad, dx) and torch.equal(leaves[1].grad, dw)
    only = x.clone().requires_grad_()
    fn.apply(only, w).backward(dy)
    assert torch.equal(only.grad, dx)
    # of a sum: a dy whose rows all are one element
    leaf = x.clone().requires_grad_()
    fn.apply(leaf, w).sum().backward()
    assert torch.equal(leaf.grad, capi.linear_backward(torch.ones_like(dy), x, w)[0])


def test_the_documented_function_is_captured_with_its_backward_pass():
    """Autograd's worker may see the GPU for the first time while the main thread captures."""
    g = torch.Generator(device=DEV)
    g.manual_seed(2)
    x, w, dy = ((torch.randn(*s, device=DEV, generator=g)).bfloat16() for s in ((300, 64), (24, 64), (300, 24)))
    leaf = w.clone().requires_grad_()
    fn = _documented_function()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        (grad,) = torch.autograd.grad(fn.apply(x, leaf), leaf, dy)
    x.copy_(torch.randn(300, 64, device=DEV, generator=g))
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(grad, capi.linear_backward(dy, x, w)[1])
