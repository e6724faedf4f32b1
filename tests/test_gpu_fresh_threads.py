"""Calls from a host thread that has not touched the GPU before, as autograd's and a server's workers are: no context is current
there, and what a call needs of one it has to bring along."""

import threading

import pytest
import torch

from moe_bench_b200 import capi

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _operands():
    g = torch.Generator(device=DEV)
    g.manual_seed(7)
    x, w, dy, experts = ((torch.randn(*s, device=DEV, generator=g) * 0.1).bfloat16() for s in ((300, 256), (200, 256), (300, 200), (2, 200, 256)))
    return x, w, dy, experts, torch.tensor([0, 120, 300], device=DEV, dtype=torch.int32)


def _stage():
    """The first grouped stage of the layer on 64 rows of one expert."""
    g = torch.Generator(device=DEV)
    g.manual_seed(8)
    x, w1 = ((torch.randn(*s, device=DEV, generator=g) * 0.1).bfloat16() for s in ((64, 256), (1, 256, 256)))
    ids = torch.zeros(64, 1, device=DEV, dtype=torch.int32)
    counts, prefix, sorted_ids, _ = capi.align(ids, None, 1)
    rows = x.new_zeros(sorted_ids.shape[0], 256)
    rows[:64] = x
    out, status = rows.new_zeros(rows.shape[0], 128), torch.zeros(64, device=DEV, dtype=torch.int32)

    def call():
        capi.grouped_gemm_bf16(0, rows, w1, 256, 128, counts, prefix, sorted_ids, None, out, status)
        return (out,)

    return call


CALLS = {
    "linear": lambda x, w, dy, experts, off: (capi.linear(x, w),),
    "linear of few rows": lambda x, w, dy, experts, off: (capi.linear(x[:5], w),),
    "linear_backward": lambda x, w, dy, experts, off: capi.linear_backward(dy, x, w, want_db=False)[:2],
    "linear_backward with db": lambda x, w, dy, experts, off: capi.linear_backward(dy, x, w),
    "grouped_linear": lambda x, w, dy, experts, off: (capi.grouped_linear(x, experts, off),),
    "grouped_linear_backward": lambda x, w, dy, experts, off: capi.grouped_linear_backward(dy, x, experts, off),
    "layer_norm": lambda x, w, dy, experts, off: capi.layer_norm(x),
}


@pytest.mark.parametrize("name", [*CALLS, "layer's first stage"])
def test_first_call_of_a_thread(name):
    operands, got = _operands(), []
    call = (lambda: CALLS[name](*operands)) if name in CALLS else _stage()
    expect = [t.clone() for t in call()]
    torch.cuda.synchronize()

    def work():
        try:
            got.append(call())
        except Exception as e:  # the thread's end would hide it
            got.append(e)

    thread = threading.Thread(target=work)
    thread.start()
    thread.join()
    torch.cuda.synchronize()
    assert not isinstance(got[0], Exception), got[0]
    assert all(torch.equal(a, b) for a, b in zip(got[0], expect))


def test_first_call_of_a_thread_into_a_capture():
    """The stream is being captured by another thread, in the mode that is strictest about what others call."""
    x, w = _operands()[:2]
    expect, failed = capi.linear(x, w), []
    out = torch.zeros_like(expect)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        stream = torch.cuda.current_stream()

        def work():
            try:
                with torch.cuda.stream(stream):
                    capi.linear(x, w, out=out)
            except Exception as e:
                failed.append(e)

        thread = threading.Thread(target=work)
        thread.start()
        thread.join()
    assert not failed, failed[0]
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, expect)
