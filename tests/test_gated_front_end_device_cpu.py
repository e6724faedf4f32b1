"""The gated front end on tensors of another GPU than the current one: every call of it has to be made with that GPU current,
the selection too, which launches on the current device whatever stream it is given.  Host side only, with the device faked."""

import contextlib

import torch

from moe_bench_b200 import capi, gating


def test_every_call_is_made_on_the_hidden_states_device(monkeypatch):
    current, seen = [0], {}

    @contextlib.contextmanager
    def device(index):
        before, current[0] = current[0], index
        yield
        current[0] = before

    class Hidden:
        def get_device(self):
            return 1

    def record(name, result):
        def call(*args, **kwargs):
            seen[name] = current[0]
            return result
        return call

    monkeypatch.setattr(capi, "_current_device", lambda: current[0])
    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(capi, "layer_norm", record("norm", ("x", None, None)))
    monkeypatch.setattr(capi, "linear", record("gate", "logits"))
    monkeypatch.setattr(capi, "route_topk", record("selection", ("ids", "weights")))
    assert gating.route_hidden(Hidden(), gating.GateParams(weight=None), 2) == ("x", "ids", "weights")
    assert seen == {"norm": 1, "gate": 1, "selection": 1} and current == [0]
