"""CPU tests: the calls that moe_synth.RoutedStack and VocabHead make, seen at
a handle that only notes them."""
import contextlib
import types

import pytest
import torch
from torch.utils._python_dispatch import TorchDispatchMode

import ft_hip
import moe_synth

SHAPE = moe_synth.Shape("small-moe", 64, 32, 8, 2, 2, 901)


class NotedHandle:
    """Stands for a Q4Gemv: calls is a list of (method, positional arguments, keyword arguments, noted())."""

    def __init__(self, noted=lambda: None):
        self.calls, self.device, self.noted = [], 0, noted

    def sample_tokens_workspace_bytes(self, vocab, n):
        return 256

    def __getattr__(self, name):
        def method(*args, **kw):
            self.calls.append((name, args, kw, self.noted()))
        return method


def model(g, bias=None):
    """What RoutedStack reads of a SyntheticMoE."""
    s, n_layers = SHAPE, SHAPE.n_layers
    m = types.SimpleNamespace(g=g, shape=s, L=n_layers, device="cpu", layout=ft_hip.LAYOUT_Q4R, expert_bytes=4, gu_bytes=2,
                              banks=torch.zeros(n_layers * s.n_experts * 4, dtype=torch.uint8),
                              routers=torch.zeros((n_layers, s.n_experts, s.hidden)), bias=bias)
    m.layer_bias = lambda l: moe_synth.SyntheticMoE.layer_bias(m, l)
    return m


@pytest.fixture
def streams(monkeypatch):
    """torch's streams as names: streams.current is the one that torch would launch on."""
    now = types.SimpleNamespace(current="device 1's")

    @contextlib.contextmanager
    def stream(s):
        before, now.current = now.current, s
        yield
        now.current = before

    monkeypatch.setattr(torch.cuda, "stream", stream)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda d=None: now.current if d is None else f"device {d}'s")
    return now


@pytest.mark.parametrize("with_bias", [False, True])
def test_router_logits_take_the_models_bias(streams, with_bias):
    g = NotedHandle()
    bias = torch.arange(SHAPE.n_layers * SHAPE.n_experts, dtype=torch.float32).view(SHAPE.n_layers, -1)
    r = moe_synth.RoutedStack(model(g, bias if with_bias else None), 3)
    for l in range(SHAPE.n_layers):
        g.calls.clear()
        r.layer(l, r.branch, None, 3)
        (kw,) = [kw for name, _, kw, _ in g.calls if name == "gemv_f32_rows_dev"]
        given = kw.get("bias")
        assert torch.equal(given, bias[l]) if with_bias else given is None


class Ops(TorchDispatchMode):
    """Notes torch's own operations that write, beside the handle's calls."""

    def __init__(self, g):
        super().__init__()
        self.g = g

    def __torch_dispatch__(self, func, kinds, args=(), kwargs=None):
        if func._schema.is_mutable:
            self.g.calls.append((str(func), args, {}, self.g.noted()))
        return func(*args, **(kwargs or {}))


@pytest.mark.parametrize("given,expected", [("side", "side"), (None, "device 0's")])
@pytest.mark.parametrize("what", ["layer", "run", "head"])
def test_every_launch_is_on_one_stream(streams, what, given, expected):
    """With another stream and another device current, whatever a call launches, torch's clearing of the branch among
    it, is on the given stream, or on that of the handle's device."""
    g = NotedHandle(lambda: streams.current)
    if what == "head":
        w = torch.zeros(16, dtype=torch.uint8)
        head = moe_synth.VocabHead(g, w, None, 100, 64, 3)
        call = lambda: head.run(torch.zeros(3, 64), None, 3, torch.zeros(3), stream=given)  # noqa: E731
    else:
        r = moe_synth.RoutedStack(model(g), 3)
        x = torch.zeros(3, SHAPE.hidden)
        call = (lambda: r.layer(0, x, None, 3, stream=given)) if what == "layer" else lambda: r.run(x, 3, stream=given)
    with Ops(g):
        g.calls.clear()
        call()
    assert len(g.calls) >= 3
    for name, _, kw, current in g.calls:
        on = kw.get("stream") or current  # a call without a stream goes to the current one
        assert on == current == expected, name
    assert streams.current == "device 1's"
