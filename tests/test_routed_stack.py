"""CPU tests: the calls that moe_synth.RoutedStack and VocabHead make, seen at
a handle that only notes them."""
import types

import pytest
import torch

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


@pytest.mark.parametrize("with_bias", [False, True])
def test_router_logits_take_the_models_bias(with_bias):
    g = NotedHandle()
    bias = torch.arange(SHAPE.n_layers * SHAPE.n_experts, dtype=torch.float32).view(SHAPE.n_layers, -1)
    r = moe_synth.RoutedStack(model(g, bias if with_bias else None), 3)
    for l in range(SHAPE.n_layers):
        g.calls.clear()
        r.layer(l, r.branch, None, 3)
        (kw,) = [kw for name, _, kw, _ in g.calls if name == "gemv_f32_rows_dev"]
        given = kw.get("bias")
        assert torch.equal(given, bias[l]) if with_bias else given is None
