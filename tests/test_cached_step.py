"""CPU tests: the calls that moe_synth.CachedAttention and VocabHead's rules
make, seen at a handle that only notes them."""
import pytest
import torch

import moe_synth
from test_routed_stack import NotedHandle, Ops, streams  # noqa: F401 (a fixture)


class Noted(NotedHandle):
    def kv_page_bytes(self, page, heads, dim):
        return heads * page * (2 * dim + 8)

    def attention_workspace_bytes(self, *_):
        return 256


def attention(g, n_q=1):
    return moe_synth.CachedAttention(g, 4, 2, 64, 6, 16, 3, n_q=n_q, window=9, device="cpu")


@pytest.mark.parametrize("given,expected", [("side", "side"), (None, "device 0's")])
@pytest.mark.parametrize("what", ["attention", "head"])
def test_every_launch_is_on_one_stream(streams, what, given, expected):  # noqa: F811
    g = Noted(lambda: streams.current)
    if what == "head":
        head = moe_synth.VocabHead(g, torch.zeros(16, dtype=torch.uint8), None, 100, 64, 3)
        call = lambda: head.run(torch.zeros(3, 64), None, 3, torch.zeros(3), stream=given, rules=dict(mask=None))  # noqa: E731
    else:
        a, ints = attention(g), torch.zeros((3, 2), dtype=torch.int32)
        call = lambda: a.run(torch.zeros(3, 512), ints[:, 0], ints, ints[:, 0], 3, stream=given)  # noqa: E731
    with Ops(g):
        g.calls.clear()
        call()
    assert [name for name, *_ in g.calls] == (["add_rmsnorm", "gemv_q4r_idx", "adjust_logits", "sample_tokens"]
                                              if what == "head" else ["kv_write", "attention"])
    for name, _, kw, current in g.calls:
        assert (kw.get("stream") or current) == current == expected, name


def test_the_rows_columns_go_where_they_belong(streams):  # noqa: F811
    g = Noted()
    a = attention(g, n_q=2)
    qkv, ints = torch.arange(6 * 512, dtype=torch.float32).view(6, 512), torch.zeros((3, 2), dtype=torch.int32)
    a.run(qkv, ints.view(-1), ints, ints[:, 0], 3)
    (_, w, _, _), (_, t, kw, _) = g.calls
    assert torch.equal(w[0], qkv[:, 256:384]) and torch.equal(w[1], qkv[:, 384:]) and w[4] == 6
    assert torch.equal(t[0], qkv[:, :256]) and t[6] == 3 and kw["n_q"] == 2 and kw["window"] == 9
    assert a.out.shape == (6, 256) and a.cache.shape == (6, 2 * 16 * 136)


def test_without_rules_the_logits_are_drawn_from_as_they_are(streams):  # noqa: F811
    g = Noted()
    head = moe_synth.VocabHead(g, torch.zeros(16, dtype=torch.uint8), None, 100, 64, 3)
    for rules in (None, {}):
        g.calls.clear()
        head.run(torch.zeros(3, 64), None, 3, torch.zeros(3), rules=rules)
        assert "adjust_logits" not in [name for name, *_ in g.calls]
