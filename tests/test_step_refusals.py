"""CPU tests: the operators around the expert section refuse bad arguments
before any GPU call (no pointer below is ever dereferenced)."""
import ctypes

import pytest

import ft_hip

P = ctypes.c_void_p(0x1000)
ODD = ctypes.c_void_p(0x1002)
BIG = 1 << 62


def _err(rc):
    return rc, ft_hip.lib().ft_hip_last_error().decode()


NORM = dict(ctx=None, stream=None, x=P, x_type=0, x_stride=64, x_w=None, residual=P, residual_stride=64, h=P,
            h_stride=64, w=P, eps=1e-6, y=P, y_stride=64, q8=P, hidden=64, n=2)


@pytest.mark.parametrize("change,code,word", [
    (dict(hidden=0), "SHAPE", "hidden"), (dict(hidden=-32), "SHAPE", "hidden"), (dict(hidden=16416), "SHAPE", "hidden"),
    (dict(hidden=48), "SHAPE", "multiple of 32"), (dict(n=-1), "SHAPE", "n="), (dict(n=1 << 22), "SHAPE", "n="),
    (dict(n=BIG), "SHAPE", "n="), (dict(x_type=3), "INVALID", "x_type"), (dict(x_type=-1), "INVALID", "x_type"),
    (dict(eps=-1e-6), "SHAPE", "eps"), (dict(eps=float("nan")), "SHAPE", "eps"),
    (dict(eps=float("inf")), "SHAPE", "eps"), (dict(x_stride=63), "SHAPE", "x_stride"),
    (dict(x_stride=0), "SHAPE", "x_stride"), (dict(x_stride=BIG), "SHAPE", "x_stride"),
    (dict(residual_stride=1), "SHAPE", "residual_stride"), (dict(residual_stride=BIG), "SHAPE", "residual_stride"),
    (dict(h_stride=-64), "SHAPE", "h_stride"), (dict(y_stride=60), "SHAPE", "y_stride"),
    (dict(y_stride=BIG), "SHAPE", "y_stride"),
    (dict(x=ODD), "SHAPE", "aligned"), (dict(q8=ODD), "SHAPE", "aligned"), (dict(h=ODD), "SHAPE", "aligned"),
    (dict(x_type=2, x=ctypes.c_void_p(0x1001)), "SHAPE", "aligned"), (dict(x_type=2, x=ODD), "INVALID", "null"),
    (dict(h=None, y=None, q8=None), "INVALID", "no output|null"), (dict(x=None), "INVALID", "null"),
    (dict(), "INVALID", "null"),  # all right but for the context
])
def test_add_rmsnorm(change, code, word):
    rc, msg = _err(ft_hip.lib().ft_hip_add_rmsnorm(*{**NORM, **change}.values()))
    assert rc == getattr(ft_hip, "E_" + code), msg
    assert any(w in msg for w in word.split("|")), msg


ROUTE = dict(ctx=None, stream=None, logits=P, stride=128, bias=None, expert_scale=None, score=0, n_groups=8,
             top_groups=4, group_rank=2, renorm=1, scale=1.0, ids=P, wts=P, n_experts=128, top_k=8, n_seqs=3)


@pytest.mark.parametrize("change,code,word", [
    (dict(n_experts=0), "SHAPE", "n_experts"), (dict(n_experts=1025), "SHAPE", "n_experts"),
    (dict(n_experts=BIG), "SHAPE", "n_experts"), (dict(n_groups=0), "SHAPE", "n_groups"),
    (dict(n_groups=-1), "SHAPE", "n_groups"), (dict(n_groups=3), "SHAPE", "n_groups"),
    (dict(n_groups=128), "SHAPE", "n_groups"), (dict(top_groups=0), "SHAPE", "top_groups"),
    (dict(top_groups=9), "SHAPE", "top_groups"), (dict(top_k=0), "SHAPE", "top_k"), (dict(top_k=33), "SHAPE", "top_k"),
    (dict(n_groups=32, top_groups=1, top_k=5), "SHAPE", "top_k"), (dict(group_rank=0), "SHAPE", "group_rank"),
    (dict(group_rank=3), "SHAPE", "group_rank"), (dict(score=2), "INVALID", "score"), (dict(renorm=2), "SHAPE", "renorm"),
    (dict(scale=float("inf")), "SHAPE", "scale"), (dict(scale=float("nan")), "SHAPE", "scale"),
    (dict(n_seqs=-1), "SHAPE", "n_seqs"), (dict(n_seqs=BIG), "SHAPE", "n_seqs"), (dict(stride=127), "SHAPE", "stride"),
    (dict(stride=BIG), "SHAPE", "stride"), (dict(ids=None), "INVALID", "null"), (dict(logits=None), "INVALID", "null"),
    (dict(wts=None), "INVALID", "null"), (dict(), "INVALID", "null"),
])
def test_route_experts(change, code, word):
    rc, msg = _err(ft_hip.lib().ft_hip_route_experts(*{**ROUTE, **change}.values()))
    assert rc == getattr(ft_hip, "E_" + code), msg
    assert word in msg, msg


SAMPLE = dict(ctx=None, stream=None, logits=P, logits_type=0, stride=1000, vocab=1000, n=4, temperature=None,
              top_k=None, top_p=None, min_p=None, u=P, tokens=P, logprobs=None, workspace=P, workspace_bytes=1 << 40)


@pytest.mark.parametrize("change,code,word", [
    (dict(vocab=0), "SHAPE", "vocab"), (dict(vocab=(1 << 21) + 1), "SHAPE", "vocab"), (dict(vocab=BIG), "SHAPE", "vocab"),
    (dict(n=-1), "SHAPE", "n="), (dict(n=65536), "SHAPE", "n="), (dict(n=BIG), "SHAPE", "n="),
    (dict(logits_type=3), "INVALID", "logits_type"), (dict(stride=999), "SHAPE", "stride"),
    (dict(stride=BIG), "SHAPE", "stride"), (dict(logits=ODD), "SHAPE", "aligned"),
    (dict(logits_type=1, logits=ctypes.c_void_p(0x1001)), "SHAPE", "aligned"),
    (dict(workspace=ctypes.c_void_p(0x1008)), "SHAPE", "workspace"), (dict(workspace_bytes=0), "SHAPE", "workspace"),
    (dict(u=None), "INVALID", "null"), (dict(tokens=None), "INVALID", "null"), (dict(logits=None), "INVALID", "null"),
    (dict(workspace=None), "INVALID", "null"), (dict(), "INVALID", "null"),
])
def test_sample_tokens(change, code, word):
    rc, msg = _err(ft_hip.lib().ft_hip_sample_tokens(*{**SAMPLE, **change}.values()))
    assert rc == getattr(ft_hip, "E_" + code), msg
    assert word in msg, msg


def test_sample_tokens_workspace():
    f = ft_hip.lib().ft_hip_sample_tokens_workspace_bytes
    assert f(0, 1) == f(1, -1) == f((1 << 21) + 1, 1) == f(1, 65536) == 0
    assert 0 < f(1, 1) <= f(262144, 1) <= f(262144, 256) <= f(1 << 21, 65535)
    rc, msg = _err(ft_hip.lib().ft_hip_sample_tokens(*{**SAMPLE, "workspace_bytes": f(1000, 4) - 1}.values()))
    assert rc == ft_hip.E_SHAPE and "needed" in msg
