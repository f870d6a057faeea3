"""CPU tests: what the norm, the routing and the draw refuse of the memory they
are given, before any GPU call (no pointer below is ever dereferenced)."""
import ctypes

import pytest

import ft_hip
from test_step_refusals import NORM, ROUTE, SAMPLE

# each refused for the missing context alone
FREE = {"add_rmsnorm": NORM, "route_experts": ROUTE, "sample_tokens": SAMPLE}


def call(name, **change):
    """(code, message) of an entry point with its usual arguments changed."""
    rc = getattr(ft_hip.lib(), "ft_hip_" + name)(*{**FREE[name], **change}.values())
    return rc, ft_hip.lib().ft_hip_last_error().decode()


@pytest.mark.parametrize("name,argument", [
    ("route_experts", a) for a in ("logits", "bias", "expert_scale", "ids", "wts")] + [
    ("sample_tokens", a) for a in ("temperature", "top_k", "top_p", "min_p", "u", "tokens", "logprobs")] + [
    ("add_rmsnorm", a) for a in ("x", "x_w", "residual", "h", "w", "y", "q8")])
@pytest.mark.parametrize("at", [0x1001, 0x1002, 0x1003])
def test_pointers_that_are_not_aligned(name, argument, at):
    rc, msg = call(name, **{argument: ctypes.c_void_p(at)})
    assert rc == ft_hip.E_SHAPE and "aligned" in msg, msg
