"""CPU tests: what the norm, the routing and the draw refuse of the memory they
are given, before any GPU call (no pointer below is ever dereferenced)."""
import ctypes
import os
import subprocess

import numpy as np
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


@pytest.fixture(scope="module")
def overlap():
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    subprocess.run(["make", "-s", "-C", os.path.join(root, "oracle")], check=True)
    f = ctypes.CDLL(os.path.join(root, "oracle", "_build", "liboverlapcheck.so")).oc_overlap
    f.argtypes = [ctypes.c_uint64, ctypes.c_int64, ctypes.c_int64, ctypes.c_int64] * 2
    return f


def test_rows_that_overlap(overlap):
    """Against the bytes themselves, for rows of the same and of other strides, side by side and interleaved."""
    rng = np.random.default_rng(4)
    met = [0, 0]
    for i in range(20000):
        spans = []
        for _ in "ab":
            n, size = int(rng.integers(1, 7)), int(rng.integers(1, 9))
            spans.append([int(rng.integers(100, 140)), n, size + int(rng.integers(0, 12)), size])
        if i % 2:
            spans[1][2] = max(spans[0][2], spans[1][3])
            spans[0][2] = max(spans[1][2], spans[0][3])
        sets = [{at + r * stride + j for r in range(n) for j in range(size)} for at, n, stride, size in spans]
        want = bool(sets[0] & sets[1])
        assert overlap(*spans[0], *spans[1]) == overlap(*spans[1], *spans[0]) == want, spans
        met[want] += 1
    assert min(met) > 3000


def test_rows_that_overlap_far_apart(overlap):
    """Strides and addresses at the limits of what the entry points take."""
    top, far = (1 << 57) - 4096, (1 << 63) // 8
    assert not overlap(0, 2, 8, 8, 4096, 2, 8, 8)  # no pointer: no rows
    assert not overlap(4096, 0, 8, 8, 4096, 1, 8, 8) and not overlap(4096, 1, 8, 8, 4096, 1, 8, 0)
    assert overlap(top, 2, far, 64, top, 1, 64, 64) and not overlap(top, 2, far, 64, top + 64, 1, 64, 64)
    assert overlap(top, 2, far, 64, top + far + 63, 1, 64, 1) and not overlap(top, 2, far, 64, top + far + 64, 1, 64, 1)
    assert not overlap(top, 4194303, 1 << 39, 64, top + 64, 4194303, 1 << 39, (1 << 39) - 64)
    assert overlap(top, 4194303, 1 << 39, 64, top + 64, 4194303, 1 << 39, (1 << 39) - 63)


ROOM = ctypes.create_string_buffer(4096)  # stands for a context, which no refused call reads
CTX = ctypes.cast(ROOM, ctypes.c_void_p)

# x, residual, h, y: 2 rows of 64 f32 (256 bytes) a KiB apart in one buffer, weights and blocks (160 bytes) behind it
LAID = dict(NORM, ctx=CTX, x=ctypes.c_void_p(0x10000), residual=ctypes.c_void_p(0x10100),
            h=ctypes.c_void_p(0x10200), y=ctypes.c_void_p(0x10300), x_stride=256, residual_stride=256, h_stride=256,
            y_stride=256, w=ctypes.c_void_p(0x20000), x_w=ctypes.c_void_p(0x20100), q8=ctypes.c_void_p(0x20200))


@pytest.mark.parametrize("change", [
    dict(h=0x10004), dict(h=0x100fc), dict(h=0x10104), dict(h=0x10500), dict(y=0x10504), dict(h=0x10304),
    dict(y=0x10204), dict(h=0x10300), dict(y=0x20004), dict(h=0x200fc), dict(y=0x20100), dict(h=0x20204),
    dict(h=0x10000, h_stride=64), dict(y=0x10100, y_stride=128), dict(h=0x10000, x_type=1), dict(y=0x10040, x_type=2),
    dict(q8=0x10040), dict(q8=0x10440), dict(q8=0x10300), dict(q8=0x2009c), dict(q8=0x20180), dict(q8=0x10000),
    dict(w=0x10300), dict(x_w=0x10200), dict(n=1, y=0x10080), dict(n=1, h=0x101fc),
])
def test_add_rmsnorm_refuses_outputs_that_overlap(change):
    """Every case is refused before any GPU call."""
    change = {k: ctypes.c_void_p(v) if k in ("x", "residual", "h", "y", "w", "x_w", "q8") else v
              for k, v in change.items()}
    rc = ft_hip.lib().ft_hip_add_rmsnorm(*{**LAID, **change}.values())
    msg = ft_hip.lib().ft_hip_last_error().decode()
    assert rc == ft_hip.E_SHAPE and "overlap" in msg, msg


def refused(name, usual, change):
    """Message of a call that has to be refused as a bad shape; whole numbers in place of pointers."""
    now = {k: ctypes.c_void_p(v) if isinstance(usual[k], ctypes.c_void_p) and isinstance(v, int) else v
           for k, v in {**usual, **change}.items()}
    rc = getattr(ft_hip.lib(), "ft_hip_" + name)(*now.values())
    msg = ft_hip.lib().ft_hip_last_error().decode()
    assert rc == ft_hip.E_SHAPE, msg
    return msg


# 3 rows of 128 f32 (512 bytes) a KiB apart; ids and weights of 3 x 8 (96 bytes)
ROUTED = dict(ROUTE, ctx=CTX, logits=ctypes.c_void_p(0x10000), stride=256, bias=ctypes.c_void_p(0x20000),
              expert_scale=ctypes.c_void_p(0x20200), ids=ctypes.c_void_p(0x20400), wts=ctypes.c_void_p(0x20460))


@pytest.mark.parametrize("change", [
    dict(ids=0x10000), dict(wts=0x10000), dict(ids=0x101fc), dict(wts=0x103a4), dict(ids=0x109fc), dict(ids=0x20000),
    dict(wts=0x201fc), dict(ids=0x203fc), dict(wts=0x201a4), dict(wts=0x20400), dict(wts=0x2045c), dict(ids=0x204bc),
])
def test_route_experts_refuses_outputs_that_overlap(change):
    assert "overlap" in refused("route_experts", ROUTED, change)


# 4 rows of 9000 logits (f32) 9216 apart, settings and outputs of 16 bytes each, the workspace behind
SAMPLED = dict(SAMPLE, ctx=CTX, logits=ctypes.c_void_p(0x100000), stride=9216, vocab=9000,
               temperature=ctypes.c_void_p(0x200000), top_k=ctypes.c_void_p(0x200010), top_p=ctypes.c_void_p(0x200020),
               min_p=ctypes.c_void_p(0x200030), u=ctypes.c_void_p(0x200040), tokens=ctypes.c_void_p(0x200050),
               logprobs=ctypes.c_void_p(0x200060), workspace=ctypes.c_void_p(0x300000))


@pytest.mark.parametrize("change", [
    dict(tokens=0x100000), dict(logprobs=0x108c9c), dict(tokens=0x109000 - 0x4), dict(logprobs=0x200050),
    dict(logprobs=0x200044, u=0x200080), dict(logprobs=0x20005c), dict(workspace=0x100000), dict(workspace=0x108c90),
    dict(workspace=0x200000), dict(workspace=0x1ffff0), dict(workspace=0x200040), dict(workspace=0x200050),
    dict(workspace=0x200060), dict(tokens=0x200004), dict(tokens=0x200014), dict(logprobs=0x20001c),
    dict(logprobs=0x200024), dict(tokens=0x200034), dict(tokens=0x20003c), dict(logprobs=0x200044),
])
def test_sample_tokens_refuses_memory_that_overlaps(change):
    assert "overlap" in refused("sample_tokens", SAMPLED, change)


@pytest.mark.parametrize("name,change", [
    ("add_rmsnorm", dict(x=None, residual=None, h=None, y=None, q8=None, n=0)), ("add_rmsnorm", dict(n=0)),
    ("route_experts", dict(logits=None, ids=None, wts=None, n_seqs=0)), ("route_experts", dict(n_seqs=0)),
    ("sample_tokens", dict(logits=None, u=None, tokens=None, workspace=None, n=0)), ("sample_tokens", dict(n=0)),
])
def test_no_rows(name, change):
    """Nothing to do, also where an empty batch has no address; what is wrong of a shape or a handle stays refused."""
    rc, msg = call(name, ctx=CTX, **change)
    assert rc == ft_hip.OK, msg
    rc, msg = call(name, **change)
    assert rc == ft_hip.E_INVALID and "null" in msg, msg
    bad = dict(add_rmsnorm=dict(hidden=0), route_experts=dict(top_k=0), sample_tokens=dict(vocab=0))[name]
    assert call(name, ctx=CTX, **{**change, **bad})[0] == ft_hip.E_SHAPE
