"""CPU tests: what the Python methods of the norm, the routing and the draw
make of their tensors, seen at a library that only notes its arguments.

The handle's device is -1, which is what a tensor on the CPU names as its own.
"""
import types

import pytest
import torch

import ft_hip

STREAM = types.SimpleNamespace(cuda_stream=0)


class Noted:
    """Stands for the library: calls maps an entry point to its last arguments."""

    def __init__(self):
        self.calls = {}

    def __getattr__(self, name):
        def entry(*args):
            self.calls[name] = args
            return ft_hip.OK
        return entry


@pytest.fixture
def noted(monkeypatch):
    noted = Noted()
    monkeypatch.setattr(ft_hip, "lib", lambda: noted)
    g = ft_hip.Q4Gemv.__new__(ft_hip.Q4Gemv)
    g._ctx, g.device = None, -1
    return g, noted.calls


def norm(g, calls, x, hidden, n, **kw):
    """(x_stride, residual_stride, h_stride, y_stride) of a call."""
    g.add_rmsnorm(x, None, hidden, n, 1e-6, stream=STREAM, **kw)
    a = calls["ft_hip_add_rmsnorm"]
    return a[4], a[7], a[9], a[13]


def route(g, calls, logits, n_experts, n):
    ids, wts = torch.zeros((n, 2), dtype=torch.int32), torch.zeros((n, 2))
    g.route_experts(logits, ids, wts, n_experts, 2, n, stream=STREAM)
    return calls["ft_hip_route_experts"][3]


def sample(g, calls, logits, vocab, n, workspace=None):
    u, tokens = torch.zeros(n), torch.zeros(n, dtype=torch.int32)
    ws = torch.zeros(1 << 10, dtype=torch.uint8) if workspace is None else workspace
    g.sample_tokens(logits, vocab, n, u, tokens, ws, stream=STREAM)
    return calls["ft_hip_sample_tokens"][4]


LAYOUTS = [  # shape, rows, width, stride
    ((3, 64), 3, 64, 64), ((3, 72), 3, 64, 72), ((192,), 3, 64, 64), ((200,), 3, 64, 64),
    ((3, 1, 64), 3, 64, 64), ((3, 1, 72), 3, 64, 72), ((1, 3, 72), 3, 64, 72), ((2, 3, 72), 5, 64, 72),
    ((3, 4, 16), 3, 64, 64), ((3, 5, 16), 3, 64, 80), ((1, 3, 4, 16), 3, 64, 64), ((3, 1, 1, 65), 3, 64, 65),
    ((1, 1, 72), 1, 64, 72), ((3, 1, 128), 3, 64, 128), ((6, 1, 32), 3, 64, 64),
]


@pytest.mark.parametrize("shape,n,width,stride", LAYOUTS)
def test_the_row_stride_is_the_tensors(noted, shape, n, width, stride):
    """The same for each operator and each of the norm's tensors: a padded row is as long as it is stored."""
    t = torch.zeros(shape)
    assert norm(*noted, t, width, n, residual=t, h=torch.zeros(shape), y=torch.zeros(shape)) == (stride,) * 4
    assert route(*noted, t, width, n) == stride
    assert sample(*noted, t, width, n) == stride
    assert sample(*noted, t.half(), width, n) == stride


@pytest.mark.parametrize("shape,n,width", [
    ((3, 1, 63), 3, 64), ((2, 1, 72), 3, 64), ((3, 5, 16), 4, 64), ((6, 1, 32), 2, 64), ((2, 2, 2), 1, 64),
    ((7, 1, 32), 3, 64), ((191,), 3, 64), ((3, 63), 3, 64),
])
def test_rows_that_a_tensor_does_not_hold_are_refused(noted, shape, n, width):
    t, whole = torch.zeros(shape), torch.zeros(n, width)
    for call in (lambda: norm(*noted, t, width, n, h=whole), lambda: norm(*noted, whole, width, n, residual=t, h=whole),
                 lambda: norm(*noted, whole, width, n, h=t), lambda: norm(*noted, whole, width, n, y=t),
                 lambda: route(*noted, t, width, n), lambda: sample(*noted, t, width, n)):
        with pytest.raises(ft_hip.FtHipError) as e:
            call()
        assert e.value.code == ft_hip.E_SHAPE


def test_views_of_more_dimensions_that_are_not_contiguous_are_refused(noted):
    t = torch.zeros(3, 1, 72)[:, :, :64]
    for call in (norm, route, sample):
        with pytest.raises(ft_hip.FtHipError):
            call(*noted, t, 64, 3)


def test_a_workspace_with_gaps_is_refused(noted):
    """Its count says nothing of the memory behind it: bytes between would be overwritten, or bytes past its end."""
    logits = torch.zeros(2, 9000)
    for ws in (torch.zeros(1 << 11, dtype=torch.uint8)[::2], torch.zeros(1, dtype=torch.uint8).expand(1 << 20),
               torch.zeros((8, 64), dtype=torch.uint8).t(), torch.zeros((4, 64), dtype=torch.uint8)[:, :32]):
        with pytest.raises(ft_hip.FtHipError, match="workspace") as e:
            sample(*noted, logits, 9000, 2, ws)
        assert e.value.code == ft_hip.E_SHAPE
    sample(*noted, logits, 9000, 2, torch.zeros((8, 64), dtype=torch.uint8)[4:])  # a run of rows has none
    assert noted[1]["ft_hip_sample_tokens"][15] == 4 * 64
