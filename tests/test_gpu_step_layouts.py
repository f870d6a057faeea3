"""The norm, the routing and the draw on rows inside tensors of three
dimensions, padded as a head or a router leaves them: the same bits as on rows
one after the other, and what lies between the rows stays as it was."""
import numpy as np
import pytest
import torch

import ft_hip

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def rows(n, width, seed, scale=1.0):
    return torch.from_numpy((scale * np.random.default_rng(seed).standard_normal((n, width))).astype(np.float32)).to(DEV)


def padded(a, pad, shape=None, dtype=torch.float32):
    """a [n, width] inside [n, 1, width + pad] (seen as `shape`), 60 in between."""
    n, width = a.shape
    t = torch.full((n, 1, width + pad), 60.0, dtype=dtype, device=DEV)
    t[:, 0, :width] = a
    return t if shape is None else t.view(shape)


@pytest.mark.parametrize("pad", [0, 1, 64])
@pytest.mark.parametrize("n", [1, 3])
def test_draw(gemv, n, pad):
    for V, dtype in ((9000, torch.float32), (700, torch.bfloat16)):
        l = rows(n, V, V + n, 3.0)
        u = torch.linspace(0.1, 0.9, n, device=DEV)
        ws = torch.empty(gemv.sample_tokens_workspace_bytes(V, n), dtype=torch.uint8, device=DEV)
        got = []
        for logits in (l.to(dtype), padded(l, pad, dtype=dtype), padded(l, pad, (1, n, V + pad), dtype)):
            tokens, lp = torch.zeros(n, dtype=torch.int32, device=DEV), torch.zeros(n, device=DEV)
            gemv.sample_tokens(logits, V, n, u, tokens, ws, logprobs=lp)
            got.append((tokens, lp))
        torch.cuda.synchronize()
        for tokens, lp in got[1:]:
            assert torch.equal(tokens, got[0][0]) and torch.equal(lp, got[0][1])


@pytest.mark.parametrize("pad", [0, 1, 64])
def test_routing(gemv, pad):
    n, E = 5, 96
    l = rows(n, E, pad)
    got = []
    for logits in (l, padded(l, pad), padded(l, pad, (n, 1, 1, E + pad))):
        ids, wts = torch.zeros((n, 6), dtype=torch.int32, device=DEV), torch.zeros((n, 6), device=DEV)
        gemv.route_experts(logits, ids, wts, E, 6, n, score=ft_hip.SCORE_SIGMOID)
        got.append((ids, wts))
    torch.cuda.synchronize()
    for ids, wts in got[1:]:
        assert torch.equal(ids, got[0][0]) and torch.equal(wts, got[0][1])


@pytest.mark.parametrize("pad", [0, 1, 64])
def test_norm(gemv, pad):
    n, H = 4, 320
    x, r, w = rows(n, H, 1), rows(n, H, 2), rows(1, H, 3)[0]
    h, y, q8 = torch.zeros((n, H), device=DEV), torch.zeros((n, H), device=DEV), torch.zeros(n * 400, dtype=torch.uint8,
                                                                                             device=DEV)
    gemv.add_rmsnorm(x, w, H, n, 1e-6, residual=r, h=h, y=y, q8=q8)
    xp, rp, hp, yp = (padded(a, pad) for a in (x, r, r, r))
    qp = torch.zeros_like(q8)
    gemv.add_rmsnorm(xp, w, H, n, 1e-6, residual=rp, h=hp, y=yp, q8=qp)
    torch.cuda.synchronize()
    assert torch.equal(hp[:, 0, :H], h) and torch.equal(yp[:, 0, :H], y) and torch.equal(qp, q8)
    for t in (hp, yp):
        assert bool((t[:, 0, H:] == 60.0).all())


def test_norm_of_heads(gemv):
    """A branch as attention leaves it, [rows, heads, values]: a row is all of its heads."""
    n, H = 3, 256
    x = rows(n, H, 5)
    y, yh = torch.zeros((n, H), device=DEV), torch.zeros((n, 4, 64), device=DEV)
    gemv.add_rmsnorm(x, None, H, n, 1e-6, y=y)
    gemv.add_rmsnorm(x.view(n, 4, 64), None, H, n, 1e-6, y=yh)
    torch.cuda.synchronize()
    assert torch.equal(yh.view(n, H), y)


def test_norm_of_rows_side_by_side(gemv):
    """x, residual, h and y as columns of one buffer, and with strides of their own in one: no row overlaps another."""
    n, H = 5, 64
    x, r, w = rows(n, H, 7), rows(n, H, 8), rows(1, H, 9)[0]
    h, y, q8 = torch.zeros((n, H), device=DEV), torch.zeros((n, H), device=DEV), torch.zeros(n * 80, dtype=torch.uint8,
                                                                                             device=DEV)
    gemv.add_rmsnorm(x, w, H, n, 1e-6, residual=r, h=h, y=y, q8=q8)
    one = torch.zeros((n, 4 * H), device=DEV)
    xs, rs, hs, ys = (one[:, i * H:(i + 1) * H] for i in range(4))
    xs.copy_(x)
    rs.copy_(r)
    qs = torch.zeros_like(q8)
    gemv.add_rmsnorm(xs, w, H, n, 1e-6, residual=rs, h=hs, y=ys, q8=qs)
    torch.cuda.synchronize()
    assert torch.equal(hs, h) and torch.equal(ys, y) and torch.equal(qs, q8)
    assert torch.equal(xs, x) and torch.equal(rs, r)
    # x in steps of 3 H from 0, h in steps of 6 H from H: never the same place
    one = torch.zeros(2 * 3 * H * n, device=DEV)
    xs, hs = one.as_strided((n, H), (3 * H, 1)), one.as_strided((n, H), (6 * H, 1), H)
    xs.copy_(x)
    gemv.add_rmsnorm(xs, w, H, n, 1e-6, residual=r, h=hs)
    torch.cuda.synchronize()
    assert torch.equal(hs, h) and torch.equal(xs, x)
    # h on the residual and y on x, with q8: rows on rows
    xi, ri, qi = x.clone(), r.clone(), torch.zeros_like(q8)
    gemv.add_rmsnorm(xi, w, H, n, 1e-6, residual=ri, h=ri, y=xi, q8=qi)
    torch.cuda.synchronize()
    assert torch.equal(ri, h) and torch.equal(xi, y) and torch.equal(qi, q8)


@pytest.mark.parametrize("V", [700, 20000])
def test_draw_into_the_settings_arrays(gemv, V):
    """tokens over top_k and logprobs over the random numbers: as into arrays of their own."""
    n = 40
    l, ws = rows(n, V, V, 3.0), torch.empty(gemv.sample_tokens_workspace_bytes(V, n), dtype=torch.uint8, device=DEV)
    u, k = torch.linspace(0, 0.99, n, device=DEV), torch.arange(n, dtype=torch.int32, device=DEV) * 3
    t = torch.linspace(0, 2, n, device=DEV)
    tokens, lp = torch.zeros(n, dtype=torch.int32, device=DEV), torch.zeros(n, device=DEV)
    gemv.sample_tokens(l, V, n, u, tokens, ws, temperature=t, top_k=k, logprobs=lp)
    gemv.sample_tokens(l, V, n, u, k, ws, temperature=t, top_k=k, logprobs=u)
    torch.cuda.synchronize()
    assert torch.equal(k, tokens) and torch.equal(u, lp)


def test_routing_into_the_gaps_between_rows(gemv):
    """ids and weights where padded rows of logits leave room: no row is touched."""
    E, k = 64, 4
    one = torch.full((2, 256), 60.0, device=DEV)
    one[:, :E] = rows(2, E, 2)
    before = one[:, :E].clone()
    ids, wts = one[0, 128:128 + 2 * k].view(torch.int32), one[0, 200:200 + 2 * k]
    want = torch.zeros((2, k), dtype=torch.int32, device=DEV), torch.zeros((2, k), device=DEV)
    gemv.route_experts(one[:, :E].contiguous(), *want, E, k, 2)
    gemv.route_experts(one[:, :E], ids, wts, E, k, 2)
    torch.cuda.synchronize()
    assert torch.equal(ids.view(2, k), want[0]) and torch.equal(wts.view(2, k), want[1])
    assert torch.equal(one[:, :E], before)


def test_an_empty_batch(gemv):
    """Tensors without rows, as slices of a batch of none: nothing is done, nothing refused."""
    f, i = torch.empty((0, 64), device=DEV), torch.empty((0, 4), dtype=torch.int32, device=DEV)
    gemv.add_rmsnorm(f, None, 64, 0, 1e-6, residual=f, h=torch.empty_like(f), y=torch.empty_like(f),
                     q8=torch.empty(0, dtype=torch.uint8, device=DEV))
    gemv.add_rmsnorm(torch.empty((0, 1, 72), dtype=torch.float16, device=DEV), None, 64, 0, 1e-6, h=f)
    gemv.route_experts(f, i, f[:, :4].contiguous(), 64, 4, 0)
    for V in (64, 9000):
        ws = torch.empty(gemv.sample_tokens_workspace_bytes(V, 0), dtype=torch.uint8, device=DEV)
        none = torch.empty(0, device=DEV)
        gemv.sample_tokens(torch.empty((0, V), device=DEV), V, 0, none, none.int(), ws, temperature=none, logprobs=none)
    torch.cuda.synchronize()
