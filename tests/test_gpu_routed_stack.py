"""moe_synth.RoutedStack beside the layer entry point, on a model whose router
has the Zipf bias and on one without."""
import numpy as np
import pytest
import torch

import ft_hip
import moe_synth
from test_gpu_norm import check_q8, host
from test_gpu_step import SMALL, VOCAB, batch, head_of, settings, stack_of

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("zipf_s", [None, 1.1])
def test_a_layer_routes_as_moe_layer_does(gemv, monkeypatch, zipf_s):
    """Softmax over the top-k asked of route_experts, against ft_hip_moe_layer with its input norm.

    There a logit is (W x) inv, here W (x inv): H products and sums in f32 with one rounding more on either side, so
    the two differ by at most B = (H + 3) 2^-24 sum |W y| (each of the sums' roundings is at most 2^-24 of that sum).
    Rows in which neighbours among the k + 1 largest logits are closer than 2 B may be routed either way and are
    passed over; a weight's logits are off by B each, and it has the roundings of two f32 softmaxes, under 2^-20."""
    monkeypatch.setitem(moe_synth.ZIPF_TAU, (SMALL.name, 1.1), 0.895)
    H, E, K, n = SMALL.hidden, SMALL.n_experts, SMALL.top_k, 24
    m = moe_synth.SyntheticMoE(gemv, SMALL, zipf_s=zipf_s, w_sigma=0.1, r_sigma=0.1)
    assert (m.bias is not None) == (zipf_s is not None)
    r = moe_synth.RoutedStack(m, n)
    ids, wts = torch.zeros((n, K), dtype=torch.int32, device=DEV), torch.zeros((n, K), device=DEV)
    x_out, ws = torch.zeros((n, H), device=DEV), m.workspace(n)
    for l in range(m.L):
        x = batch(n, H, 50 + l)
        r.layer(l, x, None, n)
        gemv.set_input_norm(1)
        try:
            m.layer(l, x, x_out, ids, wts, ws, n)
            torch.cuda.synchronize()
        finally:
            gemv.set_input_norm(0)
        check_q8(r.q8x, host(r.h), None)
        y, w = host(r.y).astype(np.float64), host(m.routers[l]).astype(np.float64)
        B = (H + 3) * 2.0 ** -24 * (np.abs(y) @ np.abs(w).T).max()
        exact = y @ w.T + (0.0 if m.bias is None else host(m.bias[l]).astype(np.float64))
        assert np.max(np.abs(host(r.logits) - exact)) <= B + 2.0 ** -24 * np.abs(exact).max()
        top = -np.sort(-exact, axis=1)[:, :K + 1]
        clear = np.min(top[:, :-1] - top[:, 1:], axis=1) > 2 * B + 2.0 ** -22 * np.abs(exact).max()
        assert clear.sum() >= n // 2
        assert np.array_equal(host(r.ids)[clear], host(ids)[clear])
        off = np.abs(host(r.wts) - host(wts))[clear] / host(wts)[clear]
        assert off.max() <= 4 * B + 2.0 ** -20
        # the experts' sums: a quant of the input and one of the activation may round a half the other way, each by a
        # step of 1/127 of its block's largest: together under 2 %
        branch, layer = host(r.branch)[clear], (host(x_out) - host(x))[clear]
        assert np.max(np.abs(branch - layer)) <= 0.02 * np.abs(layer).max()


def test_two_of_many_experts_carry_a_zipf_model(gemv, monkeypatch):
    """The bias does what it is there for: the popular experts are chosen more often than without it."""
    monkeypatch.setitem(moe_synth.ZIPF_TAU, (SMALL.name, 1.1), 0.895)
    n, share = 64, []
    for zipf_s in (None, 1.1):
        m = moe_synth.SyntheticMoE(gemv, SMALL, zipf_s=zipf_s, w_sigma=0.1, r_sigma=0.1)
        r = moe_synth.RoutedStack(m, n, score=ft_hip.SCORE_SIGMOID)
        r.layer(0, batch(n, SMALL.hidden, 3), None, n)
        popular = moe_synth.zipf_ranks(SMALL, m.L)[0] <= SMALL.top_k
        share.append(popular[host(r.ids)].mean())
    assert share[1] > share[0]


def test_a_step_on_a_stream_that_is_not_current(gemv):
    """All of a step on the given stream, behind what that stream already holds."""
    n, H = 6, SMALL.hidden
    r, head = stack_of(gemv, n), head_of(gemv, H, VOCAB, n)
    x, s = batch(n, H, 70), settings(n, 70)
    want = [t.clone() for t in (*head.run(*r.run(x, n), n, **s), r.branch, r.h)]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for _ in range(3):
        with torch.cuda.stream(side):
            r.branch.fill_(7.0)
            r.h.fill_(7.0)
        tokens, logprobs = head.run(*r.run(x, n, stream=side), n, stream=side, **s)
        side.synchronize()
        assert all(torch.equal(a, b) for a, b in zip((tokens, logprobs, r.branch, r.h), want))
    assert torch.cuda.current_stream() != side


def test_a_step_of_no_sequences(gemv):
    r, head = stack_of(gemv, 2), head_of(gemv, SMALL.hidden, VOCAB, 2)
    none = torch.empty((0, SMALL.hidden), device=DEV)
    before = [t.clone() for t in (r.h, r.ids, head.tokens)]
    tokens, logprobs = head.run(*r.run(none, 0), 0, torch.empty(0, device=DEV))
    torch.cuda.synchronize()
    assert tokens.shape == logprobs.shape == (0,)
    assert all(torch.equal(a.view(torch.int32), t.view(torch.int32)) for a, t in zip(before, (r.h, r.ids, head.tokens)))
