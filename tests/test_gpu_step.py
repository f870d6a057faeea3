"""The operators around the expert section together, as a decode step runs
them: moe_synth.RoutedStack (norm with q8, router, route_experts, the experts'
GEMVs, per layer) and moe_synth.VocabHead (norm with q8, head GEMV, draw).

Every stage is checked from what the stage before it left, with the checks of
the operators' own tests; a captured step has to repeat the eager one's bits on
new inputs, and a smaller batch on the same buffers those of a stack of its own.
"""
import numpy as np
import pytest
import torch

import ft_hip
import moe_synth
from test_gpu_norm import blocks, check_q8, check_y, host
from test_gpu_route import SUB, WT, reference as route_reference
from test_gpu_sample import reference as draw_reference

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
SMALL = moe_synth.Shape("small-moe", 256, 64, 16, 4, 2, 901)
VOCAB = 9000
ROUTE = dict(score=ft_hip.SCORE_SIGMOID, n_groups=4, top_groups=2, group_rank=2, renorm=True, scale=2.5)


def head_of(gemv, hidden, vocab, max_seqs, seed=3):
    rb = ft_hip.row_bytes(hidden, ft_hip.LAYOUT_Q4R)
    w = torch.empty(vocab * rb, dtype=torch.uint8, device=DEV)
    gemv.gen_q4_rows(moe_synth.tensor_key(902, 0, seed, 1), 0, vocab, hidden, moe_synth.gen_scale(0.2), w,
                     ft_hip.LAYOUT_Q4R)
    norm = torch.from_numpy((1 + 0.2 * np.random.default_rng(seed).standard_normal(hidden)).astype(np.float32)).to(DEV)
    return moe_synth.VocabHead(gemv, w, norm, vocab, hidden, max_seqs)


def settings(n, seed):
    rng = np.random.default_rng(seed)
    f = lambda v: torch.tensor(np.asarray(v, np.float32), device=DEV)  # noqa: E731
    return dict(u=f(rng.random(n)), temperature=f(rng.uniform(0.5, 1.5, n)), top_p=f(rng.uniform(0.5, 1.2, n)),
                top_k=torch.tensor(rng.integers(0, 80, n).astype(np.int32), device=DEV), min_p=f(rng.uniform(-0.05, 0.05, n)))


def stack_of(gemv, max_seqs, shape=SMALL, **more):
    m = moe_synth.SyntheticMoE(gemv, shape, w_sigma=0.1, r_sigma=0.1)
    rng = np.random.default_rng(17)
    bias = torch.from_numpy((0.1 * rng.standard_normal(shape.n_experts)).astype(np.float32)).to(DEV)
    norm = torch.from_numpy((1 + 0.2 * rng.standard_normal((m.L, shape.hidden))).astype(np.float32)).to(DEV)
    return moe_synth.RoutedStack(m, max_seqs, norm, **{**ROUTE, "bias": bias, **more})


def batch(n, hidden, seed):
    return torch.from_numpy(np.random.default_rng(seed).standard_normal((n, hidden)).astype(np.float32)).to(DEV)


@pytest.mark.parametrize("n", [1, 3, 17])
def test_every_stage_from_the_one_before(gemv, n):
    r, head = stack_of(gemv, n), head_of(gemv, SMALL.hidden, VOCAB, n)
    x = batch(n, SMALL.hidden, n)
    residual, branch = None, x
    for l in range(r.m.L):
        before = None if residual is None else host(residual).copy()
        add = host(branch).copy()
        r.layer(l, branch, residual, n)
        h, w = host(r.h), host(r.norm_w[l])
        assert np.array_equal(h, add if before is None else before + add)
        check_y(host(r.y), h, w)
        check_q8(r.q8x, h, w)
        logits = host(r.logits)
        want = host(r.y).astype(np.float64) @ host(r.m.routers[l]).astype(np.float64).T
        assert np.max(np.abs(logits - want)) <= 1e-5 * np.abs(want).max()
        ids, wts = route_reference(logits, SMALL.top_k, ROUTE["score"], bias=host(r.route["bias"]), G=4, tg=2, rank=2,
                                   scale=2.5)
        assert np.array_equal(host(r.ids), ids)
        assert np.all(np.abs(host(r.wts) - wts) <= WT * wts + SUB)
        # the weighted sum of the chosen experts' rows
        total = (host(r.down).reshape(n, SMALL.top_k, -1).astype(np.float64) * host(r.wts)[:, :, None]).sum(1)
        scale = (np.abs(host(r.down)).reshape(n, SMALL.top_k, -1) * host(r.wts)[:, :, None]).sum(1)
        assert np.all(np.abs(host(r.branch) - total) <= 2.0 ** -21 * scale + 1e-30)  # 4 products and 4 sums in f32
        residual, branch = r.h, r.branch
    s = settings(n, n)
    tokens, logprobs = head.run(branch, residual, n, **s)
    check_q8(head.q8, host(residual) + host(branch), host(head.norm_w))
    logits = host(head.logits).astype(np.float64)
    for i in range(n):
        want, lp = draw_reference(logits[i], float(s["temperature"][i]), int(s["top_k"][i]), float(s["top_p"][i]),
                                  float(s["min_p"][i]), float(s["u"][i]))
        assert int(tokens[i]) == want
        assert abs(float(logprobs[i]) - lp) <= 2.0 ** -24 * abs(lp) * (1 + 1e-6) + 1e-12


def test_the_head_reads_the_q8_that_the_norm_wrote(gemv):
    """Logits of the chain against the dequantized blocks and rows in 64 bits (f32 sums of 8 blocks: 1e-6)."""
    n, H = 5, SMALL.hidden
    head = head_of(gemv, H, VOCAB, n)
    head.run(batch(n, H, 8), batch(n, H, 9), n, settings(n, 2)["u"])
    d, _, qs = blocks(head.q8, n, H)
    xq = (d[:, :, None].astype(np.float64) * qs).reshape(n, H)
    raw = host(head.weights).reshape(VOCAB, -1)
    scales = raw[:, :2 * (H // 32)].copy().view(np.float16).astype(np.float64)
    q = raw[:, ft_hip.q4r_scales_bytes(H):].reshape(VOCAB, H // 32, 16).astype(int)
    w = (np.concatenate([q & 15, q >> 4], 2) - 8) * scales[:, :, None]
    want = xq @ w.reshape(VOCAB, H).T
    assert np.max(np.abs(host(head.logits) - want)) <= 1e-6 * np.abs(xq).max() * np.abs(w).max() * H


def test_captured_step_repeats_the_eager_one(gemv):
    n, H = 9, SMALL.hidden
    r, head = stack_of(gemv, n), head_of(gemv, H, VOCAB, n)
    x, s = batch(n, H, 0), settings(n, 0)

    def step():
        return head.run(*r.run(x, n), n, **s)

    step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        captured = step()
    for seed in range(1, 5):
        x.copy_(batch(n, H, seed))
        for name, v in settings(n, seed).items():
            s[name].copy_(v)
        g.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in captured] + [r.h.clone(), head.logits.clone()]
        want = [t.clone() for t in step()] + [r.h.clone(), head.logits.clone()]
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), seed


def test_smaller_batch_on_the_same_buffers(gemv):
    """A batch that shrinks between steps: what a stack of its own size gives, and the rows behind it stay."""
    H = SMALL.hidden
    r, head = stack_of(gemv, 12), head_of(gemv, H, VOCAB, 12)
    head.run(*r.run(batch(12, H, 1), 12), 12, **settings(12, 1))
    torch.cuda.synchronize()
    for n in (5, 1):
        keep = [t[n:].clone() for t in (r.h, r.ids, head.logits, head.tokens)]
        x, s = batch(n, H, 40 + n), settings(n, 40 + n)
        got = [t.clone() for t in head.run(*r.run(x, n), n, **s)]
        r2, head2 = stack_of(gemv, n), head_of(gemv, H, VOCAB, n)
        want = head2.run(*r2.run(x, n), n, **s)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        assert all(torch.equal(a, t[n:]) for a, t in zip(keep, (r.h, r.ids, head.logits, head.tokens)))


def test_two_steps_on_two_streams(gemv):
    """Two batches at once, each with its own buffers and workspace, as one after the other."""
    H = SMALL.hidden
    parts = [(stack_of(gemv, 6), head_of(gemv, H, VOCAB, 6), batch(6, H, 60 + i), settings(6, 60 + i)) for i in range(2)]
    want = []
    for r, head, x, s in parts:
        want.append([t.clone() for t in head.run(*r.run(x, 6), 6, **s)])
        torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in parts]
    for _ in range(3):
        for st, (r, head, x, s) in zip(streams, parts):
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                head.run(*r.run(x, 6), 6, **s)
    torch.cuda.synchronize()
    for (r, head, x, s), w in zip(parts, want):
        assert torch.equal(head.tokens, w[0]) and torch.equal(head.logprobs, w[1])


def test_routing_of_the_layer_entry_point(gemv):
    """With softmax over the top-k asked of route_experts, a layer's choice is moe_layer's on the same normed input
    (its router: W x * inv; here W (x * inv): the choice may only differ where logits are within rounding)."""
    shape = SMALL
    r = stack_of(gemv, 8, score=ft_hip.SCORE_SOFTMAX, n_groups=1, top_groups=1, group_rank=1, scale=1.0, bias=None)
    r.norm_w = None
    x = batch(8, shape.hidden, 77)
    r.layer(0, x, None, 8)
    ids, wts = torch.zeros((8, shape.top_k), dtype=torch.int32, device=DEV), torch.zeros((8, shape.top_k), device=DEV)
    gemv.topk_router_dev(r.logits, None, ids, wts, shape.n_experts, shape.top_k, 8)
    assert torch.equal(ids, r.ids)
    assert float(((wts - r.wts).abs() / wts).max()) < 2.0 ** -20
    assert np.array_equal(blocks(r.q8x, 8, shape.hidden)[2].shape, (8, shape.hidden // 32, 32))


def far(n, width, stride, dtype):
    """n rows of width values, `stride` values apart, in a buffer that is nothing else."""
    return torch.empty((n - 1) * stride + width, dtype=dtype, device=DEV).as_strided((n, width), (stride, 1))


def test_rows_further_apart_than_32_bits(gemv):
    """Row offsets past 2^32 bytes and 2^31 values: as on rows one after the other."""
    rng = np.random.default_rng(5)
    H, E, V = 320, 64, 9000
    x, w = batch(2, H, 1).half(), batch(1, H, 2)[0]
    xf, yf = far(2, H, (1 << 31) + 8, torch.float16), far(2, H, (1 << 30) + 64, torch.float32)
    xf.copy_(x)
    y, q8, q8f = torch.empty((2, H), device=DEV), *(torch.zeros(2 * 400, dtype=torch.uint8, device=DEV) for _ in "ab")
    gemv.add_rmsnorm(x, w, H, 2, 1e-6, y=y, q8=q8)
    gemv.add_rmsnorm(xf, w, H, 2, 1e-6, y=yf, q8=q8f)
    assert torch.equal(y, yf) and torch.equal(q8, q8f)
    del xf, yf
    l = batch(3, E, 3)
    lf = far(3, E, (1 << 30) + 4, torch.float32)
    lf.copy_(l)
    out = [(torch.zeros((3, 4), dtype=torch.int32, device=DEV), torch.zeros((3, 4), device=DEV)) for _ in "ab"]
    for logits, (ids, wts) in zip((l, lf), out):
        gemv.route_experts(logits, ids, wts, E, 4, 3, score=ft_hip.SCORE_SIGMOID)
    assert torch.equal(out[0][0], out[1][0]) and torch.equal(out[0][1], out[1][1])
    del lf
    l = torch.from_numpy((3 * rng.standard_normal((2, V))).astype(np.float32)).to(DEV).bfloat16()
    lf = far(2, V, (1 << 31) + 8, torch.bfloat16)
    lf.copy_(l)
    ws = torch.empty(gemv.sample_tokens_workspace_bytes(V, 2), dtype=torch.uint8, device=DEV)
    out = [(torch.zeros(2, dtype=torch.int32, device=DEV), torch.zeros(2, device=DEV)) for _ in "ab"]
    for logits, (tokens, lp) in zip((l, lf), out):
        gemv.sample_tokens(logits, V, 2, torch.full((2,), 0.7, device=DEV), tokens, ws,
                           top_p=torch.full((2,), 0.9, device=DEV), logprobs=lp)
    assert torch.equal(out[0][0], out[1][0]) and torch.equal(out[0][1], out[1][1])


def test_most_rows_of_the_norm(gemv):
    """2^22 - 1 rows of one value: y = x / sqrt(x x + eps), each rounded once."""
    n = (1 << 22) - 1
    x = torch.from_numpy(np.random.default_rng(3).standard_normal((n, 1)).astype(np.float32)).to(DEV)
    y = torch.empty_like(x)
    gemv.add_rmsnorm(x, None, 1, n, 1e-6, y=y)
    want = x.double() / torch.sqrt(x.double() ** 2 + float(np.float32(1e-6)))
    assert float(((y.double() - want).abs() / want.abs().clamp_min(1e-30)).max()) <= 2.0 ** -24 * (1 + 1e-6)


def test_two_threads_on_one_handle(gemv):
    """Calls of two host threads at once, each on a stream, buffers and workspace of its own, as one after the other."""
    import threading
    H = SMALL.hidden
    parts = [(stack_of(gemv, 4), head_of(gemv, H, VOCAB, 4), batch(4, H, 80 + i), settings(4, 80 + i)) for i in range(2)]
    want = []
    for r, head, x, s in parts:
        want.append([t.clone() for t in head.run(*r.run(x, 4), 4, **s)])
    torch.cuda.synchronize()
    failed = []

    def work(part, w):
        try:
            r, head, x, s = part
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for _ in range(10):
                    got = head.run(*r.run(x, 4), 4, **s)
                    with pytest.raises(ft_hip.FtHipError, match="n_groups"):
                        gemv.route_experts(r.logits, r.ids, r.wts, SMALL.n_experts, 4, 4, n_groups=3)
                stream.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(got, w))
        except BaseException as e:  # noqa: BLE001 - handed to the test's own thread
            failed.append(e)

    threads = [threading.Thread(target=work, args=p) for p in zip(parts, want)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed
