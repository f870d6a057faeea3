"""The cache, the attention and the rules on logits together, as a decode loop
runs them: qkv GEMV, moe_synth.CachedAttention, q8, o_proj, moe_synth.VocabHead
with rules. Every stage is checked from what the stage before it left."""
import numpy as np
import pytest
import torch

import ft_hip
import moe_synth
from test_gpu_adjust_logits import inputs as rules_of, reference as adjusted
from test_gpu_attention import Batch, definition
from test_gpu_kv import E4M3, I8, Layout, host
from test_gpu_sample import reference as draw_reference

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
H, HEADS, KV, DIM, PAGE, VOCAB, N = 256, 4, 2, 64, 16, 3000, 3
ROW = (HEADS + 2 * KV) * DIM


def q4r(gemv, rows, k, seed):
    w = torch.empty(rows * ft_hip.row_bytes(k, ft_hip.LAYOUT_Q4R), dtype=torch.uint8, device=DEV)
    gemv.gen_q4_rows(moe_synth.tensor_key(903, 0, seed, 1), 0, rows, k, moe_synth.gen_scale(0.1), w, ft_hip.LAYOUT_Q4R)
    return w


class Step:
    """One layer and the head, for N sequences behind a prefix."""

    def __init__(self, gemv, kind, shared):
        self.g, self.kind = gemv, kind
        self.wq, self.wo = q4r(gemv, ROW, H, 1), q4r(gemv, H, HEADS * DIM, 2)
        self.head = moe_synth.VocabHead(gemv, q4r(gemv, VOCAB, H, 3), None, VOCAB, H, N)
        self.pages = 4 * N + 2
        self.att = moe_synth.CachedAttention(gemv, HEADS, KV, DIM, self.pages, PAGE, N, cache_type=kind, device=DEV)
        order = np.random.default_rng(4).permutation(self.pages).astype(np.int32)
        self.tables = torch.from_numpy(order[:4 * N].reshape(N, 4).copy()).to(DEV)
        self.prefix = torch.from_numpy(order[4 * N:].copy()).to(DEV) if shared else None
        self.prefix_len = torch.full((1,), 21, dtype=torch.int32, device=DEV) if shared else None
        f = lambda *s: torch.zeros(s, device=DEV)  # noqa: E731
        self.x, self.qkv, self.o, self.u = f(N, H), f(N, ROW), f(N, H), f(N)
        self.q8 = [torch.zeros(N * k // 32 * ft_hip.Q8_BLK, dtype=torch.uint8, device=DEV) for k in (H, HEADS * DIM)]
        self.zero = torch.zeros(N, dtype=torch.int32, device=DEV)
        self.slots, self.lens = (torch.zeros(N, dtype=torch.int32, device=DEV) for _ in range(2))
        _, s = rules_of(np.random.default_rng(5), N, VOCAB, 40, 6, True)
        self.host_rules, self.rules = s, {k: torch.from_numpy(v).to(DEV) for k, v in s.items()}
        if shared:
            rows = torch.from_numpy(np.random.default_rng(6).standard_normal((21, ROW)).astype(np.float32)).to(DEV)
            at = np.arange(21)
            slots = torch.from_numpy((order[4 * N:][at // PAGE] * PAGE + at % PAGE).astype(np.int32)).to(DEV)
            self.att.write(rows, slots, 21)
        torch.cuda.synchronize()

    def feed(self, t):
        """Inputs of the sequences' t-th token; the second joins late."""
        rng = np.random.default_rng(100 + t)
        self.x.copy_(torch.from_numpy(rng.standard_normal((N, H)).astype(np.float32)))
        self.u.copy_(torch.from_numpy(rng.random(N).astype(np.float32)))
        lens = np.array([t + 1, max(0, t - 2), t + 1], np.int32)
        tab = host(self.tables)
        slots = [tab[i, (n - 1) // PAGE] * PAGE + (n - 1) % PAGE if n else -1 for i, n in enumerate(lens)]
        self.lens.copy_(torch.from_numpy(lens))
        self.slots.copy_(torch.tensor(slots, dtype=torch.int32))
        torch.cuda.synchronize()
        return lens

    def run(self, stream=None):
        g = self.g
        with moe_synth._current(g, stream):
            g.quantize_q8(self.x, H, self.q8[0], H, N)
            g.gemv_q4r_idx(self.wq, 0, 0, self.zero, None, N, self.q8[0], H // 32, self.qkv, ROW, ROW, H)
            out = self.att.run(self.qkv, self.slots, self.tables, self.lens, N, self.prefix, self.prefix_len, stream=stream)
            g.quantize_q8(out, HEADS * DIM, self.q8[1], HEADS * DIM, N)
            g.gemv_q4r_idx(self.wo, 0, 0, self.zero, None, N, self.q8[1], HEADS * DIM // 32, self.o, H, H, HEADS * DIM)
        return self.head.run(self.o, self.x, N, self.u, stream=stream, rules=self.rules)


@pytest.mark.parametrize("shared", [False, True])
@pytest.mark.parametrize("kind", [I8, E4M3])
def test_every_stage_from_the_one_before(gemv, kind, shared):
    s, lay = Step(gemv, kind, shared), Layout(PAGE, KV, DIM)
    want_cache = host(s.att.cache).reshape(-1).copy()
    for t in range(20):  # past a page's end
        lens = s.feed(t)
        tokens, logprobs = s.run()
        torch.cuda.synchronize()
        qkv = host(s.qkv).astype(np.float64)
        slots = host(s.slots)
        live = slots >= 0
        k, v = (qkv[live, (HEADS + i * KV) * DIM:(HEADS + (i + 1) * KV) * DIM].reshape(-1, KV, DIM) for i in (0, 1))
        lay.put(want_cache, slots[live], k, v, kind)
        assert np.array_equal(host(s.att.cache).reshape(-1), want_cache)
        out, tol, _, _ = definition(qkv[:, :HEADS * DIM], want_cache, lay, kind, host(s.tables), lens,
                                    host(s.prefix) if shared else None, 21, 1, HEADS, DIM ** -0.5, 0, torch.float32, s.pages)
        assert np.all(np.abs(host(s.att.out) - out) <= tol)
        # the rules were applied in place: the head's GEMV again, then the formula
        logits = torch.empty_like(s.head.logits)
        gemv.gemv_q4r_idx(s.head.weights, 0, 0, s.head.slots, None, N, s.head.q8, H // 32, logits, VOCAB, VOCAB, H)
        want = adjusted(host(logits), VOCAB, **s.host_rules)
        assert np.array_equal(host(s.head.logits), want)
        for i in range(N):
            token, lp = draw_reference(want[i].astype(np.float64), 1.0, 0, 1.0, 0.0, float(s.u[i]))
            assert int(tokens[i]) == token and abs(float(logprobs[i]) - lp) <= 2.0 ** -23 * abs(lp) + 1e-9


@pytest.mark.parametrize("shared", [False, True])
def test_captured_steps_repeat_the_eager_ones(gemv, shared):
    """One step captured, replayed as the sequences grow, with eager work and another stream between."""
    s, e = Step(gemv, I8, shared), Step(gemv, I8, shared)
    s.feed(0)
    s.run()
    torch.cuda.synchronize()
    s.att.cache.copy_(e.att.cache)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = s.run()
    side = torch.cuda.Stream()
    for t in range(18):
        s.feed(t), e.feed(t)
        want = e.run(side if t % 4 == 3 else None)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip((*captured, s.att.out, s.head.logits), (*want, e.att.out, e.head.logits)))
        assert torch.equal(s.att.cache, e.att.cache)


def test_several_layers_and_sequences_share_a_workspace_one_after_the_other(gemv):
    """Batches of other sizes on one workspace, in turn: the same bits as on workspaces of their own."""
    batches = [Batch(gemv, [30 + i, 200, 7][:3 - i % 2], PAGE, 2, 2, 64, I8, torch.float32, prefix=40 * (i % 2), seed=30 + i)
               for i in range(4)]
    want = [b.run() for b in batches]
    ws = max((b.workspace() for b in batches), key=len)
    torch.cuda.synchronize()
    for _ in range(2):
        for b, w in zip(batches, want):
            got = b.run(workspace=ws)
            torch.cuda.synchronize()
            assert torch.equal(got[0], w[0]) and torch.equal(got[1], w[1])
