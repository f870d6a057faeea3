"""ft_hip_adjust_logits against its formula, bit for bit: every operation of it
rounds once, in f32."""
import numpy as np
import pytest
import torch

import ft_hip

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F = np.float32


def host(t):
    return t.detach().cpu().numpy()


def dev(a):
    return None if a is None else torch.from_numpy(np.ascontiguousarray(a)).to(DEV)


def reference(x, vocab, history=None, history_len=None, repetition=None, presence=None, frequency=None, bias_ids=None, bias=None,
              mask=None):
    out = x.astype(F).copy()
    for i in range(len(out)):
        if history is not None:
            h = history[i][:max(0, min(len(history[i]), history_len[i] if history_len is not None else 1 << 30))]
            ids, count = np.unique(h[(h >= 0) & (h < vocab)], return_counts=True)
            y = out[i, ids]
            if repetition is not None:
                with np.errstate(all="ignore"):
                    y = np.where(y > 0, y / repetition[i], y * repetition[i]).astype(F)
            p = F(0.0) if presence is None else presence[i]
            f = F(0.0) if frequency is None else frequency[i]
            out[i, ids] = y - (p + f * count.astype(F))
        if bias is not None:
            add = {}
            for t, b in zip(bias_ids[i], bias[i]):
                if 0 <= t < vocab:
                    add[t] = F(add[t] + b) if t in add else b
            for t, b in add.items():
                out[i, t] += b
        if mask is not None:
            bits = np.unpackbits(mask[i].view(np.uint8), bitorder="little")[:vocab]
            out[i, bits == 0] = -np.inf
    return out


def inputs(rng, n, vocab, history=0, bias=0, mask=False, dtype=torch.float32):
    x = torch.from_numpy(rng.standard_normal((n, vocab)).astype(F) * F(3)).to(dtype)
    s = {}
    if history:
        s["history"] = (vocab * rng.random((n, history)) ** 4).astype(np.int32)
        s["history_len"] = rng.integers(0, history + 1, n).astype(np.int32)
        s["repetition"] = rng.uniform(0.8, 1.6, n).astype(F)
        s["presence"], s["frequency"] = rng.uniform(-0.5, 1, n).astype(F), rng.uniform(-0.2, 0.5, n).astype(F)
    if bias:
        s["bias_ids"] = rng.integers(-2, vocab + 2, (n, bias)).astype(np.int32)
        s["bias"] = rng.standard_normal((n, bias)).astype(F) * F(5)
    if mask:
        s["mask"] = rng.integers(-2 ** 31, 2 ** 31, (n, (vocab + 31) // 32)).astype(np.int32)
    return x, s


def check(gemv, x, s, vocab, out=None, place=None):
    n = len(x)
    want = reference(host(x.float())[:, :vocab], vocab, **s)
    given = x.to(DEV) if place is None else place
    out = torch.full((n, vocab), 5.0, device=DEV) if out is None else out
    gemv.adjust_logits(given, out, vocab, n, **{k: dev(v) for k, v in s.items()})
    torch.cuda.synchronize()
    got = host(out)[:, :vocab]
    assert np.array_equal(np.isnan(got), np.isnan(want))
    assert np.array_equal(np.nan_to_num(got, nan=1.0), np.nan_to_num(want, nan=1.0))


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n,vocab,history,bias,mask", [
    (1, 1, 1, 1, True), (1, 31, 5, 0, True), (3, 33, 0, 4, False), (2, 2047, 100, 3, True), (5, 2048, 1, 1, False),
    (4, 2049, 3000, 0, False), (2, 8193, 50, 1024, True), (300, 8191, 40, 5, True), (64, 50021, 700, 30, True),
    (9, 262144, 2000, 17, False), (1, 262144, 20000, 300, True), (33, 262144, 20000, 1024, True), (40, 262143, 0, 0, True), (3, 5000, 0, 0, True), (2, 5000, 0, 0, False)])
def test_against_the_formula(gemv, dtype, n, vocab, history, bias, mask):
    x, s = inputs(np.random.default_rng(n * 7 + vocab), n, vocab, history, bias, mask, dtype)
    check(gemv, x, s, vocab)


@pytest.mark.parametrize("keep", [("history",), ("history", "repetition"), ("history", "presence"), ("history", "frequency"),
                                  ("history", "history_len", "presence", "frequency"), ("bias_ids", "bias"), ("mask",)])
def test_each_alone(gemv, keep):
    x, s = inputs(np.random.default_rng(3), 3, 4100, 60, 5, True)
    check(gemv, x, {k: s[k] for k in keep}, 4100)


def test_tokens_that_are_none_and_lengths_out_of_range(gemv):
    x, s = inputs(np.random.default_rng(5), 6, 3000, 50, 9)
    s["history"][:, ::5] = [[-1], [3000], [2 ** 31 - 1], [-2 ** 31], [-7], [5000]]
    s["history_len"] = np.array([0, -3, 51, 2 ** 31 - 1, -2 ** 31, 50], np.int32)
    s["bias_ids"][:, 0] = [-1, 3000, 2 ** 31 - 1, -2 ** 31, 2999, 0]
    check(gemv, x, s, 3000)


def test_the_same_token_again_and_again(gemv):
    """All of a history one token, at a chunk's ends too; a token biased many times, in order."""
    vocab = 20000
    for token in (0, 2047, 2048, 8191, 8192, vocab - 1):
        x, s = inputs(np.random.default_rng(token), 2, vocab, 3000, 64)
        s["history"][:] = token
        s["bias_ids"][:, ::2] = token
        check(gemv, x, s, vocab)


def test_infinities_nan_and_zero(gemv):
    x, s = inputs(np.random.default_rng(7), 2, 4000, 300, 20, True)
    for i, v in enumerate((np.inf, -np.inf, np.nan, 0.0, -0.0, 1e-45, 3e38)):
        x[:, i::11] = float(v)
    s["repetition"][:] = 0.5, 2.0
    s["bias"][0, :3] = np.inf, -np.inf, np.nan
    with np.errstate(all="ignore"):
        check(gemv, x, s, 4000)


def test_in_place_rows_apart_and_off_their_vectors(gemv):
    rng = np.random.default_rng(8)
    for off, width, vocab in ((0, 3000, 3000), (1, 3001, 2999), (4, 3016, 3001), (3, 6001, 2900)):
        x, s = inputs(rng, 4, vocab, 90, 6, True)
        buf = torch.full((4, width + 4), 2.0, device=DEV)
        rows = buf[:, off:off + vocab]
        rows.copy_(x)
        check(gemv, x, s, vocab, rows, rows)
        left = torch.ones_like(buf, dtype=torch.bool)
        left[:, off:off + vocab] = False
        assert torch.all(buf[left] == 2.0)
    # lists that are columns of wider ones
    x, s = inputs(rng, 3, 1000, 40, 0, True)
    wide = {k: dev(np.concatenate([s[k], s[k]], 1))[:, :s[k].shape[1]] for k in ("history", "mask")}
    out = torch.empty((3, 1000), device=DEV)
    gemv.adjust_logits(x.to(DEV), out, 1000, 3, history=wide["history"], mask=wide["mask"], presence=dev(s["presence"]))
    torch.cuda.synchronize()
    assert np.array_equal(host(out), reference(host(x), 1000, history=s["history"], mask=s["mask"], presence=s["presence"]))


def test_replayed_with_new_settings_and_drawn_from(gemv):
    """Adjusted and drawn from in one captured run; what a mask forbids is never drawn."""
    rng = np.random.default_rng(9)
    n, vocab = 5, 9000
    x, s = inputs(rng, n, vocab, 200, 8, True)
    d = {k: dev(v) for k, v in s.items()}
    logits, out, u = x.to(DEV), torch.empty((n, vocab), device=DEV), torch.rand(n, device=DEV)
    tokens = torch.empty(n, dtype=torch.int32, device=DEV)
    ws = torch.empty(gemv.sample_tokens_workspace_bytes(vocab, n), dtype=torch.uint8, device=DEV)
    top_k = torch.full((n,), 3, dtype=torch.int32, device=DEV)

    def step(stream=None):
        gemv.adjust_logits(logits, out, vocab, n, stream=stream, **d)
        gemv.sample_tokens(out, vocab, n, u, tokens, ws, top_k=top_k, stream=stream)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    side = torch.cuda.Stream()
    for i in range(4):
        x, s = inputs(rng, n, vocab, 200, 8, True)
        logits.copy_(x)
        for k, v in s.items():
            d[k].copy_(torch.from_numpy(v))
        torch.cuda.synchronize()
        if i == 2:
            step(side)
        else:
            graph.replay()
        torch.cuda.synchronize()
        want = reference(host(x), vocab, **s)
        assert np.array_equal(host(out), want)
        best = np.sort(want, 1)[:, -3]
        for r, t in enumerate(host(tokens)):
            assert want[r, t] >= best[r] and want[r, t] > -np.inf


def test_a_row_that_the_mask_leaves_empty(gemv):
    x, s = inputs(np.random.default_rng(10), 3, 500, 0, 0, True)
    s["mask"][1] = 0
    check(gemv, x, s, 500)


def test_no_rows(gemv):
    none = torch.empty((0, 100), device=DEV)
    gemv.adjust_logits(none, none, 100, 0)
    torch.cuda.synchronize()


@pytest.mark.parametrize("n,vocab", [(8400, 1000), (65535, 129), (1025, 8192), (513, 16385)])
def test_many_rows_of_a_small_vocabulary(gemv, n, vocab):
    """Values enough for the longest chunks, rows that fill a part of one or a little more."""
    x, s = inputs(np.random.default_rng(n), n, vocab, 30, 7, True)
    check(gemv, x, s, vocab)
