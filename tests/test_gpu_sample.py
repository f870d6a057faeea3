"""ft_hip_sample_tokens against its definition in 64 bits (numpy, row by row).

Tokens must be equal. Both sides sum f64 weights in their own order, so a token
may only differ where u times the kept sum lies within about 1e-13 of a running
sum, or a limit that close to a border; the inputs are fixed by their seeds, and
where sums meet a limit exactly (equal logits) both are exact. A log probability
is rounded once: 2^-24 of it, plus the sums' 1e-12.
"""
import numpy as np
import pytest
import torch

import ft_hip

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
INF, NAN = np.inf, np.nan
LOWEST = float(np.finfo(np.float32).min)


def host(t):
    torch.cuda.synchronize()
    return t.cpu().numpy()


def reference(row, t=1.0, k=0, p=1.0, m=0.0, u=0.5):
    """(token, log probability) of one row of float64 logits."""
    row = row.astype(np.float64)
    V = len(row)
    ok = row > -INF
    if not ok.any():
        return -1, NAN
    M = row[ok].max()
    if not t > 0:
        return int(np.flatnonzero(row == M)[0]), 0.0
    with np.errstate(all="ignore"):
        e = np.exp((row - M) / np.float64(t)) if t < INF else np.where(np.isinf(M), 0.0, 1.0) * np.ones(V)
    e = np.where(row == M, 1.0, np.where(ok & ~np.isinf(M), e, 0.0))
    order = np.argsort(np.where(ok, -row, INF), kind="stable")
    n = int(ok.sum())
    if 0 < k < V:
        n = min(n, k)
    s = e[order[:n]]
    if p < 1:
        c = np.cumsum(s)
        n = min(n, int((c < max(p, 0.0) * c[-1]).sum()) + 1)
    if m > 0:
        n = max(1, min(n, int((s[:n] >= min(m, 1.0)).sum())))
    kept = np.sort(order[:n])
    c = np.cumsum(e[kept])
    u = min(u, 1.0) if u > 0 else 0.0
    at = np.flatnonzero(c > u * c[-1])
    at = int(at[0]) if len(at) else int(np.flatnonzero(e[kept] > 0)[-1])
    return int(kept[at]), float(np.log(e[kept[at]] / c[-1]))


def draw(gemv, logits, n, vocab, u, stream=None, ws=None, **settings):
    """Tokens and log probabilities through the library; settings: sequences of n, or None."""
    arr = {a: None if v is None else torch.tensor(np.asarray(v, np.int32 if a == "top_k" else np.float32), device=DEV)
           for a, v in settings.items()}
    tokens = torch.full((n + 1,), -5, dtype=torch.int32, device=DEV)
    logprobs = torch.full((n + 1,), 7.0, device=DEV)
    if ws is None:
        ws = torch.full((gemv.sample_tokens_workspace_bytes(vocab, n),), 0xA5, dtype=torch.uint8, device=DEV)
    gemv.sample_tokens(logits, vocab, n, torch.tensor(np.asarray(u, np.float32), device=DEV), tokens, ws,
                       logprobs=logprobs, stream=stream, **arr)
    tok, lp = host(tokens), host(logprobs)
    assert tok[n] == -5 and lp[n] == 7.0
    return tok[:n], lp[:n]


def check(gemv, logits, u, t=None, k=None, p=None, m=None, dev=None):
    """logits: a CPU tensor [n, V]; settings: sequences of n or None. dev: the same on the GPU, laid out another way."""
    n, V = logits.shape
    tok, lp = draw(gemv, logits.to(DEV) if dev is None else dev, n, V, u, temperature=t, top_k=k, top_p=p, min_p=m)
    rows = logits.double().numpy()
    f = lambda v, i, off: off if v is None else float(np.float32(v[i]))  # noqa: E731
    for i in range(n):
        s = dict(t=f(t, i, 1.0), k=0 if k is None else int(k[i]), p=f(p, i, 1.0), m=f(m, i, 0.0), u=f(u, i, 0.5))
        want, want_lp = reference(rows[i], **s)
        assert tok[i] == want, (i, s, tok[i], want)
        if np.isnan(want_lp):
            assert np.isnan(lp[i])
        else:
            assert abs(lp[i] - want_lp) <= 2.0 ** -24 * abs(want_lp) * (1 + 1e-6) + 1e-12, (i, s, lp[i], want_lp)
    return tok, lp


def model_logits(rng, n, V, level=None):
    """A bulk of sd 2.5 and up to 64 tokens that stand out, falling with their rank."""
    l = 2.5 * rng.standard_normal((n, V))
    h = min(64, V)
    for i in range(n):
        top = (20.0 if rng.random() < 0.6 else 11.0) if level is None else level
        l[i, rng.permutation(V)[:h]] = top - 1.5 * np.log(np.arange(1, h + 1)) + 0.5 * rng.standard_normal(h)
    return l.astype(np.float32)


SETTINGS = {
    "plain": lambda rng, n: {},
    "hot": lambda rng, n: dict(t=rng.uniform(0.3, 3, n)),
    "top_k": lambda rng, n: dict(k=rng.integers(1, 100, n)),
    "big_k": lambda rng, n: dict(k=rng.integers(100, 20000, n), t=rng.uniform(0.5, 2, n)),
    "top_p": lambda rng, n: dict(p=rng.uniform(0.1, 0.999, n)),
    "min_p": lambda rng, n: dict(m=10.0 ** rng.uniform(-4, -0.3, n), t=rng.uniform(0.5, 2, n)),
    "chat": lambda rng, n: dict(t=0.8 * np.ones(n), k=64 * np.ones(n), p=0.95 * np.ones(n)),
    "all": lambda rng, n: dict(t=rng.uniform(0.3, 2, n), k=rng.integers(-1, 3000, n), p=rng.uniform(0.3, 1.2, n),
                               m=rng.uniform(-0.1, 0.1, n)),
    "greedy": lambda rng, n: dict(t=np.where(rng.random(n) < 0.5, 0.0, 1.0)),
    "cold": lambda rng, n: dict(t=10.0 ** rng.uniform(-3, -0.5, n), k=rng.integers(0, 60, n), p=rng.uniform(0.5, 1.1, n)),
}


@pytest.mark.parametrize("settings", list(SETTINGS))
@pytest.mark.parametrize("V", [1, 2, 3, 63, 64, 65, 500, 1023, 1024, 1025, 4096, 8193, 50021])
def test_against_the_definition(gemv, settings, V):
    rng = np.random.default_rng(V + 1000 * list(SETTINGS).index(settings))
    n = 9
    l = torch.from_numpy(model_logits(rng, n, V))
    check(gemv, l, rng.random(n), **SETTINGS[settings](rng, n))


@pytest.mark.parametrize("settings", list(SETTINGS))
@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
def test_whole_vocabulary(gemv, settings, type):
    rng = np.random.default_rng(7 + list(SETTINGS).index(settings))
    n, V = 6, 262144
    l = torch.from_numpy(model_logits(rng, n, V)).to(TYPES[type])
    check(gemv, l, rng.random(n), **SETTINGS[settings](rng, n))


@pytest.mark.parametrize("settings", ["plain", "top_p", "all", "chat"])
@pytest.mark.parametrize("n,V", [(200, 1500), (70, 32003), (300, 64)])
def test_many_rows(gemv, settings, n, V):
    rng = np.random.default_rng(n + V)
    l = torch.from_numpy(model_logits(rng, n, V))
    check(gemv, l, rng.random(n), **SETTINGS[settings](rng, n))


@pytest.mark.parametrize("V", [300000, 1 << 21])
def test_larger_vocabularies(gemv, V):
    rng = np.random.default_rng(V)
    l = torch.from_numpy(model_logits(rng, 4, V))
    check(gemv, l, rng.random(4), t=[1.0, 0.7, 1.5, 1.0], k=[0, 50, 0, 5000], p=[1.0, 0.9, 0.95, 0.8])


@pytest.mark.parametrize("V", [2, 7, 64, 1000, 4097, 50000, 262144])
def test_equal_logits(gemv, V):
    """All equal: every sum is exact, the borders are met exactly, and the cut is by index."""
    us = [0.0, 0.25, 0.5, 0.999]
    for p in (0.5, 0.25, 1.0, 0.0, 0.3):
        for k in (0, 1, 2, V // 2, V):
            l = torch.full((4, V), 1.7)
            check(gemv, l, us, p=[p] * 4, k=[k] * 4, t=[1.0, 0.3, 2.0, 0.7])


@pytest.mark.parametrize("type", ["f32", "bf16"])
@pytest.mark.parametrize("V", [100, 5000, 262144])
def test_few_distinct_logits(gemv, type, V):
    """Thousands of equal values on the border of top-k, top-p and min-p."""
    rng = np.random.default_rng(V)
    n = 12
    l = torch.from_numpy(np.round(rng.standard_normal((n, V)) * 2).astype(np.float32) / 2).to(TYPES[type])
    check(gemv, l, rng.random(n), k=rng.integers(0, V, n), p=rng.uniform(0.05, 1.0, n))
    check(gemv, l, rng.random(n), p=rng.uniform(0.05, 1.0, n))
    check(gemv, l, rng.random(n), m=rng.uniform(0.01, 1.0, n), k=rng.integers(0, V, n))


@pytest.mark.parametrize("V", [5, 130, 9000, 262144])
def test_masked_and_nonfinite_rows(gemv, V):
    rng = np.random.default_rng(V)
    l = (3 * rng.standard_normal((12, V))).astype(np.float32)
    l[0] = -INF
    l[1] = NAN
    l[2, rng.random(V) < 0.5] = -INF
    l[3, rng.random(V) < 0.5] = NAN
    l[4] = LOWEST
    l[5] = -INF
    l[5, V - 1] = -3.0
    l[6, [1, V - 2]] = INF
    l[7] = LOWEST
    l[7, V // 2] = 0.0
    l[8] = -INF
    l[8, [0, V - 1]] = LOWEST
    l[9, :] = -0.0
    l[9, ::2] = 0.0
    l[10] *= 1e36
    l[11, V // 2:] = -INF
    l = torch.from_numpy(l)
    for s in (dict(), dict(k=[3] * 12), dict(p=[0.7] * 12), dict(m=[0.2] * 12), dict(t=[0.0] * 12),
              dict(k=[V // 2] * 12, p=[0.5] * 12, m=[0.01] * 12), dict(t=[INF] * 12), dict(t=[INF] * 12, p=[0.5] * 12)):
        for u in (0.0, 0.4, 0.999999):
            tok, _ = check(gemv, l, [u] * 12, **s)
            assert tok[0] == tok[1] == -1


def test_settings_out_of_range(gemv):
    rng = np.random.default_rng(5)
    l = torch.from_numpy(model_logits(rng, 10, 3000, level=9.0))
    us = rng.random(10)
    check(gemv, l, us, t=[-1.0, NAN, 0.0, -0.0, -INF, INF, 1e-30, 1e30, 1e-45, 3e38])
    check(gemv, l, us, k=[0, -1, -2 ** 31, 3000, 3001, 2 ** 31 - 1, 1, 2, 2999, 5])
    check(gemv, l, us, p=[0.0, -1.0, NAN, 1.0, 2.0, INF, -INF, 1e-30, 1 - 2.0 ** -24, 0.5])
    check(gemv, l, us, m=[0.0, -1.0, NAN, 1.0, 2.0, INF, -INF, 1e-30, 1 - 2.0 ** -24, 0.5])
    check(gemv, l, [0.0, -1.0, NAN, 1.0, 2.0, INF, -INF, 1e-30, 1 - 2.0 ** -24, 0.5])
    check(gemv, l, [0.0, -1.0, NAN, 1.0, 2.0, INF, -INF, 1e-30, 1 - 2.0 ** -24, 0.5], k=[7] * 10, p=[0.9] * 10)


@pytest.mark.parametrize("V", [40, 3000, 70000])
@pytest.mark.parametrize("s", [dict(), dict(k=20), dict(p=0.8), dict(m=0.05), dict(t=1.4, p=0.99)])
def test_the_draw_runs_through_the_kept_tokens(gemv, V, s):
    """One row of logits, u from 0 to 1: the tokens rise, and their shares are the probabilities to 1/n."""
    rng = np.random.default_rng(V)
    n = 400
    l = torch.from_numpy(np.repeat(model_logits(rng, 1, V, level=13.0), n, 0))
    tok, lp = check(gemv, l, np.arange(n) / n, **{a: [v] * n for a, v in s.items()})
    assert np.all(np.diff(tok) >= 0)
    for token in np.unique(tok):
        assert abs((tok == token).mean() - np.exp(lp[tok == token][0])) <= 1.0 / n + 1e-6


@pytest.mark.parametrize("descending", [False, True])
@pytest.mark.parametrize("V", [6000, 262144])
def test_sorted_vocabularies(gemv, descending, V):
    """The largest logits side by side at one end."""
    rng = np.random.default_rng(V)
    l = np.sort(model_logits(rng, 6, V), axis=1)
    l = torch.from_numpy((l[:, ::-1] if descending else l).copy())
    check(gemv, l, rng.random(6), k=[1, 64, 700, 5000, 0, 0], p=[1, 0.9, 0.99, 0.9, 0.9, 1.0], m=[0, 0, 0, 0, 0, 0.001])


@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("off,pad", [(0, 0), (1, 0), (0, 1), (3, 5), (0, 8)])
def test_strides_and_offsets(gemv, type, off, pad):
    rng = np.random.default_rng(off + 10 * pad)
    n, V = 5, 9001
    l = torch.from_numpy(model_logits(rng, n, V)).to(TYPES[type])
    flat = torch.full((n * (V + pad) + off,), 60.0, dtype=TYPES[type], device=DEV)
    view = flat[off:].view(n, V + pad)[:, :V]
    view.copy_(l)
    before = flat.clone()
    check(gemv, l, rng.random(n), t=[0.8] * n, k=[50, 0, 0, 7, 0], p=[0.9, 0.9, 1.0, 1.0, 0.5], dev=view)
    assert torch.equal(before, flat)


def test_same_bits_on_another_stream_and_captured(gemv):
    rng = np.random.default_rng(11)
    n, V = 12, 40000
    l = torch.from_numpy(model_logits(rng, n, V)).to(DEV)
    u = torch.rand(n, device=DEV)
    s = {a: torch.tensor(np.asarray(v), dtype=torch.int32 if a == "top_k" else torch.float32, device=DEV)
         for a, v in dict(temperature=rng.uniform(0, 2, n), top_k=rng.integers(-5, 100, n),
                          top_p=rng.uniform(0.5, 1.2, n), min_p=rng.uniform(-0.1, 0.1, n)).items()}

    def call(ws=None):
        tokens, lp = torch.zeros(n, dtype=torch.int32, device=DEV), torch.zeros(n, device=DEV)
        ws = torch.empty(gemv.sample_tokens_workspace_bytes(V, n), dtype=torch.uint8, device=DEV) if ws is None else ws
        gemv.sample_tokens(l, V, n, u, tokens, ws, logprobs=lp, **s)
        return tokens, lp

    first = call()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = call()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, other))
    ws = torch.empty(gemv.sample_tokens_workspace_bytes(V, n), dtype=torch.uint8, device=DEV)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        captured = call(ws)
    for seed in (1, 2, 3):
        l.copy_(torch.from_numpy(model_logits(np.random.default_rng(seed), n, V)))
        u.uniform_()
        g.replay()
        want = call()  # eager, with a workspace of its own
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(captured, want))


def test_without_logprobs_or_settings(gemv):
    rng = np.random.default_rng(1)
    l = torch.from_numpy(model_logits(rng, 3, 1234))
    u = torch.rand(3, device=DEV)
    tokens, ws = torch.zeros(3, dtype=torch.int32, device=DEV), torch.zeros(1 << 20, dtype=torch.uint8, device=DEV)
    gemv.sample_tokens(l.to(DEV), 1234, 3, u, tokens, ws)
    want = [reference(l[i].double().numpy(), u=float(u[i]))[0] for i in range(3)]
    assert list(host(tokens)) == want
    gemv.sample_tokens(l.to(DEV), 1234, 0, u, tokens, ws)  # no rows: nothing
    assert list(host(tokens)) == want


def test_refused_by_the_python_side(gemv):
    l = torch.zeros((4, 100), device=DEV)
    one = torch.ones(4, device=DEV)
    tokens = torch.zeros(4, dtype=torch.int32, device=DEV)
    ws = torch.zeros(gemv.sample_tokens_workspace_bytes(100, 4), dtype=torch.uint8, device=DEV)
    bad = [dict(logits=l[:3]), dict(logits=l.double()), dict(logits=l[:, :99]), dict(u=one[:3]), dict(u=one.half()),
           dict(tokens=one), dict(tokens=tokens.long()), dict(temperature=tokens), dict(top_k=one),
           dict(top_p=one.double()), dict(min_p=one[::2]), dict(logprobs=tokens), dict(workspace=ws[:-1])]
    for change in bad:
        kw = dict(logits=l, u=one, tokens=tokens, workspace=ws)
        kw.update(change)
        with pytest.raises(ft_hip.FtHipError) as e:
            gemv.sample_tokens(kw.pop("logits"), 100, 4, kw.pop("u"), kw.pop("tokens"), kw.pop("workspace"), **kw)
        assert e.value.code in (ft_hip.E_SHAPE, ft_hip.E_INVALID), change


@pytest.mark.parametrize("settings", list(SETTINGS))
@pytest.mark.parametrize("V", [8191, 8192])
def test_longest_rows_of_one_launch(gemv, settings, V):
    rng = np.random.default_rng(V + 1000 * list(SETTINGS).index(settings))
    n = 5
    check(gemv, torch.from_numpy(model_logits(rng, n, V)).half(), rng.random(n), **SETTINGS[settings](rng, n))


def test_more_rows_than_the_workspace_holds(gemv):
    """Rows that share the workspace one batch after the other: as each alone."""
    rng = np.random.default_rng(21)
    n, V = 1030, 8201
    l = torch.from_numpy(model_logits(rng, n, V)).to(DEV)
    u = rng.random(n)
    s = dict(temperature=rng.uniform(0, 2, n), top_k=rng.integers(-50, 100, n), top_p=rng.uniform(0.5, 1.2, n),
             min_p=rng.uniform(-0.1, 0.1, n))
    assert gemv.sample_tokens_workspace_bytes(V, n) == gemv.sample_tokens_workspace_bytes(V, 512)
    tok, lp = draw(gemv, l, n, V, u, **s)
    for a, b in ((0, 3), (510, 515), (1000, 1030)):
        part = draw(gemv, l[a:b], b - a, V, u[a:b], **{k: v[a:b] for k, v in s.items()})
        assert np.array_equal(tok[a:b], part[0]) and np.array_equal(lp[a:b], part[1])


def test_one_row_of_logits_for_several_draws(gemv):
    """A batch that is the same row again and again, and one that rises in u: as a call each."""
    rng = np.random.default_rng(8)
    for V in (700, 30000):
        l = torch.from_numpy(model_logits(rng, 1, V)).to(DEV)
        u = [0.3, 0.3, 0.9, 0.3]
        tok, lp = draw(gemv, l.repeat(4, 1), 4, V, u, top_p=[0.9] * 4)
        assert tok[0] == tok[1] == tok[3] and lp[0] == lp[1] == lp[3]
        for i in range(4):
            one = draw(gemv, l, 1, V, u[i:i + 1], top_p=[0.9])
            assert one[0][0] == tok[i] and one[1][0] == lp[i]


def test_tensors_of_another_device_are_refused(gemv):
    l = torch.zeros((4, 100), device=DEV)
    one = torch.ones(4, device=DEV)
    tokens = torch.zeros(4, dtype=torch.int32, device=DEV)
    ws = torch.zeros(gemv.sample_tokens_workspace_bytes(100, 4), dtype=torch.uint8, device=DEV)
    for change in (dict(logits=l.cpu()), dict(logits=l.int()), dict(u=one.cpu()), dict(tokens=tokens.cpu()),
                   dict(workspace=ws.cpu()), dict(temperature=one.cpu()), dict(top_k=tokens.cpu()),
                   dict(top_p=one.cpu()), dict(min_p=one.cpu()), dict(logprobs=one.cpu()),
                   dict(u=one[:1].expand(4))):
        kw = dict(dict(logits=l, u=one, tokens=tokens, workspace=ws), **change)
        with pytest.raises(ft_hip.FtHipError) as e:
            gemv.sample_tokens(kw.pop("logits"), 100, 4, kw.pop("u"), kw.pop("tokens"), kw.pop("workspace"), **kw)
        assert e.value.code in (ft_hip.E_SHAPE, ft_hip.E_INVALID), change
