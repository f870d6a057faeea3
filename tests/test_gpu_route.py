"""ft_hip_route_experts against its definition in 64 bits (numpy).

ids must be equal (equal scores go to the lower index). A weight is rounded
once from f64: half a step of f32, 2^-24 of it; the f64 exps and sums before
it are off by a few 2^-53 each, under 1e-13 over 1024 experts.
"""
import numpy as np
import pytest
import torch

import ft_hip

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
WT = 2.0 ** -24 + 1e-13
SUB = 2.0 ** -150


def dev(a):
    return None if a is None else torch.from_numpy(np.ascontiguousarray(a)).to(DEV)


def host(t):
    torch.cuda.synchronize()
    return t.cpu().numpy()


def reference(l, k, score, bias=None, G=1, tg=1, rank=1, renorm=True, scale=1.0, es=None):
    l = l.astype(np.float64)
    n, E = l.shape
    ids, wts = np.zeros((n, k), np.int32), np.zeros((n, k))
    for t in range(n):
        row = l[t]
        ok = row > -np.inf  # False for NaN
        with np.errstate(all="ignore"):
            if score == ft_hip.SCORE_SOFTMAX:
                m = row[ok].max() if ok.any() else 0.0
                s = np.where(row == m, 1.0, np.exp(row - m))
                s = s / s[ok].sum()
            else:
                s = 1.0 / (1.0 + np.exp(-row))
            c = s + (0.0 if bias is None else bias.astype(np.float64))
        c = np.where(ok & ~np.isnan(c), c, -np.inf)
        if G > 1:
            best = -np.sort(-c.reshape(G, -1), axis=1)
            gs = best[:, 0].copy()
            if rank == 2:
                two = best[:, 1] > -np.inf
                gs[two] += best[two, 1]
            opened = np.argsort(-gs, kind="stable")[:tg]
            closed = np.ones(G, bool)
            closed[opened] = False
            c[np.repeat(closed, E // G)] = -np.inf
        order = np.argsort(-c, kind="stable")[:k]
        order = order[c[order] > -np.inf]
        w = s[order]
        if renorm:
            w = w / w.sum() if w.sum() > 0 else 0.0 * w
        ids[t, :len(order)] = order
        wts[t, :len(order)] = w * np.float64(np.float32(scale))
        if es is not None:
            wts[t, :len(order)] *= es[order].astype(np.float64)
    return ids, wts


def check(gemv, l, k, score, stride=None, **kw):
    n, E = l.shape
    ids = torch.full((n + 1, k), -5, dtype=torch.int32, device=DEV)
    wts = torch.full((n + 1, k), 7.0, device=DEV)
    names = dict(bias="bias", G="n_groups", tg="top_groups", rank="group_rank", renorm="renorm", scale="scale",
                 es="expert_scale")
    args = {names[a]: dev(v) if a in ("bias", "es") else v for a, v in kw.items()}
    ld = dev(l)
    if stride:
        wide = torch.full((n, stride), 50.0, device=DEV)
        wide[:, :E] = ld
        ld = wide[:, :E]
    gemv.route_experts(ld, ids, wts, E, k, n, score=score, **args)
    want_ids, want = reference(l, k, score, **kw)
    got_ids, got = host(ids), host(wts)
    assert np.array_equal(got_ids[:n], want_ids)
    assert np.all(np.abs(got[:n] - want) <= WT * np.abs(want) + SUB)
    assert np.all(got_ids[n] == -5) and np.all(got[n] == 7.0)  # rows behind the last stay
    return got_ids[:n], got[:n]


SHAPES = [  # experts, top_k, groups, top_groups
    (1, 1, 1, 1), (2, 2, 1, 1), (8, 2, 1, 1), (8, 8, 1, 1), (16, 4, 4, 2), (33, 5, 1, 1), (60, 4, 1, 1),
    (64, 6, 8, 3), (96, 8, 3, 2), (128, 8, 1, 1), (128, 1, 1, 1), (160, 6, 8, 3), (255, 32, 1, 1), (256, 8, 8, 4),
    (256, 32, 64, 8), (300, 12, 4, 1), (384, 8, 1, 1), (512, 10, 16, 4), (1000, 7, 1, 1), (1024, 32, 32, 4),
]


@pytest.mark.parametrize("score", [ft_hip.SCORE_SOFTMAX, ft_hip.SCORE_SIGMOID])
@pytest.mark.parametrize("E,k,G,tg", SHAPES)
def test_against_the_definition(gemv, score, E, k, G, tg):
    rng = np.random.default_rng(E * 31 + k)
    for n in (1, 5, 67):
        l = rng.standard_normal((n, E)).astype(np.float32) * 1.5
        bias = (0.1 * rng.standard_normal(E)).astype(np.float32)
        es = rng.uniform(0.5, 1.5, E).astype(np.float32)
        rank = 2 if E // G >= 2 else 1
        check(gemv, l, k, score, bias=bias, G=G, tg=tg, rank=rank, renorm=True, scale=2.5)
        check(gemv, l, k, score, G=G, tg=tg, rank=1, renorm=False, es=es)
        check(gemv, l, k, score, bias=bias, es=es, scale=0.7, stride=E + 3)


@pytest.mark.parametrize("score", [ft_hip.SCORE_SOFTMAX, ft_hip.SCORE_SIGMOID])
def test_many_tokens(gemv, score):
    rng = np.random.default_rng(8)
    l = rng.standard_normal((4099, 256)).astype(np.float32)
    bias = (0.1 * rng.standard_normal(256)).astype(np.float32)
    check(gemv, l, 8, score, bias=bias, G=8, tg=4, rank=2)
    check(gemv, l[:, :128].copy(), 8, score)


@pytest.mark.parametrize("score", [ft_hip.SCORE_SOFTMAX, ft_hip.SCORE_SIGMOID])
@pytest.mark.parametrize("E,G,tg", [(8, 1, 1), (64, 8, 2), (128, 1, 1), (256, 8, 4), (512, 1, 1)])
def test_equal_scores_go_to_the_lower_index(gemv, score, E, G, tg):
    rng = np.random.default_rng(E)
    k = min(8, tg * (E // G))
    check(gemv, np.zeros((3, E), np.float32), k, score, G=G, tg=tg, rank=2)
    l = rng.integers(-2, 3, (50, E)).astype(np.float32)
    check(gemv, l, k, score, G=G, tg=tg, rank=2)
    check(gemv, l, k, score, G=G, tg=tg, rank=1, renorm=False, bias=rng.integers(0, 2, E).astype(np.float32))


@pytest.mark.parametrize("score", [ft_hip.SCORE_SOFTMAX, ft_hip.SCORE_SIGMOID])
@pytest.mark.parametrize("E,G,tg", [(8, 1, 1), (64, 8, 2), (128, 4, 2), (1024, 1, 1)])
def test_masked_and_nonfinite(gemv, score, E, G, tg):
    """Rows with few or no experts left, +inf, NaN, the lowest f32, huge logits."""
    rng = np.random.default_rng(E + G)
    k = 6
    l = rng.standard_normal((10, E)).astype(np.float32)
    l[0] = -np.inf
    l[1] = np.nan
    l[2] = -np.inf
    l[2, E - 1] = 0.5
    l[3, ::2] = np.nan
    l[4, 3] = np.inf
    l[5, [1, E - 2]] = np.inf
    l[6] = np.finfo(np.float32).min
    l[7, :] = -np.inf
    l[7, [0, E // 2, E - 1]] = [3.0, -2.0, 1.0]
    l[8] *= 1e30
    l[9, 1:] = np.finfo(np.float32).min
    for rank in (1, 2):
        ids, wts = check(gemv, l, k, score, G=G, tg=tg, rank=rank)
        assert not ids[:2].any() and not wts[:2].any()
        bias = np.zeros(E, np.float32)
        bias[:E // 2] = -np.inf
        bias[E - 1] = np.nan
        check(gemv, l, k, score, G=G, tg=tg, rank=rank, bias=bias)


def test_agrees_with_topk_router(gemv):
    """Softmax scores renormalised over the chosen are the softmax over the top-k: the same ids, weights within
    the f32 roundings of that launch (exp, sum of 8, quotient: under 2^-20)."""
    rng = np.random.default_rng(2)
    n, E, k = 40, 128, 8
    l, es = dev(rng.standard_normal((n, E)).astype(np.float32)), dev(rng.uniform(0.5, 2, E).astype(np.float32))
    ids, wts = torch.zeros((2, n, k), dtype=torch.int32, device=DEV), torch.zeros((2, n, k), device=DEV)
    gemv.topk_router_dev(l, es, ids[0], wts[0], E, k, n)
    gemv.route_experts(l, ids[1], wts[1], E, k, n, expert_scale=es)
    assert torch.equal(ids[0], ids[1])
    assert float(((wts[0] - wts[1]).abs() / wts[0]).max()) < 2.0 ** -20


def test_same_bits_on_another_stream_and_captured(gemv):
    rng = np.random.default_rng(3)
    n, E, k = 65, 256, 8
    l, bias = dev(rng.standard_normal((n, E)).astype(np.float32)), dev(0.1 * rng.standard_normal(E).astype(np.float32))
    kw = dict(score=ft_hip.SCORE_SIGMOID, bias=bias, n_groups=8, top_groups=4, group_rank=2)

    def call():
        ids, wts = torch.zeros((n, k), dtype=torch.int32, device=DEV), torch.zeros((n, k), device=DEV)
        gemv.route_experts(l, ids, wts, E, k, n, **kw)
        return ids, wts

    first = call()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = call()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, other))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        captured = call()
    for seed in (1, 2, 3):
        l.copy_(dev(np.random.default_rng(seed).standard_normal((n, E)).astype(np.float32)))
        g.replay()
        want = call()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(captured, want))


def test_refused_by_the_python_side(gemv):
    l = torch.zeros((4, 16), device=DEV)
    ids, wts = torch.zeros((4, 2), dtype=torch.int32, device=DEV), torch.zeros((4, 2), device=DEV)
    bad = [dict(logits=l[:3]), dict(logits=l.half()), dict(ids=ids[:3]), dict(ids=ids.long()), dict(wts=wts.half()),
           dict(wts=wts[:, :1]), dict(bias=l[0, :15]), dict(expert_scale=l[0].double())]
    for change in bad:
        kw = dict(logits=l, ids=ids, wts=wts)
        kw.update(change)
        with pytest.raises(ft_hip.FtHipError) as e:
            gemv.route_experts(kw.pop("logits"), kw.pop("ids"), kw.pop("wts"), 16, 2, 4, **kw)
        assert e.value.code in (ft_hip.E_SHAPE, ft_hip.E_INVALID), change


@pytest.mark.parametrize("score", [ft_hip.SCORE_SOFTMAX, ft_hip.SCORE_SIGMOID])
@pytest.mark.parametrize("E", [6, 40, 300])
def test_scores_that_vanish(gemv, score, E):
    """Scores below the smallest number of f64 are equal (0 in 64 bits): the lower index first, weight 0."""
    l = np.full((3, E), -1000.0, np.float32)
    l[0, E - 1], l[0, 3] = 2.0, -900.0
    l[1, E // 2], l[1, 0] = 300.0, -1100.0
    l[2] = -3.0e38
    l[2, 1:3] = 3.0e38
    ids, wts = torch.zeros((3, 3), dtype=torch.int32, device=DEV), torch.zeros((3, 3), device=DEV)
    gemv.route_experts(dev(l), ids, wts, E, 3, 3, score=score)
    assert ids.tolist() == [[E - 1, 0, 1], [E // 2, 0, 1], [1, 2, 0]]
    assert wts.tolist() == [[1.0, 0.0, 0.0], [1.0, 0.0, 0.0], [0.5, 0.5, 0.0]]


def test_tensors_of_another_device_or_kind_are_refused(gemv):
    l = torch.zeros((4, 16), device=DEV)
    ids, wts = torch.zeros((4, 2), dtype=torch.int32, device=DEV), torch.zeros((4, 2), device=DEV)
    for change in (dict(logits=l.cpu()), dict(logits=l.int()), dict(ids=ids.cpu()), dict(wts=wts.cpu()),
                   dict(ids=wts), dict(wts=ids), dict(bias=l[0].cpu()), dict(bias=l[0].int()),
                   dict(expert_scale=l[0].cpu())):
        kw = dict(dict(logits=l, ids=ids, wts=wts), **change)
        with pytest.raises(ft_hip.FtHipError) as e:
            gemv.route_experts(kw.pop("logits"), kw.pop("ids"), kw.pop("wts"), 16, 2, 4, **kw)
        assert e.value.code in (ft_hip.E_SHAPE, ft_hip.E_INVALID), change
