"""The steps of a decode step that stand around the expert section, as cases that can be timed and compared.

Each case is one call of an operator of ft_hip.Q4Gemv on data as a decode loop or a prompt's chunk holds it:

  norm    the residual addition and RMS norm in front of a section (sandwich: the branch is normed before it is added),
          with the f32 row for the router and the q8 blocks for the q4 GEMVs (add_rmsnorm)
  route   experts chosen from router logits: softmax or sigmoid scores, a selection bias, groups of experts, top-k,
          renormalised and scaled weights (route_experts)
  sample  a token drawn from the vocabulary head's logits with temperature, top-k, top-p and min-p from a given
          random number (sample_tokens)

run() takes the plain torch form of each where `own` is false. Hidden sizes, expert counts and the 262,144-token
vocabulary are those of moe_synth's shapes; the others are generic.
"""
import math
import os
import sys

import torch

own = False

DEV = "cuda:0"
EPS = 1e-6
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # one new token of one conversation: the norm in front of its expert section, bound by latency
        dict(name="norm_token", kind="norm", n=1, hidden=2816, type="f32", sandwich=False, y=True),
        # sixty-four conversations decoding together, the attention's output in bf16, normed before it is added
        dict(name="norm_batch64", kind="norm", n=64, hidden=2816, type="bf16", sandwich=True, y=True),
        # a ragged chunk of a prompt where only the q4 GEMVs read the result
        dict(name="norm_chunk777", kind="norm", n=777, hidden=4096, type="f16", sandwich=False, y=False),
        # long prompts of a batch in one pass: the largest call, bound by memory
        dict(name="norm_prompt", kind="norm", n=16384, hidden=2816, type="f32", sandwich=True, y=True),
        # one new token's experts among 128
        dict(name="route_token", kind="route", n=1, experts=128, top_k=8, score="softmax", groups=1, top_groups=1,
             rank=1, bias=False, renorm=True, expert_scale=True),
        # a decoding batch on a model with groups of experts and a bias that balances them
        dict(name="route_batch64", kind="route", n=64, experts=256, top_k=8, score="sigmoid", groups=8, top_groups=4,
             rank=2, bias=True, renorm=True, expert_scale=False),
        # an odd chunk of a prompt, weights that are shares of all experts
        dict(name="route_chunk5003", kind="route", n=5003, experts=128, top_k=8, score="softmax", groups=1,
             top_groups=1, rank=1, bias=True, renorm=False, expert_scale=False),
        # long prompts in one pass, groups and bias
        dict(name="route_prompt", kind="route", n=16384, experts=256, top_k=8, score="sigmoid", groups=8, top_groups=4,
             rank=2, bias=True, renorm=True, expert_scale=False),
        # one conversation's next token, with the usual settings of a chat
        dict(name="sample_chat", kind="sample", n=1, vocab=262144, type="f32", filters="chat", masked=False),
        # a smaller vocabulary of odd size, logits of a bf16 head, a grammar that forbids part of the vocabulary
        dict(name="sample_masked9", kind="sample", n=9, vocab=50021, type="bf16", filters="min_p", masked=True),
        # a server's batch whose requests all have settings of their own
        dict(name="sample_mixed64", kind="sample", n=64, vocab=262144, type="f32", filters="mixed", masked=False),
        # the largest batch, nucleus sampling over the whole vocabulary
        dict(name="sample_nucleus256", kind="sample", n=256, vocab=262144, type="f32", filters="nucleus", masked=False),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["norm", "route", "sample"])
    if kind == "norm":
        hidden = 32 * _log_int(rng, 8, 256)
        return dict(kind=kind, n=_log_int(rng, 1, max(1, 16384 * 2816 // max(hidden, 2816))), hidden=hidden,
                    type=rng.choice(["f32", "f16", "bf16"]), sandwich=rng.random() < 0.5, y=rng.random() < 0.7)
    if kind == "route":
        groups = rng.choice([1, 1, 4, 8])
        experts = groups * rng.randint(max(2, 32 // groups), 320 // groups)
        top_groups = groups if groups == 1 else rng.randint(2, groups - 1)
        return dict(kind=kind, n=_log_int(rng, 1, 16384 * 256 // max(experts, 256)), experts=experts,
                    top_k=rng.randint(1, min(12, top_groups * (experts // groups))),
                    score=rng.choice(["softmax", "sigmoid"]), groups=groups, top_groups=top_groups,
                    rank=rng.choice([1, 2]), bias=rng.random() < 0.5, renorm=rng.random() < 0.6,
                    expert_scale=rng.random() < 0.3)
    vocab = _log_int(rng, 1000, 262144)
    return dict(kind=kind, n=_log_int(rng, 1, 255), vocab=vocab, type=rng.choice(["f32", "f32", "f16", "bf16"]),
                filters=rng.choice(["chat", "min_p", "mixed", "nucleus"]), masked=rng.random() < 0.3)


# ---- inputs, from the seed alone ----

def _inputs(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed * 7919 + 17)
    randn = lambda *s: torch.randn(s, generator=g, device=DEV)  # noqa: E731
    rand = lambda *s: torch.rand(s, generator=g, device=DEV)  # noqa: E731
    n, st = case["n"], {}
    if case["kind"] == "norm":
        h = case["hidden"]
        # a residual stream that has grown, with a few large channels, and a branch's output of about 1
        st["residual"] = randn(n, h).mul_(3.0).mul_(1.0 + 20.0 * (rand(h) > 0.995))
        st["x"] = randn(n, h).to(TYPES[case["type"]])
        st["w"] = 1.0 + 0.3 * randn(h)
        st["x_w"] = 0.5 + 0.2 * randn(h) if case["sandwich"] else None
    elif case["kind"] == "route":
        e = case["experts"]
        st["logits"] = randn(n, e) + 0.5 * randn(e)
        st["bias"] = 0.1 * randn(e) if case["bias"] else None
        st["expert_scale"] = 0.5 + rand(e) if case["expert_scale"] else None
    else:
        v = case["vocab"]
        logits = randn(n, v).mul_(2.5)
        # most rows know what comes next: 64 tokens stand out, falling with their rank; a quarter hardly does
        level = torch.where(rand(n, 1) < 0.25, 11.0, 20.0)
        at = torch.randint(0, v, (n, 64), generator=g, device=DEV)
        rank = torch.arange(1, 65, device=DEV, dtype=torch.float32)
        logits.scatter_(1, at, level - 1.5 * rank.log() + 0.5 * randn(n, 64))
        if case["masked"]:
            logits.masked_fill_(rand(n, v) < 0.3, -math.inf)
        st["logits"] = logits.to(TYPES[case["type"]])
        one, off = torch.ones(n, device=DEV), torch.zeros(n, device=DEV)
        u = rand(n, 4)
        kind = case["filters"]
        st["temperature"], st["top_k"], st["top_p"], st["min_p"] = one * 0.8, off.int(), one.clone(), off.clone()
        if kind == "chat":
            st["top_k"], st["top_p"] = (64 * one).int(), 0.95 * one
        elif kind == "min_p":
            st["temperature"], st["min_p"] = 1.2 * one, 0.02 * one
        elif kind == "nucleus":
            st["top_p"] = 0.9 * one
        else:  # each request its own; one in ten greedy
            st["temperature"] = torch.where(u[:, 0] < 0.1, off, 0.5 + u[:, 0])
            st["top_k"] = torch.where(u[:, 1] < 0.5, 1 + 200 * u[:, 1], off).int()
            st["top_p"] = torch.where(u[:, 2] < 0.7, 0.3 + u[:, 2], one)
            st["min_p"] = torch.where(u[:, 3] < 0.3, 0.2 * u[:, 3], off)
        st["u"] = rand(n)
    return st


def prepare(case, seed):
    st = dict(_inputs(case, seed), case=case)
    n = case["n"]
    if case["kind"] == "norm":  # the buffers that a decode loop keeps
        h = case["hidden"]
        st["h"] = torch.empty(n, h, device=DEV)
        st["y"] = torch.empty(n, h, device=DEV) if case["y"] else None
        st["q8"] = torch.empty(n * (h // 32) * 40, dtype=torch.uint8, device=DEV)
    elif case["kind"] == "route":
        st["ids"] = torch.empty(n, case["top_k"], dtype=torch.int32, device=DEV)
        st["wts"] = torch.empty(n, case["top_k"], device=DEV)
    else:
        st["tokens"], st["logprobs"] = torch.empty(n, dtype=torch.int32, device=DEV), torch.empty(n, device=DEV)
    return st


# ---- one pass ----

def _handle(st):
    """The library's handle and the workspace, as a program keeps them beside its buffers."""
    if "g" not in st:
        path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "freetoken-rs_amd")
        if path not in sys.path:
            sys.path.insert(0, path)
        import ft_hip
        st["g"], case = ft_hip.Q4Gemv(0), st["case"]
        if case["kind"] == "route":
            st["score"] = {"softmax": ft_hip.SCORE_SOFTMAX, "sigmoid": ft_hip.SCORE_SIGMOID}[case["score"]]
        if case["kind"] == "sample":
            st["ws"] = torch.empty(st["g"].sample_tokens_workspace_bytes(case["vocab"], case["n"]), dtype=torch.uint8,
                                   device=DEV)
    return st["g"]


def _blocks(q8, n, hidden):
    """The q8 blocks {f32 d; i32 qsum; i8 qs[32]} as what they hold, views of the buffer: the scales, the whole
    numbers' sums and the whole numbers."""
    words = q8.view(torch.float32).view(n, hidden // 32, 10)
    return {"d": words[:, :, 0], "qsum": q8.view(torch.int32).view(n, hidden // 32, 10)[:, :, 1],
            "qs": q8.view(torch.int8).view(n, hidden // 32, 40)[:, :, 8:]}


def _norm(st):
    case, x = st["case"], st["x"].double()
    if st["x_w"] is not None:
        x = x * torch.rsqrt(x.square().mean(1, keepdim=True) + EPS) * st["x_w"]
    h = (x + st["residual"]).float()
    inv = torch.rsqrt(h.square().mean(1, keepdim=True) + EPS)
    # the blocks' roundings are borders: in 64 bits
    u = (h * st["w"]).double().view(case["n"], -1, 32)
    amax = u.abs().amax(2, keepdim=True)
    q = torch.where(amax > 0, 127.0 * u.abs() / amax + 0.5, 0.0).floor().mul(u.sign()).to(torch.int8)
    out = {"h": h, "d": amax[:, :, 0].div(127.0).mul(inv).float(), "qs": q, "qsum": q.sum(2, dtype=torch.int32)}
    if case["y"]:
        out["y"] = h * inv * st["w"]
    return out


def _route(st):
    case, l = st["case"], st["logits"].double()  # which expert comes first is a border: in 64 bits
    n, e, groups = case["n"], case["experts"], case["groups"]
    if case["score"] == "softmax":
        s = (l - l.amax(1, keepdim=True)).exp()
        s = s / s.sum(1, keepdim=True)
    else:
        s = 1.0 / (1.0 + (-l).exp())
    c = s if st["bias"] is None else s + st["bias"]
    if groups > 1:
        by = c.view(n, groups, e // groups)
        best = by.sort(dim=2, descending=True).values[:, :, :case["rank"]].sum(2)
        first = best.sort(dim=1, descending=True, stable=True).indices[:, :case["top_groups"]]
        open_ = torch.zeros(n, groups, dtype=torch.bool, device=DEV).scatter_(1, first, True)
        c = torch.where(open_.unsqueeze(2), by, -math.inf).view(n, e)
    ids = c.sort(dim=1, descending=True, stable=True).indices[:, :case["top_k"]]
    w = s.gather(1, ids)
    if case["renorm"]:
        w = w / w.sum(1, keepdim=True)
    w = w * 2.5
    if st["expert_scale"] is not None:
        w = w * st["expert_scale"][ids]
    return {"ids": ids.int(), "wts": w.float()}


def _sample(st):
    # where the cumulative sums pass top_p and the random number is a border: in 64 bits
    l = st["logits"].double()
    n, v = l.shape
    top = l.amax(1, keepdim=True)
    t = st["temperature"].double().unsqueeze(1)
    greedy = t <= 0
    e = ((l - top) / torch.where(greedy, 1.0, t)).exp()
    order = l.sort(dim=1, descending=True, stable=True).indices
    es, rank = e.gather(1, order), torch.arange(v, device=DEV)
    k = st["top_k"].unsqueeze(1)
    k = torch.where(greedy, 1, torch.where(k <= 0, v, k))
    es = es * (rank < k)
    c = es.cumsum(1)
    before = torch.cat([torch.zeros_like(c[:, :1]), c[:, :-1]], 1)
    p = st["top_p"].double().unsqueeze(1)
    m = st["min_p"].double().clamp(max=1).unsqueeze(1)
    keep = (es > 0) & ((p >= 1) | (rank == 0) | (before < p * c[:, -1:])) & (es >= m)
    w = torch.zeros_like(es).scatter_(1, order, es * keep)
    c = w.cumsum(1)
    token = (c <= st["u"].double().unsqueeze(1) * c[:, -1:]).sum(1, keepdim=True).clamp(max=v - 1)
    return {"tokens": token[:, 0].int(), "logprobs": (w.gather(1, token) / c[:, -1:]).log()[:, 0].float()}


def run(st):
    case = st["case"]
    if own:
        g = _handle(st)
        if case["kind"] == "norm":
            g.add_rmsnorm(st["x"], st["w"], case["hidden"], case["n"], EPS, residual=st["residual"], h=st["h"],
                          y=st["y"], q8=st["q8"], x_w=st["x_w"])
            if "blocks" not in st:  # views of the buffer that it keeps
                st["blocks"] = _blocks(st["q8"], case["n"], case["hidden"])
            out = dict(st["blocks"], h=st["h"])
            if case["y"]:
                out["y"] = st["y"]
            return out
        if case["kind"] == "route":
            g.route_experts(st["logits"], st["ids"], st["wts"], case["experts"], case["top_k"], case["n"],
                            score=st["score"], bias=st["bias"], n_groups=case["groups"],
                            top_groups=case["top_groups"], group_rank=case["rank"], renorm=case["renorm"], scale=2.5,
                            expert_scale=st["expert_scale"])
            return {"ids": st["ids"], "wts": st["wts"]}
        g.sample_tokens(st["logits"], case["vocab"], case["n"], st["u"], st["tokens"], st["ws"],
                        temperature=st["temperature"], top_k=st["top_k"], top_p=st["top_p"], min_p=st["min_p"],
                        logprobs=st["logprobs"])
        return {"tokens": st["tokens"], "logprobs": st["logprobs"]}
    return _norm(st) if case["kind"] == "norm" else _route(st) if case["kind"] == "route" else _sample(st)


# ---- what a pass cannot do without ----

def work(case):
    n = case["n"]
    size = {"f32": 4, "f16": 2, "bf16": 2}
    if case["kind"] == "norm":
        h = case["hidden"]
        per = size[case["type"]] + 4 + 4 + (4 if case["y"] else 0) + 40 / 32
        return {"bytes": n * h * per + h * (8 if case["sandwich"] else 4),
                "flops": n * h * (14 if case["sandwich"] else 10)}
    if case["kind"] == "route":
        e = case["experts"]
        return {"bytes": n * (e * 4 + case["top_k"] * 8) + e * 4 * (case["bias"] + case["expert_scale"]),
                "flops": n * e * 6}
    return {"bytes": n * (case["vocab"] * size[case["type"]] + 28), "flops": n * case["vocab"] * 6}


# ---- the same in 64 bits, from the definitions ----

def exact(case, seed):
    st = _inputs(case, seed)
    n = case["n"]
    if case["kind"] == "norm":
        def rms(v):
            return (v * v).sum(1, keepdim=True).div_(v.shape[1]).add_(EPS).sqrt_()
        x = st["x"].to(torch.float64)
        if case["sandwich"]:
            x = x / rms(x) * st["x_w"].to(torch.float64)
        h = x + st["residual"].to(torch.float64)
        del x
        y = h / rms(h) * st["w"].to(torch.float64)
        d = y.reshape(n, case["hidden"] // 32, 32).abs().max(dim=2).values / 127.0
        out = {"h": h, "d": d, "qs": None, "qsum": None}  # the whole numbers have to be equal
        if case["y"]:
            out["y"] = y
        return out
    if case["kind"] == "route":
        l = st["logits"].to(torch.float64)
        s = torch.softmax(l, dim=1) if case["score"] == "softmax" else torch.sigmoid(l)
        c = s.clone() if st["bias"] is None else s + st["bias"].to(torch.float64)
        if case["groups"] > 1:
            size = case["experts"] // case["groups"]
            of = torch.stack([c[:, i * size:(i + 1) * size].topk(case["rank"], dim=1).values.sum(1)
                              for i in range(case["groups"])], dim=1)
            last = of.topk(case["top_groups"], dim=1).values[:, -1:]
            c.masked_fill_((of < last).repeat_interleave(size, dim=1), -math.inf)
        ids = c.topk(case["top_k"], dim=1).indices
        w = torch.gather(s, 1, ids)
        if case["renorm"]:
            w /= w.sum(1, keepdim=True)
        w *= 2.5
        if case["expert_scale"]:
            w *= st["expert_scale"].to(torch.float64)[ids]
        return {"ids": ids.int(), "wts": w}
    tokens, logprobs = [], []
    for i in range(n):  # row by row, on the probabilities themselves
        row = st["logits"][i].to(torch.float64)
        t, k, p, m, u = (float(st[name][i]) for name in ("temperature", "top_k", "top_p", "min_p", "u"))
        if t <= 0:
            tokens.append(int((row == row.max()).nonzero()[0]))
            logprobs.append(0.0)
            continue
        prob = torch.softmax(row / t, dim=0)
        falling, order = torch.sort(row, descending=True, stable=True)
        share = prob[order]
        kept = int(k) if 0 < k < row.numel() else row.numel()
        total = torch.cumsum(share[:kept], 0)
        if p < 1:
            kept = min(kept, int((total < p * total[-1]).sum()) + 1)
        kept = min(kept, int((share[:kept] >= m * share[0]).sum()))
        kept = min(kept, int((share[:kept] > 0).sum()))
        index = torch.sort(order[:kept]).values
        total = torch.cumsum(prob[index], 0)
        at = min(int(torch.searchsorted(total, total[-1:] * u, right=True)), kept - 1)
        tokens.append(int(index[at]))
        logprobs.append(math.log(float(prob[index[at]] / total[-1])))
    return {"tokens": torch.tensor(tokens, dtype=torch.int32), "logprobs": torch.tensor(logprobs, dtype=torch.float64)}
