"""What stands between a decode step's projections and its draw, as cases that can be timed and compared.

Each case is one call of an operator of ft_hip.Q4Gemv on data as a decode loop holds it:

  write   keys and values quantised into the pages of a cache, a scale a token and head (kv_write)
  read    tokens of the cache read back (kv_read)
  attn    attention of a batch's newest tokens over the quantised cache, with a prefix that all sequences share, a
          window, and sequences of their own lengths (attention)
  logits  penalties for repeated tokens, biases and a grammar's mask on a vocabulary's logits, in front of the draw
          (adjust_logits)

run() takes the plain torch form of each where `own` is false. 16 query heads on 8 key heads of 256 are the widths of
moe_synth's dense projections, the 262,144-token vocabulary is its head's; the other sizes are generic.

A page of P tokens holds, for each key head, P x D bytes of keys, P x D of values, P f32 scales of the keys and P of
the values. Keys lie as [P / 16][D / 16][16 tokens][16 dimensions], values as [P / 16][D / 64][4 groups][64 dimensions]
[4 tokens]. i8: the byte is q + 128, the value q times the scale; e4m3: the byte is the code, the scale a power of two.
"""
import math
import os
import sys

import torch

own = False

DEV = "cuda:0"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # one new token of one conversation, from the f32 projections: bound by latency
        dict(name="write_token", kind="write", n=1, heads=8, dim=256, page=64, cache="i8", type="f32"),
        # the chunks of several long prompts in one pass: the largest write, bound by memory
        dict(name="write_prompt", kind="write", n=16387, heads=8, dim=128, page=64, cache="e4m3", type="bf16"),
        # a short, odd number of tokens read back
        dict(name="read_few", kind="read", n=333, heads=4, dim=64, page=16, cache="i8", type="f16"),
        # a long prompt's keys and values in 16 bits, for a pass that wants them wide
        dict(name="read_prompt", kind="read", n=32768, heads=8, dim=256, page=128, cache="e4m3", type="bf16"),
        # one conversation's next token on the widths of the dense projections: bound by latency
        dict(name="attn_token", kind="attn", n=1, heads=16, kv_heads=8, dim=256, page=64, cache="i8", type="f32",
             own=777, n_q=1, window=0, prefix=0, padded=False, lse=False),
        # one conversation with a very long history: a long axis and few rows
        dict(name="attn_long", kind="attn", n=1, heads=32, kv_heads=8, dim=128, page=64, cache="e4m3", type="bf16",
             own=131071, n_q=1, window=0, prefix=0, padded=False, lse=False),
        # sixty-four conversations of all lengths decoding together
        dict(name="attn_batch64", kind="attn", n=64, heads=16, kv_heads=8, dim=256, page=64, cache="i8", type="f32",
             own=4096, n_q=1, window=0, prefix=0, padded=False, lse=False),
        # a layer with a sliding window in a padded batch that verifies three guessed tokens
        dict(name="attn_window", kind="attn", n=45, heads=24, kv_heads=8, dim=64, page=16, cache="i8", type="f16",
             own=9000, n_q=3, window=1024, prefix=0, padded=True, lse=True),
        # sixty-four conversations behind one system prompt
        dict(name="attn_prefix64", kind="attn", n=64, heads=16, kv_heads=8, dim=256, page=64, cache="i8", type="f32",
             own=512, n_q=1, window=0, prefix=8192, padded=False, lse=False),
        # the largest batch, behind a long document that all ask about
        dict(name="attn_prefix256", kind="attn", n=256, heads=64, kv_heads=8, dim=128, page=128, cache="e4m3",
             type="bf16", own=300, n_q=1, window=0, prefix=16390, padded=False, lse=True),
        # one conversation's logits with a penalty for repeated tokens and a few biased ones
        dict(name="logits_chat", kind="logits", n=1, vocab=262144, type="f32", history=1500, bias=20, mask=False),
        # a server's batch whose answers follow grammars
        dict(name="logits_grammar64", kind="logits", n=64, vocab=262144, type="bf16", history=6000, bias=100,
             mask=True),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["write", "read", "attn", "attn", "attn", "logits"])
    base = dict(kind=kind, page=rng.choice([16, 32, 64, 128]), cache=rng.choice(["i8", "e4m3"]),
                type=rng.choice(["f32", "f16", "bf16"]), dim=rng.choice([64, 128, 256]))
    if kind in ("write", "read"):
        base["heads"] = rng.choice([1, 2, 3, 4, 8])
        most = (16387 if kind == "write" else 32768) * 1024 // (base["heads"] * base["dim"])
        return dict(base, n=_log_int(rng, 1, min(65536, most)))
    if kind == "logits":
        vocab = _log_int(rng, 1000, 262144)
        return dict(kind=kind, n=_log_int(rng, 1, 64), vocab=vocab, type=base["type"],
                    history=_log_int(rng, 1, 20000) if rng.random() < 0.8 else 0,
                    bias=rng.choice([0, 1, 17, 300]), mask=rng.random() < 0.5)
    kv = rng.choice([1, 2, 4, 8])
    n, heads = _log_int(rng, 1, 256), kv * rng.choice([1, 2, 3, 4, 8])
    n_q = rng.choice([1, 1, 1, 2, 5])
    most = min(131071, 2097152 * 1024 // (n * kv * base["dim"] * 8))  # tokens of the longest
    longest = min(16390, 16390 * 256 * 64 * 128 // (n * n_q * heads * base["dim"]))
    prefix = _log_int(rng, 1, longest) if rng.random() < 0.5 else 0
    return dict(base, n=n, heads=heads, kv_heads=kv, own=max(n_q, _log_int(rng, 1, most)), n_q=n_q,
                window=_log_int(rng, 1, 8192) if rng.random() < 0.3 else 0, prefix=prefix,
                padded=rng.random() < 0.3, lse=rng.random() < 0.5)


# ---- inputs, from the seed alone ----

def _lens(case):
    """The sequences' lengths in falling shares of the longest, in an order that the seed decides; a padded batch ends
    some of them at 0."""
    n, most, n_q = case["n"], case["own"], case["n_q"]
    lens = [max(n_q, int(round(most * (1.0 - i / n) ** 2))) for i in range(n)]
    if case["padded"]:
        lens = [0 if i % 7 == 3 else v for i, v in enumerate(lens)]
    return lens


def _pages_of(case, tokens):
    return (tokens + case["page"] - 1) // case["page"]


def _cache(case, n_pages, g):
    """A cache in use: quantised normal values, scales that vary by token, the first tokens' keys larger."""
    h, d, p = case.get("kv_heads", case.get("heads")), case["dim"], case["page"]
    cache = torch.empty((n_pages, h, p * (2 * d + 8)), dtype=torch.uint8, device=DEV)
    v = _views(cache, case)
    at = 0
    while at < n_pages:  # a few hundred MiB of normal values at a time
        to = min(n_pages, at + max(1, (1 << 26) // (h * p * 2 * d)))
        x = torch.randn((to - at, h, 2 * p * d), generator=g, device=DEV)
        if case["cache"] == "i8":
            cache[at:to, :, :2 * p * d] = x.mul_(36.0).round_().clamp_(-127, 127).add_(128).to(torch.uint8)
            scale = 1.0 / 36.0
        else:
            cache[at:to, :, :2 * p * d] = x.mul_(64.0).to(torch.float8_e4m3fn).view(torch.uint8)
            scale = 1.0 / 64.0
        at = to
    for name in ("ks", "vs"):
        s = torch.randint(-1, 2, v[name].shape, generator=g, device=DEV).float().exp2_().mul_(scale)
        if case["cache"] == "i8":
            s *= 0.75 + 0.5 * torch.rand(v[name].shape, generator=g, device=DEV)
        v[name].copy_(s)
    return cache


def _views(cache, case):
    """The cache's parts where they lie; e4m3 codes as what they stand for."""
    h, d, p = case.get("kv_heads", case.get("heads")), case["dim"], case["page"]
    n = cache.shape[0]
    q = cache if case["cache"] == "i8" else cache.view(torch.float8_e4m3fn)
    f = cache.view(torch.float32)
    return {"k": q[:, :, :p * d].view(n, h, p // 16, d // 16, 16, 16),
            "v": q[:, :, p * d:2 * p * d].view(n, h, p // 16, d // 64, 4, 64, 4),
            "ks": f[:, :, p * d // 2:p * d // 2 + p], "vs": f[:, :, p * d // 2 + p:]}


def _inputs(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed * 7919 + 29)
    randn = lambda *s: torch.randn(s, generator=g, device=DEV)  # noqa: E731
    rand = lambda *s: torch.rand(s, generator=g, device=DEV)  # noqa: E731
    kind, st = case["kind"], {}
    if kind in ("write", "read"):
        n, h, d = case["n"], case["heads"], case["dim"]
        pages = _pages_of(case, n + 5) + 2
        order = torch.randperm(pages, generator=g, device=DEV)
        at = torch.arange(5, n + 5, device=DEV)  # a sequence that goes on behind its first five tokens
        st["slots"] = (order[at // case["page"]] * case["page"] + at % case["page"]).int()
        st["cache"] = _cache(case, pages, g)
        if kind == "write":
            # the keys' and values' columns of a row of projections; a few large channels in the keys
            rows = randn(n, 2 * h * d)
            rows[:, :h * d] *= 1.0 + 8.0 * (rand(h * d) > 0.98)
            rows = rows.to(TYPES[case["type"]])
            st["k"], st["v"] = rows[:, :h * d], rows[:, h * d:]
    elif kind == "attn":
        lens = _lens(case)
        width = _pages_of(case, case["own"])
        order = torch.randperm(case["n"], generator=g, device=DEV)
        lens = torch.tensor(lens, dtype=torch.int32, device=DEV)[order]
        need = (lens + case["page"] - 1) // case["page"]
        first = need.cumsum(0) - need
        shared = _pages_of(case, case["prefix"])
        pages = sum(_pages_of(case, v) for v in _lens(case)) + shared + 1
        where = torch.randperm(pages, generator=g, device=DEV).int()
        col = torch.arange(width, device=DEV)
        at = torch.where(col < need[:, None], first[:, None] + col, pages - 1)
        st["tables"], st["lens"] = where[at], lens
        st["prefix"] = where[pages - 1 - shared:pages - 1].clone() if shared else None
        st["prefix_len"] = torch.full((1,), case["prefix"], dtype=torch.int32, device=DEV) if shared else None
        st["cache"] = _cache(case, pages, g)
        # queries that look for some keys more than for others
        st["q"] = (1.5 * randn(case["n"] * case["n_q"], case["heads"] * case["dim"])).to(TYPES[case["type"]])
    else:
        n, v = case["n"], case["vocab"]
        st["logits"] = randn(n, v).mul_(2.5).to(TYPES[case["type"]])
        if case["history"]:
            # words by a falling law, the same ones again and again
            st["history"] = (v * rand(n, case["history"]) ** 6).int().clamp_(0, v - 1)
            st["history_len"] = (case["history"] * (0.2 + 0.8 * rand(n))).int().clamp_(min=1)
            st["repetition"], st["presence"], st["frequency"] = 1.0 + 0.4 * rand(n), 0.5 * rand(n), 0.3 * rand(n)
        if case["bias"]:
            ids = rand(n, v).topk(case["bias"], dim=1).indices
            st["bias_ids"] = torch.where(rand(n, case["bias"]) < 0.2, -1, ids).int()  # some places are free
            st["bias"] = 4.0 * randn(n, case["bias"])
        if case["mask"]:
            st["mask"] = torch.randint(-2 ** 31, 2 ** 31, (n, (v + 31) // 32), generator=g, device=DEV).int()
    return st


def prepare(case, seed):
    st = dict(_inputs(case, seed), case=case)
    n = case["n"]
    if case["kind"] == "read":  # the buffers that a decode loop keeps
        for name in "kv":
            st[name] = torch.empty((n, case["heads"] * case["dim"]), dtype=TYPES[case["type"]], device=DEV)
    elif case["kind"] == "attn":
        st["out"] = torch.empty_like(st["q"])
        st["lse"] = torch.empty((n * case["n_q"], case["heads"]), device=DEV) if case["lse"] else None
    elif case["kind"] == "logits":
        st["out"] = torch.empty((n, case["vocab"]), device=DEV)
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
        if case["kind"] != "logits":
            st["cache_type"] = {"i8": ft_hip.KV_I8, "e4m3": ft_hip.KV_E4M3}[case["cache"]]
        if case["kind"] == "attn":
            st["ws"] = torch.empty(st["g"].attention_workspace_bytes(case["n"], case["n_q"], case["heads"],
                                                                     case["kv_heads"], case["dim"]),
                                   dtype=torch.uint8, device=DEV)
    return st["g"]


def _rows_of(view, slots, page, value):
    """A view of the cache's keys, values or scales, by token: [..., heads, ...]; with the tokens' places in it."""
    at, o = slots // page, slots % page
    if value == "k":
        return view.permute(0, 2, 4, 1, 3, 5), (at, o // 16, o % 16)
    if value == "v":
        return view.permute(0, 2, 4, 6, 1, 3, 5), (at, o // 16, o % 16 // 4, o % 4)
    return view.permute(0, 2, 1), (at, o)


def _quantised(x, cache):
    """(codes, scales) of rows of values [n, heads, dim]. The roundings are borders: in 64 bits."""
    u = x.double()
    a = u.abs().amax(2, keepdim=True)
    one = torch.where(a > 0, a, 1.0)
    if cache == "i8":
        q = (127.0 * u.abs() / one + 0.5).floor() * u.sign()
        return (q + 128).to(torch.uint8), (a / 127.0).float()[:, :, 0]
    mant, ex = torch.frexp(one)
    scale = torch.ldexp(torch.ones_like(one), ex - 9 + (mant > 0.875))
    y = u.abs() / scale
    step = torch.ldexp(torch.ones_like(y), torch.frexp(y).exponent.clamp(min=-5) - 4)  # 8 steps to a power of two
    y = torch.copysign((y / step).round() * step, u)
    return y.float().to(torch.float8_e4m3fn), torch.where(a > 0, scale, 0.0).float()[:, :, 0]


def _write(st):
    case, n = st["case"], st["case"]["n"]
    views, slots = _views(st["cache"], case), st["slots"].long()
    raw = dict(views, k=views["k"].view(torch.uint8), v=views["v"].view(torch.uint8))
    for name, inner in (("k", 16), ("v", 64)):
        q, scale = _quantised(st[name].view(n, case["heads"], case["dim"]), case["cache"])
        view, at = _rows_of(raw[name], slots, case["page"], name)
        view[at] = q.view(torch.uint8).view(n, case["heads"], case["dim"] // inner, inner)
        view, at = _rows_of(raw[name + "s"], slots, case["page"], "s")
        view[at] = scale
    return views


def _tokens(cache, case, slots, heads):
    """Keys and values of tokens in 32 bits: [..., heads, dim]."""
    views = _views(cache, case)
    out = []
    for name in "kv":
        view, at = _rows_of(views[name].view(torch.uint8), slots, case["page"], name)
        q = view[at]
        q = q.float() - 128.0 if case["cache"] == "i8" else q.view(torch.float8_e4m3fn).float()
        view, at = _rows_of(views[name + "s"], slots, case["page"], "s")
        out.append(q.reshape(*slots.shape, heads, case["dim"]) * view[at].unsqueeze(-1))
    return out


def _read(st):
    case = st["case"]
    k, v = _tokens(st["cache"], case, st["slots"].long(), case["heads"])
    return {"k": k.to(TYPES[case["type"]]).view(case["n"], -1), "v": v.to(TYPES[case["type"]]).view(case["n"], -1)}


def _attn(st):
    case = st["case"]
    n, n_q, kv, d, page = case["n"], case["n_q"], case["kv_heads"], case["dim"], case["page"]
    group, most, shared = case["heads"] // kv, case["own"], case["prefix"]
    lens = st["lens"].long()
    # rows of queries by key head: [n, kv, n_q * group, d]
    q = st["q"].float().view(n, n_q, kv, group, d).transpose(1, 2).reshape(n, kv, n_q * group, d) / math.sqrt(d)
    j = torch.arange(most, device=DEV)
    slots = st["tables"].long()[:, j // page] * page + j % page
    k, v = _tokens(st["cache"], case, slots, kv)
    k, v = k.permute(0, 2, 3, 1).contiguous(), v.transpose(1, 2).contiguous()
    o = lens[:, None] - n_q + torch.arange(n_q, device=DEV)  # the queries' places among their own tokens
    seen = (o[:, :, None] >= 0) & (j <= o[:, :, None])
    if case["window"]:
        seen &= j > o[:, :, None] - case["window"]
    s = torch.where(seen[:, None, :, None, :], torch.matmul(q, k).view(n, kv, n_q, group, most), -math.inf)
    if shared:
        i = torch.arange(shared, device=DEV)
        pk, pv = _tokens(st["cache"], case, st["prefix"].long()[i // page] * page + i % page, kv)
        rows = q.transpose(0, 1).reshape(kv, n * n_q * group, d)
        ps = torch.matmul(rows, pk.permute(1, 2, 0).contiguous()).view(kv, n, n_q, group, shared).transpose(0, 1)
        seen = (o[:, :, None] >= 0).expand(n, n_q, shared)
        if case["window"]:
            seen = seen & (i > shared + o[:, :, None] - case["window"])
        ps = torch.where(seen[:, None, :, None, :], ps, -math.inf)
        m = torch.maximum(s.amax(4, keepdim=True), ps.amax(4, keepdim=True))
    else:
        m = s.amax(4, keepdim=True)
    m = torch.where(m > -math.inf, m, 0.0)
    s = (s - m).exp()
    total = s.sum(4, keepdim=True)
    out = torch.matmul(s.view(n, kv, n_q * group, most), v).view(n, kv, n_q, group, d)
    if shared:
        ps = (ps - m).exp()
        total = total + ps.sum(4, keepdim=True)
        rows = ps.transpose(0, 1).reshape(kv, n * n_q * group, shared)
        out = out + torch.matmul(rows, pv.transpose(0, 1).contiguous()).view(kv, n, n_q, group, d).transpose(0, 1)
    lse = (m + total.log())[..., 0]
    out = torch.where(total > 0, out / total, 0.0)
    out = {"out": out.transpose(1, 2).reshape(n * n_q, -1).to(st["q"].dtype)}
    if case["lse"]:
        out["lse"] = lse.transpose(1, 2).reshape(n * n_q, -1)
    return out


def _logits(st):
    case = st["case"]
    n, v = case["n"], case["vocab"]
    x = st["logits"].float()
    if case["history"]:
        live = torch.arange(case["history"], device=DEV) < st["history_len"][:, None]
        count = torch.zeros((n, v), dtype=torch.int32, device=DEV).scatter_add_(1, st["history"].long(), live.int())
        rep = st["repetition"][:, None]
        y = torch.where(x > 0, x / rep, x * rep) - (st["presence"][:, None] + st["frequency"][:, None] * count)
        x = torch.where(count > 0, y, x)
    if case["bias"]:
        free = st["bias_ids"] < 0
        add = torch.zeros((n, v), device=DEV)
        add.scatter_add_(1, torch.where(free, 0, st["bias_ids"]).long(), torch.where(free, 0.0, st["bias"]))
        x = x + add
    if case["mask"]:
        i = torch.arange(v, device=DEV)
        x = torch.where((st["mask"][:, i // 32] >> (i % 32)) & 1 == 1, x, -math.inf)
    return {"out": x}


def run(st):
    case = st["case"]
    if own:
        g = _handle(st)
        if case["kind"] == "write":
            g.kv_write(st["k"], st["v"], st["slots"], st["cache"], case["n"], case["heads"], case["dim"], case["page"],
                       cache_type=st["cache_type"])
            if "views" not in st:  # views of the buffer that it keeps
                st["views"] = _views(st["cache"], case)
            return st["views"]
        if case["kind"] == "read":
            g.kv_read(st["cache"], st["slots"], st["k"], st["v"], case["n"], case["heads"], case["dim"], case["page"],
                      cache_type=st["cache_type"])
            return {"k": st["k"], "v": st["v"]}
        if case["kind"] == "attn":
            g.attention(st["q"], st["cache"], st["tables"], st["lens"], st["out"], st["ws"], case["n"], case["heads"],
                        case["kv_heads"], case["dim"], case["page"], case["dim"] ** -0.5, n_q=case["n_q"],
                        window=case["window"], prefix=st["prefix"], prefix_len=st["prefix_len"], lse=st["lse"],
                        cache_type=st["cache_type"])
            return {"out": st["out"], "lse": st["lse"]} if case["lse"] else {"out": st["out"]}
        g.adjust_logits(st["logits"], st["out"], case["vocab"], case["n"], history=st.get("history"),
                        history_len=st.get("history_len"), repetition=st.get("repetition"),
                        presence=st.get("presence"), frequency=st.get("frequency"), bias_ids=st.get("bias_ids"),
                        bias=st.get("bias"), mask=st.get("mask"))
        return {"out": st["out"]}
    return {"write": _write, "read": _read, "attn": _attn, "logits": _logits}[case["kind"]](st)


# ---- what a pass cannot do without ----

def work(case):
    n, size = case["n"], {"f32": 4, "f16": 2, "bf16": 2}[case["type"]]
    if case["kind"] in ("write", "read"):
        values = 2 * n * case["heads"] * case["dim"]
        return {"bytes": values * (size + 1) + 8 * n * case["heads"] + 4 * n, "flops": 4 * values}
    if case["kind"] == "logits":
        each = 4 * case["history"] + 8 * case["bias"] + (case["vocab"] / 8 if case["mask"] else 0)
        return {"bytes": n * (case["vocab"] * (size + 4) + each), "flops": n * (case["vocab"] + case["history"])}
    n_q, w, shared = case["n_q"], case["window"], case["prefix"]
    own_tokens, pairs, least = 0, 0, shared
    for length in _lens(case):
        if not length:
            continue
        own_tokens += min(length, w + n_q - 1) if w else length
        for o in range(length - n_q, length):
            pairs += min(o + 1 + shared, w) if w else o + 1 + shared
        least = min(least, max(0, shared + length - n_q + 1 - w) if w else 0)
    token = case["kv_heads"] * (2 * case["dim"] + 8)
    q = n * n_q * case["heads"]
    return {"bytes": (own_tokens + shared - least) * token + 2 * size * q * case["dim"] + (4 * q if case["lse"] else 0),
            "flops": 4 * pairs * case["heads"] * case["dim"]}


# ---- the same in 64 bits, from the definitions ----

def _wide(cache, case, slots, heads):
    """Keys and values of tokens [heads, tokens, dim], from the bytes' addresses."""
    d, p = case["dim"], case["page"]
    flat, floats = cache.reshape(-1), cache.reshape(-1).view(torch.float32)
    base = (slots // p)[None, :] * heads + torch.arange(heads, device=DEV)[:, None]  # the head's block in its page
    base = base * (p * (2 * d + 8))
    o, i = (slots % p)[None, :, None], torch.arange(d, device=DEV)
    places = (o // 16 * 16 * d + i // 16 * 256 + o % 16 * 16 + i % 16,
              p * d + o // 16 * 16 * d + i // 64 * 1024 + o % 16 // 4 * 256 + i % 64 * 4 + o % 4)
    out = []
    for at, place in enumerate(places):
        code = flat[base[:, :, None] + place]
        q = code.to(torch.float64) - 128 if case["cache"] == "i8" else code.view(torch.float8_e4m3fn).to(torch.float64)
        out.append(q * floats[(base + 2 * p * d + at * 4 * p) // 4 + (slots % p)[None, :]].to(torch.float64)[:, :, None])
    return out


def exact(case, seed):
    st = _inputs(case, seed)
    n, kind = case["n"], case["kind"]
    if kind == "write":
        return None  # codes and scales are roundings that have to be equal
    if kind == "read":
        k, v = _wide(st["cache"], case, st["slots"].long(), case["heads"])
        return {"k": k.transpose(0, 1).reshape(n, -1), "v": v.transpose(0, 1).reshape(n, -1)}
    if kind == "logits":
        x = st["logits"].to(torch.float64)
        for i in range(n):  # row by row, token by token of the lists
            row = x[i]
            if case["history"]:
                seen, count = st["history"][i, :int(st["history_len"][i])].long().unique(return_counts=True)
                r, p, f = (float(st[name][i]) for name in ("repetition", "presence", "frequency"))
                was = row[seen]
                row[seen] = torch.where(was > 0, was / r, was * r) - p - f * count
            if case["bias"]:
                used = st["bias_ids"][i] >= 0
                row[st["bias_ids"][i][used].long()] += st["bias"][i][used].to(torch.float64)
            if case["mask"]:
                bits = (st["mask"][i].to(torch.int64)[:, None] >> torch.arange(32, device=DEV)) & 1
                row[bits.view(-1)[:case["vocab"]] == 0] = -math.inf
        return {"out": x}
    n_q, kv, d, page, w, shared = (case[name] for name in ("n_q", "kv_heads", "dim", "page", "window", "prefix"))
    group = case["heads"] // kv
    q = st["q"].to(torch.float64).view(n, n_q, kv, group, d)
    out = torch.zeros((n, n_q, kv, group, d), dtype=torch.float64, device=DEV)
    lse = torch.full((n, n_q, kv, group), -math.inf, dtype=torch.float64, device=DEV)
    if shared:
        i = torch.arange(shared, device=DEV)
        pk, pv = _wide(st["cache"], case, st["prefix"].long()[i // page] * page + i % page, kv)
        pk = pk.transpose(1, 2).contiguous()
    lens = st["lens"].tolist()
    for i in range(n):  # sequence by sequence, over the prefix and its own tokens in one row
        length = lens[i]
        if not length:
            continue
        j = torch.arange(length, device=DEV)
        k, v = _wide(st["cache"], case, st["tables"][i].long()[j // page] * page + j % page, kv)
        for t in range(max(0, n_q - length), n_q):
            s = torch.bmm(q[i, t], k.transpose(1, 2).contiguous())
            if shared:
                s = torch.cat([torch.bmm(q[i, t], pk), s], 2)
            s /= math.sqrt(d)
            at = shared + length - n_q + t
            s[:, :, at + 1:] = -math.inf
            if w:
                s[:, :, :max(0, at + 1 - w)] = -math.inf
            lse[i, t] = torch.logsumexp(s, 2)
            p = torch.softmax(s, 2)
            out[i, t] = torch.bmm(p[:, :, shared:].contiguous(), v)
            if shared:
                out[i, t] += torch.bmm(p[:, :, :shared].contiguous(), pv)
    answer = {"out": out.reshape(n * n_q, -1)}
    if case["lse"]:
        answer["lse"] = lse.reshape(n * n_q, -1)
    return answer
