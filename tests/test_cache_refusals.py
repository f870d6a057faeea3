"""CPU tests: the cache, the attention over it and the rules on logits refuse bad
arguments and memory before any GPU call (no pointer below is dereferenced), and
their Python methods hand on what a tensor holds."""
import ctypes
import types

import pytest
import torch

import ft_hip

P = ctypes.c_void_p
BIG = 1 << 62
STREAM = types.SimpleNamespace(cuda_stream=0)
ROOM = ctypes.create_string_buffer(4096)  # stands for a context, which no refused call reads
CTX = ctypes.cast(ROOM, P)

# 2 rows of 2 heads of 64 f32 (512 bytes), 1 KiB apart; a cache of 3 pages of 16 tokens (4352 bytes each)
WRITE = dict(ctx=None, stream=None, k=P(0x10000), k_stride=256, v=P(0x10200), v_stride=256, type=0, slots=P(0x20000),
             cache=P(0x30000), cache_type=0, n_pages=3, page_tokens=16, n_heads=2, head_dim=64, n=2)
READ = dict(ctx=None, stream=None, cache=P(0x30000), cache_type=0, n_pages=3, page_tokens=16, n_heads=2, head_dim=64,
            slots=P(0x20000), k=P(0x10000), k_stride=256, v=P(0x10200), v_stride=256, type=0, n=2)
# 2 sequences with 1 query on 4 heads of 64 f32 (1 KiB), tables of 2 pages
ATTEND = dict(ctx=None, stream=None, q=P(0x10000), q_stride=256, type=0, cache=P(0x30000), cache_type=0, n_pages=3,
              page_tokens=16, n_kv_heads=2, head_dim=64, tables=P(0x20000), table_stride=4, table_pages=2,
              lens=P(0x20100), prefix=P(0x20200), prefix_pages=2, prefix_len=P(0x20300), n_seqs=2, n_q=1, n_heads=4,
              scale=0.125, window=0, out=P(0x11000), out_stride=256, lse=P(0x12000), workspace=P(0x100000000),
              workspace_bytes=1 << 40)
# 2 rows of 100 f32 (400 bytes), 512 bytes apart
ADJUST = dict(ctx=None, stream=None, logits=P(0x10000), logits_type=0, logits_stride=128, vocab=100, n=2,
              history=P(0x20000), history_stride=8, history_max=8, history_len=P(0x20100), repetition=P(0x20110),
              presence=P(0x20120), frequency=P(0x20130), bias_ids=P(0x20200), bias=P(0x20300), n_bias=3,
              mask=P(0x20400), mask_stride=4, out=P(0x11000), out_stride=128)
USUAL = dict(kv_write=WRITE, kv_read=READ, attention=ATTEND, adjust_logits=ADJUST)


def call(name, **change):
    usual = USUAL[name]
    now = {k: P(v) if isinstance(usual[k], P) and isinstance(v, int) else v for k, v in {**usual, **change}.items()}
    rc = getattr(ft_hip.lib(), "ft_hip_" + name)(*now.values())
    return rc, ft_hip.lib().ft_hip_last_error().decode()


CACHE = [(dict(page_tokens=0), "SHAPE", "page_tokens"), (dict(page_tokens=8), "SHAPE", "page_tokens"),
         (dict(page_tokens=48), "SHAPE", "page_tokens"), (dict(page_tokens=512), "SHAPE", "page_tokens"),
         (dict(page_tokens=-16), "SHAPE", "page_tokens"), (dict(head_dim=32), "SHAPE", "head_dim"),
         (dict(head_dim=192), "SHAPE", "head_dim"), (dict(head_dim=0), "SHAPE", "head_dim"),
         (dict(n_pages=0), "SHAPE", "n_pages"), (dict(n_pages=-1), "SHAPE", "n_pages"),
         (dict(n_pages=1 << 27), "SHAPE", "n_pages"), (dict(n_pages=BIG), "SHAPE", "n_pages"),
         (dict(cache_type=2), "INVALID", "cache_type"), (dict(cache_type=-1), "INVALID", "cache_type"),
         (dict(type=3), "INVALID", "type"), (dict(cache=0x30008), "SHAPE", "aligned"), (dict(cache=None), "INVALID", "null")]
ROWS = CACHE + [(dict(n_heads=0), "SHAPE", "n_heads"), (dict(n_heads=257), "SHAPE", "n_heads"),
                (dict(n=-1), "SHAPE", "n="), (dict(n=(1 << 20) + 1), "SHAPE", "n="), (dict(n=BIG), "SHAPE", "n="),
                (dict(k_stride=127), "SHAPE", "k_stride"), (dict(v_stride=0), "SHAPE", "v_stride"),
                (dict(k_stride=BIG), "SHAPE", "k_stride"), (dict(k=0x10002), "SHAPE", "aligned"),
                (dict(type=1, v=0x10201), "SHAPE", "aligned"), (dict(slots=0x20002), "SHAPE", "aligned"),
                (dict(k=None), "INVALID", "null"), (dict(v=None), "INVALID", "null"), (dict(slots=None), "INVALID", "null")]
ATTENDED = CACHE + [
    (dict(n_kv_heads=0), "SHAPE", "n_kv_heads"), (dict(n_kv_heads=257), "SHAPE", "n_kv_heads"),
    (dict(n_heads=3), "SHAPE", "n_heads"), (dict(n_heads=0), "SHAPE", "n_heads"), (dict(n_heads=4098), "SHAPE", "n_heads"),
    (dict(n_seqs=-1), "SHAPE", "n_seqs"), (dict(n_seqs=4097), "SHAPE", "n_seqs"), (dict(n_q=0), "SHAPE", "n_q"),
    (dict(n_q=65), "SHAPE", "n_q"), (dict(table_pages=0), "SHAPE", "table_pages"), (dict(table_stride=1), "SHAPE", "table_stride"),
    (dict(table_pages=1 << 28, table_stride=1 << 28), "SHAPE", "table_pages"), (dict(table_stride=BIG), "SHAPE", "table_stride"),
    (dict(n_seqs=4096, table_pages=1 << 26, table_stride=1 << 26), "SHAPE", "table_pages"),
    (dict(prefix_pages=0), "SHAPE", "prefix_pages"), (dict(prefix_pages=-1), "SHAPE", "prefix_pages"),
    (dict(prefix_pages=BIG), "SHAPE", "prefix_pages"),
    (dict(prefix_pages=1 << 26, table_pages=1 << 26, table_stride=1 << 26), "SHAPE", "prefix_pages"),
    (dict(window=-1), "SHAPE", "window"), (dict(window=1 << 31), "SHAPE", "window"), (dict(scale=float("nan")), "SHAPE", "scale"),
    (dict(scale=float("inf")), "SHAPE", "scale"), (dict(q_stride=255), "SHAPE", "q_stride"),
    (dict(out_stride=255), "SHAPE", "out_stride"), (dict(out_stride=BIG), "SHAPE", "out_stride"),
    (dict(workspace_bytes=0), "SHAPE", "workspace"), (dict(workspace=0x100000008), "SHAPE", "aligned"),
    (dict(q=0x10002), "SHAPE", "aligned"), (dict(out=0x11002), "SHAPE", "aligned"), (dict(tables=0x20002), "SHAPE", "aligned"),
    (dict(lens=0x20102), "SHAPE", "aligned"), (dict(prefix=0x20202), "SHAPE", "aligned"),
    (dict(prefix_len=0x20302), "SHAPE", "aligned"), (dict(lse=0x12002), "SHAPE", "aligned"),
    (dict(q=None), "INVALID", "null"), (dict(tables=None), "INVALID", "null"), (dict(lens=None), "INVALID", "null"),
    (dict(out=None), "INVALID", "null"), (dict(workspace=None), "INVALID", "null"), (dict(prefix_len=None), "INVALID", "null")]
ADJUSTED = [
    (dict(vocab=0), "SHAPE", "vocab"), (dict(vocab=(1 << 21) + 1), "SHAPE", "vocab"), (dict(n=-1), "SHAPE", "n="),
    (dict(n=65536), "SHAPE", "n="), (dict(logits_type=3), "INVALID", "logits_type"), (dict(logits_stride=99), "SHAPE", "logits_stride"),
    (dict(out_stride=99), "SHAPE", "out_stride"), (dict(out_stride=BIG), "SHAPE", "out_stride"),
    (dict(history_max=0), "SHAPE", "history"), (dict(history_max=(1 << 24) + 1, history_stride=1 << 25), "SHAPE", "history"),
    (dict(history_stride=7), "SHAPE", "history"), (dict(history_stride=BIG), "SHAPE", "history"),
    (dict(n_bias=-1), "SHAPE", "n_bias"), (dict(n_bias=1025), "SHAPE", "n_bias"), (dict(mask_stride=3), "SHAPE", "mask"),
    (dict(mask_stride=BIG), "SHAPE", "mask"), (dict(logits=0x10002), "SHAPE", "aligned"),
    (dict(logits_type=2, logits=0x10001), "SHAPE", "aligned"), (dict(bias_ids=None), "INVALID", "null"),
    (dict(bias=None), "INVALID", "null"), (dict(logits=None), "INVALID", "null"), (dict(out=None), "INVALID", "null")]
ADJUSTED += [({a: 0x20002 + i}, "SHAPE", "aligned") for i, a in enumerate(
    ("out", "history", "history_len", "repetition", "presence", "frequency", "bias_ids", "bias", "mask")) if (0x20002 + i) % 4]


@pytest.mark.parametrize("name,change,code,word", [(n, *c) for n, cases in (
    ("kv_write", ROWS), ("kv_read", ROWS), ("attention", ATTENDED), ("adjust_logits", ADJUSTED)) for c in cases])
def test_bad_arguments(name, change, code, word):
    """With a context where only that would be missing otherwise."""
    rc, msg = call(name, **{"ctx": CTX, **change})
    assert rc == getattr(ft_hip, "E_" + code), msg
    assert word in msg, msg


@pytest.mark.parametrize("name", USUAL)
def test_no_context(name):
    rc, msg = call(name)
    assert rc == ft_hip.E_INVALID and "null" in msg, msg


@pytest.mark.parametrize("name,change", [
    ("kv_write", dict(k=0x30000)), ("kv_write", dict(v=0x33100)), ("kv_write", dict(slots=0x332fc)),
    ("kv_read", dict(k=0x30000)), ("kv_read", dict(v=0x2fc00)), ("kv_read", dict(slots=0x33000)),
    ("kv_read", dict(v=0x10004)), ("kv_read", dict(v=0x105fc)), ("kv_read", dict(slots=0x10400)),
    ("kv_read", dict(slots=0x103fc - 0x200)),
    ("attention", dict(out=0x10000)), ("attention", dict(out=0x10400)), ("attention", dict(out=0x30000)),
    ("attention", dict(out=0x332fc, out_stride=256)), ("attention", dict(out=0x1fc04)), ("attention", dict(out=0x200fc - 0x3f8)),
    ("attention", dict(lse=0x10000)), ("attention", dict(lse=0x20100)), ("attention", dict(lse=0x2020c - 0x20)),
    ("attention", dict(lse=0x20300)), ("attention", dict(lse=0x11000)), ("attention", dict(workspace=0x10000)),
    ("attention", dict(workspace=0x11000)), ("attention", dict(workspace=0x12000)), ("attention", dict(workspace=0x1fff0)),
    ("adjust_logits", dict(out=0x10004)), ("adjust_logits", dict(out=0x10000, logits_type=2)),
    ("adjust_logits", dict(out=0x10000, out_stride=256)), ("adjust_logits", dict(out=0x20000)),
    ("adjust_logits", dict(out=0x1ff80)), ("adjust_logits", dict(out=0x20410)), ("adjust_logits", dict(out=0x20300)),
    ("adjust_logits", dict(out=0x20134)),
])
def test_memory_that_overlaps(name, change):
    rc, msg = call(name, ctx=CTX, **change)
    assert rc == ft_hip.E_SHAPE and "overlap" in msg, msg


@pytest.mark.parametrize("name,count,pointers", [
    ("kv_write", "n", ("k", "v", "slots", "cache")), ("kv_read", "n", ("k", "v", "slots", "cache")),
    ("attention", "n_seqs", ("q", "cache", "tables", "lens", "out", "workspace")),
    ("adjust_logits", "n", ("logits", "out", "bias", "bias_ids"))])
def test_no_rows(name, count, pointers):
    """Nothing to do, also where an empty batch has no address; a bad shape stays refused."""
    none = {count: 0, **{p: None for p in pointers}}
    assert call(name, ctx=CTX, **none)[0] == ft_hip.OK
    assert call(name, **none)[0] == ft_hip.E_INVALID
    bad = dict(vocab=0) if name == "adjust_logits" else dict(head_dim=65)
    assert call(name, ctx=CTX, **{**none, **bad})[0] == ft_hip.E_SHAPE


def test_sizes():
    L = ft_hip.lib()
    assert L.ft_hip_kv_page_bytes(64, 8, 256) == 8 * 64 * (2 * 256 + 8)
    for bad in ((0, 8, 256), (24, 8, 256), (64, 0, 256), (64, 8, 80), (64, 257, 64), (512, 8, 64)):
        assert L.ft_hip_kv_page_bytes(*bad) == -1
    f = L.ft_hip_attention_workspace_bytes
    assert 0 < f(0, 1, 8, 8, 64) <= f(1, 1, 8, 8, 64) <= f(64, 1, 16, 8, 64) <= f(64, 1, 16, 8, 256) <= f(4096, 1, 16, 8, 256)
    for bad in ((-1, 1, 8, 8, 64), (4097, 1, 8, 8, 64), (1, 0, 8, 8, 64), (1, 65, 8, 8, 64), (1, 1, 9, 8, 64), (1, 1, 8, 0, 64),
                (1, 1, 8, 8, 96), (1, 1, 0, 1, 64), (BIG, 1, 8, 8, 64), (1, 1, BIG, 8, 64)):
        assert f(*bad) == 0
    need = f(2, 1, 4, 2, 64)
    assert call("attention", ctx=CTX, workspace_bytes=need - 1)[0] == ft_hip.E_SHAPE


# ---- the Python methods, seen at a library that notes its arguments ----

class Noted:
    def __init__(self):
        self.calls = {}

    def __getattr__(self, name):
        def entry(*args):
            self.calls[name] = args
            return 16 * (2 * 64 + 8) * 2 if name == "ft_hip_kv_page_bytes" else ft_hip.OK
        return entry


@pytest.fixture
def noted(monkeypatch):
    noted = Noted()
    monkeypatch.setattr(ft_hip, "lib", lambda: noted)
    g = ft_hip.Q4Gemv.__new__(ft_hip.Q4Gemv)
    g._ctx, g.device = None, -1
    return g, noted.calls


PAGE = 16 * (2 * 64 + 8) * 2


def ints(*shape):
    return torch.zeros(shape, dtype=torch.int32)


def test_columns_of_a_row_of_projections(noted):
    g, calls = noted
    rows, cache = torch.zeros(3, 512), torch.zeros((5, PAGE), dtype=torch.uint8)
    k, v = rows[:, 256:384], rows[:, 384:]
    g.kv_write(k, v, ints(3), cache, 3, 2, 64, 16, ft_hip.KV_E4M3, stream=STREAM)
    a = calls["ft_hip_kv_write"]
    assert (a[2], a[3], a[4], a[5], a[6]) == (k.data_ptr(), 512, v.data_ptr(), 512, ft_hip.TYPE_F32)
    assert a[9:] == (ft_hip.KV_E4M3, 5, 16, 2, 64, 3)
    g.kv_read(cache, ints(3), k, v, 3, 2, 64, 16, stream=STREAM)
    a = calls["ft_hip_kv_read"]
    assert a[4:8] == (5, 16, 2, 64) and (a[10], a[12]) == (512, 512)
    out, lse = torch.zeros(3, 256), torch.zeros(3, 4)
    tables = ints(4, 9)[:, 2:7]
    g.attention(rows[:, :256], cache, tables, ints(3), out, torch.zeros(64, dtype=torch.uint8), 3, 4, 2, 64, 16, 0.5, lse=lse,
                window=7, stream=STREAM)
    a = calls["ft_hip_attention"]
    assert (a[3], a[7], a[11], a[12], a[13]) == (512, 5, tables.data_ptr(), 9, 5)
    assert a[15:18] == (None, 0, None) and a[18:23] == (3, 1, 4, 0.5, 7) and a[24:26] == (256, lse.data_ptr())


def test_tensors_that_do_not_hold_what_is_asked(noted):
    g, _ = noted
    cache, ws = torch.zeros((5, PAGE), dtype=torch.uint8), torch.zeros(64, dtype=torch.uint8)
    k, out = torch.zeros(3, 128), torch.zeros(3, 256)
    write = lambda **c: g.kv_write(**{**dict(k=k, v=k, slots=ints(3), cache=cache, n=3, n_heads=2, head_dim=64,  # noqa: E731
                                             page_tokens=16, stream=STREAM), **c})
    read = lambda **c: g.kv_read(**{**dict(k=k, v=k, slots=ints(3), cache=cache, n=3, n_heads=2, head_dim=64,  # noqa: E731
                                           page_tokens=16, stream=STREAM), **c})
    for f in (write, read):
        f()
        for bad in (dict(v=k.half()), dict(k=k[:2]), dict(k=k[:, :127]), dict(slots=ints(2)), dict(slots=torch.zeros(3)),
                    dict(slots=ints(3).long()), dict(cache=cache[:, ::2]), dict(k=k.double(), v=k.double()),
                    dict(slots=ints(6)[::2])):
            with pytest.raises(ft_hip.FtHipError):
                f(**bad)
    attend = lambda **c: g.attention(**{**dict(  # noqa: E731
        q=out, cache=cache, tables=ints(3, 2), lens=ints(3), out=out.clone(), workspace=ws, n_seqs=3, n_heads=4, n_kv_heads=2,
        head_dim=64, page_tokens=16, scale=1.0, stream=STREAM), **c})
    attend()
    for bad in (dict(out=out.half()), dict(q=out[:2]), dict(n_q=2), dict(tables=ints(2, 2)), dict(tables=ints(6)),
                dict(tables=ints(3, 2).float()), dict(tables=ints(2, 3).t()), dict(lens=ints(2)), dict(lens=torch.zeros(3)),
                dict(prefix=torch.zeros(3)), dict(prefix=ints(2), prefix_len=ints(0)), dict(lse=torch.zeros(3, 3)),
                dict(lse=ints(3, 4)), dict(workspace=ws[::2]), dict(cache=cache.t()), dict(tables=ints(1, 2).expand(3, 2))):
        with pytest.raises(ft_hip.FtHipError):
            attend(**bad)
    logits = torch.zeros(3, 100)
    adjust = lambda **c: g.adjust_logits(**{**dict(logits=logits, out=logits, vocab=100, n=3, stream=STREAM), **c})  # noqa: E731
    adjust()
    adjust(history=ints(3, 7), history_len=ints(3), repetition=torch.ones(3), bias=torch.zeros(3, 2), bias_ids=ints(3, 2),
           mask=ints(3, 4))
    for bad in (dict(out=logits.half()), dict(out=logits[:2]), dict(history=ints(2, 7)), dict(history=torch.zeros(3, 7)),
                dict(history=ints(3, 7).long()), dict(history_len=ints(2)), dict(repetition=torch.ones(2)),
                dict(presence=ints(3)), dict(frequency=torch.ones(3).double()), dict(bias=torch.zeros(3, 2)),
                dict(bias_ids=ints(3, 2)), dict(bias=torch.zeros(3, 2), bias_ids=ints(3, 3)),
                dict(bias=torch.zeros(6), bias_ids=ints(6)), dict(mask=ints(3, 3)), dict(mask=ints(2, 4)),
                dict(mask=torch.zeros(3, 4)), dict(bias=torch.zeros(2, 2), bias_ids=ints(2, 2))):
        with pytest.raises(ft_hip.FtHipError):
            adjust(**bad)


def test_a_single_row_of_one_column(noted):
    g, calls = noted
    g.adjust_logits(torch.zeros(1, 30), torch.zeros(1, 30), 30, 1, history=ints(1, 1), mask=ints(1, 1), stream=STREAM)
    a = calls["ft_hip_adjust_logits"]
    assert a[8:10] == (1, 1) and a[18] == 1
