"""ft_hip_attention against its definition in 64 bits, on what the cache holds.

Tolerances, from the arithmetic (u = 2^-24, D dimensions, per column):
  a score's products are exact; its sum over D (twice D where q is two f16) in
  f32, in any order, is off by at most 2 D u A, A = |scale| sum |q k|; q's two
  halves leave 2^-22 of q (16-bit types: nothing), the scales' three products and
  the subtraction of the maximum 4 u of A + M, M the largest score: together
  ds = (2 D u + 2^-22 + 4 u) A + 4 u M. exp2 and its argument's factor: 4 u more.
  Each weight is then off by the factor exp(ds) and, as f16, by 2^-11 (two f16:
  2^-22); the sums over n tokens, pieces and steps, in f32, by n u at most.
  f16 steps no finer than 2^-24: in units of 2^-7 of the largest scale dv (or
  less) each weight p dv leaves up to 2^-25, which is 2^-32 max |v| of its token's
  part at most, over a sum of p of at least 1.
  out = sum w v / sum w: off by at most (2 ds' + 2^-11 or 2^-22 + 2 n u + 8 u) sum p |v|
  + n 2^-32 max |v|, ds' = ds + 4 u, and half a step of its type. lse: ds' + n u,
  and 4 u of itself.
These are bounds; the errors come in all signs, and their root mean square over
the outputs is held to an eighth of the bound's.
"""
import numpy as np
import pytest
import torch

import ft_hip
from test_gpu_kv import E4M3, I8, Layout, host

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24


def definition(q, cache, layout, kind, tables, lens, prefix, prefix_len, n_q, heads, scale, window, dtype, n_pages):
    """(out, its tolerance, lse, its tolerance) in 64 bits, sequence by sequence."""
    n, kv, dim, page = len(lens), layout.heads, layout.dim, layout.page
    group = heads // kv
    q = q.astype(np.float64).reshape(n, n_q, kv, group, dim)
    out, tol = np.zeros(q.shape), np.zeros(q.shape)
    lse, ltol = np.full(q.shape[:-1], -np.inf), np.zeros(q.shape[:-1])
    plen = 0 if prefix is None else min(max(int(prefix_len), 0), len(prefix) * page)
    eps = {torch.float32: 2.0 ** -22, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -11}[dtype]
    split = 2.0 ** -22 if dtype == torch.float32 else 0.0

    def tokens(pages, count):
        at = np.arange(count)
        ids = np.asarray(pages, np.int64)[at // page]
        ok = (ids >= 0) & (ids < n_pages)
        return np.where(ok, ids, 0) * page + at % page, ok

    pk = pv = None
    if plen:
        ps, pok = tokens(prefix, plen)
        pk, pv = layout.get(cache, ps, kind)
    for i in range(n):
        own = min(max(int(lens[i]), 0), tables.shape[1] * page)
        if not own:
            continue
        slots, ok = tokens(tables[i], own)
        k, v = layout.get(cache, slots, kind)
        if plen:
            k, v, ok = np.concatenate([pk, k]), np.concatenate([pv, v]), np.concatenate([pok, ok])
        for t in range(max(0, n_q - own), n_q):
            at = plen + own - n_q + t
            lo = max(0, at + 1 - window) if window else 0
            live = np.flatnonzero(ok[lo:at + 1]) + lo
            if not len(live):
                continue
            kk, vv = k[live], v[live]
            s = scale * np.einsum("hgd,jhd->hgj", q[i, t], kk)
            A = abs(scale) * np.einsum("hgd,jhd->hgj", np.abs(q[i, t]), np.abs(kk)).max(2)
            M = s.max(2)
            p = np.exp(s - M[:, :, None])
            total = p.sum(2)
            out[i, t] = np.einsum("hgj,jhd->hgd", p, vv) / total[:, :, None]
            lse[i, t] = M + np.log(total)
            ds = (2 * dim * U + split + 4 * U) * A + 4 * U * np.abs(M) + 4 * U
            size = np.einsum("hgj,jhd->hgd", p, np.abs(vv)) / total[:, :, None]
            half = torch.finfo(dtype).eps / 2
            # max |v| as the formats allow it: the scale times its largest number, which is at most twice max |x|
            most = 2.0 * np.abs(vv).max((0, 2))[:, None, None]
            tol[i, t] = ((2 * ds + eps + (2 * len(live) + 8) * U)[:, :, None] * size + len(live) * 2.0 ** -32 * most
                         + half * np.abs(out[i, t])
                         + float(torch.finfo(dtype).smallest_normal) * half * 2)
            ltol[i, t] = ds + len(live) * U + 4 * U * np.abs(lse[i, t])
    flat = lambda a: a.reshape(n * n_q, -1)  # noqa: E731
    return flat(out), flat(tol), flat(lse), flat(ltol)


class Batch:
    """A cache with tokens in random pages, everything else of it garbage: bytes that are NaN codes and scales that
    are NaN and infinities."""

    def __init__(self, gemv, lens, page, kv, group, dim, kind, dtype, prefix=0, n_q=1, seed=0, spread=1.0, width=None):
        rng = np.random.default_rng(seed)
        self.g, self.kv, self.heads, self.dim, self.page, self.kind, self.dtype, self.n_q = (
            gemv, kv, kv * group, dim, page, kind, dtype, n_q)
        self.lens, self.n = np.asarray(lens, np.int32), len(lens)
        self.layout = Layout(page, kv, dim)
        need = [-(-max(0, int(x)) // page) for x in lens]
        shared = -(-prefix // page)
        self.n_pages = sum(need) + shared + 2
        where = rng.permutation(self.n_pages).astype(np.int32)
        width = max(1, max(need, default=0)) if width is None else width
        # places behind a sequence's pages name pages of others, or none
        self.tables = rng.choice(np.array([-1, 0, self.n_pages - 1, self.n_pages, 2 ** 31 - 1], np.int32), (self.n, width))
        at = shared
        for i, c in enumerate(need):
            self.tables[i, :c] = where[at:at + c]
            at += c
        self.prefix = where[:shared] if shared else None
        self.prefix_len = prefix
        garbage = rng.integers(0, 256, self.n_pages * kv * self.layout.block, dtype=np.uint8)
        f = garbage.view(np.float32)
        pages = np.arange(self.n_pages * page)
        for value in (0, 1):
            f[self.layout.scales_at(pages, value)] = rng.choice(np.array([np.nan, np.inf, -np.inf, 1e30], np.float32),
                                                                (len(pages), kv))
            if kind == E4M3:
                garbage[self.layout.at(pages, value)] = rng.choice(np.array([0x7F, 0xFF, 1], np.uint8),
                                                                   (len(pages), kv, dim))
        self.cache = torch.from_numpy(garbage).to(DEV)
        slots = [self.places(self.tables[i], int(x)) for i, x in enumerate(lens) if x > 0]
        if shared:
            slots.append(self.places(self.prefix, prefix))
        if slots:
            slots = np.concatenate(slots).astype(np.int32)
            x = rng.standard_normal((2, len(slots), kv * dim)) * np.exp(spread * rng.uniform(-1, 1, (2, len(slots), 1)))
            x[0] += rng.standard_normal(kv * dim)  # channels that all keys share
            k, v = (torch.from_numpy(y.astype(np.float32)).to(DEV) for y in x)
            gemv.kv_write(k, v, torch.from_numpy(slots).to(DEV), self.cache, len(slots), kv, dim, page, kind)
        q = rng.standard_normal((self.n * n_q, self.heads * dim)).astype(np.float32)
        self.q = torch.from_numpy(q).to(dtype).to(DEV)
        torch.cuda.synchronize()

    def places(self, pages, count):
        at = np.arange(count)
        return np.asarray(pages, np.int64)[at // self.page] * self.page + at % self.page

    def workspace(self):
        return torch.full((self.g.attention_workspace_bytes(self.n, self.n_q, self.heads, self.kv, self.dim),), 0xFF,
                          dtype=torch.uint8, device=DEV)

    def tensors(self):
        t = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(DEV)  # noqa: E731
        return dict(tables=t(self.tables), lens=t(self.lens),
                    prefix=None if self.prefix is None else t(self.prefix.astype(np.int32)),
                    prefix_len=None if self.prefix is None else t(np.array([self.prefix_len], np.int32)))

    def run(self, window=0, scale=None, q=None, out=None, lse=True, workspace=None, stream=None, **given):
        q = self.q if q is None else q
        out = torch.full_like(self.q, 9.0) if out is None else out
        lse = torch.full((self.n * self.n_q, self.heads), 9.0, device=DEV) if lse is True else lse
        t = given if len(given) == 4 else {**self.tensors(), **given}  # none made where a capture has them all
        self.g.attention(q, self.cache, t["tables"], t["lens"], out, self.workspace() if workspace is None else workspace, self.n,
                         self.heads, self.kv, self.dim, self.page, self.dim ** -0.5 if scale is None else scale, n_q=self.n_q,
                         window=window, prefix=t["prefix"], prefix_len=t["prefix_len"], lse=lse, cache_type=self.kind,
                         stream=stream)
        return out, lse

    def want(self, window=0, scale=None, lens=None, tables=None, prefix_len=None):
        return definition(host(self.q.float()), host(self.cache), self.layout, self.kind,
                          self.tables if tables is None else tables, self.lens if lens is None else lens, self.prefix,
                          self.prefix_len if prefix_len is None else prefix_len, self.n_q, self.heads,
                          self.dim ** -0.5 if scale is None else scale, window, self.dtype, self.n_pages)

    def check(self, window=0, scale=None, **kw):
        out, lse = self.run(window, scale, **kw)
        torch.cuda.synchronize()
        self.close(out, lse, self.want(window, scale))
        return out, lse

    def close(self, out, lse, want):
        o, tol, l, ltol = want
        got = host(out.float()).astype(np.float64)
        off = np.abs(got - o)
        beyond = np.argwhere(~(off <= tol))
        assert len(beyond) == 0, (len(beyond), beyond[:4].tolist(), float(np.nanmax(off / np.maximum(tol, 1e-300))))
        half = torch.finfo(self.dtype).eps / 2 * np.abs(o)
        if tol.any():  # beside the last rounding
            assert np.sqrt(np.mean(np.maximum(off - half, 0) ** 2)) <= np.sqrt(np.mean((tol - half) ** 2)) / 8
        if lse is not None:
            got = host(lse).astype(np.float64)
            none = np.isneginf(l)
            assert np.array_equal(np.isneginf(got), none)
            assert np.all(np.abs(got[~none] - l[~none]) <= ltol[~none])


TYPES = [torch.float32, torch.float16, torch.bfloat16]


@pytest.mark.parametrize("kind", [I8, E4M3])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_types_and_head_sizes(gemv, kind, dtype, dim):
    Batch(gemv, [1, 77, 300], 32, 2, 2, dim, kind, dtype, seed=dim).check()


@pytest.mark.parametrize("length", [1, 2, 15, 16, 17, 31, 32, 33, 47, 48, 49, 63, 64, 65, 127, 128, 129, 1000, 1023, 1024, 1025])
def test_lengths(gemv, length):
    Batch(gemv, [length], 16, 1, 4, 64, I8, torch.float32, seed=length).check()


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("kind", [I8, E4M3])
def test_pages(gemv, page, kind):
    """Sequences that end everywhere in their last page."""
    Batch(gemv, [1, page - 1, page, page + 1, 3 * page + 5, 4 * page - 17 if page > 16 else 50], page, 2, 3, 128, kind,
          torch.bfloat16, seed=page, width=9).check()


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("group", [1, 2, 3, 7, 8, 9, 16, 17, 40])
def test_query_heads_on_a_key_head(gemv, dtype, group):
    Batch(gemv, [90, 33], 16, 2, group, 64, I8, dtype, seed=group).check()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n_q,group", [(2, 1), (3, 2), (5, 3), (8, 4), (64, 1), (17, 8)])
def test_several_new_tokens(gemv, dtype, n_q, group):
    """Each sees what is before it; sequences shorter than the new tokens are padded at their front."""
    Batch(gemv, [n_q, 100 + n_q, 1, n_q - 1, 0, 40], 16, 2, group, 64, E4M3, dtype, n_q=n_q, seed=n_q).check()


@pytest.mark.parametrize("window", [1, 2, 15, 16, 17, 100, 299, 300, 301, 5000])
@pytest.mark.parametrize("n_q", [1, 4])
def test_window(gemv, window, n_q):
    Batch(gemv, [300, 7, 450, 0, 33], 32, 2, 2, 64, I8, torch.float32, n_q=n_q, seed=window).check(window=window)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("prefix", [1, 16, 31, 100, 1025])
@pytest.mark.parametrize("n,n_q,group", [(1, 1, 2), (3, 1, 8), (20, 1, 2), (37, 2, 3)])
def test_shared_prefix(gemv, dtype, prefix, n, n_q, group):
    rng = np.random.default_rng(n)
    lens = rng.integers(n_q, 90, n)
    lens[0] = n_q
    if n > 2:
        lens[[1, n - 1]] = 0, 1
    Batch(gemv, lens, 32, 2, group, 64, I8 if n % 2 else E4M3, dtype, prefix=prefix, n_q=n_q, seed=prefix).check()


@pytest.mark.parametrize("dim", [128, 256])
@pytest.mark.parametrize("kind", [I8, E4M3])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_shared_prefix_at_other_head_sizes(gemv, dim, kind, dtype):
    Batch(gemv, [60, 1, 200, 31, 5], 64, 2, 4, dim, kind, dtype, prefix=333, seed=dim).check()


@pytest.mark.parametrize("window", [1, 20, 64, 130, 400, 900])
def test_a_window_into_the_prefix(gemv, window):
    """Sequences whose window ends in the prefix, in their own tokens, and at the border."""
    Batch(gemv, [5, 64, 63, 65, 1, 0, 128, 129, 400, 90], 16, 1, 3, 64, I8, torch.float32, prefix=500, n_q=2,
          seed=window).check(window=window)


def test_the_prefix_equals_the_same_tokens_at_each_sequences_front(gemv):
    """The shared pages in every table, against the prefix: the same definition, within both tolerances."""
    b = Batch(gemv, [70, 3, 200, 41], 16, 2, 2, 128, E4M3, torch.float32, prefix=160, seed=5)
    out, lse = b.check()
    t = b.tensors()
    whole = torch.cat([t["prefix"].expand(4, -1), t["tables"]], 1).contiguous()
    out2, lse2 = b.run(tables=whole, lens=t["lens"] + 160, prefix=None, prefix_len=None)
    torch.cuda.synchronize()
    _, tol, _, ltol = b.want()
    assert np.all(np.abs(host(out) - host(out2)) <= 2 * tol) and np.all(np.abs(host(lse) - host(lse2)) <= 2 * ltol)


@pytest.mark.parametrize("kind", [I8, E4M3])
def test_a_long_sequence_on_the_whole_device(gemv, kind):
    Batch(gemv, [40000], 64, 4, 2, 64, kind, torch.float32, seed=3).check()


def test_ragged_batch_with_a_long_tail(gemv):
    rng = np.random.default_rng(11)
    lens = np.concatenate([[9000, 2500], rng.integers(0, 60, 300)])
    Batch(gemv, lens, 16, 2, 2, 64, I8, torch.bfloat16, seed=1).check()


def test_more_sequences_than_threads(gemv):
    rng = np.random.default_rng(12)
    Batch(gemv, rng.integers(0, 40, 1100), 16, 1, 2, 64, I8, torch.float32, prefix=40, seed=2).check()


def test_scores_far_apart(gemv):
    """A maximum that comes late and raises everything, and one that is alone; large and small scales of values."""
    for seed, spread in ((1, 3.0), (2, 5.0)):
        b = Batch(gemv, [500, 64, 33], 32, 2, 2, 64, I8, torch.float32, seed=seed, spread=spread)
        b.check(scale=1.0)
        b.check(scale=-0.7)
        b.check(scale=0.0)
    b.q *= 50.0
    b.check(scale=1.0)


@pytest.mark.parametrize("dtype", TYPES)
def test_large_and_small_queries(gemv, dtype):
    b = Batch(gemv, [100, 40], 16, 1, 4, 64, I8, dtype, seed=8)
    for f in (2.0 ** -12, 2.0 ** 12) if dtype == torch.float16 else (1e-30, 1e30):
        q = b.q.clone()
        b.q = (q.float() * f).to(dtype)
        b.check(scale=1.0 / f)
        b.q = q
    b.q[0] = 0.0
    b.check()


@pytest.mark.parametrize("kind", [I8, E4M3])
@pytest.mark.parametrize("n,group,prefix", [(200, 4, 0), (100, 20, 0), (150, 6, 60)])
def test_each_weight_of_f32_queries(gemv, kind, n, group, prefix):
    """Values of one number at a dimension of their own, so that each output is a single token's weight: with a small
    scale the bound is a few 2^-16 of it, and a weight that loses its second half in one of thousands shows."""
    lens = [4] * n if prefix else [60 + i % 5 for i in range(n)]
    b = Batch(gemv, lens, 16, 1, group, 64, kind, torch.float32, prefix=prefix, seed=60)
    rng = np.random.default_rng(61)
    rows = [(b.places(b.tables[i], x), np.arange(x) + prefix) for i, x in enumerate(lens)]
    if prefix:
        rows.append((b.places(b.prefix, prefix), np.arange(prefix)))
    slots = np.concatenate([r[0] for r in rows]).astype(np.int32)
    v = np.zeros((len(slots), 64), np.float32)
    v[np.arange(len(slots)), np.concatenate([r[1] for r in rows]) % 64] = rng.uniform(0.5, 2.0, len(slots))
    k = rng.standard_normal((len(slots), 64)).astype(np.float32)
    t = lambda a: torch.from_numpy(a).to(DEV)  # noqa: E731
    gemv.kv_write(t(k), t(v), t(slots), b.cache, len(slots), 1, 64, 16, kind)
    b.check(scale=2.0 ** -6)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n_q,prefix", [(1, 0), (1, 100), (4, 100), (4, 0)])
def test_rows_of_other_sizes_do_not_reach_each_other(gemv, dtype, n_q, prefix):
    """Queries far smaller and far larger than their neighbours', and rows that are no numbers: the others' results are
    what they were, bit for bit."""
    b = Batch(gemv, [60, 9, 100, 33, 20], 16, 2, 2, 64, I8, dtype, prefix=prefix, n_q=n_q, seed=40)
    want, lse = b.check()
    big = 6e4 if dtype == torch.float16 else 1e30
    q = b.q.clone()
    b.q[n_q] *= 1e-4 if dtype == torch.float16 else 1e-25
    b.q[2 * n_q, 5] = big
    b.q[3 * n_q] = float("inf")
    b.q[4 * n_q, 130] = float("-inf")
    out, got = b.run()
    torch.cuda.synchronize()
    same = [i for i in range(5 * n_q) if i not in (n_q, 2 * n_q, 3 * n_q, 4 * n_q)]
    assert torch.equal(out[same], want[same]) and torch.equal(got[same], lse[same])
    o, tol, _, _ = b.want()
    assert np.all(np.abs(host(out.float())[n_q] - o[n_q]) <= tol[n_q])
    assert torch.equal(out[4 * n_q, :128], want[4 * n_q, :128]) and torch.equal(q[0], b.q[0])


def test_nan_and_infinities_reach_those_who_see_them_alone(gemv):
    """Rows of NaN in the cache (what a NaN leaves there) in front of a window, behind a query, and in sight."""
    b = Batch(gemv, [100, 100, 100], 16, 1, 2, 64, E4M3, torch.float32, n_q=3, seed=9)
    bad = [(0, 10), (1, 99), (2, 97)]  # before the window; the last token; the first query's own
    slots = torch.tensor([b.places(b.tables[i], 100)[at] for i, at in bad], dtype=torch.int32, device=DEV)
    nan = torch.full((3, 64), float("nan"), device=DEV)
    for k, v in ((nan, torch.ones_like(nan)), (torch.ones_like(nan), nan)):
        gemv.kv_write(k, v, slots, b.cache, 3, 1, 64, 16, E4M3)
        out, lse = b.run(window=50)
        torch.cuda.synchronize()
        got = host(torch.isnan(out).all(1)).reshape(3, 3)
        assert got.tolist() == [[False] * 3, [False, False, True], [True] * 3]
        assert np.array_equal(host(torch.isnan(out).any(1)).reshape(3, 3), got)
        want = b.want(window=50)
        sees = ~got.reshape(-1)
        assert np.all(np.abs(host(out)[sees] - want[0][sees]) <= want[1][sees])
    q = b.q.clone()
    b = Batch(gemv, [100, 100, 100], 16, 1, 2, 64, E4M3, torch.float32, n_q=3, seed=9)
    b.q[4, 70] = float("nan")
    out, _ = b.run()
    torch.cuda.synchronize()
    assert torch.isnan(out[4, 64:]).all() and torch.isfinite(out[4, :64]).all()
    assert torch.isfinite(out[[i for i in range(9) if i != 4]]).all() and torch.equal(q[0], b.q[0])


def test_pages_that_are_not_in_the_cache(gemv):
    """Their tokens count as not seen, in the middle, at the end and all of them; nothing else is read."""
    b = Batch(gemv, [100, 100, 100, 100], 16, 2, 2, 64, I8, torch.float32, prefix=64, seed=10)
    b.tables[0, 2] = -1
    b.tables[1, 6] = b.n_pages
    b.tables[2, :] = 2 ** 31 - 1
    b.tables[3, 3:5] = -2 ** 31
    b.check()
    b.prefix[1] = -5
    b.check()
    b.prefix[:] = b.n_pages
    out, lse = b.check()
    assert torch.all(out[2] == 0) and torch.all(torch.isneginf(lse[2]))


def test_lengths_out_of_range(gemv):
    """Taken as at least 0 and at most what the pages hold."""
    b = Batch(gemv, [64, 64, 64, 64], 16, 1, 2, 64, I8, torch.float32, prefix=48, seed=13)
    lens = np.array([-1, 2 ** 31 - 1, 65, -2 ** 31], np.int32)
    for plen in (-3, 49, 2 ** 31 - 1):
        t = dict(lens=torch.from_numpy(lens).to(DEV), prefix_len=torch.tensor([plen], dtype=torch.int32, device=DEV))
        out, lse = b.run(**t)
        torch.cuda.synchronize()
        b.close(out, lse, b.want(lens=lens, prefix_len=plen))


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_apart_and_off_their_vectors(gemv, dtype):
    """Queries as columns of a row of projections, outputs between other columns, tables of a wider one."""
    b = Batch(gemv, [50, 7, 90], 16, 2, 3, 64, I8, dtype, prefix=20, seed=14)
    want = b.check()
    w = b.heads * b.dim
    for off, width in ((0, w + 8), (8, w + 24), (1, w + 1), (3, w + 10)):
        rows, outs = (torch.full((4, width), 2.0, dtype=dtype, device=DEV) for _ in range(2))
        q, out = rows[:, off:off + w], outs[:, off:off + w]
        q[:3].copy_(b.q)
        wide = torch.full((5, b.tables.shape[1] + 3), 99, dtype=torch.int32, device=DEV)
        wide[:3, 1:1 + b.tables.shape[1]].copy_(torch.from_numpy(b.tables))
        got, lse = b.run(q=q, out=out, tables=wide[:, 1:1 + b.tables.shape[1]])
        torch.cuda.synchronize()
        assert torch.equal(got[:3], want[0]) and torch.equal(lse, want[1])
        left = torch.ones_like(outs, dtype=torch.bool)
        left[:3, off:off + w] = False
        assert torch.all(outs[left] == 2.0)


def test_without_lse_and_with_any_workspace(gemv):
    b = Batch(gemv, [500, 20], 16, 2, 2, 64, I8, torch.float32, prefix=300, seed=15)
    want, _ = b.check()
    for fill in (0, 0x7F):
        ws = b.workspace().fill_(fill)
        guard = torch.full((ws.numel() + 512,), 0x55, dtype=torch.uint8, device=DEV)
        guard[256:-256].copy_(ws)
        out, _ = b.run(lse=None, workspace=guard[256:-256])
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        assert torch.all(guard[:256] == 0x55) and torch.all(guard[-256:] == 0x55)


def test_the_same_bits_alone_and_again(gemv):
    """The same call again and again, other work between."""
    b = Batch(gemv, [3000, 20, 700], 16, 2, 2, 64, E4M3, torch.float32, prefix=300, seed=16)
    want = b.check()
    other = Batch(gemv, [100] * 5, 16, 2, 2, 64, E4M3, torch.float32, seed=17)
    ws = max(b.workspace(), other.workspace(), key=len)
    for _ in range(3):
        other.run(workspace=ws)
        got = b.run(workspace=ws)
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_replayed_as_the_sequences_grow(gemv):
    """Captured once; every replay's token is written first, lengths and prefix change between, other graphs and eager
    calls use the same workspace one after the other."""
    b = Batch(gemv, [200, 200, 200], 16, 2, 2, 64, I8, torch.float32, prefix=64, seed=18)
    t, ws = b.tensors(), b.workspace()
    out, lse = torch.empty_like(b.q), torch.empty((3, 4), device=DEV)
    rng = np.random.default_rng(19)
    k, v = (torch.zeros((3, 128), device=DEV) for _ in range(2))
    slots = torch.zeros(3, dtype=torch.int32, device=DEV)

    def step(stream=None):
        gemv.kv_write(k, v, slots, b.cache, 3, 2, 64, 16, I8, stream=stream)
        b.run(out=out, lse=lse, workspace=ws, stream=stream, **t)

    lens = np.array([1, 40, 100], np.int32)
    plen = 64

    def feed():
        for x in (k, v, b.q):
            x.copy_(torch.from_numpy(rng.standard_normal(tuple(x.shape)).astype(np.float32)))
        t["lens"].copy_(torch.from_numpy(lens))
        t["prefix_len"].fill_(plen)
        at = [b.places(b.tables[i], int(n))[-1] if n else -1 for i, n in enumerate(lens)]
        slots.copy_(torch.tensor(at, dtype=torch.int32))
        torch.cuda.synchronize()

    feed()
    step()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            step()
        graphs.append(g)
    side = torch.cuda.Stream()
    for i in range(8):
        lens = np.array([1 + i, 40 + 20 * i, 0 if i % 3 == 1 else 100 + i], np.int32)
        plen = [64, 0, 1, 33][i % 4]
        feed()
        if i % 3 == 2:
            step(side)
        else:
            graphs[i % 2].replay()
        torch.cuda.synchronize()
        b.close(out, lse, b.want(lens=lens, prefix_len=plen))


def test_two_calls_at_once_with_a_workspace_each(gemv):
    one = Batch(gemv, [3000, 20, 700], 16, 2, 2, 64, E4M3, torch.float32, prefix=300, seed=20)
    two = Batch(gemv, [900, 2000], 16, 2, 4, 64, I8, torch.bfloat16, seed=21)
    want = [one.check(), two.check()]
    streams = [torch.cuda.Stream() for _ in range(2)]
    ws = [one.workspace(), two.workspace()]
    for _ in range(5):
        # made and filled before either call: that is the current stream's work
        given = [dict(b.tensors(), out=torch.full_like(b.q, 9.0), lse=torch.full_like(w[1], 9.0))
                 for b, w in zip((one, two), want)]
        torch.cuda.synchronize()
        got = [b.run(workspace=w, stream=s, **g) for b, w, s, g in zip((one, two), ws, streams, given)]
        torch.cuda.synchronize()
        for g, w in zip(got, want):
            assert torch.equal(g[0], w[0]) and torch.equal(g[1], w[1])


def test_a_cache_whose_bytes_pass_32_bits(gemv):
    page, kv, dim = 256, 8, 256
    b = Batch(gemv, [300], page, kv, 2, dim, I8, torch.float32, seed=22)
    out, lse = b.check()
    pages = (5 << 30) // (page * kv * (2 * dim + 8))
    big = torch.empty((pages, kv * b.layout.block), dtype=torch.uint8, device=DEV)
    small = b.cache.view(b.n_pages, -1)
    tables = torch.tensor([[pages - 1, pages - 7]], dtype=torch.int32, device=DEV)
    for at, page_id in zip(tables[0].tolist(), b.tables[0].tolist()):
        big[at].copy_(small[page_id])
    b.cache = big
    got = b.run(tables=tables)
    torch.cuda.synchronize()
    assert torch.equal(got[0], out) and torch.equal(got[1], lse)


def test_no_sequences(gemv):
    none = torch.empty((0, 128), device=DEV)
    ints = torch.empty(0, dtype=torch.int32, device=DEV)
    cache = torch.zeros(2 * 16 * 136, dtype=torch.uint8, device=DEV)
    gemv.attention(none, cache, torch.empty((0, 1), dtype=torch.int32, device=DEV), ints, none.clone(),
                   torch.empty(gemv.attention_workspace_bytes(0, 1, 2, 1, 64), dtype=torch.uint8, device=DEV), 0, 2, 1, 64, 16, 1.0)
    torch.cuda.synchronize()
