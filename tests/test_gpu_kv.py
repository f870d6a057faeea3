"""ft_hip_kv_write and ft_hip_kv_read against the formats in 64 bits: codes and
scales bit for bit, places byte for byte, everything else of the cache as it was."""
import numpy as np
import pytest
import torch

import ft_hip

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
I8, E4M3 = ft_hip.KV_I8, ft_hip.KV_E4M3
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def host(t):
    return t.detach().cpu().numpy()


# ---- the formats, in numpy ----

E4M3_VALUES = np.array([(-1.0) ** (c >> 7) * ((c & 7) * 2.0 ** -9 if c >> 3 & 15 == 0 else (8 + (c & 7)) * 2.0 ** ((c >> 3 & 15) - 10))
                        for c in range(256)])
E4M3_VALUES[[0x7F, 0xFF]] = np.nan


def quantise(x, kind):
    """(bytes, scales) of rows [..., dim] of f64 values."""
    a = np.abs(x).max(-1)
    with np.errstate(invalid="ignore"):
        bad, a = ~np.isfinite(a), np.where(np.isfinite(a), a, 0.0)
    x = np.where(bad[..., None], 0.0, x)
    one = np.where(a > 0, a, 1.0)[..., None]
    if kind == I8:
        q = np.sign(x) * np.floor(127.0 * np.abs(x) / one + 0.5)
        d = np.float32(a / 127.0)
        codes = (q + 128).astype(np.uint8)
    else:
        m, e = np.frexp(one)  # one = m 2^e, m in [1/2, 1)
        e = np.maximum(e - 9 + (m > 0.875), -126)
        y = np.abs(x) / np.ldexp(1.0, e)
        step = np.ldexp(1.0, np.maximum(np.frexp(y)[1] - 1, -6) - 3)
        y = np.rint(y / step) * step  # halves to even
        positive = E4M3_VALUES[:127]
        codes = np.searchsorted(positive, y).astype(np.uint8)
        assert np.array_equal(positive[codes], y)
        codes |= np.where(np.signbit(x), 128, 0).astype(np.uint8)
        d = np.where(a > 0, np.ldexp(1.0, e[..., 0]), 0.0).astype(np.float32)
    return codes, np.where(bad, np.float32(np.nan), d)


class Layout:
    """Bytes of a cache by slot, head and dimension, as the header gives them."""

    def __init__(self, page, heads, dim):
        self.page, self.heads, self.dim = page, heads, dim
        self.block = page * (2 * dim + 8)

    def at(self, slots, value):
        """[n, heads, dim] places of bytes."""
        slots = np.asarray(slots, np.int64)
        o, d = (slots % self.page)[:, None, None], np.arange(self.dim)
        base = ((slots // self.page)[:, None] * self.heads + np.arange(self.heads))[:, :, None] * self.block
        tile = o // 16 * 16 * self.dim
        if value:
            return base + self.page * self.dim + tile + d // 64 * 1024 + o % 16 // 4 * 256 + d % 64 * 4 + o % 4
        return base + tile + d // 16 * 256 + o % 16 * 16 + d % 16

    def scales_at(self, slots, value):
        """[n, heads] places of f32."""
        slots = np.asarray(slots, np.int64)
        base = ((slots // self.page)[:, None] * self.heads + np.arange(self.heads)) * self.block
        return (base + 2 * self.page * self.dim + 4 * self.page * value) // 4 + (slots % self.page)[:, None]

    def put(self, cache, slots, k, v, kind):
        """Writes rows [n, heads, dim] into a numpy cache."""
        for value, x in enumerate((k, v)):
            codes, d = quantise(np.asarray(x, np.float64), kind)
            cache[self.at(slots, value)] = codes
            cache.view(np.float32)[self.scales_at(slots, value)] = d

    def get(self, cache, slots, kind):
        """(k, v) [n, heads, dim] as f64."""
        out = []
        for value in (0, 1):
            codes = cache[self.at(slots, value)]
            q = codes.astype(np.float64) - 128 if kind == I8 else E4M3_VALUES[codes]
            with np.errstate(invalid="ignore"):  # scales of places never written may be anything
                out.append(q * cache.view(np.float32)[self.scales_at(slots, value)].astype(np.float64)[:, :, None])
        return out


def same_bits(a, b):
    return np.array_equal(a.view(np.uint8), b.view(np.uint8))


def same_cache(got, want, layout):
    """Every byte, with NaN scales as NaN."""
    g, w = got.view(np.float32).copy(), want.view(np.float32).copy()
    pages = np.arange(got.size // (layout.block * layout.heads) * layout.page)
    for value in (0, 1):
        at = layout.scales_at(pages, value)
        assert np.array_equal(np.isnan(g[at]), np.isnan(w[at]))
        for x in (g, w):
            s = x[at]
            s[np.isnan(s)] = np.float32(7.0)
            x[at] = s
    return same_bits(g, w)


def rows_of(rng, n, width, dtype):
    x = rng.standard_normal((n, width)) * np.exp(rng.uniform(-3, 3, (n, 1)))
    return torch.from_numpy(x.astype(np.float32)).to(dtype).to(DEV)


def check_write(gemv, k, v, slots, page, heads, dim, kind, pages, seed=0, n=None):
    lay = Layout(page, heads, dim)
    before = np.random.default_rng(seed).integers(0, 256, pages * heads * lay.block, dtype=np.uint8)
    cache = torch.from_numpy(before.copy()).to(DEV)
    slots = np.asarray(slots, np.int32)
    n = len(slots) if n is None else n
    gemv.kv_write(k, v, torch.from_numpy(slots).to(DEV), cache, n, heads, dim, page, kind)
    torch.cuda.synchronize()
    want, live = before.copy(), (slots[:n] >= 0) & (slots[:n] < pages * page)
    wide = lambda t: host(t.float())[:n].astype(np.float64).reshape(n, heads, dim)[live]  # noqa: E731
    lay.put(want, slots[:n][live], wide(k), wide(v), kind)
    got = host(cache)
    assert same_cache(got, want, lay)
    return cache


@pytest.mark.parametrize("kind", [I8, E4M3])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("page,heads,dim,n", [(16, 1, 64, 1), (64, 8, 256, 1), (16, 3, 128, 5), (32, 2, 256, 37), (128, 4, 64, 130),
                                              (256, 1, 128, 300), (64, 8, 128, 16)])
def test_write_and_read(gemv, kind, dtype, page, heads, dim, n):
    rng = np.random.default_rng(n * dim + heads)
    pages = (n + 20) // page + 3
    first = 7
    order = rng.permutation(pages)
    at = np.arange(first, first + n)
    slots = order[at // page] * page + at % page
    k, v = rows_of(rng, n, heads * dim, dtype), rows_of(rng, n, heads * dim, dtype)
    cache = check_write(gemv, k, v, slots, page, heads, dim, kind, pages)
    # read back: the products q d, rounded to f32 and then to the type: half a step of each
    ko, vo = torch.empty_like(k), torch.empty_like(v)
    gemv.kv_read(cache, torch.from_numpy(slots.astype(np.int32)).to(DEV), ko, vo, n, heads, dim, page, kind)
    torch.cuda.synchronize()
    half = torch.finfo(dtype).eps / 2 + 2.0 ** -24
    least = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    for got, want, x in zip((ko, vo), Layout(page, heads, dim).get(host(cache), slots, kind), (k, v)):
        got, x = host(got.float()).reshape(n, heads, dim), host(x.float()).reshape(n, heads, dim)
        assert np.all(np.abs(got - want) <= half * np.abs(want) + least)
        # and what the format keeps: half a step of a / 127, or 2^-4 of a value (2^-10 of the scale below 2^-6 of it)
        a = np.abs(x).max(2, keepdims=True)
        lost = a / 254 if kind == I8 else np.maximum(2.0 ** -4 * np.abs(x), 2.0 ** -10 * a / 224)
        assert np.all(np.abs(got - x) <= lost * (1 + 2.0 ** -20) + (half + 2.0 ** -23) * np.abs(x) + least)


@pytest.mark.parametrize("dim,dtype,kind", [(64, torch.float32, E4M3), (64, torch.float16, I8), (64, torch.bfloat16, E4M3),
                                            (128, torch.float16, E4M3), (128, torch.float32, I8), (256, torch.bfloat16, I8)])
def test_many_rows_with_parts_left_over(gemv, dim, dtype, kind):
    """65604 rows: four of a token's 142 parts a wavefront, and two at its end."""
    rng = np.random.default_rng(dim)
    page, heads, n = 32, 71, 924
    pages = n // page + 2
    order = rng.permutation(pages)
    at = np.arange(2, n + 2)
    slots = (order[at // page] * page + at % page).astype(np.int32)
    slots[[5, 100, 101]] = -1, pages * page, 2 ** 31 - 1
    k, v = rows_of(rng, n, heads * dim, dtype), rows_of(rng, n, heads * dim, dtype)
    cache = check_write(gemv, k, v, slots, page, heads, dim, kind, pages)
    ko, vo = torch.full_like(k, 9.0), torch.full_like(v, 9.0)
    gemv.kv_read(cache, torch.from_numpy(slots).to(DEV), ko, vo, n, heads, dim, page, kind)
    torch.cuda.synchronize()
    live = (slots >= 0) & (slots < pages * page)
    for got, want in zip((ko, vo), Layout(page, heads, dim).get(host(cache), slots[live], kind)):
        exact = torch.from_numpy(want.reshape(int(live.sum()), -1).astype(np.float32)).to(dtype)
        assert torch.equal(got.cpu()[live], exact) and bool((got.cpu()[~live] == 9.0).all())


@pytest.mark.parametrize("kind", [I8, E4M3])
def test_scattered_skipped_and_out_of_range_slots(gemv, kind):
    rng = np.random.default_rng(4)
    page, heads, dim, pages, n = 32, 2, 128, 6, 61
    slots = rng.permutation(pages * page)[:n]
    slots[[0, 9, 17]] = -1
    slots[[3, 30]] = pages * page, 2 ** 31 - 1
    slots[12] = -2 ** 31
    slots[20:24] = [40, 41, 42, 43]       # a group in order,
    slots[24:28] = [47, 46, 45, 44]       # one backwards,
    slots[28:30] = [pages * page - 1, 0]  # the last place and the first
    first = {}
    for i, s in enumerate(slots):  # each place once: what equal slots leave is nobody's to say
        if s in first:
            slots[first[s]] = -1
        first[s] = i
    k, v = rows_of(rng, n, heads * dim, torch.float32), rows_of(rng, n, heads * dim, torch.float32)
    cache = check_write(gemv, k, v, slots, page, heads, dim, kind, pages)
    out = [torch.full((n, heads * dim), 7.0, device=DEV) for _ in range(2)]
    gemv.kv_read(cache, torch.from_numpy(slots.astype(np.int32)).to(DEV), *out, n, heads, dim, page, kind)
    torch.cuda.synchronize()
    live = (slots >= 0) & (slots < pages * page)
    for got, want in zip(out, Layout(page, heads, dim).get(host(cache), slots[live], kind)):
        got = host(got).reshape(n, heads, dim)
        assert np.all(got[~live] == 7.0)
        assert np.all(np.abs(got[live] - want) <= 2.0 ** -24 * np.abs(want))


@pytest.mark.parametrize("start", range(8))
@pytest.mark.parametrize("n", [1, 2, 3, 4, 5, 8, 19])
def test_every_start_in_a_group(gemv, start, n):
    """Runs of tokens from every place of a group, ended in every place."""
    rng = np.random.default_rng(start * 100 + n)
    k, v = rows_of(rng, n, 64, torch.float16), rows_of(rng, n, 64, torch.float16)
    check_write(gemv, k, v, 16 + start + np.arange(n), 16, 1, 64, I8, 4)


@pytest.mark.parametrize("kind", [I8, E4M3])
@pytest.mark.parametrize("dtype", TYPES)
def test_rows_apart_and_off_their_vectors(gemv, kind, dtype):
    """Columns of a wider row, from odd places on; rows behind n stay unread and unwritten."""
    rng = np.random.default_rng(6)
    page, heads, dim, n = 16, 2, 64, 23
    for off, width in ((0, 512), (1, 517), (4, 516), (3, 259)):
        rows = rows_of(rng, n + 2, 2 * width, dtype)
        k, v = rows[:, off:off + heads * dim], rows[:, width + off:width + off + heads * dim]
        cache = check_write(gemv, k, v, 5 + np.arange(n), page, heads, dim, kind, 3, n=n)
        out = torch.full((n + 2, 2 * width), 3.0, dtype=dtype, device=DEV)
        ko, vo = out[:, off:off + heads * dim], out[:, width + off:width + off + heads * dim]
        gemv.kv_read(cache, torch.arange(5, 5 + n, dtype=torch.int32, device=DEV), ko, vo, n, heads, dim, page, kind)
        whole = [torch.empty((n, heads * dim), dtype=dtype, device=DEV) for _ in range(2)]
        gemv.kv_read(cache, torch.arange(5, 5 + n, dtype=torch.int32, device=DEV), *whole, n, heads, dim, page, kind)
        torch.cuda.synchronize()
        assert torch.equal(ko[:n], whole[0]) and torch.equal(vo[:n], whole[1])
        left = torch.ones_like(out, dtype=torch.bool)
        left[:n, off:off + heads * dim] = False
        left[:n, width + off:width + off + heads * dim] = False
        assert torch.all(out[left] == 3.0)


def special_rows(dim):
    """f32 rows of 8-bit formats' hard values."""
    f = np.float32
    rng = np.random.default_rng(9)
    x = rng.standard_normal((24, dim)).astype(f)
    x[0] = 0.0
    x[1] = -0.0
    x[2, 3] = np.nan
    x[3, 5] = np.inf
    x[4, 6], x[4, 7] = -np.inf, np.nan
    x[5] = 0.0
    x[5, 1] = f(1e-45)                         # the smallest subnormal alone
    x[6] = x[6] * f(1e-39)                     # subnormals
    x[7] = x[7] * f(1e38)
    x[8, 0] = np.finfo(f).max
    x[9] = f(-3.5)                             # all equal
    x[10, 0], x[10, 1:] = f(127.0), (np.arange(dim - 1) % 127 + 0.5).astype(f)       # i8's halves
    x[11, 0], x[11, 1:] = f(127.0), -(np.arange(dim - 1) % 127 + 0.5).astype(f)
    x[12, 0], x[12, 1:] = f(254.0), np.nextafter((2 * (np.arange(dim - 1) % 127) + 1).astype(f), f(0))  # just below
    x[13, 0], x[13, 1:] = f(254.0), np.nextafter((2 * (np.arange(dim - 1) % 127) + 1).astype(f), f(1e9))
    x[14, 0] = f(448.0)                        # e4m3's scale of 1, all codes and the halves between them
    halves = (E4M3_VALUES[:126] + E4M3_VALUES[1:127]) / 2
    x[14, 1:] = np.resize(halves, dim - 1)
    x[15, 0], x[15, 1:] = f(448.0), -np.resize(halves, dim - 1)[::-1]
    x[16, 0], x[16, 1:] = f(448.0), np.resize(E4M3_VALUES[:127], dim - 1)
    x[17, 0], x[17, 1:] = np.nextafter(f(448.0), f(500)), np.resize(halves, dim - 1)  # the next scale
    x[18, 0], x[18, 1:] = f(448.0), np.nextafter(np.resize(halves, dim - 1).astype(f), f(0))
    x[19, 0], x[19, 1:] = f(-448.0), np.nextafter(np.resize(halves, dim - 1).astype(f), f(1e9))
    x[20] = np.ldexp(x[20], -118)
    x[20, 0] = np.ldexp(f(1.9), -118)
    x[21] = 0.0
    x[21, 0] = 1.0
    x[22, :] = np.ldexp(f(1.0), -rng.integers(0, 30, dim)).astype(f)
    x[23] = np.where(rng.random(dim) < 0.5, f(1.0), f(-1.0)) * np.resize(halves, dim).astype(f) * f(1.75)
    return x


@pytest.mark.parametrize("kind", [I8, E4M3])
@pytest.mark.parametrize("dim", [64, 256])
def test_zeros_halves_subnormals_infinities_and_nan(gemv, kind, dim):
    x = torch.from_numpy(special_rows(dim)).to(DEV)
    v = x.flip(0).contiguous()
    cache = check_write(gemv, x, v, 3 + np.arange(24), 16, 1, dim, kind, 2)
    out = [torch.empty_like(x) for _ in range(2)]
    gemv.kv_read(cache, torch.arange(3, 27, dtype=torch.int32, device=DEV), *out, 24, 1, dim, 16, kind)
    torch.cuda.synchronize()
    got = host(out[0])
    assert np.all(np.isnan(got[2:5])) and np.all(got[:2] == 0)
    # else f32(q d), bit for bit: d = f32(a / 127) may lie 2^-24 of itself above a / 127, and where a is the largest f32
    # 127 d then lies at or past half a step over it, which rounds to inf
    for x, want in zip(out, Layout(16, 1, dim).get(host(cache), 3 + np.arange(24), kind)):
        with np.errstate(over="ignore"):
            want = want.reshape(24, dim).astype(np.float32)
        assert np.array_equal(host(x), want, equal_nan=True)
        assert np.isinf(want).sum() <= 1


def test_every_16_bit_value(gemv):
    """All finite f16 and bf16 values as single values of a row whose largest is 1, 127 and 448 of their kind."""
    for dtype in (torch.float16, torch.bfloat16):
        x = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(dtype).float()
        x = x[torch.isfinite(x) & (x.abs() <= 448)]
        x = torch.cat([x, torch.zeros(-len(x) % 63)]).view(-1, 63)
        x = torch.cat([torch.full((len(x), 1), 448.0), x], 1).to(dtype).to(DEV)
        for kind in (I8, E4M3):
            check_write(gemv, x, x, np.arange(len(x)), 256, 1, 64, kind, len(x) // 256 + 1)


def test_a_cache_whose_bytes_pass_32_bits(gemv):
    page, heads, dim = 256, 8, 256
    pages = (5 << 30) // (page * heads * (2 * dim + 8))
    lay = Layout(page, heads, dim)
    cache = torch.zeros((pages, heads * lay.block), dtype=torch.uint8, device=DEV)
    slots = np.array([0, pages * page - 1, pages * page - 2, (pages - 1) * page, pages // 2 * page + 5], np.int32)
    rng = np.random.default_rng(8)
    k, v = rows_of(rng, 5, heads * dim, torch.float32), rows_of(rng, 5, heads * dim, torch.float32)
    gemv.kv_write(k, v, torch.from_numpy(slots).to(DEV), cache, 5, heads, dim, page, I8)
    out = [torch.empty_like(k) for _ in range(2)]
    gemv.kv_read(cache, torch.from_numpy(slots).to(DEV), *out, 5, heads, dim, page, I8)
    torch.cuda.synchronize()
    for x, got in zip((k, v), out):
        codes, d = quantise(host(x).astype(np.float64).reshape(5, heads, dim), I8)
        want = ((codes.astype(np.float64) - 128) * d[:, :, None]).reshape(5, -1)
        assert np.all(np.abs(host(got) - want) <= 2.0 ** -24 * np.abs(want))
    # the pages between hold nothing
    touched = sorted({int(s) // page for s in slots})
    for p in range(pages):
        if p not in touched and (p < 4 or p > pages - 4 or p % 501 == 0):
            assert not cache[p].any()


def test_replayed_on_new_tokens_and_on_another_stream(gemv):
    rng = np.random.default_rng(10)
    page, heads, dim, n = 16, 2, 64, 9
    lay = Layout(page, heads, dim)
    k, v = rows_of(rng, n, heads * dim, torch.float32), rows_of(rng, n, heads * dim, torch.float32)
    slots = torch.arange(n, dtype=torch.int32, device=DEV)
    cache = torch.zeros(8 * heads * lay.block, dtype=torch.uint8, device=DEV)
    out = [torch.zeros_like(k) for _ in range(2)]

    def step(stream=None):
        gemv.kv_write(k, v, slots, cache, n, heads, dim, page, E4M3, stream=stream)
        gemv.kv_read(cache, slots, *out, n, heads, dim, page, E4M3, stream=stream)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    want = np.zeros_like(host(cache))
    lay.put(want, np.arange(n), host(k).reshape(n, heads, dim), host(v).reshape(n, heads, dim), E4M3)
    side = torch.cuda.Stream()
    for i in range(1, 5):
        k.copy_(rows_of(rng, n, heads * dim, torch.float32))
        v.copy_(rows_of(rng, n, heads * dim, torch.float32))
        slots.add_(n)
        torch.cuda.synchronize()
        if i == 3:
            step(side)
            side.synchronize()
        else:
            graph.replay()
        torch.cuda.synchronize()
        lay.put(want, host(slots), host(k).reshape(n, heads, dim), host(v).reshape(n, heads, dim), E4M3)
        assert same_cache(host(cache), want, lay)
        for got, x in zip(out, lay.get(want, host(slots), E4M3)):
            assert np.array_equal(host(got).reshape(n, heads, dim), x)


@pytest.mark.parametrize("kind", [I8, E4M3])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_narrow_rows_are_rounded_from_f32(gemv, kind, dtype):
    """f32(q d) and then the type, where one rounding of q d would now and then be another number."""
    n, heads, dim = 5000, 4, 64
    x = (torch.randn(2, n, heads * dim, generator=torch.Generator().manual_seed(5)) * 3.0).to(DEV)
    layout, slots = Layout(16, heads, dim), torch.arange(n, dtype=torch.int32, device=DEV)
    cache = torch.zeros(313 * heads * layout.block, dtype=torch.uint8, device=DEV)
    gemv.kv_write(x[0], x[1], slots, cache, n, heads, dim, 16, kind)
    out = [torch.empty_like(x[0], dtype=dtype) for _ in range(2)]
    gemv.kv_read(cache, slots, *out, n, heads, dim, 16, kind)
    torch.cuda.synchronize()
    for got, want in zip(out, layout.get(host(cache), np.arange(n), kind)):  # 8 bits times 24: exact in 64 bits
        assert torch.equal(got.cpu(), torch.from_numpy(want.reshape(n, -1).astype(np.float32)).to(dtype))


def test_no_tokens(gemv):
    cache = torch.full((2 * 16 * 136,), 9, dtype=torch.uint8, device=DEV)
    none = torch.empty((0, 64), device=DEV)
    slots = torch.empty(0, dtype=torch.int32, device=DEV)
    gemv.kv_write(none, none, slots, cache, 0, 1, 64, 16)
    gemv.kv_read(cache, slots, none, none.clone(), 0, 1, 64, 16)
    torch.cuda.synchronize()
    assert torch.all(cache == 9)
