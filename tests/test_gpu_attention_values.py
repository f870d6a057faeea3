"""ft_hip_attention on values of every size: the definition and tolerances are test_gpu_attention's.

What those leave out: numbers below the smallest normal one. A piece of a row leaves its average and the pieces are
joined in f32, each rounded to half of the type's smallest step at most: (pieces + 2) 2^-150 beside the rest, and a
piece has at least one token. A weight times a scale is held to 2^-151 at least, which a value's 8 bits multiply:
n 2^-151 max |q|.
"""
import numpy as np
import pytest
import torch

from test_gpu_attention import DEV, Batch, host
from test_gpu_kv import E4M3, I8

pytestmark = pytest.mark.gpu


def put(b, slots, k=None, v=None):
    """Rows of keys and values in place of what the cache has in these slots; None: normal ones, by the slot."""
    each = [np.random.default_rng(int(x)).standard_normal((2, b.kv * b.dim)) for x in slots]
    k, v = (torch.from_numpy((np.stack([e[j] for e in each]) if x is None else x).astype(np.float32)).to(DEV)
            for j, x in enumerate((k, v)))
    b.g.kv_write(k, v, torch.tensor(np.asarray(slots), dtype=torch.int32, device=DEV), b.cache, len(slots), b.kv, b.dim,
                 b.page, b.kind)


def all_slots(b):
    own = [b.places(b.tables[i], int(x)) for i, x in enumerate(b.lens) if x > 0]
    if b.prefix is not None:
        own.append(b.places(b.prefix, b.prefix_len))
    return np.concatenate(own)


def close(b, out, want, subnormal=0.0):
    o, tol, _, _ = want
    got = host(out.float()).astype(np.float64)
    off = np.abs(got - o)
    assert np.all(off <= tol + subnormal), (float(np.nanmax(off / (tol + subnormal))), np.argwhere(~(off <= tol + subnormal))[:4].tolist())


@pytest.mark.parametrize("kind", [I8, E4M3])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("prefix", [0, 100])
@pytest.mark.parametrize("size", [1e-24, 1e-27, 1e-30, 1e-33, 1e-36, 1e-38, 1e-41])
def test_small_values(gemv, kind, dtype, prefix, size):
    """Down to scales that are no normal numbers: no less exact than others, as far as outputs have the bits."""
    b = Batch(gemv, [100, 40, 700, 1], 16, 1, 4, 64, kind, dtype, prefix=prefix, seed=70)
    slots = all_slots(b)
    rng = np.random.default_rng(71)
    put(b, slots, v=size * (rng.uniform(0.5, 1.5, (len(slots), 64)) * rng.choice([-1.0, 1.0, 1.0], (len(slots), 64))))
    out, _ = b.run()
    torch.cuda.synchronize()
    want = b.want()
    assert np.abs(want[0]).max() > size / 8
    codes = 127.0 if kind == I8 else min(448.0, 1.1 * (1.5 * size * 2.0 ** 126 + 2.0 ** -9))  # |v| / d, d at least 2^-126
    close(b, out, want, (700 + prefix + 2) * 2.0 ** -150 + (700 + prefix) * 2.0 ** -151 * codes)


@pytest.mark.parametrize("kind", [I8, E4M3])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,prefix", [(1, 0), (5, 0), (3, 300), (70, 200)])
def test_the_largest_values(gemv, kind, dtype, n, prefix):
    """Averages of numbers whose sum leaves f32's range."""
    b = Batch(gemv, [3000, 40, 1, 90, 700][:n] if n < 6 else [60] * n, 16, 1, 4, 64, kind, dtype, prefix=prefix, seed=72)
    slots = all_slots(b)
    rng = np.random.default_rng(73)
    put(b, slots, v=rng.uniform(2e38, 3e38, (len(slots), 64)) * np.where(np.arange(64) % 3 == 0, -1.0, 1.0))
    out, _ = b.run()
    torch.cuda.synchronize()
    close(b, out, b.want())


@pytest.mark.parametrize("kind", [I8, E4M3])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n_q,window,prefix", [(4, 0, 0), (4, 50, 0), (1, 50, 0), (3, 0, 64), (2, 90, 64), (1, 90, 64)])
def test_scales_of_tokens_that_a_query_does_not_see(gemv, kind, dtype, n_q, window, prefix):
    """Values far larger than the rest, behind a query or before its window: nothing of them reaches it, not in its
    last bit."""
    lens = [100, 77, 60, 20]
    b = Batch(gemv, lens, 16, 1, 2, 64, kind, dtype, prefix=prefix, n_q=n_q, seed=74)
    put(b, all_slots(b))
    plain, lse = b.check(window=window)
    # of each sequence: its newest token, if several are new, and the last one that its last query's window leaves out
    big, before = [], []
    for i, x in enumerate(lens):
        at = prefix + x - window - 1 if window else -1  # among prefix and own tokens
        for place in ([x - 1] if n_q > 1 else []) + ([at - prefix] if at >= prefix else []):
            big.append(b.places(b.tables[i], x)[place])
        before.append(at if window else -1)
    shared = [at for at in before if 0 <= at < prefix]
    if shared:  # the prefix's token that the shortest window end leaves out, and others still see
        big.append(b.places(b.prefix, prefix)[min(shared)])
    put(b, big, v=np.full((len(big), b.kv * 64), 1e30))
    out, got = b.run(window=window)
    torch.cuda.synchronize()
    out, plain = host(out.float()).reshape(4, n_q, -1), host(plain.float()).reshape(4, n_q, -1)
    checked = 0
    for i, x in enumerate(lens):
        for t in range(n_q):
            place = prefix + x - n_q + t
            lo = max(0, place + 1 - window) if window else 0
            sees = [prefix + x - 1] if n_q > 1 else []
            if before[i] >= prefix:
                sees.append(before[i])
            if shared:
                sees.append(min(shared))
            if not any(lo <= s <= place for s in sees):
                assert np.array_equal(out[i, t], plain[i, t]), (i, t)
                checked += 1
    assert checked
    assert torch.equal(got, lse)  # what a query sees of keys is the same


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kind", [I8, E4M3])
@pytest.mark.parametrize("bad", [float("inf"), float("-inf")])
def test_a_query_of_infinities_beside_large_values(gemv, dtype, kind, bad):
    """Its scores are no numbers or infinities; whichever values they fall on, the other rows' results are what they
    were. Rows enough that a lane holds several, a prefix that ends inside a step."""
    b = Batch(gemv, [5] * 40, 16, 1, 2, 64, kind, dtype, prefix=75, seed=76)
    put(b, all_slots(b))
    put(b, b.places(b.prefix, 75)[-1:], v=np.full((1, 64), 1e30))
    want, lse = b.check()
    for row in (0, 33):  # q k is minus or plus infinity by the key's sign
        q = b.q.clone()
        q[row] = 0.0
        q[row, ::64] = bad
        out, got = b.run(q=q)
        torch.cuda.synchronize()
        same = [i for i in range(40) if i != row]
        assert torch.equal(out[same], want[same]) and torch.equal(got[same], lse[same])


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("lens", [[131071], [70001], [40000] + [20] * 300, [131071] + [9] * 19])
def test_more_pieces_than_are_joined_at_once(gemv, dtype, lens):
    """One key head, so that all wavefronts have a piece of the long row; its largest scores are first or late: what was
    joined before is scaled, or what comes after."""
    group = 16 if len(lens) == 20 else 2
    b = Batch(gemv, lens, 64, 1, group, 64, I8, dtype, seed=75)
    q = host(b.q.float())[0].reshape(group, 64)
    places = b.places(b.tables[0], lens[0])
    for at, score in ((7, 16.0), (lens[0] - 100, 24.0), (lens[0] // 2, 40.0)):
        put(b, [places[at]], k=(8.0 * score / float(q[0] @ q[0]) * q[0])[None], v=np.full((1, 64), 3.0))
        b.check()


@pytest.mark.parametrize("lens,prefix", [([40], 0), ([5000], 0), ([90], 700), ([40000] + [20] * 300, 0)])
def test_no_number_shows_whatever_its_weight(gemv, lens, prefix):
    """A value that is NaN, seen with a weight that is 0 in f32 as all weights of its piece are."""
    b = Batch(gemv, lens, 16, 1, 2, 64, E4M3, torch.float32, prefix=prefix, seed=77)
    top = b.places(b.tables[0], lens[0])[-1]
    q = host(b.q)[0].reshape(2, 64)
    put(b, [top], k=(1000.0 * q.sum(0) / float(q[0] @ q[0]))[None])  # first among its row's by far
    out, lse = b.check(scale=50.0)
    first = b.places(b.prefix, prefix) if prefix else b.places(b.tables[0], lens[0])
    put(b, first[:1], v=np.full((1, 64), np.nan))
    got, same = b.run(scale=50.0)
    torch.cuda.synchronize()
    assert torch.isnan(got[0]).all() and torch.equal(same, lse)
    assert torch.equal(got[1:].isnan().all(1), torch.full((len(lens) - 1,), bool(prefix), device=DEV))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kind", [I8, E4M3])
@pytest.mark.parametrize("lens,prefix", [([50], 0), ([2000], 0), ([60, 3], 500)])
def test_keys_as_large_as_scores_allow(gemv, dtype, kind, lens, prefix):
    """The scale times the largest query and key just under 2^120: each row's largest score is alone, and its value the output."""
    b = Batch(gemv, lens, 16, 1, 2, 64, kind, dtype, prefix=prefix, seed=78)
    slots = all_slots(b)
    rng = np.random.default_rng(79)
    q = host(b.q.float()).astype(np.float64).reshape(len(lens), 2, 64)
    size = 2.0 ** 119 / (np.abs(q).max() / 8.0)
    put(b, slots, k=size * rng.uniform(-1, 1, (len(slots), 64)))
    out, lse = b.run()
    torch.cuda.synchronize()
    shared, pv = b.layout.get(host(b.cache), b.places(b.prefix, prefix), kind) if prefix else (np.zeros((0, 1, 64)),) * 2
    for i, n in enumerate(lens):
        k, v = b.layout.get(host(b.cache), b.places(b.tables[i], n), kind)
        k, v = np.concatenate([shared, k])[:, 0], np.concatenate([pv, v])[:, 0]
        for h in range(2):
            s = k @ q[i, h] / 8.0
            first = np.argsort(s)[::-1][:2]
            assert s[first[0]] - s[first[1]] > 1e-5 * s[first[0]]  # or its rounding might choose
            want = torch.from_numpy(v[first[0]]).to(dtype).double().numpy()
            got = host(out.double()).reshape(len(lens), 2, 64)[i, h]
            assert np.all(np.abs(got - want) <= (2.0 ** -21 + torch.finfo(dtype).eps) * np.abs(want))
            assert abs(host(lse)[i, h] / s[first[0]] - 1) < 1e-5
