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
