"""Top-k around the limits between a draw's ways through a row: the number of
64-value segments, shares of it, and the 8192 values that a workgroup lists."""
import numpy as np
import pytest
import torch

from test_gpu_sample import check, model_logits

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("V", [8193, 50021, 131072, 262144])
@pytest.mark.parametrize("p", [None, 0.9])
def test_top_k_around_the_segments(gemv, V, p):
    segs = (V + 63) // 64
    ks = sorted({int(segs * x) + d for x in (0.5, 0.75, 0.81, 0.875, 0.95, 1.0) for d in (-1, 0, 1)})
    rng = np.random.default_rng(V)
    n = len(ks)
    l = torch.from_numpy(np.repeat(model_logits(rng, 1, V, level=9.0), n, 0))
    check(gemv, l, rng.random(n), k=ks, t=rng.uniform(0.6, 2, n), p=None if p is None else [p] * n)


@pytest.mark.parametrize("k", [6000, 6162, 6163, 8191, 8192, 8193, 20000, 32767, 32768, 32769])
def test_top_k_of_the_largest_vocabulary(gemv, k):
    rng = np.random.default_rng(k)
    l = torch.from_numpy(model_logits(rng, 1, 1 << 21, level=9.0))
    check(gemv, l, [0.7], k=[k], t=[1.3])
    check(gemv, l, [0.3], k=[k], m=[0.02])


@pytest.mark.parametrize("V", [131072, 262144])
@pytest.mark.parametrize("kind", ["around zero", "uniform", "below zero", "sorted"])
def test_top_k_of_rows_whose_maxima_lie_otherwise(gemv, V, kind):
    """Maxima on both sides of 0, close to one bound, and the largest values side by side."""
    segs = (V + 63) // 64
    ks = [segs // 2, segs * 3 // 4, int(segs * 0.81), int(segs * 0.87), segs * 15 // 16]
    rng = np.random.default_rng(V + len(kind))
    l = rng.uniform(-5, 5, (len(ks), V)) if kind == "uniform" else 2.5 * rng.standard_normal((len(ks), V))
    l = np.sort(l, 1) if kind == "sorted" else l - dict(zip(("around zero", "below zero"), (5.0, 40.0))).get(kind, 0.0)
    check(gemv, torch.from_numpy(l.astype(np.float32)), rng.random(len(ks)), k=ks, t=[1.0, 0.5, 2.0, 1.0, 1.5])


def test_rows_of_either_way_in_one_batch(gemv):
    """Row by row the scan leaves the maxima alone or fills the bins; the finish reads what is there."""
    rng = np.random.default_rng(3)
    n, V = 64, 40000
    l = torch.from_numpy(model_logits(rng, n, V))
    k = rng.choice([0, 1, 300, 540, 546, 547, 548, 600, 625, 700, 30000], n)
    check(gemv, l, rng.random(n), k=k, t=np.where(rng.random(n) < 0.1, 0.0, rng.uniform(0.5, 2, n)),
          p=rng.uniform(0.3, 1.3, n))
