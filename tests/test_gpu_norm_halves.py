"""The q8 quotients of ft_hip_add_rmsnorm that lie nearest to a half.

127 u / a of two f32 numbers, |u| <= a, is a half exactly or at least 2^-32 of
itself away from one; the pairs below are as near as that allows, on either
side of each half, found by the whole numbers' equation and rounded as
fractions.
"""
from fractions import Fraction

import numpy as np
import pytest
import torch

from test_gpu_norm import DEV, blocks

pytestmark = pytest.mark.gpu


def nearest_to_halves():
    """(m, u, a) with 127 u / a next to m + 1/2: u = U 2^-s, a = A of 24 bits, 254 U - (2 m + 1) A 2^s = +-1 (s = 0) or
    +-2 (both sides are even)."""
    out = []
    for m in range(127):
        odd = 2 * m + 1
        if odd == 127:  # 254 U - 127 A 2^s is a multiple of 127: the nearest is no nearer than usual
            continue
        for s in range(9):
            k, step = (254, odd) if s == 0 else (127, odd << (s - 1))
            if not k // 2 <= step < 2 * k:  # U / A has to be in (1/2, 2)
                continue
            for sign in (1, -1):
                first = pow(k, -1, step) * sign % step
                for U in range((1 << 23) + (first - (1 << 23)) % step, 1 << 24, step * 4099):
                    A = (k * U - sign) // step
                    assert k * U - step * A == sign
                    if 1 << 23 <= A < 1 << 24 and U <= A << s:
                        out.append((m, Fraction(U, 1 << s), Fraction(A)))
    return out


def test_quotients_nearest_to_a_half(gemv):
    pairs = nearest_to_halves()
    assert {m for m, _, _ in pairs} == set(range(127)) - {63}
    # one more such pair, and the f32 numbers next to it
    a, u = np.float32(127 * 131000 - 1), np.float32(128 * 131000 - 1) * np.float32(2.0 ** -8)
    pairs += [(0, Fraction(float(v)), Fraction(float(a))) for v in (u, np.nextafter(u, np.float32(0)), np.nextafter(u, a))]
    n = 0
    for scale in (0, -40, 60):
        x = np.zeros((len(pairs), 32), np.float32)
        want = np.zeros((len(pairs), 32), np.int64)
        for i, (_, u, a) in enumerate(pairs):
            x[i, :3] = [float(a) * 2.0 ** scale, float(u) * 2.0 ** scale, -float(u) * 2.0 ** scale]
            q = int(127 * u / a + Fraction(1, 2))
            want[i, :3] = [127, q, -q]
            n += abs(127 * u / a - (q - Fraction(1, 2))) <= Fraction(1, 1 << 25)
        q8 = torch.zeros(len(pairs) * 40, dtype=torch.uint8, device=DEV)
        gemv.add_rmsnorm(torch.from_numpy(x).to(DEV), None, 32, len(pairs), 1e-6, q8=q8)
        assert np.array_equal(blocks(q8, len(pairs), 32)[2][:, 0], want)
    assert n > 100


def test_quotients_of_subnormal_numbers(gemv):
    """Whole numbers of 2^-149: 127 u / 254 is u / 2, a half for every odd u."""
    u = np.arange(0, 254 + 1, dtype=np.int64)
    u = np.concatenate([u, -u])
    u = np.concatenate([u, np.zeros(-len(u) % 31, np.int64)]).reshape(-1, 31)
    x = np.concatenate([np.full((len(u), 1), 254), u], 1)
    q8 = torch.zeros(len(x) * 40, dtype=torch.uint8, device=DEV)
    gemv.add_rmsnorm(torch.from_numpy((x * 2.0 ** -149).astype(np.float32)).to(DEV), None, 32, len(x), 1e-6, q8=q8)
    assert np.array_equal(blocks(q8, len(x), 32)[2][:, 0], np.sign(x) * ((np.abs(x) + 1) // 2))
