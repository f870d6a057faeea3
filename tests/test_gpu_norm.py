"""ft_hip_add_rmsnorm against its definition in 64 bits (numpy).

h is rounded once from f64 (with no branch norm it is one f32 addition, the
same bits); y and the scales d are checked from the kernel's own h, so their
only error is one rounding: half a step of f32, 2^-24 of the value, plus the
f64 arithmetic's few 2^-53 (1e-14 below covers them, of the largest term).
The quants are those of u = f32(h * w), 127 u / a rounded half away: 127 |u| is
exact in f64 and the f64 quotient is right at halves, so they must be equal.
"""
import numpy as np
import pytest
import torch

import ft_hip

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
EPS = 1e-6
HALF = 2.0 ** -24 * (1 + 1e-6)
SUB = 2.0 ** -150
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).to(DEV)


def host(t):
    torch.cuda.synchronize()
    return t.cpu().numpy()


def blocks(q8, n, hidden):
    raw = host(q8).reshape(n, hidden // 32, 40)
    return (raw[:, :, :4].copy().view(np.float32)[:, :, 0], raw[:, :, 4:8].copy().view(np.int32)[:, :, 0],
            raw[:, :, 8:].copy().view(np.int8))


def check_h(h, x, residual, x_w, eps=EPS):
    """x as f64 values; the kernel's h against the definition."""
    if x_w is None:
        want = x.astype(np.float32) if residual is None else residual + x.astype(np.float32)
        assert np.array_equal(h, want)
        return
    b = x / np.sqrt((x * x).mean(1, keepdims=True) + eps) * x_w.astype(np.float64)
    r = 0.0 if residual is None else residual.astype(np.float64)
    assert np.all(np.abs(h - (r + b)) <= HALF * np.abs(r + b) + 1e-14 * (np.abs(r) + np.abs(b)) + SUB)


def check_y(y, h, w, eps=EPS):
    h = h.astype(np.float64)
    want = h / np.sqrt((h * h).mean(1, keepdims=True) + eps) * (1.0 if w is None else w.astype(np.float64))
    assert np.all(np.abs(y - want) <= (HALF + 1e-14) * np.abs(want) + SUB)


def check_q8(q8, h, w, eps=EPS):
    n, hidden = h.shape
    d, qsum, qs = blocks(q8, n, hidden)
    u = (h if w is None else h * w).astype(np.float64).reshape(n, -1, 32)
    a = np.abs(u).max(2, keepdims=True)
    q = np.floor(np.divide(127.0 * np.abs(u), a, out=np.zeros_like(u), where=a > 0) + 0.5) * np.sign(u)
    assert np.array_equal(qs, q.astype(np.int8))
    assert np.array_equal(qsum, q.sum(2).astype(np.int32))
    h = h.astype(np.float64)
    want = a[:, :, 0] / 127.0 / np.sqrt((h * h).mean(1, keepdims=True) + eps)
    assert np.all(np.abs(d - want) <= (HALF + 1e-14) * want + SUB)


def run(gemv, x, residual, w, x_w, n, hidden, outs="hyq", eps=EPS, stream=None):
    h = torch.full((n, hidden), 7.0, device=DEV) if "h" in outs else None
    y = torch.full((n, hidden), 7.0, device=DEV) if "y" in outs else None
    q8 = torch.full((n * (hidden // 32) * 40,), 7, dtype=torch.uint8, device=DEV) if "q" in outs else None
    gemv.add_rmsnorm(x, w, hidden, n, eps, residual=residual, h=h, y=y, q8=q8, x_w=x_w, stream=stream)
    return h, y, q8


def inputs(n, hidden, seed, type="f32"):
    rng = np.random.default_rng(seed)
    x = torch.from_numpy(rng.standard_normal((n, hidden)).astype(np.float32)).to(TYPES[type])
    r = (3 * rng.standard_normal((n, hidden))).astype(np.float32)
    w = (1 + 0.3 * rng.standard_normal(hidden)).astype(np.float32)
    x_w = (0.5 + 0.2 * rng.standard_normal(hidden)).astype(np.float32)
    return x, r, w, x_w


@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("sandwich", [False, True])
@pytest.mark.parametrize("n,hidden", [(1, 32), (3, 64), (2, 2816), (65, 2816), (5, 4096), (2, 8224), (3, 16384),
                                      (2500, 288), (9000, 32)])
def test_against_the_definition(gemv, type, sandwich, n, hidden):
    x, r, w, x_w = inputs(n, hidden, 11 * hidden + n, type)
    xw = x_w if sandwich else None
    h, y, q8 = run(gemv, x.to(DEV), dev(r), dev(w), None if xw is None else dev(xw), n, hidden)
    hh = host(h)
    check_h(hh, x.double().numpy(), r, xw)
    check_y(host(y), hh, w)
    check_q8(q8, hh, w)


@pytest.mark.parametrize("hidden", [1, 2, 3, 5, 63, 64, 65, 100, 1027, 2815, 16383])
@pytest.mark.parametrize("sandwich", [False, True])
def test_odd_rows_without_blocks(gemv, hidden, sandwich):
    n = 3
    x, r, w, x_w = inputs(n, hidden, hidden)
    xw = x_w if sandwich else None
    h, y, _ = run(gemv, x.to(DEV), dev(r), dev(w), None if xw is None else dev(xw), n, hidden, "hy")
    hh = host(h)
    check_h(hh, x.double().numpy(), r, xw)
    check_y(host(y), hh, w)


@pytest.mark.parametrize("outs", ["h", "y", "q", "hq", "yq", "hy"])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("weight", [False, True])
def test_optional_arguments(gemv, outs, residual, weight):
    n, hidden = 4, 704
    x, r, w, _ = inputs(n, hidden, 5)
    w = w if weight else None
    h, y, q8 = run(gemv, x.to(DEV), dev(r) if residual else None, None if w is None else dev(w), None, n, hidden, outs)
    hh = x.numpy() + r if residual else x.numpy()
    if h is not None:
        assert np.array_equal(host(h), hh)
    if y is not None:
        check_y(host(y), hh, w)
    if q8 is not None:
        check_q8(q8, hh, w)


@pytest.mark.parametrize("off,pad", [(0, 8), (1, 0), (0, 3), (2, 5)])
@pytest.mark.parametrize("type", ["f32", "bf16"])
def test_strides_and_offsets(gemv, off, pad, type):
    """Rows inside wider tensors, aligned or not; the values between the rows stay as they were."""
    n, hidden = 5, 320
    x, r, w, x_w = inputs(n, hidden, 77, type)

    def wide(a, dtype):
        t = torch.full((n * (hidden + pad) + off,), 9.0, dtype=dtype, device=DEV)
        v = t[off:].view(n, hidden + pad)[:, :hidden]
        if a is not None:
            v.copy_(a)
        return t, v

    _, xv = wide(x, TYPES[type])
    _, rv = wide(torch.from_numpy(r), torch.float32)
    ht, hv = wide(None, torch.float32)
    yt, yv = wide(None, torch.float32)
    q8 = torch.zeros(n * (hidden // 32) * 40 + 4, dtype=torch.uint8, device=DEV)[4:]
    gemv.add_rmsnorm(xv, dev(w), hidden, n, EPS, residual=rv, h=hv, y=yv, q8=q8, x_w=dev(x_w))
    hh = host(hv.contiguous())
    check_h(hh, x.double().numpy(), r, x_w)
    check_y(host(yv.contiguous()), hh, w)
    check_q8(q8.clone(), hh, w)
    for t in (ht, yt):
        flat = host(t)
        assert np.all(flat[:off] == 9.0)
        if pad:
            assert np.all(flat[off:].reshape(n, hidden + pad)[:, hidden:] == 9.0)


def test_rows_behind_the_last_stay(gemv):
    n, hidden = 3, 256
    x, r, w, _ = inputs(n + 2, hidden, 3)
    h = torch.full((n + 2, hidden), 7.0, device=DEV)
    q8 = torch.full(((n + 2) * 8 * 40,), 7, dtype=torch.uint8, device=DEV)
    gemv.add_rmsnorm(x.to(DEV), dev(w), hidden, n, EPS, residual=dev(r), h=h, q8=q8)
    assert np.all(host(h)[n:] == 7.0) and np.all(host(q8)[n * 320:] == 7)
    gemv.add_rmsnorm(x.to(DEV), dev(w), hidden, 0, EPS, h=h)  # no rows: nothing
    assert np.all(host(h)[n:] == 7.0)


@pytest.mark.parametrize("hidden", [320, 2816, 16384])
def test_in_place(gemv, hidden):
    """h over the residual, y over x: as with buffers of their own."""
    n = 6
    x, r, w, x_w = inputs(n, hidden, hidden)
    for xw in (None, dev(x_w)):
        h, y, q8 = run(gemv, x.to(DEV), dev(r), dev(w), xw, n, hidden)
        xi, ri, qi = x.to(DEV), dev(r), torch.zeros_like(q8)
        gemv.add_rmsnorm(xi, dev(w), hidden, n, EPS, residual=ri, h=ri, y=xi, q8=qi, x_w=xw)
        assert torch.equal(ri, h) and torch.equal(xi, y) and torch.equal(qi, q8)


def test_halves_and_zero_blocks(gemv):
    """Values whose quotient is a half exactly, all-zero blocks and rows, subnormals."""
    x = np.zeros((4, 96), np.float32)
    x[0, :32] = 127 * np.linspace(-1, 1, 32)
    x[0, 1:9] = np.array([0.5, -0.5, 1.5, 2.5, -2.5, 63.5, -63.5, 126.5], np.float32)
    x[0, 0] = 127
    x[0, 32:64] = np.array([4.0, 2.0, -2.0, 1.0] * 8)  # 127 / 2 = 63.5
    x[1, 40] = 1e-3
    x[2, :] = np.float32(1e-42)
    w = np.ones(96, np.float32)
    for eps in (EPS, 0.0):
        rows = x if eps else x[:3]
        h, y, q8 = run(gemv, dev(rows), None, None, None, len(rows), 96, eps=eps)
        check_q8(q8, rows, None, eps)
        check_y(host(y), rows, w, eps)
    assert list(blocks(q8, 3, 96)[2][0, 0, 1:9]) == [1, -1, 2, 3, -3, 64, -64, 127]


def test_nonfinite_rows(gemv):
    """NaN and inf stay in their rows; quants are 0 where the block has no maximum to divide by."""
    n, hidden = 3, 64
    x, r, w, _ = inputs(n, hidden, 9)
    x = x.numpy()
    x[0, 5] = np.nan
    x[1, 40] = np.inf
    h, y, q8 = run(gemv, dev(x), None, dev(w), None, n, hidden)
    d, qsum, qs = blocks(q8, n, hidden)
    assert np.all(np.isnan(host(y)[0])) and np.all(np.isnan(d[0])) and qs[0, 0, 5] == 0
    assert np.isnan(host(y)[1, 40]) and np.all(host(y)[1, :40] == 0) and d[1, 0] == 0
    assert np.isnan(d[1, 1]) and not qs[1, 1].any() and qsum[1, 1] == 0
    check_y(host(y)[2:], x[2:], w)
    for i in (0, 1):  # the quants of blocks without NaN or inf do not depend on the row's sum
        b = 1 - i
        u = (x[i, 32 * b:32 * b + 32] * w[32 * b:32 * b + 32]).astype(np.float64)
        assert np.array_equal(qs[i, b], np.floor(127 * np.abs(u) / np.abs(u).max() + 0.5) * np.sign(u))


def test_large_values_do_not_overflow(gemv):
    n, hidden = 2, 128
    x = (np.random.default_rng(1).uniform(-3, 3, (n, hidden)) * 1e38).astype(np.float32)
    h, y, q8 = run(gemv, dev(x), None, None, None, n, hidden)
    check_y(host(y), x, None)
    check_q8(q8, x, None)


def test_blocks_are_those_of_quantize_q8_on_y(gemv):
    """Beside ft_hip_quantize_q8 on y: quants within one (it rounds y, d and 1/d first), scales within
    2^-23 (one rounding here, y's and the quotient's there: 3 * 2^-24, and its reciprocal is not in d)."""
    n, hidden = 7, 2816
    x, r, w, _ = inputs(n, hidden, 21)
    _, y, q8 = run(gemv, x.to(DEV), dev(r), dev(w), None, n, hidden)
    other = torch.zeros_like(q8)
    gemv.quantize_q8(y, hidden, other, hidden, n)
    d, _, qs = blocks(q8, n, hidden)
    d2, _, qs2 = blocks(other, n, hidden)
    assert np.all(np.abs(d - d2) <= 3 * HALF * d)
    assert np.max(np.abs(qs.astype(int) - qs2.astype(int))) <= 1
    assert np.mean(qs != qs2) < 1e-3


def test_same_bits_each_time_on_another_stream_and_captured(gemv):
    n, hidden = 33, 2816
    x, r, w, x_w = inputs(n, hidden, 4)
    xd, rd, wd, xwd = x.to(DEV), dev(r), dev(w), dev(x_w)
    first = run(gemv, xd, rd, wd, xwd, n, hidden)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        again = run(gemv, xd, rd, wd, xwd, n, hidden)
        explicit = run(gemv, xd, rd, wd, xwd, n, hidden, stream=s)
    torch.cuda.synchronize()
    h, y, q8 = (torch.zeros_like(t) for t in first)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        gemv.add_rmsnorm(xd, wd, hidden, n, EPS, residual=rd, h=h, y=y, q8=q8, x_w=xwd)
    for seed in (5, 6, 4):
        x2 = inputs(n, hidden, seed)[0].to(DEV)
        xd.copy_(x2)
        g.replay()
        want = run(gemv, x2, rd, wd, xwd, n, hidden)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip((h, y, q8), want)), seed
    for other in (again, explicit, (h, y, q8)):
        assert all(torch.equal(a, b) for a, b in zip(first, other))


def test_refused_by_the_python_side(gemv):
    x, r, w, _ = inputs(4, 64, 1)
    xd, rd, wd = x.to(DEV), dev(r), dev(w)
    q8 = torch.zeros(4 * 2 * 40, dtype=torch.uint8, device=DEV)
    bad = [dict(x=xd[:3]), dict(x=xd.double()), dict(x=xd.t()), dict(h=rd[:, :32]), dict(y=rd.half()),
           dict(q8=q8[:-1]), dict(w=wd[:63]), dict(x_w=wd[:1]), dict(residual=rd.flatten()[:-1])]
    for change in bad:
        kw = dict(x=xd, w=wd, residual=rd, h=torch.zeros_like(rd), y=None, q8=q8, x_w=None)
        kw.update(change)
        with pytest.raises(ft_hip.FtHipError) as e:
            gemv.add_rmsnorm(kw.pop("x"), kw.pop("w"), 64, 4, EPS, **kw)
        assert e.value.code in (ft_hip.E_SHAPE, ft_hip.E_INVALID), change


def test_outputs_beside_an_input_are_refused(gemv):
    """An output may lie on an input's rows, not across them: another stride or type would mix rows; nor on the other
    output."""
    n, hidden = 4, 64
    x, r, w, _ = inputs(n, hidden, 2)
    xd, rd, wd = x.to(DEV), dev(r), dev(w)
    wide = torch.zeros((n, 96), device=DEV)
    wide[:, :hidden] = rd
    across = wide.flatten()[:n * hidden].view(n, hidden)  # the same start, rows 64 apart
    x16 = torch.zeros((n, 2 * hidden), dtype=torch.float16, device=DEV)
    on_x16 = x16.view(torch.float32)
    before = wide.clone()
    for kw in (dict(residual=wide[:, :hidden], h=across), dict(residual=wide[:, :hidden], y=across),
               dict(x=wide[:, :hidden], h=across), dict(x=wide[:, :hidden], y=across), dict(h=wide, y=wide),
               dict(x=x16, h=on_x16), dict(x=x16, y=on_x16)):
        kw = dict(dict(x=xd, residual=rd), **kw)
        with pytest.raises(ft_hip.FtHipError) as e:
            gemv.add_rmsnorm(kw.pop("x"), wd, hidden, n, EPS, **kw)
        assert e.value.code == ft_hip.E_SHAPE
    torch.cuda.synchronize()
    assert torch.equal(before, wide)
    # a single row has no stride to differ in
    h = torch.empty((1, hidden), device=DEV)
    gemv.add_rmsnorm(xd, wd, hidden, 1, EPS, residual=rd, h=h)
    gemv.add_rmsnorm(xd, wd, hidden, 1, EPS, residual=wide[:, :hidden], h=across)
    assert torch.equal(across[:1], h)


def test_tensors_of_another_device_or_kind_are_refused(gemv):
    x, r, w, _ = inputs(4, 64, 3)
    xd, rd, wd = x.to(DEV), dev(r), dev(w)
    q8 = torch.zeros(4 * 2 * 40, dtype=torch.uint8)
    for change in (dict(x=x), dict(residual=rd.cpu()), dict(h=rd.cpu()), dict(y=rd.cpu()), dict(w=wd.cpu()),
                   dict(x_w=wd.cpu()), dict(q8=q8), dict(x=xd.int()), dict(residual=rd.int()), dict(w=wd.int())):
        kw = dict(dict(x=xd, w=wd, residual=rd, h=torch.zeros_like(rd)), **change)
        with pytest.raises((ft_hip.FtHipError)) as e:
            gemv.add_rmsnorm(kw.pop("x"), kw.pop("w"), 64, 4, EPS, **kw)
        assert e.value.code in (ft_hip.E_SHAPE, ft_hip.E_INVALID), change
