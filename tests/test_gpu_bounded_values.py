"""Values at the ends of their types, and weights far below the largest, in the attention of a cache of fixed size."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from tests.bounded_model import HALF, TINY
from tests.test_gpu_bounded import DT, Setup, f64, within

pytestmark = pytest.mark.gpu

INF = float("inf")


def take_caches(s):
    s.model.k, s.model.v = s.caches()


def attend_with_infinities(s, Hq, q=None):
    """Against the model: finite where it is (other elements of the same keys among them), and the same infinities and NaN."""
    c, m = s.cache, s.model
    take_caches(s)
    q = s.randn(m.rows, Hq, m.D, std=1.5) if q is None else q
    out = f64(c.attend(q.cuda()))
    with np.errstate(invalid="ignore"):
        want, tol, wt = m.attend(f64(q), m.D ** -0.5, s.dtype, None, s.there)
    finite = np.isfinite(want)
    within(np.where(finite, out, 0), np.where(finite, want, 0), np.where(finite, tol, 0))
    assert np.array_equal(out[~finite], want[~finite], equal_nan=True)
    s.check_meta(wt)
    return want


@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("D", [16, 64, 128, 256])
@pytest.mark.parametrize("n,paged", [(1, False), (40, True), (513, False), (1500, True)])
def test_infinite_values(n, paged, D, dtype):
    """+inf, -inf and both in one element, NaN in another; every other element of these keys counts as ever."""
    s = Setup(n + D, 2, 2, D, n + 20, [n, max(1, n // 2)], dtype, paged)
    v = s.cache.values
    block, at = (lambda r, i: (int(s.cache.block_table[r, i // 16]), i % 16)) if paged else (lambda r, i: (r, i)), n // 3
    b, i = block(0, at)
    v[b, 0, i, 3], v[b, 0, i, 5], v[b, 1, i, 2] = INF, -INF, float("nan")
    b, i = block(0, n - 1)
    v[b, 0, i, 7], v[b, 0, i, 3] = INF, INF
    b, i = block(0, 0)
    v[b, 0, i, 7] = -INF
    want = attend_with_infinities(s, 6)
    assert (want[0, :3, 3] == INF).all() and np.isnan(want[0, 3:, 2]).all() and np.isfinite(want[1]).all()
    if n > 1:
        assert (want[0, :3, 5] == -INF).all() and np.isnan(want[0, :3, 7]).all()


@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("first", [True, False])
@pytest.mark.parametrize("n", [20, 60, 1200])
def test_infinite_values_of_keys_that_weigh_little(n, first, dtype):
    """40 nats below the largest score, in front of it and behind it: an infinite value is infinite at any weight."""
    D = 64
    s = Setup(n, 1, 1, D, n, [n], dtype)
    top, low = (n - 2, 1) if first else (1, n - 2)
    k = torch.zeros(n, D)
    k[:, 0], k[top, 0], k[low, 0] = torch.rand(n, generator=s.g), 20.0, -20.0
    s.cache.keys[0, 0] = k.to(DT[dtype]).cuda()
    s.cache.values[0, 0, low, 1] = -INF
    q = torch.zeros(1, 2, D, dtype=DT[dtype])
    q[..., 0] = 8.0
    assert (attend_with_infinities(s, 2, q)[0, :, 1] == -INF).all()


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("n,top,low", [(20, 18, 1), (20, 1, 18), (60, 58, 1), (500, 3, 490), (1200, 1198, 1), (1200, 1, 1198), (1200, 300, 310)])
def test_infinite_values_of_keys_whose_weight_32_bits_do_not_hold(n, top, low, dtype):
    """200 nats below the largest score, in the same tile, wave and slice and in others."""
    D = 64
    s = Setup(n, 1, 1, D, n, [n], dtype)
    k = torch.zeros(n, D)
    k[:, 0], k[top, 0], k[low, 0] = torch.rand(n, generator=s.g), 100.0, -100.0
    s.cache.keys[0, 0] = k.to(DT[dtype]).cuda()
    s.cache.values[0, 0, low, 1], s.cache.values[0, 0, low, 2] = -INF, INF
    q = torch.zeros(1, 2, D, dtype=DT[dtype])
    q[..., 0] = 8.0
    want = attend_with_infinities(s, 2, q)
    assert (want[0, :, 1] == -INF).all() and (want[0, :, 2] == INF).all()


# ---- float16: weights far below the largest

def exact(q, k, v):
    s = k @ q / len(q) ** 0.5
    p = np.exp(s - s.max())
    p /= p.sum()
    return p, p @ v


def tolerance(q, k, v, p, o):
    """What 32 bits leave in scores and sums (as the model has it: D products and sums, the exponent to base 2 twice; a sum of at most 256 terms in a row: 24 keys' worth of a wave's three tiles in a lane and
    96 in a matrix instruction's, twice for the two terms, then 4 waves and up to 64 slices); P as two float16 numbers, half a step of half a step of each
    or half of float16's smallest number, of which the largest weight of the 32 keys of a tile is at least 2^26; the output's own rounding."""
    n, u = len(p), 2.0 ** -24
    off = (len(q) + 4) * u * float((np.abs(k) @ np.abs(q)).max()) / len(q) ** 0.5 + 4 * u * (1 + float(np.abs(k @ q).max()) / len(q) ** 0.5)
    tile = np.repeat(np.maximum.reduceat(p, np.arange(0, n, 32)), 32)[:n]
    t = (2 * off + (2 * min(n, 256) + 16) * u + 2 * HALF["float16"] ** 2) * (p @ np.abs(v)) + 2.0 ** -27 * (tile @ np.abs(v))
    return t + (np.abs(o) + t) * HALF["float16"] + TINY["float16"]


@pytest.mark.parametrize("gap", [8.0, 13.0, 16.0, 18.0])
@pytest.mark.parametrize("n,at", [(50, 0), (500, 0), (2000, 1999), (20000, 0), (20000, 11111)])
def test_weights_far_below_the_largest(n, at, gap):
    """One key takes nearly all of the weight and its value is nothing: the output is what the others hold, each of them `gap` nats below."""
    D, Hq = 64, 4
    s = Setup(n + at, 1, 1, D, n, [n], "float16")
    k = torch.randn((n, D), generator=s.g) * 0.02
    k[:, 0], k[at, 0] = 0, gap
    v = 1 + torch.rand((n, D), generator=s.g)
    v[at] = 0
    s.cache.keys[0, 0], s.cache.values[0, 0] = k.half().cuda(), v.half().cuda()
    q = s.randn(1, Hq, D)
    q[..., 0] = 8.0                                       # 8 gap / sqrt(64)
    out = f64(s.cache.attend(q.cuda()))[0]
    kk, vv = f64(s.cache.keys)[0, 0], f64(s.cache.values)[0, 0]
    for h in range(Hq):
        p, o = exact(f64(q)[0, h], kk, vv)
        within(out[h], o, tolerance(f64(q)[0, h], kk, vv, p, o))


@pytest.mark.parametrize("n", [300, 5000])
def test_widely_spread_scores(n):
    """Scores over 30 nats, values that grow as their weights fall, to float16's largest."""
    D, Hq = 64, 5
    s = Setup(n, 2, 1, D, n, [n, n - 1], "float16")
    k = torch.zeros((2, n, D))
    k[..., 0] = -30 * torch.rand((2, n), generator=s.g)
    v = torch.randn((2, n, D), generator=s.g) * torch.exp(-k[..., :1]).clamp_max(20000.0)
    s.cache.keys[:, 0], s.cache.values[:, 0] = k.half().cuda(), v.clamp(-65504, 65504).half().cuda()
    q = torch.zeros(2, Hq, D, dtype=torch.float16)
    q[..., 0] = 8.0
    out = f64(s.cache.attend(q.cuda()))
    for r in range(2):
        kk, vv = f64(s.cache.keys)[r, 0, :n - r], f64(s.cache.values)[r, 0, :n - r]
        for h in range(Hq):
            p, o = exact(f64(q)[r, h], kk, vv)
            within(out[r, h], o, tolerance(f64(q)[r, h], kk, vv, p, o))


# ---- nothing to see

@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("n", [40, 1500])
def test_scores_of_minus_infinity_alone(n, dtype):
    """Nothing to see: zeros, whatever the values hold."""
    s = Setup(n, 2, 1, 64, n, [n, n], dtype)
    c = s.cache
    c.keys[0] = -INF
    c.values[0] = INF
    before = c.weights.clone()
    q = torch.rand((2, 4, 64), generator=s.g).add_(0.5).to(DT[dtype]).cuda()
    out = c.attend(q)
    assert (out[0] == 0).all() and torch.equal(c.weights[0], before[0])
    assert torch.isfinite(out[1]).all() and not torch.equal(c.weights[1], before[1])


# ---- values near the largest of their type

@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("n", [40, 700])
def test_values_of_the_types_size(n, dtype):
    """An average of numbers near the type's largest is no larger than they are, in whatever order the scores rise."""
    D = 64
    s = Setup(n, 2, 1, D, n, [n, n], dtype)
    c = s.cache
    k = torch.zeros((2, n, D))
    k[0, :, 0], k[1, :, 0] = torch.linspace(-4, 4, n), 0.5
    c.keys[:, 0] = k.to(DT[dtype]).cuda()
    big = torch.finfo(DT[dtype]).max * 0.9
    sign = torch.where(torch.rand((2, 1, n, D), generator=s.g) < 0.7, 1.0, -1.0)
    sign[..., 0] = 1
    c.values.copy_((sign.double() * big).to(DT[dtype]))
    q = torch.zeros(2, 4, D, dtype=DT[dtype])
    q[..., 0] = 8.0
    want = attend_with_infinities(s, 4, q)
    assert np.isfinite(want).all()


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("n", [40, 700])
def test_values_that_are_next_to_nothing(n, dtype):
    """2^-98 and less of it: their sums keep their bits."""
    s = Setup(n, 2, 1, 64, n, [n, n], dtype)
    s.cache.values.copy_((torch.randn((2, 1, n, 64), generator=s.g).double() * 2.0 ** -98).to(DT[dtype]))
    attend_with_infinities(s, 4)
