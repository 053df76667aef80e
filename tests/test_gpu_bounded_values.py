"""Values at the ends of their types in the attention of a cache of fixed size."""
from __future__ import annotations

import numpy as np
import pytest
import torch

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
