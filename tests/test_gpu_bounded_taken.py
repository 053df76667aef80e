"""Rows of a cache of fixed size that do not take all of their tokens: what follows an append asks for those that were taken alone."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from tests.bounded_model import HALF
from tests.test_gpu_bounded import Setup, angles, attend_once, f64, within

pytestmark = pytest.mark.gpu

D, HQ, HKV = 64, 4, 2
POSITIONS = 90


def cut_short(L, counts=None, paged=False):
    """Rows with slots for all of L, for some, for none; at the end of the angle tables; at no position.  -> setup, queries, tokens taken"""
    s = Setup(L, 6, HKV, D, 80, [3, 80 - max(1, L // 2), 80, 20, 20, 80 - L], "float32", paged)
    nxt = [3, 60, 85, POSITIONS - max(1, L // 3), -1, 0]
    s.cache.next_positions.copy_(torch.tensor(nxt, dtype=torch.int32))
    s.model.next[:] = nxt
    cos, sin = angles(POSITIONS, D)
    qkv = s.randn(6, L, (HQ + 2 * HKV) * D)
    asked = None if counts is None else torch.tensor(counts, dtype=torch.int32)
    before = s.model.len.copy()
    q = s.cache.append(qkv.cuda(), HQ, cos.cuda(), sin.cuda(), counts=None if asked is None else asked.cuda())
    want, dq, _ = s.model.append(f64(qkv), HQ, cos.numpy(), sin.numpy(), counts)
    taken = s.model.len - before
    within(f64(q), want, dq + (np.abs(want) + dq) * HALF["float32"])
    s.check_meta()
    assert s.cache.taken.tolist() == taken.tolist()
    s.model.k, s.model.v = s.caches()
    return s, q, taken


@pytest.mark.parametrize("paged", [False, True])
@pytest.mark.parametrize("L", [1, 2, 9, 40])
def test_prompt_weights_of_the_tokens_that_were_taken(L, paged):
    s, q, taken = cut_short(L, paged=paged)
    assert 0 in taken.tolist() and (L < 3 or any(0 < t < L for t in taken.tolist())) and L in taken.tolist()
    before = s.model.w.copy()
    s.cache.weigh(q, counts=s.cache.taken)
    s.check_meta(s.model.weigh(f64(q), D ** -0.5, taken))
    # every taken token gives each KV head's keys its query heads' weight, one each, and the others give nothing
    added = (f64(s.cache.weights) - before).sum(2)
    assert np.allclose(added, taken[:, None] * (HQ // HKV), rtol=1e-5, atol=1e-5)
    s.model.w[:] = f64(s.cache.weights)
    s.cache.weigh(q, counts=s.cache.taken, last=2)
    s.check_meta(s.model.weigh(f64(q), D ** -0.5, taken, last=2))


def test_a_step_of_full_rows_asks_for_nothing():
    s, q, taken = cut_short(1)
    attend_once(s, HQ, counts=taken)
    before = s.cache.weights.clone()
    out = s.cache.attend(q[:, 0].contiguous(), counts=s.cache.taken)
    for r in np.flatnonzero(taken == 0):
        assert (out[r] == 0).all() and torch.equal(s.cache.weights[r], before[r])
    assert (out[0] != 0).any() and not torch.equal(s.cache.weights[0], before[0])


@pytest.mark.parametrize("L", [1, 5, 40])
def test_counts_that_were_asked_for(L):
    _, _, taken = cut_short(L, [L, 1, 3, 0, 7, -2])
    assert taken[0] == L and taken[3] == 0 and taken[5] == 0


@pytest.mark.parametrize("L", [3, 60])
def test_taken_may_be_the_counts(L):
    """Both forms of the append, and a captured one: what one append took is what the next is asked to take."""
    cos, sin = (t.cuda() for t in angles(400, D))
    s = Setup(L, 3, HKV, D, 250, [0, 249, 120], "bfloat16", skip=0)
    c = s.cache
    x = s.randn(3, L, (HQ + 2 * HKV) * D).cuda()
    c.append(x, HQ, cos, sin, counts=torch.tensor([L, L, L - 1], dtype=torch.int32, device="cuda"))
    assert c.taken.tolist() == [L, 1, L - 1]
    c.append(x, HQ, cos, sin, counts=c.taken)
    assert c.taken.tolist() == [L, 0, L - 1] and c.lengths.tolist() == [2 * L, 250, 120 + 2 * (L - 1)]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q = c.append(x, HQ, cos, sin, counts=c.taken)
        c.weigh(q, counts=c.taken)
    lengths = np.array([2 * L, 250, 120 + 2 * (L - 1)])
    for _ in range(4):
        graph.replay()
        took = np.minimum([L, 0, L - 1], 250 - lengths)
        took = np.minimum(took, c.taken.cpu().numpy())
        lengths = lengths + took
        assert c.taken.tolist() == took.tolist() and c.lengths.tolist() == lengths.tolist()
