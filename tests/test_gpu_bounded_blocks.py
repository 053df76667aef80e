"""Evictions from a cache of fixed size of which some blocks are not there: what stays is a key that was there, with its own position and weight."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from tests.bounded_model import HALF, Model
from tests.test_gpu_bounded import Setup, angles, attend_once, f64, weigh_once, within

pytestmark = pytest.mark.gpu


def lose(s, places):
    """Table entries (row, block) that name no block from now on."""
    t = s.cache.block_table
    for i, (r, b) in enumerate(places):
        t[r, b] = [-1, s.cache.keys.shape[0], 2 ** 31 - 1, -2 ** 31][i % 4]
        s.there[r, b * s.block:(b + 1) * s.block] = False


def check(s, budget, first, last):
    """By the rule alone, without the model: of the keys that are there the best stay, as many as there are slots in front of the budget that are; every slot holds what belongs to the position it names."""
    c, there = s.cache, s.there
    (k0, v0), pos0, w0, len0 = s.caches(), c.positions.cpu().numpy(), f64(c.weights), c.lengths.cpu().numpy()
    nxt = c.next_positions.cpu().numpy()
    c.evict(budget, keep_first=first, keep_last=last)
    (k1, v1), pos1, w1, len1 = s.caches(), c.positions.cpu().numpy(), f64(c.weights), c.lengths.cpu().numpy()
    assert np.array_equal(len1, np.minimum(len0, budget)) and np.array_equal(nxt, c.next_positions.cpu().numpy())
    for r in range(s.model.rows):
        n, m = len0[r], len1[r]
        held, left = np.flatnonzero(there[r, :n]), np.flatnonzero(there[r, :m])
        for h in range(s.model.heads):
            def rank(i):
                apart = pos0[r, h, i] < first or pos0[r, h, i] >= nxt[r] - last
                return (not apart, np.inf if np.isnan(w0[r, h, i]) else -w0[r, h, i], i)
            best = sorted(held.tolist(), key=rank)[:len(left)] if n > budget else held.tolist()
            slot_of = {int(pos0[r, h, i]): i for i in held}
            came = [slot_of[int(p)] for p in pos1[r, h, left]]
            assert sorted(came) == sorted(best)
            assert np.array_equal(w1[r, h, left], w0[r, h, came], equal_nan=True)
            assert np.array_equal(k1[r, h, left], k0[r, h, came]) and np.array_equal(v1[r, h, left], v0[r, h, came])
            gone = np.flatnonzero(~there[r])
            assert np.array_equal(pos1[r, h, gone], pos0[r, h, gone]) and np.array_equal(w1[r, h, gone], w0[r, h, gone], equal_nan=True)
    s.model.k, s.model.v = k1, v1
    s.model.pos[:], s.model.w[:], s.model.len[:] = pos1, w1, len1


@pytest.mark.parametrize("cap,lens,budget,first,last,lost", [
    (32, [32], 16, 0, 4, [(0, 1)]),                                                    # the newest keys, kept by their positions, are not there
    (32, [32], 16, 0, 4, [(0, 0)]),                                                    # no slot in front of the budget is there
    (32, [32, 31], 16, 0, 4, [(0, 0), (0, 1), (1, 1)]),                                # nothing is there
    (200, [200, 150, 190], 100, 4, 8, [(0, 1), (1, 6), (2, 11), (0, 3), (1, 8), (2, 0)]),
    (200, [200, 150, 190], 100, 120, 8, [(0, 1), (1, 6), (2, 11), (0, 3), (1, 8), (2, 0)]),        # more protected keys than slots
    (200, [200, 199, 101], 99, 95, 0, [(0, 0), (0, 1), (1, 12), (2, 6)]),              # protected keys and lost slots pass the budget together
    (70, [70, 67, 66], 66, 2, 3, [(0, 4), (1, 4), (2, 4), (0, 0)]),                    # few leave; the budget lies inside a lost block
    (70, [70, 68, 69], 66, 0, 0, [(1, 0), (2, 3)]),
    (50, [50, 50], 48, 0, 1, [(0, 3), (1, 1)]),                                        # exactly the lost ones leave
    (3000, [3000, 2500], 1000, 4, 32, [(0, 3), (0, 100), (1, 62), (1, 63), (0, 187)]),
    (38000, [38000, 37000], 20000, 4, 32, [(0, 0), (0, 2000), (1, 1250), (1, 1249)])])             # ranks in the workspace
def test_evict_with_lost_blocks(cap, lens, budget, first, last, lost):
    s = Setup(cap + budget, len(lens), 2, 32, cap, lens, "bfloat16", True, spoil=False)
    lose(s, lost)
    check(s, budget, first, last)
    assert s.cache._tickets.tolist() == [0] * len(lens)


@pytest.mark.parametrize("kind", ["equal", "ties", "special"])
@pytest.mark.parametrize("n,budget", [(70, 67), (300, 120)])
def test_evict_with_lost_blocks_and_odd_weights(kind, n, budget):
    s = Setup(n, 2, 2, 16, n, [n, n - 1], "float32", True, spoil=False)
    shape = s.model.w.shape
    w = {"equal": lambda: torch.full(shape, 0.25), "ties": lambda: torch.randint(0, 3, shape, generator=s.g).float(),
         "special": lambda: torch.tensor([float("nan"), float("inf"), -float("inf"), 0.0, 1.0, 1e-45])[torch.randint(0, 6, shape, generator=s.g)]}[kind]()
    s.cache.weights.copy_(w)
    lose(s, [(0, 1), (1, n // 16)])
    check(s, budget, 2, 3)


@pytest.mark.parametrize("budget", [24, 40])
def test_tokens_beyond_the_blocks_of_a_row(budget):
    """A row runs past the blocks that it was given: those tokens are nowhere, and no key that left comes back in their place."""
    D, Hq, Hkv = 64, 4, 2
    s = Setup(5, 2, Hkv, D, 64, [30, 45], "bfloat16", True, spoil=False)
    lose(s, [(0, 2), (0, 3)])
    c, m = s.cache, s.model
    m.pos[:] = np.arange(64)
    c.positions.copy_(torch.arange(64))
    cos, sin = angles(200, D)
    for step in range(6):
        qkv = s.randn(2, 3, (Hq + 2 * Hkv) * D)
        q = c.append(qkv.cuda(), Hq, cos.cuda(), sin.cuda())
        want, dq, _ = m.append(f64(qkv), Hq, cos.numpy(), sin.numpy())
        within(f64(q), want, dq + (np.abs(want) + dq) * HALF["bfloat16"])
        s.check_meta()
        m.k, m.v = s.caches()
        attend_once(s, Hq)
        m.w[:] = f64(c.weights)
        check(s, budget, 1, 4)
    attend_once(s, Hq)
    m.w[:] = f64(c.weights)
    weigh_once(s, 4, Hq)


def test_the_models_eviction_follows_the_rule():
    """The oracle of the other tests on the same ground."""
    s = Setup(9, 3, 2, 16, 130, [130, 100, 77], "float32", True, spoil=False)
    lose(s, [(0, 0), (0, 7), (1, 3), (1, 6), (2, 4)])
    m = Model(*s.caches(), s.model.len, s.model.next, s.model.pos, s.model.w)
    m.evict(60, 3, 5, s.there)
    check(s, 60, 3, 5)
    assert np.array_equal(m.pos, s.model.pos) and np.array_equal(m.w, s.model.w) and np.array_equal(m.len, s.model.len)
    for x, y in ((m.k, s.model.k), (m.v, s.model.v)):
        assert np.array_equal(x[:, :, :60], y[:, :, :60])
