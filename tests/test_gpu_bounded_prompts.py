"""Long prompts in a cache of fixed size: the weights of all of their queries or of the last ones alone, in many units, slices and joins; 16-bit appends of whole prompts."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from tests.bounded_model import HALF, TINY, U
from tests.test_gpu_bounded import DT, Setup, angles, copies, f64, within

pytestmark = pytest.mark.gpu


def weigh_64(s, q, counts, last):
    """The model's weigh, a matrix per row and head at a time: adds to its weights, returns the tolerance (the same bound for every query)."""
    m, q, scale = s.model, f64(q), s.model.D ** -0.5
    G, tol = q.shape[2] // m.heads, np.zeros_like(m.w)
    for r in range(m.rows):
        n, c = m.held(r), min(max(int(counts[r]), 0), q.shape[1])
        i = np.arange(max(0, c - last) if last else 0, c)
        for h in range(m.heads):
            k = np.where(s.there[r, :n, None], m.k[r, h, :n], 0)
            for x in q[r, i][:, h * G:(h + 1) * G].transpose(1, 0, 2):
                sees = (np.arange(n) <= (n - c + i)[:, None]) & s.there[r, :n]
                a = np.where(sees, scale * (x @ k.T), -np.inf)
                some = sees.any(1)
                top = np.where(some, a.max(1, initial=-np.inf), 0)
                e = np.where(sees, np.exp(a - top[:, None]), 0)
                p = e / np.where(some, e.sum(1), 1)[:, None]
                size = np.where(sees, scale * (np.abs(x) @ np.abs(k).T), 0).max(1, initial=0)
                off = (m.D + 4) * U * size + 4 * U * (1 + np.abs(np.where(sees, a, 0)).max(1, initial=0))
                m.w[r, h, :n] += p.sum(0)
                tol[r, h, :n] += ((2 * off + (sees.sum(1) + 16) * U)[:, None] * p).sum(0)
    return tol + (q.shape[1] * G + 8) * U * np.abs(m.w)


def check(s, L, Hq, counts, last):
    q = s.randn(s.model.rows, L, Hq, s.model.D, std=1.5)
    before = f64(s.cache.weights)
    s.cache.weigh(q.cuda(), counts=torch.tensor(counts, dtype=torch.int32, device="cuda"), last=last)
    s.check_meta(weigh_64(s, q, counts, last))
    untouched = np.broadcast_to(~((np.arange(s.model.cap) < s.model.len[:, None]) & s.there)[:, None], s.model.w.shape)
    assert np.array_equal(f64(s.cache.weights)[untouched], before[untouched])


# several slices of the keys in the first pass and of the queries in the second, but where said otherwise
@pytest.mark.parametrize("dtype,rows,heads,G,D,cap,L,last,paged", [
    ("bfloat16", 2, 2, 4, 32, 900, 300, 100, True),                  # one slice of the queries
    ("bfloat16", 1, 2, 6, 64, 1500, 700, 200, False),
    ("float32", 2, 1, 4, 16, 1200, 1200, 333, True),
    ("float16", 2, 2, 40, 32, 600, 70, 64, False),
    ("float16", 3, 2, 5, 256, 700, 300, 130, True),
    ("float32", 2, 2, 4, 128, 900, 300, 100, False),
    ("bfloat16", 8, 4, 6, 32, 1000, 400, 150, True)])                # 128 keys a workgroup
def test_the_last_queries_of_a_long_prompt(dtype, rows, heads, G, D, cap, L, last, paged):
    lens = [cap - 97 * r for r in range(rows)]
    counts = [L - (61 * r) % L for r in range(rows)]
    check(Setup(cap + L, rows, heads, D, cap, lens, dtype, paged, bad=2 if paged else 0), L, heads * G, counts, last)


# 128 keys a workgroup of the second pass (rows x heads x cap / 128 fill the chip): one slice of the queries or several, one tile of them a head or more
@pytest.mark.parametrize("dtype,rows,heads,G,D,cap,L,paged", [
    ("bfloat16", 32, 4, 2, 16, 250, 200, True), ("float16", 32, 4, 2, 64, 250, 70, False), ("bfloat16", 16, 4, 3, 192, 500, 150, True), ("float16", 8, 4, 6, 16, 1000, 150, False),
    ("float16", 16, 4, 3, 96, 500, 130, True), ("bfloat16", 32, 8, 2, 128, 130, 130, False), ("bfloat16", 16, 4, 1, 256, 400, 100, True)])
def test_prompts_that_fill_the_chip(dtype, rows, heads, G, D, cap, L, paged):
    lens = [max(0, cap - 13 * r) for r in range(rows)]
    counts = [max(0, min(L, n) - 7 * r) for r, n in enumerate(lens)]
    check(Setup(cap + D, rows, heads, D, cap, lens, dtype, paged, bad=5 if paged else 0), L, heads * G, counts, 0)


def test_the_last_queries_do_not_depend_on_the_others():
    """The same last queries behind others, and alone: the same bits where the cut is the same."""
    s = Setup(3, 2, 2, 64, 1500, [1500, 1200], "bfloat16", True)
    q = s.randn(2, 900, 8, 64).cuda()
    a, b = copies(s), copies(s)
    a.weigh(q, last=150)
    b.weigh(q[:, -150:])
    assert torch.equal(a.weights, b.weights) and not torch.equal(a.weights, s.cache.weights)


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("paged", [False, True])
def test_a_16_bit_prompt_with_norms(dtype, paged):
    D, Hq, Hkv, L = 128, 5, 1, 700
    s = Setup(8, 2, Hkv, D, 800, [11, 90], dtype, paged, skip=3)
    cos, sin = angles(900, D)
    qn, kn = ((1 + 0.1 * torch.randn(D, generator=s.g)).to(DT[dtype]) for _ in range(2))
    qkv = s.randn(2, L, (Hq + 2 * Hkv) * D, std=2.0)
    counts = torch.tensor([L, L - 33], dtype=torch.int32)
    q = s.cache.append(qkv.cuda(), Hq, cos.cuda(), sin.cuda(), counts=counts.cuda(), q_norm=qn.cuda(), k_norm=kn.cuda())
    want, dq, dk = s.model.append(f64(qkv), Hq, cos.numpy(), sin.numpy(), counts.numpy(), q_norm=f64(qn), k_norm=f64(kn))
    within(f64(q), want, dq + (np.abs(want) + dq) * HALF[dtype] + TINY[dtype])
    s.check_meta()
    k, v = s.caches()
    new = dk > 0
    within(np.where(new, k, 0), np.where(new, s.model.k, 0), dk + (np.abs(np.where(new, s.model.k, 0)) + dk) * HALF[dtype] + TINY[dtype])
    assert np.array_equal(np.where(new, 0, k), np.where(new, 0, s.model.k), equal_nan=True) and np.array_equal(v, s.model.v, equal_nan=True)
