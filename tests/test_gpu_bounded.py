"""The operators of a cache of fixed size (mi_op_bounded_*, mlx_parallm_amd.bounded_cache) against 64-bit NumPy, slot by slot."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from tests.bounded_model import HALF, TINY, Model

pytestmark = pytest.mark.gpu

DT = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
BLOCK = 16


def f64(t):
    return t.detach().to(torch.float64).cpu().numpy()


class Setup:
    """A cache with random contents, and its model.  Paged: blocks of 16 tokens in no order, in an arena with some that belong to nobody; `bad`: how many table entries name no block.
    Slots behind the lengths hold NaN."""

    def __init__(self, seed, rows, heads, D, cap, lens, dtype="bfloat16", paged=False, bad=0, skip=7, block=BLOCK, spoil=True):
        from mlx_parallm_amd.bounded_cache import BoundedKVCache

        g = torch.Generator().manual_seed(seed)
        self.g, self.dtype, self.block = g, dtype, block
        dt = DT[dtype]
        k, v = (torch.randn((rows, heads, cap, D), generator=g).to(dt) for _ in range(2))
        lengths = torch.tensor(lens, dtype=torch.int32)
        if spoil:
            behind = torch.arange(cap) >= lengths[:, None]
            for x in (k, v):
                x.masked_fill_(behind[:, None, :, None], float("nan"))
        pos = torch.stack([torch.stack([torch.randperm(cap, generator=g) for _ in range(heads)]) for _ in range(rows)]).to(torch.int32)
        w = torch.rand((rows, heads, cap), generator=g)
        nxt = lengths + skip
        self.there = np.ones((rows, cap), bool)
        table = None
        if paged:
            per = -(-cap // block)
            n = rows * per + 3
            table = torch.randperm(n, generator=g)[:rows * per].view(rows, per)
            ka, va = (torch.full((n, heads, block, D), float("nan"), dtype=dt) for _ in range(2))
            for r in range(rows):
                for b in range(per):
                    m = min(block, cap - b * block)
                    ka[table[r, b], :, :m], va[table[r, b], :, :m] = k[r, :, b * block:b * block + m], v[r, :, b * block:b * block + m]
            table = table.to(torch.int32)
            for i in range(bad):
                r, b = i % rows, (5 * i + 1) % per
                table[r, b] = [-1, n, 2 ** 31 - 1][i % 3]
                self.there[r, b * block:(b + 1) * block] = False
            self.ka, self.va, self.table = ka, va, table.cuda()
        self.model = Model(f64(k), f64(v), lens, nxt, pos, w)
        kk, vv = (ka, va) if paged else (k, v)
        self.cache = BoundedKVCache(kk.cuda(), vv.cuda(), lengths.cuda(), nxt.cuda(), pos.cuda(), w.cuda(), table.cuda() if paged else None)

    def randn(self, *shape, std=1.0):
        return (torch.randn(shape, generator=self.g) * std).to(DT[self.dtype])

    def caches(self):
        """keys, values [rows, heads, cap, D] as they lie on the device (places without a block: the model's)"""
        out = []
        for dev, ref in ((self.cache.keys, self.model.k), (self.cache.values, self.model.v)):
            x = f64(dev)
            if self.cache.block_table is not None:
                t = self.cache.block_table.cpu().numpy()
                y = np.array(ref)
                for s in range(ref.shape[2]):
                    b = t[:, s // self.block]
                    for r in np.flatnonzero(self.there[:, s]):
                        y[r, :, s] = x[b[r], :, s % self.block]
                x = y
            out.append(x)
        return out

    def check_meta(self, w_tol=None):
        c, m = self.cache, self.model
        assert np.array_equal(c.lengths.cpu().numpy(), m.len) and np.array_equal(c.next_positions.cpu().numpy(), m.next)
        assert np.array_equal(c.positions.cpu().numpy(), m.pos)
        got = f64(c.weights)
        if w_tol is None:
            assert np.array_equal(got, m.w, equal_nan=True)
        else:
            assert np.all(np.abs(got - m.w) <= w_tol), float((np.abs(got - m.w) - w_tol).max())

    def check_same_caches(self):
        for x, y in zip(self.caches(), (self.model.k, self.model.v)):
            assert np.array_equal(x, y, equal_nan=True)


def angles(n, D, base=10000.0):
    a = np.arange(n)[:, None] * base ** (-np.arange(D // 2) / (D // 2))
    return torch.from_numpy(np.cos(a)).float(), torch.from_numpy(np.sin(a)).float()


def within(got, want, tol):
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), (int(bad.sum()), float(np.abs(got - want)[bad].max()))


# ---- append

@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("D,Hq,Hkv,norm,paged", [(16, 4, 4, False, True), (64, 5, 1, True, False), (96, 6, 2, True, True), (128, 10, 2, True, True),
                                                 (192, 3, 1, True, False), (256, 4, 2, True, False), (32, 40, 8, False, False), (128, 130, 2, True, False)])
@pytest.mark.parametrize("L", [1, 5, 37])
def test_append(dtype, D, Hq, Hkv, norm, paged, L):
    s = Setup(11, 4, Hkv, D, 59, [0, 17, 40, 3], dtype, paged)
    cos, sin = angles(59 + 40, D)
    qkv = s.randn(4, L, (Hq + 2 * Hkv) * D, std=2.0)
    counts = torch.tensor([L, max(0, L - 2), L, 0], dtype=torch.int32)
    qn, kn = (1 + s.randn(D, std=0.2).float()).to(DT[dtype]), (1 + s.randn(D, std=0.2).float()).to(DT[dtype])
    kw = dict(q_norm=qn, k_norm=kn) if norm else {}
    q = s.cache.append(qkv.cuda(), Hq, cos.cuda(), sin.cuda(), counts=counts.cuda(), eps=1e-5, **{n: t.cuda() for n, t in kw.items()})
    want, dq, dk = s.model.append(f64(qkv), Hq, cos.numpy(), sin.numpy(), counts.numpy(), eps=1e-5, **{n: f64(t) for n, t in kw.items()})
    within(f64(q), want, dq + (np.abs(want) + dq) * HALF[dtype] + TINY[dtype])
    s.check_meta()
    k, v = s.caches()
    new = dk > 0
    within(np.where(new, k, 0), np.where(new, s.model.k, 0), dk + (np.abs(np.where(new, s.model.k, 0)) + dk) * HALF[dtype] + TINY[dtype])
    assert np.array_equal(np.where(new, 0, k), np.where(new, 0, s.model.k), equal_nan=True) and np.array_equal(v, s.model.v, equal_nan=True)


@pytest.mark.parametrize("L", [1, 3, 100])
def test_append_takes_what_fits(L):
    """Full rows, positions that the tables do not hold, lengths that are none, pages that are none."""
    s = Setup(3, 5, 2, 64, 40, [40, 38, 0, 7, 20], "bfloat16", True, bad=4)
    c, m = s.cache, s.model
    c.next_positions.copy_(torch.tensor([10, 38, -3, 98, 0], dtype=torch.int32))
    m.next[:] = [10, 38, -3, 98, 0]
    c.lengths[0], m.len[0] = 55, 55                       # (counts as 40)
    cos, sin = angles(100, 64)
    qkv = s.randn(5, L, 8 * 64)
    q = c.append(qkv.cuda(), 4, cos.cuda(), sin.cuda())
    want, dq, dk = m.append(f64(qkv), 4, cos.numpy(), sin.numpy())
    within(f64(q), want, dq + (np.abs(want) + dq) * HALF["bfloat16"])
    s.check_meta()
    k, v = s.caches()
    new = (dk > 0) & s.there[:, None, :, None]
    within(np.where(new, k, 0), np.where(new, m.k, 0), dk + (np.abs(np.where(new, m.k, 0)) + dk) * HALF["bfloat16"])
    belongs = np.zeros(s.ka.shape[0], bool)
    belongs[[b for b in c.block_table.cpu().numpy().ravel() if 0 <= b < len(belongs)]] = True
    for x, y in ((c.keys, s.ka), (c.values, s.va)):      # blocks that no table names
        assert np.array_equal(f64(x)[~belongs], f64(y)[~belongs], equal_nan=True)


def test_counts_beyond_the_tokens_and_below_none():
    s = Setup(4, 3, 2, 32, 90, [10, 20, 30], "float32")
    cos, sin = angles(200, 32)
    counts = torch.tensor([7, -3, 2 ** 31 - 1], dtype=torch.int32)
    qkv = s.randn(3, 5, 8 * 32)
    q = s.cache.append(qkv.cuda(), 4, cos.cuda(), sin.cuda(), counts=counts.cuda())
    want, dq, _ = s.model.append(f64(qkv), 4, cos.numpy(), sin.numpy(), counts.numpy())
    within(f64(q), want, dq + (np.abs(want) + dq) * HALF["float32"])
    s.check_meta()
    s.model.k, s.model.v = s.caches()
    weigh_once(s, 5, 4, counts=counts.tolist())
    attend_once(s, 4, counts=counts.tolist())


def test_queries_in_other_strides_and_places():
    s = Setup(6, 2, 2, 64, 100, [100, 60], "bfloat16")
    a, b = copies(s), copies(s)
    wide = s.randn(2, 8, 3, 64).cuda()
    q = wide[:, :, 1]
    assert torch.equal(a.attend(q), b.attend(q.contiguous())) and torch.equal(a.weights, b.weights)
    p = s.randn(4, 2, 30, 64).cuda().permute(1, 2, 0, 3)                # [rows][tokens][heads][D]
    a.weigh(p)
    b.weigh(p.contiguous())
    assert torch.equal(a.weights, b.weights)
    odd = torch.zeros(2 * 8 * 64 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(2, 8, 64)
    with pytest.raises(ValueError, match="16 bytes"):
        a.attend(odd)
    with pytest.raises(ValueError, match="16 bytes"):
        a.append(torch.zeros((2, 1, 8 * 64 + 4), dtype=torch.bfloat16, device="cuda")[:, :, 4:], 4, *(t.cuda() for t in angles(10, 64)))
    assert torch.equal(a.weights, b.weights)


def test_append_strides():
    s = Setup(5, 2, 2, 32, 64, [3, 9], "float16")
    cos, sin = angles(64, 32)
    wide = s.randn(3, 2, 4, 8 * 32 + 16)                  # [token][row][other][qkv and more]
    qkv = wide[:, :, 1, 8:8 + 8 * 32].transpose(0, 1)
    q = s.cache.append(wide.cuda()[:, :, 1, 8:8 + 8 * 32].transpose(0, 1), 4, cos.cuda(), sin.cuda())
    want, dq, _ = s.model.append(f64(qkv), 4, cos.numpy(), sin.numpy())
    within(f64(q), want, dq + (np.abs(want) + dq) * HALF["float16"] + TINY["float16"])
    s.check_meta()


# ---- attend

def attend_once(s, Hq, counts=None, std=1.5, scale=None):
    m, c = s.model, s.cache
    q = s.randn(m.rows, Hq, m.D, std=std)
    before = c.weights.clone()
    n = None if counts is None else torch.tensor(counts, dtype=torch.int32)
    out = c.attend(q.cuda(), scale, counts=None if n is None else n.cuda())
    want, tol, wt = m.attend(f64(q), scale or m.D ** -0.5, s.dtype, counts, s.there)
    within(f64(out), want, tol)
    s.check_meta(wt)
    untouched = ~((np.arange(m.cap) < np.maximum(m.len, 0)[:, None]) & s.there)
    if counts is not None:
        untouched |= (np.array(counts) <= 0)[:, None]
    untouched = np.broadcast_to(untouched[:, None], m.w.shape)
    assert np.array_equal(f64(c.weights)[untouched], f64(before)[untouched])
    s.check_same_caches()


@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("D", [16, 32, 64, 96, 128, 192, 256])
@pytest.mark.parametrize("paged", [False, True])
def test_attend_types_and_heads(dtype, D, paged):
    attend_once(Setup(D, 3, 2, D, 190, [190, 77, 1], dtype, paged), 6)


@pytest.mark.parametrize("G", [1, 2, 5, 15, 16, 17, 33, 128])
@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_attend_groups(G, dtype):
    attend_once(Setup(G, 2, 2, 64, 161, [161, 130], dtype), 2 * G)


@pytest.mark.parametrize("paged", [False, True])
@pytest.mark.parametrize("n", [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 65, 127, 128, 129, 255, 257, 511, 513, 1000])
def test_attend_lengths(n, paged):
    attend_once(Setup(n, 2, 1, 64, 1003, [n, 1003 - n], "bfloat16", paged), 4)


@pytest.mark.parametrize("rows,heads", [(1, 1), (3, 1), (16, 4), (64, 8), (300, 2)])
def test_attend_rows(rows, heads):
    """From many slices a row to none, rows of every length among them."""
    attend_once(Setup(rows, rows, heads, 32, 300, [(37 * r) % 301 for r in range(rows)], "float16"), 2 * heads)


def test_attend_long():
    attend_once(Setup(8, 1, 1, 128, 20001, [20001], "bfloat16"), 4)


@pytest.mark.parametrize("rows", [2, 130])
def test_attend_leaves_out(rows):
    """Rows without new tokens, pages that are none, lengths that are none."""
    s = Setup(21, rows, 2, 64, 200, [200, 90] + [64] * (rows - 2), "bfloat16", True, bad=9)
    s.cache.lengths[1] = -4
    s.model.len[1] = -4
    attend_once(s, 8, counts=[1] * (rows - 1) + [0])


def test_attend_no_page_at_all():
    s = Setup(22, 1, 1, 64, 32, [32], "bfloat16", True)
    s.cache.block_table.fill_(-1)
    s.there[:] = False
    attend_once(s, 4)


@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
def test_attend_extreme_scores(dtype):
    """Scores far apart, and every key but one without weight; values of the type's size."""
    s = Setup(31, 2, 1, 64, 300, [300, 299], dtype)
    for x, y in ((s.cache.keys, s.model.k),):
        x[:, :, 100] *= 30
        y[:] = f64(x)
    for x, y in ((s.cache.values, s.model.v),):
        x[:, :, 5] *= 1000
        y[:] = f64(x)
    attend_once(s, 4, std=6.0)


@pytest.mark.parametrize("n", [70, 1500])
def test_attend_infinite_keys(n):
    """A key of -inf scores takes no weight; NaN anywhere in a row's keys makes that KV head's results NaN, as the formula has it, and no other's."""
    s = Setup(32, 2, 2, 64, n, [n, n], "float32")
    c = s.cache
    q = torch.randn((2, 4, 64), generator=s.g).abs().cuda()
    c.keys[0, 0, 3] = -float("inf")
    c.keys[1, 1, 40, 2] = float("nan")
    before = c.weights.clone()
    out = c.attend(q)
    p = torch.softmax((q.view(2, 2, 2, 64).double() @ c.keys.double().transpose(-1, -2)) / 8, -1)
    want = (p @ c.values.double()).view(2, 4, 64)
    assert torch.isnan(out[1, 2:]).all() and not torch.isnan(out[0]).any() and not torch.isnan(out[1, :2]).any()
    assert torch.isnan(c.weights[1, 1]).all() and c.weights[0, 0, 3] == before[0, 0, 3]
    torch.testing.assert_close(out[0].double(), want[0], rtol=1e-4, atol=1e-5)


@pytest.mark.parametrize("n", [40, 1500])
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_scores_near_the_ends_of_the_type(n, sign):
    """Scores of 1e33 and more, all above or all below zero: one key takes all the weight, of a token and of a prompt (whose last query repeats itself behind the end)."""
    s = Setup(33, 1, 1, 64, n, [n], "float32")
    c = s.cache
    c.keys[0, 0] = sign * 1e16 * (1 + torch.arange(n, device="cuda").float())[:, None]
    top = n - 1 if sign > 0 else 0
    c.weights.zero_()
    out = c.attend(torch.full((1, 2, 64), 1e17, device="cuda"))
    assert torch.equal(out, c.values[0, 0, top].expand(1, 2, 64))
    assert c.weights[0, 0, top] == 2 and c.weights.sum() == 2
    c.weights.zero_()
    c.weigh(torch.full((1, 3, 2, 64), 1e17, device="cuda"))
    want = torch.zeros(n, device="cuda")
    for i in range(3):
        want[n - 3 + i if sign > 0 else 0] += 2
    assert torch.equal(c.weights[0, 0], want)


def test_attend_beyond_32_bits():
    """Element numbers of the second row's keys pass 2^31."""
    from mlx_parallm_amd.bounded_cache import BoundedKVCache

    cap = (1 << 31) // (8 * 128) + 64
    c = BoundedKVCache.create(2, 8, 128, cap, dtype="bfloat16")
    g = torch.Generator(device="cuda").manual_seed(1)
    n = 300
    k, v = (torch.randn((8, n, 128), generator=g, device="cuda").bfloat16() for _ in range(2))
    c.keys[1, :, :n], c.values[1, :, :n] = k, v
    c.lengths[1] = n
    q = torch.randn((2, 16, 128), generator=g, device="cuda").bfloat16()
    out = c.attend(q)
    p = torch.softmax((q[1].view(8, 2, 128).double() @ k.double().transpose(1, 2)) / 128 ** 0.5, -1)
    want = (p @ v.double()).view(16, 128)
    assert (out[0] == 0).all()
    torch.testing.assert_close(out[1].double(), want, rtol=2 ** -8, atol=1e-4)
    torch.testing.assert_close(c.weights[1, :, :n].double(), p.sum(1), rtol=1e-4, atol=1e-6)
    c.positions[1, :, :n] = torch.arange(n, dtype=torch.int32, device="cuda")
    c.next_positions[1] = n
    kept = torch.sort(torch.argsort(c.weights[1, :, :n], dim=1, descending=True, stable=True)[:, :100], 1).values
    c.evict(100)
    assert c.lengths.tolist() == [0, 100]
    assert torch.equal(torch.sort(c.positions[1, :, :100], 1).values, kept.int())
    assert torch.equal(c.keys[1, :, :100], torch.gather(k, 1, c.positions[1, :, :100, None].long().expand(-1, -1, 128)))
    cos, sin = (t.cuda() for t in angles(400, 128))
    for L in (1, 20):                                     # both forms of the append, then a prompt's weights
        at = c.lengths[1].item()
        qkv = torch.randn((2, L, 32 * 128), generator=g, device="cuda").bfloat16()
        q = c.append(qkv, 16, cos, sin, counts=torch.tensor([0, L], dtype=torch.int32, device="cuda"))
        assert torch.equal(c.values[1, :, at:at + L], qkv[1, :, 24 * 128:].view(L, 8, 128).transpose(0, 1))
        want = c.weights[1, :, :at + L].double()
        x = q[1].view(L, 8, 2, 128).permute(1, 2, 0, 3).double() @ c.keys[1, :, None, :at + L].double().transpose(-1, -2) / 128 ** 0.5
        x.masked_fill_(torch.ones((L, at + L), dtype=torch.bool, device="cuda").triu(at + 1), -torch.inf)
        c.weigh(q, counts=torch.tensor([0, L], dtype=torch.int32, device="cuda"))
        torch.testing.assert_close(c.weights[1, :, :at + L].double(), want + torch.softmax(x, -1).sum((1, 2)), rtol=1e-4, atol=1e-6)


# ---- weigh

def weigh_once(s, L, Hq, counts=None, last=0, scale=None):
    m, c = s.model, s.cache
    q = s.randn(m.rows, L, Hq, m.D, std=1.5)
    before = c.weights.clone()
    n = None if counts is None else torch.tensor(counts, dtype=torch.int32)
    c.weigh(q.cuda(), scale, counts=None if n is None else n.cuda(), last=last)
    tol = m.weigh(f64(q), scale or m.D ** -0.5, counts, last, s.there)
    s.check_meta(tol)
    untouched = np.broadcast_to(~((np.arange(m.cap) < m.len[:, None]) & s.there)[:, None], m.w.shape)
    assert np.array_equal(f64(c.weights)[untouched], f64(before)[untouched])


@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("D", [16, 32, 64, 96, 128, 192, 256])
def test_weigh_types_and_heads(dtype, D):
    weigh_once(Setup(D + 1, 2, 2, D, 150, [150, 90], dtype, D % 64 == 0), 40, 6, counts=[40, 33])


@pytest.mark.parametrize("L,n", [(1, 1), (1, 70), (2, 64), (16, 16), (17, 17), (63, 63), (64, 129), (65, 65), (130, 131), (33, 500), (5, 1000)])
@pytest.mark.parametrize("paged", [False, True])
def test_weigh_lengths(L, n, paged):
    weigh_once(Setup(L + n, 2, 1, 64, n + 2, [n, n // 2], "bfloat16", paged), L, 4, counts=[min(L, n), min(L, n // 2)])


@pytest.mark.parametrize("G", [1, 3, 7, 16, 40])
def test_weigh_groups(G):
    weigh_once(Setup(G, 2, 2, 32, 100, [100, 61], "float16"), 50, 2 * G, counts=[50, 50])


@pytest.mark.parametrize("last", [1, 7, 64, 1000])
def test_weigh_last(last):
    weigh_once(Setup(last, 3, 2, 64, 120, [120, 80, 10], "bfloat16", True), 70, 4, counts=[70, 66, 0], last=last)


def test_weigh_more_queries_than_slots():
    """Queries whose slots are not there (the cache was full) see nothing; pages that are none; a row without keys."""
    weigh_once(Setup(41, 3, 1, 64, 64, [64, 20, 0], "bfloat16", True, bad=3), 50, 4)


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("D", [16, 64, 96, 128, 192, 256])
@pytest.mark.parametrize("L,G", [(1, 1), (7, 3), (16, 4), (3, 16)])
def test_weigh_few_queries(L, G, D, dtype):
    """One workgroup a row and head: few keys; pages that are none; rows with fewer keys than queries."""
    weigh_once(Setup(L + D, 3, 2, D, 120, [120, 65, 2], dtype, True, bad=4), L, 2 * G)
    weigh_once(Setup(L + D + 1, 2, 1, D, 128, [128, 0], dtype), L, G, counts=[L, max(0, L - 1)], last=2)


@pytest.mark.parametrize("dtype", ["float16", "float32"])
def test_weigh_few_queries_of_many_rows(dtype):
    weigh_once(Setup(43, 100, 2, 32, 400, [400 - 3 * r for r in range(100)], dtype, True), 5, 4, counts=[r % 6 for r in range(100)])


def test_weigh_many_rows():
    weigh_once(Setup(42, 40, 2, 16, 70, [70 - r for r in range(40)], "float32"), 9, 4)


# ---- evict

def evict_once(s, budget, first=0, last=0):
    s.cache.evict(budget, keep_first=first, keep_last=last)
    s.model.evict(budget, first, last, s.there)
    s.check_meta()
    s.check_same_caches()


@pytest.mark.parametrize("paged", [False, True])
@pytest.mark.parametrize("n,budget,first,last", [(1, 1, 0, 0), (2, 1, 0, 0), (2, 1, 1, 0), (2, 1, 0, 1), (33, 32, 4, 8), (100, 50, 0, 0), (100, 99, 4, 32), (100, 1, 0, 0),
                                                 (100, 7, 4, 3), (100, 7, 4, 32), (1500, 700, 4, 32), (4097, 4096, 0, 0), (5000, 300, 4, 200), (20, 64, 0, 0)])
def test_evict(n, budget, first, last, paged):
    s = Setup(n, 3, 2, 32, max(n + 1, 70), [n, max(0, n - 1), n // 2], "bfloat16", paged)
    evict_once(s, budget, first, last)


@pytest.mark.parametrize("dtype,D", [("float32", 16), ("float16", 256), ("bfloat16", 96), ("float32", 192)])
def test_evict_types(dtype, D):
    evict_once(Setup(D, 2, 3, D, 130, [130, 100], dtype, True), 60, 2, 5)


@pytest.mark.parametrize("n", [300, 5000, 13000, 37000])
@pytest.mark.parametrize("kind", ["equal", "zeros", "ties", "special", "negative", "near"])
def test_evict_weights(kind, n):
    """All equal, mostly zero, many equal, NaN and infinities and both zeros, below zero, neighbouring numbers."""
    s = Setup(n, 2, 1, 16, n + 9, [n, n - 7], "float32")
    g, shape = s.g, s.model.w.shape
    w = {"equal": lambda: torch.full(shape, 0.25),
         "zeros": lambda: torch.rand(shape, generator=g) * (torch.rand(shape, generator=g) > 0.9),
         "ties": lambda: torch.randint(0, 5, shape, generator=g).float() / 7,
         "special": lambda: torch.tensor([float("nan"), float("inf"), -float("inf"), 0.0, -0.0, 1.0, -float("nan"), 3.4e38, 1e-45])[torch.randint(0, 9, shape, generator=g)],
         "negative": lambda: torch.randn(shape, generator=g) * 1e-3,
         "near": lambda: (torch.full(shape, 0.1).view(torch.int32) + torch.randint(0, n, shape, generator=g).int()).view(torch.float32)}[kind]()
    s.cache.weights.copy_(w)
    s.model.w[:] = w.numpy()
    evict_once(s, n // 3, 2, 9)


@pytest.mark.parametrize("cap,n,budget", [(36864, 36860, 1000), (36865, 36865, 36800), (40000, 39990, 1000), (70000, 70000, 69999), (33000, 200, 100)])
def test_evict_large_caches(cap, n, budget):
    """On both sides of what the selection holds on chip, with much and little that moves."""
    s = Setup(77, 1, 2, 16, cap, [n], "bfloat16")
    evict_once(s, budget, 4, 64)


def test_evict_all_protected_and_odd_positions():
    """More protected keys than the budget holds, by their number or because positions occur more than once: the most weighted of them."""
    s = Setup(51, 2, 1, 16, 90, [90, 60], "float32")
    s.cache.positions.zero_()
    s.model.pos[:] = 0
    evict_once(s, 20, 4, 3)
    evict_once(Setup(55, 2, 1, 16, 90, [90, 60], "float32", skip=0), 20, 7, 2 ** 31 - 1)
    evict_once(Setup(56, 2, 2, 16, 15000, [15000, 14000], "float32", skip=0), 20, 30, 7)
    evict_once(Setup(58, 2, 1, 16, 38000, [38000, 14000], "float32", skip=0), 20, 30, 7)
    s = Setup(57, 2, 1, 16, 90, [90, 60], "float32")
    s.cache.next_positions.fill_(-2 ** 31)
    s.model.next[:] = -2 ** 31
    evict_once(s, 20, 0, 2 ** 31 - 1)


def test_evict_pages_that_are_none():
    evict_once(Setup(52, 3, 2, 32, 200, [200, 150, 190], "bfloat16", True, bad=6), 100, 4, 8)


def test_evict_a_budget_that_no_row_can_pass():
    s = Setup(53, 2, 1, 16, 50, [50, 20])
    evict_once(s, 50)
    evict_once(s, 1000)


def test_evict_twice_changes_nothing():
    s = Setup(54, 2, 2, 32, 100, [100, 90])
    evict_once(s, 40, 4, 4)
    evict_once(s, 40, 4, 4)


# ---- together

@pytest.mark.parametrize("dtype,paged,norm", [("bfloat16", True, True), ("float32", False, False), ("float16", True, False)])
def test_generation_in_a_bounded_cache(dtype, paged, norm):
    """A prompt longer than the budget, then steps at it: every call against the model, whose weights take the device's values after each comparison (an eviction
    is a comparison of numbers that two roundings may order differently)."""
    D, Hq, Hkv, R, budget = 64, 6, 2, 3, 24
    s = Setup(61, R, Hkv, D, 64, [0, 0, 0], dtype, paged, skip=0)
    c, m = s.cache, s.model
    cos, sin = angles(200, D)
    qn, kn = (1 + s.randn(D, std=0.1).float()).to(DT[dtype]), (1 + s.randn(D, std=0.1).float()).to(DT[dtype])
    kw, km = (dict(q_norm=qn.cuda(), k_norm=kn.cuda()), dict(q_norm=f64(qn), k_norm=f64(kn))) if norm else ({}, {})

    def take():
        m.w[:] = f64(c.weights)
        for x, y in zip(s.caches(), (m.k, m.v)):
            y[:] = x

    counts = torch.tensor([50, 13, 31], dtype=torch.int32)
    qkv = s.randn(R, 50, (Hq + 2 * Hkv) * D)
    q = c.append(qkv.cuda(), Hq, cos.cuda(), sin.cuda(), counts=counts.cuda(), **kw)
    want, dq, dk = m.append(f64(qkv), Hq, cos.numpy(), sin.numpy(), counts.numpy(), **km)
    within(f64(q), want, dq + (np.abs(want) + dq) * HALF[dtype] + TINY[dtype])
    take()
    c.weigh(q, counts=counts.cuda())
    s.check_meta(m.weigh(f64(q), D ** -0.5, counts.numpy()))
    take()
    evict_once(s, budget, 2, 4)
    for step in range(20):
        live = torch.tensor([1, 1, int(step % 3 > 0)], dtype=torch.int32)
        qkv = s.randn(R, 1, (Hq + 2 * Hkv) * D)
        q = c.append(qkv.cuda(), Hq, cos.cuda(), sin.cuda(), counts=live.cuda(), **kw)
        m.append(f64(qkv), Hq, cos.numpy(), sin.numpy(), live.numpy(), **km)
        take()
        s.check_meta()
        out = c.attend(q[:, 0], counts=live.cuda())
        want, tol, wt = m.attend(f64(q[:, 0]), D ** -0.5, dtype, live.numpy())
        within(f64(out), want, tol)
        s.check_meta(wt)
        take()
        evict_once(s, budget, 2, 4)
    assert c.lengths.tolist() == [24, 24, 24] and c.next_positions.tolist() == [70, 33, 44]


def test_the_frameworks_prompt_attention_reads_the_same_cache():
    """The second part of a prompt behind an eviction: mi_op_attention_prefill on the cache's arrays, offsets = lengths in front of the append."""
    import ctypes as C

    from mlx_parallm_amd import _lib as lib
    from tests.gpu_helpers import attn_shape, ptr

    D, Hq, Hkv, R, L = 128, 8, 2, 2, 20
    s = Setup(62, R, Hkv, D, 128, [60, 41], "bfloat16", True)
    c, m = s.cache, s.model
    evict_once(s, 40, 4, 8)
    cos, sin = angles(200, D)
    qkv = s.randn(R, L, (Hq + 2 * Hkv) * D)
    before = c.lengths.clone()
    q = c.append(qkv.cuda(), Hq, cos.cuda(), sin.cuda())
    m.append(f64(qkv), Hq, cos.numpy(), sin.numpy())
    m.k, m.v = s.caches()
    out = torch.empty((R, L, Hq, D), dtype=torch.bfloat16, device="cuda")
    shape = attn_shape(R, L, Hq, Hkv, D, "bfloat16", "bfloat16", 0, 128)
    torch.cuda.synchronize()
    lib.check(lib.lib().mi_op_attention_prefill(C.byref(shape), ptr(c.block_table), c.block_table.shape[1], 4, ptr(q), ptr(c.keys), ptr(c.values), ptr(before), ptr(out), D ** -0.5, 1, None, None))
    for i in range(L):
        sees = Model(m.k, m.v, before.cpu().numpy() + i + 1, m.next, m.pos, m.w)
        want, tol, _ = sees.attend(f64(q[:, i]), D ** -0.5, "bfloat16")
        within(f64(out[:, i]), want, tol + 2 ** -8 * np.abs(want) + 1e-3)      # (that kernel's own roundings; a wrong key would be off by its weight, 1 / 60)
    c.weigh(q)
    s.check_meta(m.weigh(f64(q), D ** -0.5))
    m.w[:] = f64(c.weights)
    evict_once(s, 40, 4, 8)


def steps(c, qkvs, Hq, cos, sin):
    outs = []
    for x in qkvs:
        q = c.append(x, Hq, cos, sin)
        outs.append(c.attend(q[:, 0]))
        c.evict(20, keep_first=2, keep_last=4)
    return outs


def copies(s):
    from mlx_parallm_amd.bounded_cache import BoundedKVCache

    c = s.cache
    return BoundedKVCache(*(t.clone() for t in (c.keys, c.values, c.lengths, c.next_positions, c.positions, c.weights)), c.block_table)


def same(a, b):
    for x in ("lengths", "next_positions", "positions", "weights", "keys", "values"):
        assert torch.equal(getattr(a, x).nan_to_num(), getattr(b, x).nan_to_num()), x


@pytest.mark.parametrize("cap", [40, 1000, 20000])
def test_captured_steps_are_the_eager_ones(cap):
    """A captured step, replayed with eager work of another cache in between."""
    s = Setup(71, 4, 2, 64, cap, [20, 3, cap - 10, 0], "bfloat16")
    cos, sin = (t.cuda() for t in angles(2000, 64))
    eager, other = copies(s), copies(s)
    x = torch.empty((4, 1, 12 * 64), dtype=torch.bfloat16, device="cuda")
    inputs = [s.randn(4, 1, 12 * 64).cuda() for _ in range(6)]
    want = steps(eager, inputs, 8, cos, sin)
    warm = copies(s)
    steps(warm, [inputs[0]], 8, cos, sin)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        (out,) = steps(s.cache, [x], 8, cos, sin)
    for i, y in enumerate(inputs):
        x.copy_(y)
        graph.replay()
        steps(other, [y], 8, cos, sin)
        if i % 2:
            torch.cuda.synchronize()
        assert torch.equal(out, want[i])
    same(s.cache, eager)
    same(other, eager)


def test_captured_prompt_weights():
    s = Setup(72, 2, 2, 64, 300, [300, 200], "bfloat16")
    q = s.randn(2, 100, 8, 64).cuda()
    eager = copies(s)
    for _ in range(3):
        eager.weigh(q, last=40)
    copies(s).weigh(q, last=40)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        s.cache.weigh(q, last=40)
    for _ in range(3):
        graph.replay()
        torch.randn(1000, device="cuda").sum().item()
    assert torch.equal(s.cache.weights, eager.weights)


def test_two_streams_at_once():
    s = Setup(73, 4, 2, 64, 1000, [20, 3, 900, 0], "bfloat16")
    cos, sin = (t.cuda() for t in angles(2000, 64))
    inputs = [s.randn(4, 1, 12 * 64).cuda() for _ in range(8)]
    caches, outs = [copies(s), copies(s)], [None, None]
    want = steps(s.cache, inputs, 8, cos, sin)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for i in range(2):
        with torch.cuda.stream(streams[i]):
            outs[i] = steps(caches[i], inputs, 8, cos, sin)
    torch.cuda.synchronize()
    for i in range(2):
        same(caches[i], s.cache)
        assert all(torch.equal(a, b) for a, b in zip(outs[i], want))


def test_a_new_cache_on_another_stream():
    """A cache made on one stream and evicted from at once on another, many heads racing for the row's ticket; the tickets are back at zero."""
    s = Setup(75, 40, 16, 16, 90, [90 - r for r in range(40)], "float32")
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for budget in (60, 59, 58, 30):
            evict_once(s, budget, 4, 8)
    torch.cuda.synchronize()
    assert s.cache._tickets.tolist() == [0] * 40


def test_the_same_call_twice_gives_the_same_bits():
    s = Setup(74, 3, 2, 128, 2000, [2000, 1500, 77], "bfloat16", True)
    a, b = copies(s), copies(s)
    q, p = s.randn(3, 10, 128).cuda(), s.randn(3, 300, 10, 128).cuda()
    for c in (a, b):
        c.out = c.attend(q)
        c.weigh(p, counts=torch.tensor([300, 300, 77], dtype=torch.int32, device="cuda"))
    assert torch.equal(a.out, b.out) and torch.equal(a.weights, b.weights)


def test_create_and_reset():
    from mlx_parallm_amd.bounded_cache import BoundedKVCache

    cos, sin = (t.cuda() for t in angles(100, 32))
    g = torch.Generator(device="cuda").manual_seed(4)
    x = [torch.randn((2, 5, 8 * 32), generator=g, device="cuda") for _ in range(2)]
    one, paged = (BoundedKVCache.create(2, 2, 32, 40, "float32", block_tokens=b) for b in (0, 16))
    for _ in range(2):
        outs = []
        for c in (one, paged):
            c.reset()
            c.append(x[0], 4, cos, sin)
            q = c.append(x[1], 4, cos, sin)
            outs.append(c.attend(q[:, -1]))
        assert torch.equal(outs[0], outs[1])
    assert one.lengths.tolist() == [10, 10] and paged.next_positions.tolist() == [10, 10]
