"""A cache of fixed size in 64-bit NumPy, slot by slot (what mlx_parallm_amd.bounded_cache is tested against)."""
from __future__ import annotations

import numpy as np

HALF = {"float32": 2.0 ** -24, "bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}       # half a step, relative
TINY = {"float32": 0.0, "bfloat16": 0.0, "float16": 2.0 ** -25}                     # half of float16's smallest number
U = 2.0 ** -24                                                                      # a rounding of the 32-bit arithmetic


class Model:
    """keys, values [rows, heads, cap, D], positions, weights [rows, heads, cap], lengths, following [rows]."""

    def __init__(self, keys, values, lengths, following, positions, weights):
        self.k, self.v = np.array(keys, np.float64), np.array(values, np.float64)
        self.len, self.next = np.asarray(lengths).astype(np.int64), np.asarray(following).astype(np.int64)
        self.pos, self.w = np.asarray(positions).astype(np.int64), np.asarray(weights).astype(np.float64)
        self.rows, self.heads, self.cap, self.D = self.k.shape

    def held(self, r):
        return int(min(max(self.len[r], 0), self.cap))

    def append(self, qkv, heads, cos, sin, counts=None, q_norm=None, k_norm=None, eps=1e-6):
        """-> queries, and how far 32-bit arithmetic may leave queries and keys from them before they are rounded (same shapes)."""
        R, Ln, _ = qkv.shape
        H, D = self.heads, self.D
        x = np.asarray(qkv, np.float64).reshape(R, Ln, heads + 2 * H, D)
        q, dq = np.zeros((R, Ln, heads, D)), np.zeros((R, Ln, heads, D))
        dk = np.zeros_like(self.k)
        for r in range(R):
            n = Ln if counts is None else min(int(counts[r]), Ln)
            at, first = self.held(r), int(self.next[r])
            n = max(0, 0 if first < 0 else min(n, self.cap - at, len(cos) - first))
            for t in range(n):
                for h in range(heads + H):
                    y = x[r, t, h]
                    if q_norm is not None:
                        y = y / np.sqrt(np.mean(y * y) + eps) * np.asarray(q_norm if h < heads else k_norm, np.float64)
                    a, b = y[:D // 2], y[D // 2:]
                    c, s = np.asarray(cos[first + t], np.float64), np.asarray(sin[first + t], np.float64)
                    z = np.concatenate([a * c - b * s, b * c + a * s])
                    # sum of D squares, division, square root, two products (2 D + 8 roundings at most, the norm's half under the root), then three
                    d = ((D + 8 if q_norm is not None else 0) + 3) * U * np.tile(np.abs(a) + np.abs(b), 2)
                    if h < heads:
                        q[r, t, h], dq[r, t, h] = z, d
                    else:
                        self.k[r, h - heads, at + t], dk[r, h - heads, at + t] = z, d
                self.v[r, :, at + t] = x[r, t, heads + H:]
                self.pos[r, :, at + t], self.w[r, :, at + t] = first + t, 0.0
            self.len[r], self.next[r] = at + n, first + n
        return q, dq, dk

    def probabilities(self, q, r, h, sees, there, scale):
        """softmax over the slots below `sees` that are there, and the relative error that 32 bits leave in it"""
        p = np.zeros(self.cap)
        at = np.flatnonzero((np.arange(self.cap) < sees) & there)
        if not len(at):
            return p, 0.0
        k = self.k[r, h, at]
        s = scale * (k @ q)
        e = np.exp(s - s.max())
        p[at] = e / e.sum()
        # a score: D products and sums, its scale; the exponent once more, to base 2 (2 ulp of its size); the exponential 2 ulp, the sum of all.  In both numerator and denominator
        off = (self.D + 4) * U * scale * float((np.abs(k) @ np.abs(q)).max()) + 4 * U * (1 + float(np.abs(s).max()))
        return p, 2 * off + (len(at) + 16) * U

    def attend(self, q, scale, dtype, counts=None, there=None):
        """-> output, its tolerance, tolerance of the weights"""
        R, Hq, D = q.shape
        out, tol, wt = np.zeros((R, Hq, D)), np.zeros((R, Hq, D)), np.zeros_like(self.w)
        for r in range(R):
            if counts is not None and counts[r] <= 0:
                continue
            for h in range(Hq):
                kh = h // (Hq // self.heads)
                ok = np.ones(self.cap, bool) if there is None else there[r]
                p, rel = self.probabilities(np.asarray(q[r, h], np.float64), r, kh, self.held(r), ok, scale)
                seen = p > 0
                out[r, h] = p[seen] @ self.v[r, kh, seen]
                # 16 bits: a weight is the sum of two numbers of that type (half a step of half a step), relative to 2^8 at most
                split = 0.0 if dtype == "float32" else 2 * HALF[dtype] ** 2
                size = p[seen] @ np.abs(self.v[r, kh, seen]) if seen.any() else np.zeros(D)
                tol[r, h] = (rel + split + seen.sum() * U) * size + TINY[dtype] * 2 ** 8 * np.abs(self.v[r, kh, seen]).sum(0)
                self.w[r, kh] += p
                wt[r, kh] += rel * p + 4 * U * np.abs(self.w[r, kh])
        return out, tol + (np.abs(out) + tol) * HALF[dtype] + TINY[dtype], wt + U * np.abs(self.w)

    def weigh(self, q, scale, counts=None, last=0, there=None):
        """-> tolerance of the weights"""
        R, Ln, Hq, D = q.shape
        wt = np.zeros_like(self.w)
        for r in range(R):
            n = Ln if counts is None else min(max(int(counts[r]), 0), Ln)
            ok = np.ones(self.cap, bool) if there is None else there[r]
            for i in range(max(0, n - last) if last else 0, n):
                for h in range(Hq):
                    kh = h // (Hq // self.heads)
                    p, rel = self.probabilities(np.asarray(q[r, i, h], np.float64), r, kh, self.held(r) - n + i + 1, ok, scale)
                    self.w[r, kh] += p
                    wt[r, kh] += rel * p
        asked = Ln * (Hq // self.heads) + 8
        return wt + asked * U * np.abs(self.w)

    def evict(self, budget, first=0, last=0, there=None):
        """Slots that are not there: in front of `budget` they stay as they are, behind it they leave; the other slots in front of it go to the best of the keys that are."""
        for r in range(self.rows):
            n = self.held(r)
            if n <= budget:
                continue
            lost = np.zeros(n, bool) if there is None else ~there[r, :n]
            for h in range(self.heads):
                p, w = self.pos[r, h, :n], self.w[r, h, :n]
                apart = (p < first) | (p >= self.next[r] - last)
                order = np.lexsort((np.arange(n), -np.where(np.isnan(w), -np.inf, w), ~apart))
                stays = lost & (np.arange(n) < budget)
                stays[order[~lost[order]][:budget - stays.sum()]] = True
                frm, to = np.flatnonzero(stays[budget:]) + budget, np.flatnonzero(~stays[:budget])
                self.pos[r, h, to], self.w[r, h, to] = self.pos[r, h, frm], self.w[r, h, frm]
                self.k[r, h, to], self.v[r, h, to] = self.k[r, h, frm], self.v[r, h, frm]
            self.len[r] = budget
