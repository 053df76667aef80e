"""The operators of a cache of fixed size (mlx_parallm_amd/bounded_cache.py) as cases that can be timed and checked.

A case is one call on one layer's cache: "append" (norms, rotation and append of new tokens), "attend" (attention of one new token
per row, with the weight that every key receives), "weigh" (the same weights for the queries of a prompt) and "evict" (the least
weighted keys leave).  Head layouts are those of this repository's benchmark models, of its tiny test models, or generic ones.
``run`` is the call: with ``own`` the framework's, without it the same in elementary torch operations.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

TYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16, "float32": torch.float32}
MISTRAL_7B = dict(heads=32, kv_heads=8, dim=128, norm=False)
QWEN3_14B = dict(heads=40, kv_heads=8, dim=128, norm=True)
BLOCK_TOKENS = 64                      # of the block-paged caches: the server's
EPS = 1e-6


def case(name, model, kind, rows, context, *, new=1, dtype="bfloat16", paged=False, ragged=0.0, budget=0, first=4, recent=32):
    """rows x context: keys that the rows hold before the call (append: `new` more come, weigh: the last `new` of them ask);
    ragged: the last row has that share of its keys less (its new tokens too), the others lie between."""
    return dict(model, **({"name": name} if name else {}), kind=kind, rows=rows, context=context, new=new, dtype=dtype, paged=paged, ragged=ragged,
                budget=budget, first=first, recent=recent)


def listed():
    return [
        # one user's next token: nothing but latency
        case("append_step_b1", MISTRAL_7B, "append", 1, 321),
        # a server's batch, normed heads, block-paged cache
        case("append_step_b32_paged", QWEN3_14B, "append", 32, 1025, paged=True, ragged=0.5),
        # a batch of prompts, the reference's float32 caches
        case("append_8x1024_kv32", MISTRAL_7B, "append", 8, 0, new=1024, dtype="float32"),
        # one user chatting: the latency of a token's attention
        case("attend_chat_b1", MISTRAL_7B, "attend", 1, 321),
        # the headline benchmark's attention: eight sequences, float32 caches
        case("attend_b8_kv32", MISTRAL_7B, "attend", 8, 1025, dtype="float32"),
        # a server's batch of unequal rows, one of them empty
        case("attend_b32_paged", QWEN3_14B, "attend", 32, 2048, paged=True, ragged=1.0),
        # long documents, half precision
        case("attend_b4_long_f16", MISTRAL_7B, "attend", 4, 32761, dtype="float16"),
        # which keys of a long prompt its last 64 queries look at
        case("weigh_window_8001", QWEN3_14B, "weigh", 1, 8001, new=64, paged=True),
        # whole prompts of unequal lengths
        case("weigh_4x2048", MISTRAL_7B, "weigh", 4, 2048, new=2048, ragged=0.6),
        # short prompts on float32 caches
        case("weigh_2x700_kv32", MISTRAL_7B, "weigh", 2, 700, new=700, dtype="float32"),
        # every step at the budget: one key comes, one leaves
        case("evict_step_b32", QWEN3_14B, "evict", 32, 1025, paged=True, budget=1024),
        # after a long prompt: one key in eight stays
        case("evict_8x8192", MISTRAL_7B, "evict", 8, 8192, budget=1024),
    ]


def draw(rng):
    """A case of the same kinds, sizes between the smallest and the largest listed ones."""
    def spread(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))

    heads, kv_heads, dim = rng.choice([(32, 8, 128), (40, 8, 128), (16, 8, 128), (8, 8, 128), (4, 4, 16), (5, 1, 64), (24, 1, 64), (12, 4, 96), (16, 2, 256), (8, 2, 32)])
    model = dict(heads=heads, kv_heads=kv_heads, dim=dim, norm=rng.random() < 0.5)
    kind, dtype = rng.choice(["append", "attend", "attend", "weigh", "evict"]), rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    how = dict(dtype=dtype, paged=rng.random() < 0.5, ragged=rng.choice([0.0, 0.3, 0.6, 1.0]))
    width = 131072 * 1024 // (kv_heads * dim * (2 if dtype == "float32" else 1))      # keys of a listed case's largest cache
    rows = spread(1, 32)
    if kind == "append":
        return case(None, model, kind, rows, rng.choice([0, spread(1, 2000)]), new=rng.choice([1, 1, spread(2, max(2, 6000 // rows))]), **how)
    if kind == "attend":
        return case(None, model, kind, rows, spread(1, min(32761, width // rows)), **how)
    if kind == "weigh":
        rows = spread(1, 4)
        new = spread(1, 2048 // rows)
        return case(None, model, kind, rows, new + rng.choice([0, spread(1, max(1, 4000 // rows))]), new=new, **how)
    context = spread(2, min(16384, width // (2 * rows), 524288 // (rows * kv_heads)))
    return case(None, model, kind, rows, context, budget=max(1, rng.choice([context - 1, int(context * rng.uniform(0.05, 0.95))])),
                first=rng.choice([0, 0, 4]), recent=rng.choice([0, 1, 32]), **how)


# ---- inputs ------------------------------------------------------------------------------------------------------------------

def lengths_of(c):
    """Keys and new tokens of every row."""
    keep = [1.0 - c["ragged"] * (r / (c["rows"] - 1) if c["rows"] > 1 else 0.0) for r in range(c["rows"])]
    keys = [int(round(c["context"] * k)) for k in keep]
    new = [int(math.ceil(c["new"] * k)) for k in keep]
    return keys, [min(n, k) for n, k in zip(new, keys)] if c["kind"] == "weigh" else new


def capacity_of(c):
    need = c["context"] + (c["new"] if c["kind"] == "append" else 0) + 3
    return -(-need // BLOCK_TOKENS) * BLOCK_TOKENS if c["paged"] else need


def prepare(c, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt, R, H, D, cap = TYPES[c["dtype"]], c["rows"], c["kv_heads"], c["dim"], capacity_of(c)
    keys, new = lengths_of(c)

    def normal(*shape, std=1.0, dtype=None):
        return (torch.randn(shape, generator=g, device="cuda") * std).to(dtype or dt)

    s = {"c": c, "cap": cap}
    shape = (R, H, cap, D)
    if c["paged"]:
        blocks = R * (cap // BLOCK_TOKENS) + 5                       # an arena that holds other rows' blocks too, in no order
        s["table"] = torch.randperm(blocks, generator=g, device="cuda")[:R * (cap // BLOCK_TOKENS)].to(torch.int32).view(R, -1)
        shape = (blocks, H, BLOCK_TOKENS, D)
    s["k"], s["v"] = normal(*shape), normal(*shape)
    # what changes with every token or eviction lies in one buffer: float32 weights, positions, lengths and next positions
    n = R * H * cap
    meta = torch.zeros(2 * n + 2 * R, dtype=torch.int32, device="cuda")
    weights, positions, lengths, following = meta[:n].view(torch.float32).view(R, H, cap), meta[n:2 * n].view(R, H, cap), meta[2 * n:2 * n + R], meta[2 * n + R:]
    # weights as attention leaves them: a few keys hold most of it, many have exactly nothing or the same
    weights.copy_(torch.exp(2.5 * torch.randn((R, H, cap), generator=g, device="cuda") - 4).clamp_(min=1e-3))
    weights.mul_((torch.rand((R, H, cap), generator=g, device="cuda") > 0.05).float())
    if c["kind"] == "weigh":
        weights.zero_()                                              # a prompt's first
    lengths.copy_(torch.tensor(keys, dtype=torch.int32))
    # caches that have been evicted from before: positions run ahead of slots, and slots are in no order of position
    skip = torch.randint(0, 50, (R,), generator=g, device="cuda", dtype=torch.int32)
    following.copy_(lengths + skip)
    at = torch.where(torch.arange(cap, device="cuda") < lengths[:, None, None], torch.rand((R, H, cap), generator=g, device="cuda"), 2.0)
    positions.copy_(torch.argsort(torch.argsort(at, dim=-1), dim=-1) + (skip[:, None, None] if c["kind"] == "evict" else 0))
    s.update(meta=meta, start=meta.clone(), weights=weights, positions=positions, lengths=lengths, next=following)
    counts = torch.tensor(new, dtype=torch.int32, device="cuda")
    if c["kind"] == "append":
        s["qkv"] = normal(R, c["new"], (c["heads"] + 2 * H) * D, std=1.5)
        half = D // 2
        angle = torch.arange(c["context"] + c["new"] + 64, device="cuda", dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half)
        s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
        s["counts"] = counts
        if c["norm"]:
            s["q_norm"], s["k_norm"] = 1 + normal(D, std=0.1), 1 + normal(D, std=0.1)
    elif c["kind"] == "attend":
        s["q"] = normal(R, c["heads"], D, std=1.5)
    elif c["kind"] == "weigh":
        s["q"] = normal(R, c["new"], c["heads"], D, std=1.5)
        s["counts"] = counts
    return s


# ---- the call ----------------------------------------------------------------------------------------------------------------

def run(s):
    c = s["c"]
    # append and evict change how many keys a row holds: every pass begins where the first one did
    if c["kind"] == "append":
        s["meta"][-2 * c["rows"]:].copy_(s["start"][-2 * c["rows"]:])
    elif c["kind"] == "evict":
        s["meta"].copy_(s["start"])
    if own:
        return run_own(s, c)
    return {"append": plain_append, "attend": plain_attend, "weigh": plain_weigh, "evict": plain_evict}[c["kind"]](s, c)


def run_own(s, c):
    from mlx_parallm_amd.bounded_cache import BoundedKVCache

    cache = s.get("cache")
    if cache is None:
        cache = s["cache"] = BoundedKVCache(s["k"], s["v"], s["lengths"], s["next"], s["positions"], s["weights"], block_table=s.get("table"))
    if c["kind"] == "append":
        q = cache.append(s["qkv"], c["heads"], s["cos"], s["sin"], counts=s["counts"], q_norm=s.get("q_norm"), k_norm=s.get("k_norm"), eps=EPS)
        return [q, s["k"], s["v"], s["positions"], s["weights"], s["lengths"], s["next"]]
    if c["kind"] == "attend":
        return [cache.attend(s["q"]), s["weights"]]
    if c["kind"] == "weigh":
        cache.weigh(s["q"], counts=s["counts"])
        return [s["weights"]]
    cache.evict(c["budget"], keep_first=c["first"], keep_last=c["recent"])
    return [s["k"], s["v"], s["positions"], s["weights"], s["lengths"]]


def place(s, slots):
    """Rows of the flat caches [-1][D] in which the slots [rows][kv heads][..] lie."""
    c, (R, H) = s["c"], slots.shape[:2]
    head = torch.arange(H, device="cuda")[None, :, None]
    if "table" not in s:
        return (torch.arange(R, device="cuda")[:, None, None] * H + head) * s["cap"] + slots
    block = torch.gather(s["table"].long()[:, None].expand(R, H, -1), 2, slots // BLOCK_TOKENS)
    return (block * H + head) * BLOCK_TOKENS + slots % BLOCK_TOKENS


def all_slots(s, x):
    if "table" not in s:
        return x.float()
    return x[s["table"].long()].transpose(1, 2).reshape(s["weights"].shape + x.shape[-1:]).float()


def plain_append(s, c):
    R, L, H, D, Hq = c["rows"], c["new"], c["kv_heads"], c["dim"], c["heads"]
    x = s["qkv"].view(R, L, Hq + 2 * H, D)
    qk, v = x[:, :, :Hq + H].float(), x[:, :, Hq + H:]
    if c["norm"]:
        w = torch.cat([s["q_norm"].float().expand(Hq, D), s["k_norm"].float().expand(H, D)])
        qk = qk * torch.rsqrt(qk.square().mean(-1, keepdim=True) + EPS) * w
    t = torch.arange(L, device="cuda")
    at = (s["next"][:, None] + t).long()
    cos, sin = s["cos"][at][:, :, None], s["sin"][at][:, :, None]
    a, b = qk[..., :D // 2], qk[..., D // 2:]
    qk = torch.cat([a * cos - b * sin, b * cos + a * sin], -1).to(x.dtype)
    q, k = qk[:, :, :Hq].contiguous(), qk[:, :, Hq:]
    taken = (t < s["counts"][:, None])[:, None]                       # [rows][1][tokens]
    slots = (s["lengths"][:, None] + t).long()[:, None].expand(R, H, L)
    rows = place(s, slots)
    for_cache = taken[..., None]
    kf, vf = s["k"].view(-1, D), s["v"].view(-1, D)
    kf[rows] = torch.where(for_cache, k.transpose(1, 2), kf[rows])
    vf[rows] = torch.where(for_cache, v.transpose(1, 2), vf[rows])
    s["positions"].scatter_(2, slots, torch.where(taken, at[:, None].int(), s["positions"].gather(2, slots)))
    s["weights"].scatter_(2, slots, torch.where(taken, 0.0, s["weights"].gather(2, slots)))
    s["lengths"].add_(s["counts"])
    s["next"].add_(s["counts"])
    return [q * (t < s["counts"][:, None])[:, :, None, None], s["k"], s["v"], s["positions"], s["weights"], s["lengths"], s["next"]]


def plain_attend(s, c):
    R, H, D = c["rows"], c["kv_heads"], c["dim"]
    seen = (torch.arange(s["cap"], device="cuda") < s["lengths"][:, None])[:, None, None]
    k, v = all_slots(s, s["k"]), all_slots(s, s["v"])
    x = s["q"].float().view(R, H, -1, D) @ k.transpose(-1, -2) * D ** -0.5
    x = torch.where(seen, x, -torch.inf)
    e = torch.where(seen, torch.exp(x - x.amax(-1, keepdim=True)), 0.0)
    p = e / e.sum(-1, keepdim=True).clamp_min(1e-30)
    out = p @ torch.where(seen[:, :, 0, :, None], v, 0.0)
    s["weights"].add_(p.sum(2))
    return [out.reshape(R, -1, D).to(s["q"].dtype), s["weights"]]


def plain_weigh(s, c):
    R, L, H, D = c["rows"], c["new"], c["kv_heads"], c["dim"]
    q = s["q"].float().view(R, L, H, -1, D).permute(0, 2, 3, 1, 4)                      # [rows][kv heads][group][queries][D]
    i, j = torch.arange(L, device="cuda")[:, None], torch.arange(s["cap"], device="cuda")
    n, new = s["lengths"][:, None, None], s["counts"][:, None, None]
    seen = ((i < new) & (j <= n - new + i))[:, None, None]
    x = torch.where(seen, q @ all_slots(s, s["k"])[:, :, None].transpose(-1, -2) * D ** -0.5, -torch.inf)
    e = torch.where(seen, torch.exp(x - x.amax(-1, keepdim=True)), 0.0)
    s["weights"].add_((e / e.sum(-1, keepdim=True).clamp_min(1e-30)).sum((2, 3)))
    return [s["weights"]]


def plain_evict(s, c):
    D, budget, cap = c["dim"], c["budget"], s["cap"]
    n, pos, w = s["lengths"][:, None, None], s["positions"], s["weights"]
    slot = torch.arange(cap, device="cuda").expand_as(pos)
    held = slot < n
    stays = (pos < c["first"]) | (pos >= s["next"][:, None, None] - c["recent"])
    bits = w.view(torch.int32).long()
    rank = torch.where(bits >= 0, bits, -(bits & 0x7fffffff))                            # the order of the floats
    rank = torch.where(w.isnan(), -0x7f800000, rank) + torch.where(held, torch.where(stays, 2, 1), 0) * 2 ** 33
    order = torch.argsort(rank, dim=-1, descending=True, stable=True)
    kept = torch.zeros_like(held).scatter_(2, order, (slot < budget)) & held
    left = n.clamp_max(budget)
    most = max(0, min(budget, cap - budget))                                             # moves, at most
    to = torch.argsort((~kept & (slot < left)).int(), dim=-1, descending=True, stable=True)[..., :most]
    mover = kept & (slot >= left)
    frm = torch.argsort(mover.int(), dim=-1, descending=True, stable=True)[..., :most]
    moved = torch.arange(most, device="cuda") < mover.sum(-1, keepdim=True)
    a, b = place(s, to), place(s, frm)
    for_cache = moved[..., None]
    kf, vf = s["k"].view(-1, D), s["v"].view(-1, D)
    kf[a] = torch.where(for_cache, kf[b], kf[a])
    vf[a] = torch.where(for_cache, vf[b], vf[a])
    pos.scatter_(2, to, torch.where(moved, pos.gather(2, frm), pos.gather(2, to)))
    w.scatter_(2, to, torch.where(moved, w.gather(2, frm), w.gather(2, to)))
    s["lengths"].clamp_(max=budget)
    return [s["k"], s["v"], pos, w, s["lengths"]]


# ---- what it cannot do without ----------------------------------------------------------------------------------------------

def work(c):
    es, D, H, Hq = 4 if c["dtype"] == "float32" else 2, c["dim"], c["kv_heads"], c["heads"]
    keys, new = lengths_of(c)
    if c["kind"] == "append":
        tokens = sum(new)
        return {"bytes": tokens * (2 * (Hq + 2 * H) * D * es + D * 4 + H * 8), "flops": tokens * (Hq + H) * D * (7 if c["norm"] else 3)}
    if c["kind"] == "attend":
        held = sum(keys)
        return {"bytes": held * H * (2 * D * es + 8) + 2 * c["rows"] * Hq * D * es, "flops": 4 * held * Hq * D}
    if c["kind"] == "weigh":
        pairs = sum(m * n - m * (m - 1) // 2 for n, m in zip(keys, new))
        return {"bytes": sum(keys) * H * (D * es + 8) + sum(new) * Hq * D * es, "flops": 2 * pairs * Hq * D}
    # keys that move: of those that stay, the share behind slot `budget`
    moves = sum(c["budget"] * (n - c["budget"]) / n for n in keys if n > c["budget"]) * H
    return {"bytes": sum(keys) * H * 8 + moves * (4 * D * es + 8), "flops": sum(keys) * H}


# ---- the same from the definition, in 64 bits --------------------------------------------------------------------------------

def exact(c, seed):
    s = prepare(c, seed)
    keys, new = lengths_of(c)
    H, G, D, f64 = c["kv_heads"], c["heads"] // c["kv_heads"], c["dim"], torch.float64

    def cached(x, r, h, n):
        """[n][D] of one row and head: a view of the first n slots."""
        if not c["paged"]:
            return x[r, h, :n].to(f64)
        return torch.cat([x[b, h] for b in s["table"][r].tolist()])[:n].to(f64)

    if c["kind"] == "append":
        q = torch.zeros((c["rows"], c["new"], c["heads"], D), dtype=f64, device="cuda")
        k, v, pos, w = s["k"].to(f64), s["v"].to(f64), s["positions"].clone(), s["weights"].to(f64)
        for r in range(c["rows"]):
            if not new[r]:
                continue
            x = s["qkv"][r, :new[r]].to(f64).view(new[r], -1, D)
            first = int(s["next"][r])
            for head in range(c["heads"] + 2 * H):
                y = x[:, head]
                if head < c["heads"] + H:
                    if c["norm"]:
                        y = y / torch.sqrt((y * y).mean(1, keepdim=True) + EPS) * s["q_norm" if head < c["heads"] else "k_norm"].to(f64)
                    z = torch.complex(y[:, :D // 2], y[:, D // 2:]) * torch.complex(s["cos"][first:first + new[r]].to(f64), s["sin"][first:first + new[r]].to(f64))
                    y = torch.cat([z.real, z.imag], 1)
                if head < c["heads"]:
                    q[r, :new[r], head] = y
                    continue
                h, into = (head - c["heads"]) % H, k if head < c["heads"] + H else v
                for b in range(keys[r] // BLOCK_TOKENS, -(-(keys[r] + new[r]) // BLOCK_TOKENS)) if c["paged"] else [0]:
                    lo, hi = (max(keys[r], b * BLOCK_TOKENS), min(keys[r] + new[r], (b + 1) * BLOCK_TOKENS)) if c["paged"] else (keys[r], keys[r] + new[r])
                    to = into[int(s["table"][r, b]), h, lo - b * BLOCK_TOKENS:hi - b * BLOCK_TOKENS] if c["paged"] else into[r, h, lo:hi]
                    to.copy_(y[lo - keys[r]:hi - keys[r]])
            pos[r, :, keys[r]:keys[r] + new[r]] = torch.arange(first, first + new[r], device="cuda", dtype=torch.int32)
            w[r, :, keys[r]:keys[r] + new[r]] = 0
        more = torch.tensor(new, dtype=torch.int32, device="cuda")
        return [q, k, v, pos, w, s["lengths"] + more, s["next"] + more]
    if c["kind"] in ("attend", "weigh"):
        w = s["weights"].to(f64)
        out = torch.zeros((c["rows"], c["heads"], D), dtype=f64, device="cuda")
        for r in range(c["rows"]):
            m = 1 if c["kind"] == "attend" else new[r]
            if not keys[r] or not m:
                continue
            ahead = torch.ones((m, keys[r]), dtype=torch.bool, device="cuda").triu(keys[r] - m + 1)
            for head in range(c["heads"]):
                h = head // G
                q = s["q"][r, head].to(f64)[None] if c["kind"] == "attend" else s["q"][r, :m, head].to(f64)
                p = torch.softmax((q @ cached(s["k"], r, h, keys[r]).T / math.sqrt(D)).masked_fill(ahead, -math.inf), 1)
                w[r, h, :keys[r]] += p.sum(0)
                if c["kind"] == "attend":
                    out[r, head] = (p @ cached(s["v"], r, h, keys[r]))[0]
        return [out, w] if c["kind"] == "attend" else [w]
    pos, w, k, v = s["positions"].cpu().numpy(), s["weights"].cpu().numpy(), s["k"].to(f64), s["v"].to(f64)
    following = s["next"].tolist()
    for r, n in enumerate(keys):
        if n <= c["budget"]:
            continue
        blocks = s["table"][r].tolist() if c["paged"] else None
        for h in range(H):
            p, x = pos[r, h, :n], w[r, h, :n]
            apart = (p < c["first"]) | (p >= following[r] - c["recent"])
            best = np.lexsort((np.arange(n), -np.where(np.isnan(x), -np.inf, x).astype(np.float64), ~apart))[:c["budget"]]
            stay = np.zeros(n, bool)
            stay[best] = True
            frm, to = np.flatnonzero(stay[c["budget"]:]) + c["budget"], np.flatnonzero(~stay[:c["budget"]])
            pos[r, h, to], w[r, h, to] = pos[r, h, frm], w[r, h, frm]
            f, t = torch.from_numpy(frm).cuda(), torch.from_numpy(to).cuda()
            for y in (k, v):
                if blocks is None:
                    y[r, h, t] = y[r, h, f]
                else:
                    b = s["table"][r].long()
                    y[b[t // BLOCK_TOKENS], h, t % BLOCK_TOKENS] = y[b[f // BLOCK_TOKENS], h, f % BLOCK_TOKENS]
    return [k, v, torch.from_numpy(pos).cuda(), torch.from_numpy(w).cuda().to(f64), s["lengths"].clamp(max=c["budget"])]
