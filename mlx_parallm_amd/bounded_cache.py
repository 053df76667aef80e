"""A KV cache of fixed size for one attention layer: keys that attention has looked at least make room for new ones.

The caches of the engine (``models/base.py``, ``engine.KVCache``) grow with the sequence.  ``BoundedKVCache`` holds at most a budget of
keys per row and KV head, on the kernels of ``csrc/bounded.hip`` (``mi_op_bounded_*``, include/mi355_ops.h)::

    cache = BoundedKVCache.create(rows, kv_heads, head_dim, capacity, dtype="bfloat16")
    q = cache.append(qkv, heads, cos, sin, counts=prompt_lengths)      # norms, rotation, append; [rows, L, heads, head_dim]
    ...                                                                # the prompt's attention (mi_op_attention_prefill reads the same arrays)
    cache.weigh(q, counts=cache.taken)                                 # what weight the prompt's queries give every key
    cache.evict(budget, keep_first=4, keep_last=32)
    while generating:
        q = cache.append(qkv, heads, cos, sin)                         # one token a row
        out = cache.attend(q[:, 0], counts=cache.taken)                # its attention; adds the weights
        cache.evict(budget, keep_first=4, keep_last=32)

``capacity`` holds the prompt, or the budget and what comes between two evictions.  A row that is full, or at the end of the angle tables, takes fewer tokens than it is given: ``taken`` says how many the
last append took, and with it as ``counts`` the others' queries (zeros) ask for nothing.  Everything is enqueued on torch's current stream of the cache's device, nothing waits: the lengths stay on the device, and the calls can be
captured into a HIP graph.  There are no gradients and no CPU fallback.
"""
from __future__ import annotations

import ctypes as C
from typing import Optional

import torch

from . import _lib as L

_DTYPES = {torch.float32: L.MI_F32, torch.bfloat16: L.MI_BF16, torch.float16: L.MI_F16}
_NAMES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}

# the current stream's handle: a tenth of a microsecond, where torch.cuda.current_stream() makes an object for it in 2.7 -- a fifth of a short call
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)


def _ptr(t) -> Optional[int]:
    return None if t is None else t.data_ptr()


def _whole(*numbers) -> None:
    # (ctypes cuts off what does not fit)
    for n in numbers:
        if not -2 ** 31 <= n < 2 ** 31:
            raise ValueError(f"{n}: a number of 32 bits")


class BoundedKVCache:
    """``keys`` / ``values`` [rows, kv_heads, capacity, head_dim], or -- with ``block_table`` [rows, blocks a row] int32 -- arenas
    [blocks, kv_heads, block_tokens, head_dim] as the engine's paged caches have them (block_tokens a power of two from 16 on; a block
    belongs to one row).  ``lengths``, ``next_positions`` [rows] int32: slots filled, position of the next token.  ``positions`` int32 and
    ``weights`` float32 [rows, kv_heads, capacity].  The tensors are the caller's: contiguous, on one GPU, updated in place."""

    def __init__(self, keys, values, lengths, next_positions, positions, weights, block_table=None):
        if keys.dtype not in _DTYPES or values.dtype != keys.dtype:
            raise ValueError("keys and values are both float32, bfloat16 or float16")
        if keys.dim() != 4 or values.shape != keys.shape:
            raise ValueError("keys and values have one shape, of four dimensions")
        if positions.dim() != 3:
            raise ValueError("positions: [rows, kv_heads, capacity]")
        rows, heads, cap = positions.shape
        if keys.shape[1] != heads or (block_table is None and tuple(keys.shape[:3]) != (rows, heads, cap)):
            raise ValueError(f"keys of shape {tuple(keys.shape)} do not go with positions of shape {tuple(positions.shape)}")
        if tuple(weights.shape) != (rows, heads, cap) or tuple(lengths.shape) != (rows,) or tuple(next_positions.shape) != (rows,):
            raise ValueError("weights have the shape of positions; lengths and next_positions one number a row")
        ints = [lengths, next_positions, positions] + ([] if block_table is None else [block_table])
        if any(t.dtype != torch.int32 for t in ints) or weights.dtype != torch.float32:
            raise ValueError("lengths, positions and the block table are int32, weights float32")
        if block_table is not None and (block_table.dim() != 2 or block_table.shape[0] != rows):
            raise ValueError("block_table: [rows, blocks a row]")
        for t in [keys, values, weights] + ints:
            if not t.is_contiguous():
                raise ValueError("the cache's tensors are contiguous")
            if t.device != keys.device:
                raise ValueError("the cache's tensors are on one device")
        self.keys, self.values, self.lengths, self.next_positions = keys, values, lengths, next_positions
        self.positions, self.weights, self.block_table = positions, weights, block_table
        self.rows, self.kv_heads, self.capacity, self.head_dim = rows, heads, cap, keys.shape[3]
        self.dtype, self.device, self._index = keys.dtype, keys.device, keys.device.index
        c = L.OpBoundedCache()
        c.rows, c.Hkv, c.D, c.dtype, c.cap = rows, heads, self.head_dim, _DTYPES[keys.dtype], cap
        if block_table is not None:
            tokens = keys.shape[2]
            if tokens < 16 or tokens & (tokens - 1):
                raise ValueError("block_tokens must be a power of two >= 16")
            c.n_blocks, c.bt_stride, c.bs_shift = keys.shape[0], block_table.shape[1], tokens.bit_length() - 1
        c.k, c.v, c.btab = keys.data_ptr(), values.data_ptr(), _ptr(block_table)
        c.len, c.next, c.pos, c.weight = lengths.data_ptr(), next_positions.data_ptr(), positions.data_ptr(), weights.data_ptr()
        # copied from the host, which waits: calls may come on any stream from here on (and a cache is not made while a graph is captured)
        self._tickets, self.taken = torch.zeros((2, rows), dtype=torch.int32).to(self.device)
        c.tickets = self._tickets.data_ptr()
        self._c, self._ref, self._lib = c, C.byref(c), L.lib()

    @classmethod
    def create(cls, rows: int, kv_heads: int, head_dim: int, capacity: int, dtype="bfloat16", *, block_tokens: int = 0, device="cuda") -> "BoundedKVCache":
        """An empty cache of its own tensors.  block_tokens > 0: paged, every row with blocks of its own for `capacity` slots."""
        dt = _NAMES.get(dtype) if isinstance(dtype, str) else dtype
        if dt not in _DTYPES:
            raise ValueError(f"dtype: {', '.join(_NAMES)}; got {dtype}")
        shape, table = (rows, kv_heads, capacity, head_dim), None
        if block_tokens:
            per_row = -(-capacity // block_tokens)
            shape = (rows * per_row, kv_heads, block_tokens, head_dim)
            table = torch.arange(rows * per_row, dtype=torch.int32, device=device).view(rows, per_row)
        at = dict(device=device)
        return cls(torch.zeros(shape, dtype=dt, **at), torch.zeros(shape, dtype=dt, **at), torch.zeros(rows, dtype=torch.int32, **at),
                   torch.zeros(rows, dtype=torch.int32, **at), torch.zeros((rows, kv_heads, capacity), dtype=torch.int32, **at),
                   torch.zeros((rows, kv_heads, capacity), **at), table)

    # ---- the operators

    def append(self, qkv, heads: int, cos, sin, *, counts=None, q_norm=None, k_norm=None, eps: float = 1e-6):
        """New tokens: ``qkv`` [rows, L, (heads + 2 kv_heads) * head_dim] (any strides of whole 16 bytes over rows and tokens) -> queries
        [rows, L, heads, head_dim], normed (where ``q_norm`` / ``k_norm`` [head_dim] are given) and rotated by ``cos`` / ``sin``
        [positions, head_dim / 2] float32.  ``counts`` [rows] int32: row r takes its first counts[r] tokens, the queries of the others are zeros.  A row
        takes no more than it has slots and the tables have positions; ``taken`` [rows] int32 holds from now on how many it took."""
        D, f32 = self.head_dim, torch.float32
        self._check(qkv, "qkv", self.dtype)
        rows, tokens, width = qkv.shape if qkv.dim() == 3 else (0, 0, 0)
        if rows != self.rows or tokens < 1 or width != (heads + 2 * self.kv_heads) * D or qkv.stride(2) != 1:
            raise ValueError(f"qkv: [{self.rows}, tokens, {(heads + 2 * self.kv_heads) * D}], contiguous in the last dimension")
        self._check(cos, "cos", f32)
        self._check(sin, "sin", f32)
        if cos.dim() != 2 or cos.shape[1] != D // 2 or sin.shape != cos.shape or not (cos.is_contiguous() and sin.is_contiguous()):
            raise ValueError(f"cos, sin: [positions, {D // 2}], contiguous")
        for t in (q_norm, k_norm):
            if t is not None:
                self._check(t, "norm weights", self.dtype)
                if t.shape != (D,) or not t.is_contiguous():
                    raise ValueError(f"norm weights: [{D}]")
        _whole(tokens)
        q = qkv.new_empty((rows, tokens, heads, D))
        a = L.OpBoundedTokens(qkv.data_ptr(), qkv.stride(0), qkv.stride(1), tokens, heads, self._counts(counts), _ptr(q_norm), _ptr(k_norm), eps, min(cos.shape[0], 2 ** 31 - 1),
                              cos.data_ptr(), sin.data_ptr(), q.data_ptr(), self.taken.data_ptr())
        self._call(self._lib.mi_op_bounded_append, self._ref, C.byref(a))
        return q

    def attend(self, q, scale: Optional[float] = None, *, counts=None):
        """Attention of one query per row, ``q`` [rows, heads, head_dim], over all keys that the row holds -> the same shape; adds the weight
        that every key receives to ``weights``.  scale: 1 / sqrt(head_dim).  Rows without keys, or with counts[r] <= 0 (``counts=cache.taken``: that
        took no token): zeros, and no weights."""
        self._check(q, "q", self.dtype)
        if q.dim() != 3 or q.shape[0] != self.rows or q.shape[2] != self.head_dim:
            raise ValueError(f"q: [{self.rows}, heads, {self.head_dim}]")
        q = q.contiguous()
        heads = q.shape[1]
        out = torch.empty_like(q)
        n = self._lib.mi_op_bounded_attend_ws(self._ref, heads)
        ws = self._workspace(n)
        self._call(self._lib.mi_op_bounded_attend, self._ref, q.data_ptr(), heads, self._counts(counts), self._scale(scale), out.data_ptr(), _ptr(ws), n)
        return out

    def weigh(self, q, scale: Optional[float] = None, *, counts=None, last: int = 0) -> None:
        """Adds the attention weights of a prompt's queries to ``weights``: ``q`` [rows, L, heads, head_dim], of which the first counts[r] are
        those of the row's last counts[r] slots; each sees the slots up to its own.  Behind an append: ``counts=cache.taken``.  last > 0: only the last
        `last` queries ask."""
        self._check(q, "q", self.dtype)
        if q.dim() != 4 or q.shape[0] != self.rows or q.shape[3] != self.head_dim:
            raise ValueError(f"q: [{self.rows}, tokens, heads, {self.head_dim}]")
        _whole(last, q.shape[1])
        q = q.contiguous()
        n = self._lib.mi_op_bounded_weigh_ws(self._ref, q.shape[1], q.shape[2], last)
        ws = self._workspace(n)
        self._call(self._lib.mi_op_bounded_weigh, self._ref, q.data_ptr(), q.shape[1], q.shape[2], self._counts(counts), last, self._scale(scale), _ptr(ws), n)

    def evict(self, budget: int, *, keep_first: int = 0, keep_last: int = 0) -> None:
        """At most ``budget`` keys stay per row and KV head: those at the first ``keep_first`` positions and the last ``keep_last`` before all
        others, then the most weighted (NaN least), equal ones by the lower slot.  Kept keys behind slot `budget` move into the holes in front of it.
        Slots in blocks that the table does not name have no key: in front of `budget` they stay as they are and count in it, behind it they leave."""
        _whole(budget, keep_first, keep_last)
        n = self._lib.mi_op_bounded_evict_ws(self._ref, budget)
        ws = self._workspace(n)
        self._call(self._lib.mi_op_bounded_evict, self._ref, budget, keep_first, keep_last, _ptr(ws), n)

    def reset(self) -> None:
        """Every row empty, its next token at position 0."""
        self.lengths.zero_()
        self.next_positions.zero_()

    # ---- helpers

    def _check(self, t, what: str, dtype) -> None:
        if t.dtype != dtype or t.device != self.device:
            raise ValueError(f"{what}: {dtype} on {self.device}, got {t.dtype} on {t.device}")

    def _counts(self, t) -> Optional[int]:
        if t is None:
            return None
        self._check(t, "counts", torch.int32)
        if t.shape != (self.rows,) or not t.is_contiguous():
            raise ValueError("counts: one number a row")
        return t.data_ptr()

    def _scale(self, scale) -> float:
        return self.head_dim ** -0.5 if scale is None else float(scale)

    def _workspace(self, n: int):
        # of torch's allocator, call by call: its blocks go round in the order of the stream, and a captured graph has its own
        return self.lengths.new_empty((n + 3) // 4) if n else None

    def _call(self, fn, *args) -> None:
        if self.device.type != "cuda":
            raise RuntimeError("no HIP device: the cache's tensors are on " + str(self.device))
        if torch.cuda.current_device() == self._index:
            rc = fn(*args, _raw_stream(self._index))
        else:
            with torch.cuda.device(self._index):
                rc = fn(*args, _raw_stream(self._index))
        if rc:
            L.check(rc)
