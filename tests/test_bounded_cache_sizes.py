"""Sizes of the workspaces and limits of the calls of a cache of fixed size (no GPU: nothing is launched)."""
from __future__ import annotations

import pytest
import torch

from mlx_parallm_amd import _lib as L
from mlx_parallm_amd.bounded_cache import BoundedKVCache
from tests.test_bounded_cache import P, PAGED, cache, parts, refused, tokens


@pytest.mark.parametrize("rows", [1, 8])
def test_the_workspace_of_the_last_queries_does_not_grow_with_the_prompt(rows):
    """Its statistics are those of the queries that ask: 64 of 40 heads, at most 64 slices of the keys and of the queries."""
    lib = L.lib()
    for tokens_ in (8001, 32768, 131072):
        c = cache(rows=rows, Hkv=8, D=128, cap=tokens_)
        one = rows * 40 * 64 * 8
        got = lib.mi_op_bounded_weigh_ws(c, tokens_, 40, 64)
        assert got == lib.mi_op_bounded_weigh_ws(c, 64, 40, 0) == lib.mi_op_bounded_weigh_ws(c, 64, 40, 100)
        assert one <= got <= one * 65 + 64 * rows * 8 * tokens_ * 4 + 1024
    c = cache(rows=rows, Hkv=8, D=128, cap=8001)
    assert lib.mi_op_bounded_weigh_ws(c, 8001, 40, 0) == lib.mi_op_bounded_weigh_ws(c, 8001, 40, 8001) >= rows * 40 * 8001 * 8


@pytest.mark.parametrize("call", [
    lambda c, n: c.evict(n), lambda c, n: c.evict(10, keep_first=n), lambda c, n: c.evict(10, keep_last=n),
    lambda c, n: c.weigh(torch.zeros((2, 3, 4, 64), dtype=torch.bfloat16), last=n)])
@pytest.mark.parametrize("n", [2 ** 31, 2 ** 32 + 5, 2 ** 64 + 1, -2 ** 31 - 1, -2 ** 32 + 5])
def test_numbers_of_more_than_32_bits_are_refused(call, n):
    """(The binding would cut them off: a budget of 2^32 + 5 would leave five keys, keep_last = 2^32 protect none.)"""
    with pytest.raises(ValueError, match="32 bits"):
        call(BoundedKVCache(**parts()), n)


def test_more_tokens_than_32_bits_count_are_refused():
    qkv = torch.zeros((2, 1, 8 * 64), dtype=torch.bfloat16).expand(2, 2 ** 32 + 1, 8 * 64)
    with pytest.raises(ValueError, match="32 bits"):
        BoundedKVCache(**parts()).append(qkv, 4, torch.zeros((10, 32)), torch.zeros((10, 32)))


def test_calls_of_more_threads_than_a_launch_takes_are_refused():
    """2^32 threads in a launch: the first launch of such a call would fail, and those behind it would go on with what it has not written."""
    lib = L.lib()
    at = 2 ** 32 // (8 << 2) // 2                         # tokens of 8 heads of 64, four lanes each, in two rows
    refused(lib.mi_op_bounded_append(cache(), tokens(L=at), None), -3, "too many")
    refused(lib.mi_op_bounded_weigh(cache(rows=1, Hkv=1, D=16, dtype=L.MI_F32), P, 2 ** 31 - 1, 1, None, 0, 0.1, P, 1 << 62, None), -3, "too many")
    refused(lib.mi_op_bounded_weigh(cache(rows=2000, Hkv=8, cap=1 << 20), P, 300, 8, None, 0, 0.1, P, 1 << 62, None), -3, "too many")
    for rc in (lib.mi_op_bounded_append(cache(), tokens(L=0), None), lib.mi_op_bounded_weigh(cache(), P, 0, 4, None, 0, 0.1, P, 1 << 40, None)):
        assert rc == -1


@pytest.mark.parametrize("scale", [2.4e38, 3.4e38])
def test_scales_that_are_infinite_to_base_2_are_refused(scale):
    lib = L.lib()
    refused(lib.mi_op_bounded_attend(cache(), P, 4, None, scale, P, P, 1 << 40, None), -1, "scale")
    refused(lib.mi_op_bounded_weigh(cache(), P, 3, 4, None, 0, scale, P, 1 << 40, None), -1, "scale")
