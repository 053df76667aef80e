"""Sizes of the workspaces and limits of the calls of a cache of fixed size (no GPU: nothing is launched)."""
from __future__ import annotations

import pytest

from mlx_parallm_amd import _lib as L
from tests.test_bounded_cache import P, PAGED, cache, refused, tokens


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
