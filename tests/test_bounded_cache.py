"""What the operators of a cache of fixed size refuse (no GPU: nothing is launched)."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest
import torch

from mlx_parallm_amd import _lib as L
from mlx_parallm_amd.bounded_cache import BoundedKVCache
from tests.bounded_model import Model

SOME = (C.c_char * 64)()
P = (C.addressof(SOME) + 15) & ~15                       # (never read)


def cache(**kw):
    c = L.OpBoundedCache()
    for n, v in dict(dict(rows=2, Hkv=2, D=64, dtype=L.MI_BF16, cap=100, k=P, v=P, len=P, next=P, pos=P, weight=P, tickets=P), **kw).items():
        setattr(c, n, v)
    return C.byref(c)


def tokens(**kw):
    t = L.OpBoundedTokens()
    for n, v in dict(dict(qkv=P, ld_row=512, ld_token=512, L=1, Hq=4, eps=1e-6, max_pos=100, cos_tab=P, sin_tab=P, q_out=P), **kw).items():
        setattr(t, n, v)
    return C.byref(t)


def refused(rc, code, text):
    assert rc == code, (rc, L.lib().mi_last_error())
    assert text in L.lib().mi_last_error().decode()


PAGED = dict(btab=P, n_blocks=10, bt_stride=7, bs_shift=4)


@pytest.mark.parametrize("change,code,text", [
    (dict(rows=0), -1, "rows"), (dict(rows=70000), -1, "rows"), (dict(rows=40000, Hkv=2), -1, "rows"), (dict(Hkv=0), -1, "rows"), (dict(cap=0), -1, "slots"),
    (dict(dtype=3), -1, "dtype"), (dict(D=80), -3, "head sizes"), (dict(D=512), -3, "head sizes"), (dict(k=None), -1, "null"), (dict(weight=None), -1, "null"),
    (dict(len=None), -1, "null"), (dict(tickets=None), -1, "null"), (dict(k=P + 2), -1, "aligned"), (dict(PAGED, bs_shift=3), -1, "blocks"), (dict(PAGED, n_blocks=0), -1, "blocks"),
    (dict(PAGED, bt_stride=6), -1, "blocks"), (dict(PAGED, bs_shift=30), -1, "blocks")])
def test_caches_that_every_call_refuses(change, code, text):
    lib, c = L.lib(), cache(**change)
    refused(lib.mi_op_bounded_append(c, tokens(), None), code, text)
    refused(lib.mi_op_bounded_attend(c, P, 4, None, 0.1, P, P, 1 << 40, None), code, text)
    refused(lib.mi_op_bounded_weigh(c, P, 3, 4, None, 0, 0.1, P, 1 << 40, None), code, text)
    refused(lib.mi_op_bounded_evict(c, 10, 0, 0, P, 1 << 40, None), code, text)


@pytest.mark.parametrize("change,code,text", [
    (dict(L=0), -1, "tokens"), (dict(max_pos=0), -1, "positions"), (dict(Hq=3), -1, "multiple"), (dict(Hq=0), -1, "multiple"), (dict(Hq=258), -3, "128"), (dict(qkv=None), -1, "null"),
    (dict(cos_tab=None), -1, "null"), (dict(q_norm_w=P), -1, "together"), (dict(q_norm_w=P, k_norm_w=P, eps=-1.0), -1, "eps"), (dict(qkv=P + 2), -1, "16 bytes"),
    (dict(ld_token=516), -1, "16 bytes"), (dict(L=2 ** 31 - 1), -3, "too many")])
def test_append_refuses(change, code, text):
    refused(L.lib().mi_op_bounded_append(cache(), tokens(**change), None), code, text)


def test_attend_weigh_and_evict_refuse():
    lib = L.lib()
    for scale in (0.0, -1.0, float("inf"), float("nan")):
        refused(lib.mi_op_bounded_attend(cache(), P, 4, None, scale, P, P, 1 << 40, None), -1, "scale")
        refused(lib.mi_op_bounded_weigh(cache(), P, 3, 4, None, 0, scale, P, 1 << 40, None), -1, "scale")
    refused(lib.mi_op_bounded_attend(cache(), None, 4, None, 0.1, P, P, 1 << 40, None), -1, "queries")
    refused(lib.mi_op_bounded_attend(cache(), P, 4, None, 0.1, None, P, 1 << 40, None), -1, "queries")
    refused(lib.mi_op_bounded_weigh(cache(), P, 0, 4, None, 0, 0.1, P, 1 << 40, None), -1, "tokens")
    refused(lib.mi_op_bounded_weigh(cache(), P, 3, 4, None, -1, 0.1, P, 1 << 40, None), -1, "tokens")
    for budget, first, last in ((0, 0, 0), (-5, 0, 0), (10, -1, 0), (10, 0, -1)):
        refused(lib.mi_op_bounded_evict(cache(), budget, first, last, P, 1 << 40, None), -1, "budget")


def test_sizes_of_workspaces_need_no_device():
    lib = L.lib()
    assert lib.mi_op_bounded_attend_ws(cache(k=None, cap=1000), 4) > 2 * 4 * 1000 * 4 and lib.mi_op_bounded_attend_ws(cache(), 4) == 0
    assert lib.mi_op_bounded_weigh_ws(cache(), 150, 4, 0) >= 2 * 4 * 150 * 8 and lib.mi_op_bounded_weigh_ws(cache(), 50, 4, 0) == 0
    assert lib.mi_op_bounded_evict_ws(cache(cap=1000), 300) >= 2 * 2 * 300 * 8 and lib.mi_op_bounded_evict_ws(cache(), 90) == 0
    assert lib.mi_op_bounded_attend_ws(cache(D=80), 4) == 0 and lib.mi_op_bounded_attend_ws(cache(), 3) == 0


def test_no_device_no_result():
    if torch.cuda.is_available():
        pytest.skip("GPU present")
    refused(L.lib().mi_op_bounded_evict(cache(), 10, 0, 0, P, 1 << 40, None), -4, "no HIP device")
    c = BoundedKVCache.create(2, 2, 64, 50, device="cpu")
    with pytest.raises(RuntimeError, match="no HIP device"):
        c.attend(torch.zeros((2, 4, 64), dtype=torch.bfloat16))


def parts(**kw):
    i = dict(dtype=torch.int32)
    t = dict(keys=torch.zeros((2, 2, 50, 64), dtype=torch.bfloat16), values=torch.zeros((2, 2, 50, 64), dtype=torch.bfloat16), lengths=torch.zeros(2, **i),
             next_positions=torch.zeros(2, **i), positions=torch.zeros((2, 2, 50), **i), weights=torch.zeros((2, 2, 50)))
    t.update(kw)
    return t


@pytest.mark.parametrize("change,text", [
    (dict(keys=torch.zeros((2, 2, 50, 64))), "both"), (dict(values=torch.zeros((2, 2, 49, 64), dtype=torch.bfloat16)), "one shape"),
    (dict(keys=torch.zeros((2, 2, 50, 64), dtype=torch.float64), values=torch.zeros((2, 2, 50, 64), dtype=torch.float64)), "both"),
    (dict(positions=torch.zeros((2, 2, 51), dtype=torch.int32)), "do not go"), (dict(weights=torch.zeros((2, 2, 49))), "shape of positions"),
    (dict(lengths=torch.zeros(3, dtype=torch.int32)), "one number a row"), (dict(lengths=torch.zeros(2)), "int32"), (dict(weights=torch.zeros((2, 2, 50), dtype=torch.float64)), "float32"),
    (dict(weights=torch.zeros((2, 50, 2)).transpose(1, 2)), "contiguous"), (dict(positions=torch.zeros((2, 100), dtype=torch.int32)), "capacity"),
    (dict(block_table=torch.zeros((2, 4), dtype=torch.int32)), "power of two"), (dict(block_table=torch.zeros((3, 4), dtype=torch.int32)), "blocks a row")])
def test_tensors_that_are_no_cache(change, text):
    with pytest.raises(ValueError, match=text):
        BoundedKVCache(**parts(**change))


def test_create_refuses():
    for kw in (dict(dtype="int8"), dict(dtype=torch.float64), dict(block_tokens=24), dict(block_tokens=8)):
        with pytest.raises(ValueError):
            BoundedKVCache.create(1, 1, 64, 50, **{"device": "cpu", **kw})


def test_arguments_that_do_not_fit_the_cache():
    c = BoundedKVCache(**parts())
    b = dict(dtype=torch.bfloat16)
    cos = torch.zeros((10, 32))
    qkv = torch.zeros((2, 3, 8 * 64), **b)
    for call in (lambda: c.attend(torch.zeros((2, 4, 64))), lambda: c.attend(torch.zeros((3, 4, 64), **b)), lambda: c.attend(torch.zeros((2, 4, 32), **b)),
                 lambda: c.attend(torch.zeros((2, 4, 64), **b), counts=torch.zeros(2)), lambda: c.attend(torch.zeros((2, 4, 64), **b), counts=torch.zeros(3, dtype=torch.int32)),
                 lambda: c.weigh(torch.zeros((2, 4, 64), **b)), lambda: c.append(qkv, 5, cos, cos), lambda: c.append(qkv[:, :0], 4, cos, cos),
                 lambda: c.append(qkv, 4, cos.double(), cos), lambda: c.append(qkv, 4, cos, cos[:5]), lambda: c.append(qkv, 4, cos, cos, q_norm=torch.zeros(32, **b)),
                 lambda: c.append(torch.zeros((2, 8 * 64, 3), **b).transpose(1, 2), 4, cos, cos)):
        with pytest.raises(ValueError):
            call()


def test_the_model_of_an_eviction_by_hand():
    """Slots 0..5 at positions 3 0 5 1 2 4, next 6; position 0 and the last one stay anyway: of 4 the two most weighted others, 0.9 and the first 0.5."""
    m = Model(np.arange(6.0).reshape(1, 1, 6, 1) * np.ones(16), np.zeros((1, 1, 6, 16)), [6], [6], [[[3, 0, 5, 1, 2, 4]]], [[[0.1, 0.0, 0.0, 0.5, 0.9, 0.5]]])
    m.evict(4, 1, 1)
    assert m.len[0] == 4 and m.pos[0, 0, :4].tolist() == [2, 0, 5, 1] and m.k[0, 0, :4, 0].tolist() == [4, 1, 2, 3] and m.w[0, 0, 0] == 0.9
