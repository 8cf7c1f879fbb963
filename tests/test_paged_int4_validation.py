"""Refusals of the 4-bit paged cache's C calls before they touch a device, and of their wrappers for CPU tensors."""
import ctypes

import pytest
import torch

import butterfly_b200 as bb
from butterfly_b200 import _lib

OK, BAD_SHAPE, BAD_STRIDE, BAD_DTYPE, UNSUPPORTED = _lib.OK, _lib.BAD_SHAPE, _lib.BAD_STRIDE, _lib.BAD_DTYPE, _lib.UNSUPPORTED
P = 1 << 20  # an aligned stand-in pointer: never dereferenced by a rejected call
BF = _lib.BF16


def _t(size, stride=None, data=P):
    if stride is None:
        stride, n = [0] * 4, 1
        for i in range(3, -1, -1):
            stride[i] = n
            n *= size[i]
    return _lib.Tensor4(data, (ctypes.c_int64 * 4)(*size), (ctypes.c_int64 * 4)(*stride))


POOL = (9, 2, 3, 18 * 128)


def _append(k=(1, 2, 5, 128), v=None, pool=POOL, slots=P, dt=BF, kd=P, pd=P, pool_stride=None):
    ts = [_t(k, data=kd), _t(v or k), _t(pool, pool_stride, data=pd)]
    return _lib.lib().bna_paged_append_int4(*(ctypes.byref(t) for t in ts), slots, dt, None)


def _read(k=(1, 2, 5, 128), v=None, pool=POOL, slots=P, dt=BF, kd=P, pd=P, pool_stride=None, k_stride=None):
    return _lib.lib().bna_paged_read_int4(ctypes.byref(_t(pool, pool_stride, data=pd)), slots, ctypes.byref(_t(k, k_stride, data=kd)),
                                          ctypes.byref(_t(v or k)), dt, None)


@pytest.mark.parametrize("call", [_append, _read])
def test_row_refusals(call):
    assert call(k=(1, 2, 0, 128)) == OK
    assert call(dt=7) == BAD_DTYPE and call(dt=2) == BAD_DTYPE
    assert call(k=(2, 2, 5, 128)) == BAD_SHAPE
    assert call(v=(1, 2, 6, 128)) == BAD_SHAPE
    assert call(pool=(9, 3, 3, 2304)) == BAD_SHAPE
    assert call(pool=(9, 2, 3, 2300)) == BAD_SHAPE
    assert call(pool=(0, 2, 3, 2304)) == BAD_SHAPE
    assert call(k=(1, 2, 5, 64)) == BAD_SHAPE
    assert call(k=(1, 2, 5, 96), pool=(9, 2, 3, 18 * 96)) == UNSUPPORTED
    assert call(pool=(9, 2, 1 << 28, 2304)) == UNSUPPORTED
    assert call(slots=None) == BAD_SHAPE and call(slots=P + 4) == BAD_STRIDE
    assert call(kd=P + 8) == BAD_STRIDE and call(kd=None) == BAD_SHAPE
    assert call(pd=P + 8) == BAD_STRIDE and call(pd=None) == BAD_SHAPE
    assert call(pool_stride=(0, 6912, 2304, 1)) == BAD_STRIDE        # pages over one another
    assert call(pool_stride=(13824, 6912, 2308, 1)) == BAD_STRIDE
    assert call(pool_stride=(13824, 6912, 2304, 2)) == BAD_STRIDE


def test_read_into_rows_over_one_another():
    assert _read(k_stride=(0, 0, 256, 1)) == BAD_STRIDE and _read(k_stride=(0, 640, 64, 1)) == BAD_STRIDE


def _decode(q=(3, 8, 1, 128), pool=POOL, kn=None, vn=None, active=None, out=None, dt=BF, table=P, ts=6, width=6, lens=P, window=0,
            scale=0.1, qd=P, ws=P, wsb=1 << 40, pd=P):
    new = [ctypes.byref(_t(x)) if x else None for x in (kn, vn)]
    return _lib.lib().bna_paged_decode_int4(ctypes.byref(_t(q, data=qd)), ctypes.byref(_t(pool, data=pd)), *new, active,
                                            ctypes.byref(_t(out or q)), None, 0, 0, dt, table, ts, width, lens, window, scale, ws, wsb, None)


def test_decode_refusals():
    assert _decode(q=(0, 8, 1, 128)) == OK
    assert _decode(dt=9) == BAD_DTYPE and _decode(dt=2) == BAD_DTYPE
    assert _decode(q=(3, 8, 2, 128)) == BAD_SHAPE
    assert _decode(q=(3, 7, 1, 128)) == BAD_SHAPE
    assert _decode(q=(3, 8, 1, 64)) == BAD_SHAPE
    assert _decode(q=(3, 8, 1, 80), pool=(9, 2, 3, 18 * 80)) == UNSUPPORTED
    assert _decode(pool=(9, 2, 3, 2288)) == BAD_SHAPE and _decode(pool=(9, 2, 0, 2304)) == BAD_SHAPE
    assert _decode(out=(3, 4, 1, 128)) == BAD_SHAPE
    assert _decode(kn=(3, 2, 1, 128)) == BAD_SHAPE
    assert _decode(kn=(3, 8, 1, 128), vn=(3, 8, 1, 128)) == BAD_SHAPE
    assert _decode(active=P) == BAD_SHAPE
    assert _decode(table=None) == BAD_SHAPE and _decode(lens=None) == BAD_SHAPE
    assert _decode(table=P + 2) == BAD_STRIDE and _decode(qd=P + 4) == BAD_STRIDE and _decode(pd=P + 4) == BAD_STRIDE
    assert _decode(width=0) == BAD_SHAPE and _decode(width=1 << 28) == UNSUPPORTED
    assert _decode(window=-1) == BAD_SHAPE
    assert _decode(ws=None) == _lib.CAPACITY and _decode(wsb=4096) == _lib.CAPACITY and _decode(ws=P + 8) == BAD_STRIDE
    assert _decode(scale=0.0) == BAD_SHAPE and _decode(scale=float("nan")) == BAD_SHAPE


def test_one_workspace_serves_both_kinds_of_decode():
    L = _lib.lib()
    assert 0 < L.bna_paged_decode_int4_workspace_bytes() <= L.bna_paged_decode_workspace_bytes()


def test_wrappers_refuse_cpu_tensors():
    rows = torch.zeros(4, 2, 128, dtype=torch.bfloat16)
    pool = torch.zeros(POOL, dtype=torch.uint8)
    slots = torch.zeros(4, dtype=torch.int64)
    i = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        bb.paged_append_int4(rows, rows, pool, slots)
    with pytest.raises(ValueError, match="CUDA"):
        bb.paged_read_int4(pool, slots, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        bb.paged_decode_attention_int4(rows[:1, :, None], pool, i[:, None], i)
    for bad in ((3, 2, 24, 128), (3, 2, 16, 96)):
        with pytest.raises(ValueError):
            bb.paged.int4_pool(*bad, device="cpu")
    assert bb.paged.int4_pool(3, 2, 48, 64, device="cpu").shape == (3, 2, 3, 18 * 64)


def _cache(**kw):
    a = dict(num_layers=2, num_pages=4, page_size=32, num_kv_heads=2, head_dim=64, max_requests=3, max_tokens_per_request=64, device="cpu")
    return bb.PagedKVCache(**{**a, **kw})


def test_cache_bits():
    c = _cache(cache_bits=4)
    assert [x.shape for x in c.kv_pages] == [(4, 2, 2, 18 * 64)] * 2 and not c.k_pages and not c.v_pages
    assert c.nbytes * 32 == _cache().nbytes * 9  # 4.5 bits a column for 16
    for bits in (8, 0, 32):
        with pytest.raises(ValueError, match="cache_bits"):
            _cache(cache_bits=bits)
    with pytest.raises(ValueError):
        _cache(cache_bits=4, dtype=torch.float32)
    with pytest.raises(ValueError):
        _cache(cache_bits=4, page_size=24)
    with pytest.raises(ValueError, match="4 bits"):
        _cache().read(0, torch.zeros(1, dtype=torch.int64))


def test_a_cache_takes_rows_of_its_own_type():
    c = _cache(cache_bits=4)
    rows = torch.zeros(4, 2, 64, dtype=torch.float16)
    with pytest.raises(ValueError, match="dtype"):
        c.append(0, rows, rows, torch.zeros(4, dtype=torch.int64))
    with pytest.raises(ValueError, match="dtype"):
        c.attend(0, rows[:3, :, None])
