"""Refusals of the paged-cache entry points: statuses of the C calls before they touch a device,
and the Python wrappers' errors (there is no CPU path)."""
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


def _reserve(**kw):
    a = dict(lens=P, add=P, B=4, table=P, ts=10, width=10, free=P, pages=100, nf=P, page=16, lo=2 * P, nfo=2 * P, granted=P,
             slots=P, pos=P, tokens=7, stream=None)
    a.update(kw)
    return _lib.lib().bna_paged_reserve(*a.values())


def test_reserve_refusals():
    assert _reserve(B=0, tokens=0) == OK
    assert _reserve(B=0) == BAD_SHAPE
    assert _reserve(B=-1) == BAD_SHAPE
    assert _reserve(tokens=-1) == BAD_SHAPE
    assert _reserve(tokens=1 << 31) == BAD_SHAPE
    assert _reserve(width=0, ts=0) == BAD_SHAPE
    assert _reserve(ts=9) == BAD_SHAPE
    assert _reserve(page=0) == BAD_SHAPE
    assert _reserve(pages=0) == BAD_SHAPE
    assert _reserve(B=4097) == UNSUPPORTED
    for name in ("lens", "add", "table", "free", "nf", "lo", "nfo", "granted", "slots", "pos"):
        assert _reserve(**{name: None}) == BAD_SHAPE, name
    assert _reserve(lo=P) == BAD_SHAPE and _reserve(nfo=P) == BAD_SHAPE  # not in place
    assert _reserve(table=P + 2) == BAD_STRIDE and _reserve(slots=P + 4) == BAD_STRIDE
    assert b"slot_map" in _lib.lib().bna_last_error()


def _append(k=(1, 2, 5, 128), v=None, kp=(9, 2, 16, 128), vp=None, slots=P, dt=BF, **data):
    ts = [_t(s, data=data.get(n, P)) for n, s in (("kd", k), ("vd", v or k), ("kpd", kp), ("vpd", vp or kp))]
    return _lib.lib().bna_paged_append(*(ctypes.byref(t) for t in ts), slots, dt, None)


def test_append_refusals():
    assert _append(k=(1, 2, 0, 128)) == OK
    assert _append(dt=7) == BAD_DTYPE
    assert _append(k=(2, 2, 5, 128)) == BAD_SHAPE
    assert _append(v=(1, 2, 6, 128)) == BAD_SHAPE
    assert _append(kp=(9, 3, 16, 128)) == BAD_SHAPE
    assert _append(vp=(8, 2, 16, 128)) == BAD_SHAPE
    assert _append(kp=(9, 2, 24, 128)) == UNSUPPORTED
    assert _append(k=(1, 2, 5, 96), kp=(9, 2, 16, 96)) == UNSUPPORTED
    assert _append(kp=(9, 2, 16, 64)) == BAD_SHAPE
    assert _append(slots=None) == BAD_SHAPE
    assert _append(slots=P + 4) == BAD_STRIDE
    assert _append(kd=P + 8) == BAD_STRIDE
    assert _append(vpd=None) == BAD_SHAPE
    overlapping = _t((9, 2, 16, 128), (0, 2048, 128, 1))
    row = _t((1, 2, 5, 128))
    assert _lib.lib().bna_paged_append(ctypes.byref(row), ctypes.byref(row), ctypes.byref(overlapping),
                                       ctypes.byref(overlapping), P, BF, None) == BAD_STRIDE


def _decode(q=(3, 8, 1, 128), kp=(9, 2, 16, 128), vp=None, kn=None, vn=None, active=None, out=None, dt=BF, table=P, ts=6,
            width=6, lens=P, window=0, scale=0.1, qd=P, ws=P, wsb=1 << 40):
    t = [_t(q, data=qd), _t(kp), _t(vp or kp)]
    new = [ctypes.byref(_t(x)) if x else None for x in (kn, vn)]
    o = _t(out or q)
    return _lib.lib().bna_paged_decode(*(ctypes.byref(x) for x in t), *new, active, ctypes.byref(o), None, 0, 0, dt, table, ts,
                                       width, lens, window, scale, ws, wsb, None)


def test_decode_refusals():
    assert _decode(q=(0, 8, 1, 128)) == OK
    assert _decode(dt=9) == BAD_DTYPE
    assert _decode(q=(3, 8, 2, 128)) == BAD_SHAPE        # one new token per request
    assert _decode(q=(3, 7, 1, 128)) == BAD_SHAPE        # query heads per KV head
    assert _decode(q=(3, 8, 1, 64)) == BAD_SHAPE         # head_dim of q and pool
    assert _decode(q=(3, 8, 1, 80), kp=(9, 2, 16, 80)) == UNSUPPORTED
    assert _decode(kp=(9, 2, 20, 128)) == UNSUPPORTED
    assert _decode(kp=(0, 2, 16, 128)) == BAD_SHAPE
    assert _decode(vp=(9, 2, 32, 128)) == BAD_SHAPE
    assert _decode(out=(3, 4, 1, 128)) == BAD_SHAPE
    assert _decode(kn=(3, 2, 1, 128)) == BAD_SHAPE       # k_new without v_new
    assert _decode(kn=(3, 8, 1, 128), vn=(3, 8, 1, 128)) == BAD_SHAPE
    assert _decode(active=P) == BAD_SHAPE                # active without new rows
    assert _decode(table=None) == BAD_SHAPE and _decode(lens=None) == BAD_SHAPE
    assert _decode(table=P + 2) == BAD_STRIDE and _decode(qd=P + 4) == BAD_STRIDE
    assert _decode(width=0) == BAD_SHAPE
    assert _decode(width=1 << 28) == UNSUPPORTED
    assert _decode(window=-1) == BAD_SHAPE
    assert _decode(ws=None) == _lib.CAPACITY and _decode(wsb=4096) == _lib.CAPACITY and _decode(ws=P + 8) == BAD_STRIDE
    assert _decode(scale=0.0) == BAD_SHAPE and _decode(scale=float("nan")) == BAD_SHAPE


def test_wrappers_refuse_cpu_tensors():
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        bb.paged_reserve(i, i, torch.zeros(2, 4, dtype=torch.int32), i, i[:1], page_size=16, num_tokens=0)
    pool = torch.zeros(3, 2, 16, 128, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        bb.paged_append(pool[0].transpose(0, 1), pool[0].transpose(0, 1), pool, pool, torch.zeros(16, dtype=torch.int64))
    with pytest.raises(ValueError, match="CUDA"):
        bb.paged_decode_attention(pool[:2, :, :1], pool, pool, torch.zeros(2, 4, dtype=torch.int32), i)


@pytest.mark.gpu
def test_wrappers_check_types_and_shapes():
    dev = "cuda"
    i = torch.zeros(2, dtype=torch.int32, device=dev)
    table = torch.zeros(2, 4, dtype=torch.int32, device=dev)
    pool = torch.zeros(3, 2, 16, 128, dtype=torch.bfloat16, device=dev)
    q = torch.zeros(2, 4, 1, 128, dtype=torch.bfloat16, device=dev)
    for bad in (dict(lens=i.long()), dict(add=i[:1]), dict(block_table=table.t()), dict(num_free=i), dict(free_pages=i.float())):
        a = dict(lens=i, add=i, block_table=table, free_pages=i, num_free=i[:1])
        a.update(bad)
        with pytest.raises(ValueError):
            bb.paged_reserve(**a, page_size=16, num_tokens=0)
    rows = torch.zeros(5, 2, 128, dtype=torch.bfloat16, device=dev)
    slots = torch.zeros(5, dtype=torch.int64, device=dev)
    for a in ((rows.half(), rows, slots), (rows, rows, slots[:4]), (rows, rows, slots.int()), (rows[0], rows[0], slots),
              (rows.half(), rows.half(), slots)):
        with pytest.raises(ValueError):
            bb.paged_append(a[0], a[1], pool, pool, a[2])
    kn = torch.zeros(2, 2, 1, 128, dtype=torch.bfloat16, device=dev)
    for bad in (dict(q=q.half()), dict(q=q[0]), dict(lens=i[:1]), dict(block_table=table.long()), dict(k_new=kn),
                dict(k_new=kn.half(), v_new=kn.half()), dict(k_new=kn, v_new=kn, active=i), dict(window=-2), dict(scale=-1.0),
                dict(active=torch.ones(2, dtype=torch.bool, device=dev)), dict(workspace=torch.zeros(8, device=dev))):
        a = dict(q=q, k_pages=pool, v_pages=pool.clone(), block_table=table, lens=i)
        a.update(bad)
        with pytest.raises(ValueError):
            bb.paged_decode_attention(**a)
    with pytest.raises(_lib.BnaError):
        bb.paged_decode_attention(q, pool[:, :, :8], pool[:, :, :8], table, i)
    with pytest.raises(ValueError):
        bb.PagedKVCache(num_layers=1, num_pages=2, page_size=16, num_kv_heads=1, head_dim=64, max_requests=1,
                        max_tokens_per_request=16).reserve(i[:1])
