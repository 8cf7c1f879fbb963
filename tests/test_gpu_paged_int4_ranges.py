"""Attention over the 4-bit cache where scales, scores and lengths lie far apart.

Compared with float64 arithmetic on the values s c + m, as in test_gpu_paged_int4.py, with the bar of each column taken from its
own group y of 64 columns and its own head: with G_y = sum_j p_j (15 s_jy + |m_jy|), n keys, u the type's unit roundoff (2^-8 bf16,
2^-11 fp16) and ds the score's error (there),
  * sums of p (c s + m), or of p ((15 - c) (-s) + m + 15 s), have terms of 2 G_y at most, p off by a factor of 1 +- (2 ds + 2^-20)
    and fp32 sums by n 2^-23: 2 G_y (2 ds + 2^-20 + n 2^-23);
  * a product p s is rounded to fp16, 2^-11 of itself for bf16 results and (two parts) 2^-22 for fp16 ones, and 2^-25 at least in a unit
    where the group's largest one is 2^2 or more: G_y (w + n 2^-27), w = 2^-11 or 2^-22;
  * the result is rounded once: u |ref|.
"""
import math

import pytest
import torch

from .test_gpu_paged_int4 import DEV, DTYPES, U, Case, pack, value

pytestmark = pytest.mark.gpu
W = {torch.bfloat16: 2.0 ** -11, torch.float16: 2.0 ** -22}


def _check(c, got, window=0, scale=None):
    out, lse = got
    G, dh = c.Hq // c.Hkv, c.dh
    scale = 1 / math.sqrt(dh) if scale is None else scale
    for b, ln in enumerate(c.host):
        first = max(0, ln - window) if window else 0
        k, v = c.k[b][:, first:], c.v[b][:, first:]
        n = k.shape[1]
        q = c.q[b, :, 0].double().view(c.Hkv, G, dh)
        z = scale * q @ value(k).transpose(1, 2)
        p = torch.softmax(z, -1)
        ref = p @ value(v)
        _, s, m = pack(k)
        S = scale * (q.abs() @ (15 * s.double() + m.double().abs()).repeat_interleave(64, -1).transpose(1, 2)).amax(-1, keepdim=True)
        ds = (dh + 10) * 2 ** -23 * S
        _, s, m = pack(v)
        own = (p @ (15 * s.double() + m.double().abs())).repeat_interleave(64, -1)
        bar = U[c.dtype] * ref.abs() + own * (4 * ds + 2 ** -19 + n * 2 ** -22 + W[c.dtype] + n * 2 ** -27)
        o, ls = out[b, :, 0].double().view(c.Hkv, G, dh), lse[b, :, 0].double().view(c.Hkv, G)
        assert ((o - ref).abs() <= bar).all(), (b, ln, float(((o - ref).abs() / bar).max()))
        rl = torch.logsumexp(z, -1)
        assert ((ls - rl).abs() <= ds[..., 0] + 2 ** -20 + n * 2 ** -23 + 2 ** -21 * rl.abs()).all(), (b, ln)


def _normal(seed, dtype, dh, exponents):
    """Normal rows, much alike (so that what keys lose does not cancel), times 2^exponents(key numbers [n, 1], column groups [1, groups])."""
    g = torch.Generator(device=DEV).manual_seed(seed)

    def rows(b, n):
        x = torch.randn(2, 1, dh, generator=g, device=DEV) + 0.25 * torch.randn(2, n, dh, generator=g, device=DEV)
        e = torch.as_tensor(exponents(torch.arange(n, device=DEV)[:, None], torch.arange(dh // 64, device=DEV)[None]), device=DEV)
        return (x * torch.exp2(e.expand(n, dh // 64).double()).repeat_interleave(64, -1).float()).to(dtype)

    return rows


def _levels(dtype, dh, level):
    """Keys of equal columns level(key numbers): a query of equal entries c scores c sqrt(dh) level."""
    return lambda b, n: level(torch.arange(n, device=DEV).double())[None, :, None].expand(2, n, dh).to(dtype).contiguous()


def _equal_queries(c, nats):
    """Entries of each head h such that a key of level 1 scores nats[h % len]."""
    x = torch.tensor([nats[h % len(nats)] / math.sqrt(c.dh) for h in range(c.Hq)], device=DEV)
    c.q = x[None, :, None, None].expand_as(c.q).to(c.dtype).contiguous()


@pytest.mark.parametrize("dtype,low,high", [(torch.bfloat16, 0, 20), (torch.bfloat16, 0, 24), (torch.bfloat16, -30, 0), (torch.bfloat16, 0, 90),
                                            (torch.float16, -10, 12)])
@pytest.mark.parametrize("dh,G", [(128, 2), (128, 8), (128, 16), (256, 4), (256, 7)])
def test_one_group_far_above_another(dtype, low, high, dh, G):
    for at in (0, 1):  # the group with large values
        v = _normal(high, dtype, dh, lambda j, y: torch.where(y == at, high, low))
        c = Case([40, 700, 5000], 2 * G, 2, dh=dh, dtype=dtype, v=v, seed=G)
        _check(c, c.run())


@pytest.mark.parametrize("dtype,low,high", [(torch.bfloat16, 0, 24), (torch.bfloat16, 0, 40), (torch.float16, -10, 12)])
@pytest.mark.parametrize("dh,G", [(64, 3), (128, 4), (128, 5), (256, 2)])
def test_large_values_without_weight(dtype, low, high, dh, G):
    """One key 40 nats below the others, with values far above theirs: first, in the middle, last."""
    for at in (0, 333, 1999):
        v = _normal(at, dtype, dh, lambda j, y: torch.where(j == at, high, low))
        k = _levels(dtype, dh, lambda j: -(j == at).double())
        c = Case([2000], 2 * G, 2, dh=dh, dtype=dtype, k=k, v=v)
        _equal_queries(c, [40.0])
        _check(c, c.run())


@pytest.mark.parametrize("dtype,low,high", [(torch.bfloat16, 0, 30), (torch.float16, -10, 12)])
@pytest.mark.parametrize("dh,G", [(64, 4), (128, 2), (128, 6), (256, 8)])
def test_heads_that_attend_to_different_keys(dtype, low, high, dh, G):
    """Even heads see the keys with large values, odd ones those between them, 80 nats apart."""
    v = _normal(1, dtype, dh, lambda j, y: torch.where(j % 2 == 0, high, low))
    k = _levels(dtype, dh, lambda j: torch.where(j % 2 == 0, 1.0, -1.0))
    c = Case([33, 3000], 2 * G, 2, dh=dh, dtype=dtype, k=k, v=v)
    _equal_queries(c, [40.0, -40.0])
    _check(c, c.run())


@pytest.mark.parametrize("dtype,fall", [(torch.bfloat16, 30), (torch.bfloat16, 60), (torch.float16, 20)])
@pytest.mark.parametrize("dh,G", [(64, 4), (128, 4), (128, 9), (256, 4)])
def test_scores_that_rise_as_values_fall(dtype, fall, dh, G):
    """References move often and by little, in some heads further than in others, while values lose `fall` bits."""
    n = 4000
    v = _normal(2, dtype, dh, lambda j, y: 10 - fall * j / n)
    k = _levels(dtype, dh, lambda j: j / n)
    c = Case([n], 2 * G, 2, dh=dh, dtype=dtype, k=k, v=v)
    _equal_queries(c, [100.0, 20.0, 5.0, 50.0])
    _check(c, c.run())


@pytest.mark.parametrize("dh,Hq", [(64, 4), (128, 4), (128, 8)])
def test_the_longest_table_rows(dh, Hq):
    """Windows at the end of rows of 2^31 - 16 tokens, whose columns all name one page."""
    page = 16 * 511  # 262,657 of them are 2^31 - 16
    c = Case([page], Hq, 1, dh=dh, page=page, spare=0, seed=dh)
    c.table = c.table[:, :1].expand(1, 262657).contiguous()
    assert c.table.shape[1] * page == 2 ** 31 - 16
    for ln in (2 ** 31 - 16, 2 ** 31 - 17, 2 ** 31 - 31, 2 ** 31 - 32, 2 ** 31 - 40):
        for window in (1, 20, 130):
            at = (torch.arange(ln - window, ln, device=DEV) % page)
            d = Case([window], Hq, 1, dh=dh, page=16, k=lambda b, n: c.k[0][:, at], v=lambda b, n: c.v[0][:, at])
            d.q, d.table, d.pool = c.q, c.table, c.pool
            d.lens = torch.tensor([ln], dtype=torch.int32, device=DEV)
            _check(d, d.run(window=window))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("G", [2, 8])
def test_scores_of_next_to_nothing(dtype, G):
    """Scales far below 1, and queries of zeros or of the type's smallest entries: the mean of the values."""
    for scale in (1e-12, 1e-20, 1e-30, 1e-44):
        c = Case([5, 130, 3000], 2 * G, 2, dtype=dtype, seed=G)
        c.q[:, 0] = 0
        c.q[:, 1] = torch.finfo(dtype).tiny
        _check(c, c.run(scale=scale), scale=scale)


def _check_equal(c, got, top):
    """All weight in equal parts on the keys `top` of a request alone, whose scores are equal sums and far above the others."""
    out, lse = got
    dh, G = c.dh, c.Hq // c.Hkv
    ref = value(c.v[0])[:, top].mean(1).repeat_interleave(G, 0)
    _, s, m = pack(c.v[0])
    own = (15 * s.double() + m.double().abs()).repeat_interleave(64, -1)[:, top].mean(1).repeat_interleave(G, 0)
    assert ((out[0, :, 0].double() - ref).abs() <= U[c.dtype] * ref.abs() + own * (2 ** -18 + 2 * W[c.dtype])).all()
    z = (c.q[0, :, 0].double() * value(c.k[0])[:, top[0]].repeat_interleave(G, 0)).sum(-1) / math.sqrt(dh) + math.log(len(top))
    assert ((lse[0, :, 0].double() - z).abs() <= (dh + 10) * 2 ** -22 * z.abs()).all()


@pytest.mark.parametrize("dtype,sizes", [(torch.bfloat16, (2.0 ** 26, 2.0 ** 32, 2.0 ** 50, 2.0 ** 90)), (torch.float16, (2.0 ** 22, 2.0 ** 29))])
@pytest.mark.parametrize("dh,G", [(64, 3), (128, 4), (128, 8), (256, 2)])
def test_scores_far_above_zero(dtype, sizes, dh, G):
    """Scores up to `sizes`, the largest far from the others, over groups of small and of large values."""
    high = 20 if dtype == torch.bfloat16 else 10
    for size in sizes:
        q = min(2.0 ** 14, size ** 0.5)
        k = _levels(dtype, dh, lambda j: torch.where(j % 39 == 7, 1.25, 0.25 + 0.5 * (j % 2)) * (size / q / math.sqrt(dh)))
        for sign in (1, -1):  # the group with large values
            v = _normal(3, dtype, dh, lambda j, y: sign * high * (1 - 2 * (y % 2)))
            c = Case([500], 2 * G, 2, dh=dh, dtype=dtype, k=k, v=v)
            _equal_queries(c, [q * math.sqrt(dh)])
            _check_equal(c, c.run(), list(range(7, 500, 39)))


@pytest.mark.parametrize("dh,G", [(64, 3), (128, 4), (128, 8), (256, 2)])
def test_scores_far_below_zero(dh, G):
    """Nothing but scores down to -2^106: the least low ones have all weight."""
    for size in (2.0 ** 30, 2.0 ** 98, 2.0 ** 106):
        q = min(2.0 ** 50, size ** 0.5)
        k = _levels(torch.bfloat16, dh, lambda j: -torch.where(j % 39 == 7, 0.25, 0.5 + 0.5 * (j % 2)) * (size / q / math.sqrt(dh)))
        c = Case([500], 2 * G, 2, dh=dh, k=k, v=_normal(4, torch.bfloat16, dh, lambda j, y: 0 * y))
        _equal_queries(c, [q * math.sqrt(dh)])
        _check_equal(c, c.run(), list(range(7, 500, 39)))
