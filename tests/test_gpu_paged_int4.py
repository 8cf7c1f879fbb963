"""The 4-bit paged cache on the GPU: rows into blocks and back, and one-token attention over them.

Codes, scales and minima must equal the formula's bit for bit, and so must rows read back.  Attention is compared
with float64 arithmetic on the values s c + m that the blocks stand for.  Its bars, per element, with u the unit
roundoff of the 16-bit type (2^-8 bf16, 2^-11 fp16), n the keys attended to, S the largest over the keys of
scale * sum_y (s_y sum|q_y| c + |m_y| sum|q_y|) and A = sum_j p_j (s_j c_j + |m_j|) of the column:
  * a score is an fp32 sum of dh exact products per group (tensor cores truncate: 2^-23 a step), scaled and added in
    fp32, from queries that are exact but for 2^-34 of their head's largest entry: off by ds <= (dh + 10) 2^-23 S;
  * a probability is off by a factor of 1 +- (ds + 2^-21); times the scale it is rounded to fp16, 2^-11 for bf16
    results, to two fp16 parts, 2^-22, for fp16 ones; 2^-25 at least, in units where a probability of 1 and
    the largest scale are 2^11 / 8 or more, which adds n 15 2^-25 8 2^-11 <= n 2^-29 of the largest scale;
    sums over n keys add n 2^-23; the result is rounded once:
      |out - ref| <= u |ref| + A (2 ds + w + n 2^-23) + n 2^-29 max s,   w = 2^-10 (bf16) or 2^-20 (fp16)
  * |lse - ref| <= ds + 2^-20 + n 2^-23 + 2^-21 |ref|
"""
import math

import pytest
import torch

import butterfly_b200 as bb
from butterfly_b200 import paged

pytestmark = pytest.mark.gpu
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
W = {torch.bfloat16: 2.0 ** -10, torch.float16: 2.0 ** -20}
DTYPES = [torch.bfloat16, torch.float16]
DEV = "cuda"


# ------------------------------------------------------------------------------ the format, plainly
def pack(x):
    """(codes [.., dh] int, s [.., groups], m [.., groups]) of rows, in their type."""
    f = x.double().unflatten(-1, (-1, 64))
    m, hi = f.amin(-1), f.amax(-1)
    s = ((hi.float() - m.float()) / torch.full_like(m, 15, dtype=torch.float32)).to(x.dtype)
    bad = ~torch.isfinite(f).all(-1)
    m16 = torch.where(bad, math.nan, m).to(x.dtype)
    s = torch.where(bad, math.nan, s.double()).to(x.dtype)
    use = (s > 0) & torch.isfinite(s)
    q = (f.float() - m16.float()[..., None]) / torch.where(use, s.float(), 1.0)[..., None]
    return torch.where(use[..., None], torch.round(q).clamp(0, 15), 0.0).int().flatten(-2), s, m16


def blocks_of(k, v):
    """Rows k, v [.., 16, dh] -> blocks [.., 18 dh] of bytes."""
    halves = []
    for x in (k, v):
        c, s, m = pack(x)
        words = c.unflatten(-1, (-1, 8, 8)).transpose(-3, -2).flatten(-3)  # [.., 16, (g, y, i)]
        b = (words[..., ::2] | words[..., 1::2] << 4).to(torch.uint8).flatten(-2)
        p = torch.stack([s, m], -1).flatten(-3).contiguous().view(torch.uint8)
        halves += [b, p]
    return torch.cat(halves, -1)


def value(x):
    """What rows are read as, in float64."""
    c, s, m = pack(x)
    return (c.double().unflatten(-1, (-1, 64)) * s.double()[..., None] + m.double()[..., None]).flatten(-2)


def _rows(g, *shape, dtype, scale=1.0, shift=0.0):
    return (torch.randn(*shape, generator=g, device=DEV) * scale + shift).to(dtype)


# ------------------------------------------------------------------------------ append and read
def _slots(g, pages, page, T, skip=0):
    s = torch.randperm(pages * page, generator=g, device=DEV)[:T].clone()
    s[torch.randperm(T, generator=g, device=DEV)[:skip]] = -1
    return s


def _pool(g, pages, Hkv, page, dh, token_major=False):
    shape = (pages, page // 16, Hkv, 18 * dh) if token_major else (pages, Hkv, page // 16, 18 * dh)
    p = torch.randint(0, 256, shape, generator=g, device=DEV, dtype=torch.uint8)
    return p.transpose(1, 2) if token_major else p


def _expected(pool, k, v, slots):
    """The pool after an append, written a token at a time through views of its parts."""
    want = pool.clone()
    dh, page = k.shape[-1], 16 * pool.shape[2]
    for t, slot in enumerate(slots.tolist()):
        if not 0 <= slot < pool.shape[0] * page:
            continue
        p, off = slot // page, slot % page
        block = want[p, :, off // 16]
        for half, x in ((0, k[t]), (9 * dh, v[t])):
            c, s, m = pack(x)
            words = c.unflatten(-1, (-1, 8, 8)).transpose(-3, -2).flatten(-3)
            r = off % 16
            block[:, half + r * dh // 2: half + (r + 1) * dh // 2] = (words[:, ::2] | words[:, 1::2] << 4).to(torch.uint8)
            block[:, half + 8 * dh + r * dh // 16: half + 8 * dh + (r + 1) * dh // 16] = \
                torch.stack([s, m], -1).flatten(-2).contiguous().view(torch.uint8)
    return want


def _same(pool, want, dtype, dh):
    """Equal bytes, but for the bits of NaNs."""
    if torch.equal(pool, want):
        return True
    ok = pool == want
    for at in (8 * dh, 17 * dh):
        a, b = (x[..., at:at + dh].contiguous().view(dtype) for x in (pool, want))
        nan = torch.isnan(a) & torch.isnan(b)
        ok[..., at:at + dh] |= nan.repeat_interleave(2, dim=-1)
    return bool(ok.all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dh", [64, 128, 256])
@pytest.mark.parametrize("T,Hkv,page,token_major", [(1, 1, 16, False), (77, 3, 48, True), (5, 8, 64, False)])
def test_append_and_read(dtype, dh, T, Hkv, page, token_major):
    g = torch.Generator(device=DEV).manual_seed(T + dh)
    pages = -(-T // page) + 2
    kv = _rows(g, T, 2 * Hkv, dh, dtype=dtype)
    k, v = kv[:, :Hkv], kv[:, Hkv:]
    pool = _pool(g, pages, Hkv, page, dh, token_major)
    slots = _slots(g, pages, page, T, skip=T // 5)
    want = _expected(pool, k, v, slots)
    bb.paged_append_int4(k, v, pool, slots)
    assert torch.equal(pool, want)  # the formula's bytes, and all others as they were
    got = bb.paged_read_int4(pool, slots, dtype=dtype)
    for x, y in zip(got, (k, v)):
        ref = torch.where((slots >= 0)[:, None, None], value(y), 0.0)
        assert x.dtype == dtype and torch.equal(x, ref.to(dtype))


def test_many_rows_and_any_strides():
    """Enough rows for several a thread; heads and tokens of k and v at strides of their own."""
    g = torch.Generator(device=DEV).manual_seed(3)
    T, Hkv, dh, page = 40007, 2, 128, 32
    k = _rows(g, Hkv, T, dh + 8, dtype=torch.bfloat16)[..., :dh].transpose(0, 1)
    v = _rows(g, T, Hkv + 1, dh, dtype=torch.bfloat16)[:, 1:]
    pages = -(-T // page) + 1
    pool = _pool(g, pages, Hkv, page, dh)
    slots = _slots(g, pages, page, T, skip=31)
    bb.paged_append_int4(k, v, pool, slots)
    got = bb.paged_read_int4(pool, slots, dtype=torch.bfloat16)
    for x, y in zip(got, (k, v)):
        assert torch.equal(x, torch.where((slots >= 0)[:, None, None], value(y), 0.0).to(torch.bfloat16))


@pytest.mark.parametrize("dtype", DTYPES)
def test_special_rows(dtype):
    fi = torch.finfo(dtype)
    rows = [torch.zeros(64), torch.full((64,), 3.0), torch.full((64,), -0.0), torch.full((64,), fi.max / 4),
            torch.linspace(-1, 1, 64) * fi.max / 4, torch.linspace(0, 1, 64) * fi.smallest_normal, torch.linspace(-1, 2, 64) * 2.0 ** -13,
            torch.tensor([0.0] * 63 + [1.0]), torch.tensor([100.0] * 63 + [100.5]), torch.arange(64) * 0.25, torch.arange(64) % 16 + 0.5,
            torch.tensor([math.nan] + [1.0] * 63), torch.tensor([math.inf] + [1.0] * 63), torch.tensor([-math.inf, math.inf] + [0.0] * 62),
            torch.full((64,), math.inf), torch.tensor([fi.max, fi.min] + [0.0] * 62)]
    x = torch.stack(rows).to(dtype).to(DEV)
    n = len(rows)
    # every special group beside an ordinary one, in both places
    plain = torch.randn(n, 64, device=DEV).to(dtype)
    k = torch.stack([torch.cat([x, plain], -1), torch.cat([plain, x], -1)], 1)
    v = k.flip(0).contiguous()
    pool = torch.zeros(3, 2, 1, 18 * 128, dtype=torch.uint8, device=DEV)
    slots = torch.arange(n, device=DEV) + 17
    want = _expected(pool, k, v, slots)
    bb.paged_append_int4(k, v, pool, slots)
    assert _same(pool, want, dtype, 128)
    got = bb.paged_read_int4(pool, slots, dtype=dtype)
    for a, b in zip(got, (k, v)):
        assert torch.equal(torch.nan_to_num(a, nan=-77.0), torch.nan_to_num(value(b).to(dtype), nan=-77.0))
    finite = torch.isfinite(k.double()).reshape(n, 2, 2, 64).all(-1)
    assert torch.isnan(got[0].reshape(n, 2, 2, 64)[~finite]).all()


def test_slots_outside_the_pool():
    g = torch.Generator(device=DEV).manual_seed(1)
    k, v = _rows(g, 6, 2, 64, dtype=torch.float16), _rows(g, 6, 2, 64, dtype=torch.float16)
    pool = _pool(g, 3, 2, 32, 64)
    slots = torch.tensor([-1, 96, 95, 2 ** 40, -2 ** 62, 0], device=DEV)
    want = _expected(pool, k, v, slots)
    bb.paged_append_int4(k, v, pool, slots)
    assert torch.equal(pool, want)
    got = bb.paged_read_int4(pool, slots, dtype=torch.float16)
    keep = torch.tensor([False, False, True, False, False, True], device=DEV)[:, None, None]
    for a, b in zip(got, (k, v)):
        assert torch.equal(a, torch.where(keep, value(b), 0.0).half())
    empty = torch.empty(0, 2, 64, dtype=torch.float16, device=DEV)
    none = torch.empty(0, dtype=torch.long, device=DEV)
    bb.paged_append_int4(empty, empty, pool, none)
    assert bb.paged_read_int4(pool, none, dtype=torch.float16)[0].shape == (0, 2, 64) and torch.equal(pool, want)


# ------------------------------------------------------------------------------ attention
class Case:
    """Requests of the given lengths over a shuffled pool whose unused bytes are all ones (NaN scales)."""

    def __init__(self, lens, Hq, Hkv, dh=128, page=16, dtype=torch.bfloat16, token_major=False, step=False, seed=0, spare=2, q_scale=1.0,
                 k=None, v=None):
        g = torch.Generator(device=DEV).manual_seed(seed)
        self.host, self.page, self.dh, self.Hq, self.Hkv, self.dtype = list(lens), page, dh, Hq, Hkv, dtype
        B = len(lens)
        n = [-(-x // page) for x in lens]
        P = sum(n) + spare
        ids = torch.randperm(P, generator=g, device=DEV).int()
        width = max(n + [1]) + 1
        self.table = torch.full((B, width), -1, dtype=torch.int32, device=DEV)
        shape = (P, page // 16, Hkv, 18 * dh) if token_major else (P, Hkv, page // 16, 18 * dh)
        self.pool = torch.full(shape, 255, dtype=torch.uint8, device=DEV)
        if token_major:
            self.pool = self.pool.transpose(1, 2)
        self.k, self.v, at = [], [], 0
        for b, ln in enumerate(lens):
            pages = ids[at:at + n[b]]
            at += n[b]
            self.table[b, :n[b]] = pages
            rows = [f(b, ln) if f else _rows(g, Hkv, ln, dh, dtype=dtype) for f in (k, v)]
            if ln:
                full = [torch.cat([x, torch.zeros(Hkv, n[b] * page - ln, dh, dtype=dtype, device=DEV)], 1) for x in rows]
                raw = blocks_of(*(x.unflatten(1, (-1, 16)) for x in full))  # [Hkv, blocks, 18 dh]
                last = raw[:, (ln - 1) // 16]
                for r in range((ln - 1) % 16 + 1, 16):  # tokens past the end hold NaN scales
                    for half in (0, 9 * dh):
                        last[:, half + 8 * dh + r * dh // 16: half + 8 * dh + (r + 1) * dh // 16] = 255
                raw[:, (ln - 1) // 16 + 1:] = 255
                self.pool[pages.long()] = raw.unflatten(1, (n[b], page // 16)).transpose(0, 1)
            self.k.append(rows[0])
            self.v.append(rows[1])
        self.lens = torch.tensor(lens, dtype=torch.int32, device=DEV)
        self.q = (torch.randn(B, Hq, 1, dh, generator=g, device=DEV) * q_scale).to(dtype)
        self.new = {}
        if step:
            kn, vn = (_rows(g, B, Hkv, 1, dh, dtype=dtype) for _ in range(2))
            self.new = {"k_new": kn, "v_new": vn}
            for b, ln in enumerate(lens):  # what the call has to write
                if ln:
                    self.k[b], self.v[b] = (torch.cat([x[:, :-1], y[b]], 1) for x, y in ((self.k[b], kn), (self.v[b], vn)))

    def run(self, **kw):
        return bb.paged_decode_attention_int4(self.q, self.pool, self.table, self.lens, return_lse=True, **self.new, **kw)

    def check(self, got, window=0, scale=None, rows=None):
        out, lse = got
        B, G, dh = len(self.host), self.Hq // self.Hkv, self.dh
        scale = 1 / math.sqrt(dh) if scale is None else scale
        assert out.dtype == self.dtype and out.shape == (B, self.Hq, 1, dh) and lse.shape == (B, self.Hq, 1)
        for b in range(B) if rows is None else rows:
            ln = self.host[b]
            o, ls = out[b, :, 0].double().view(self.Hkv, G, dh), lse[b, :, 0].double().view(self.Hkv, G)
            if ln == 0:
                assert (o == 0).all() and (ls == -math.inf).all()
                continue
            first = max(0, ln - window) if window else 0
            k, v = self.k[b][:, first:], self.v[b][:, first:]
            n = k.shape[1]
            q = self.q[b, :, 0].double().view(self.Hkv, G, dh)
            kv, vv = value(k), value(v)
            z = scale * q @ kv.transpose(1, 2)
            p = torch.softmax(z, -1)
            ref, rl = p @ vv, torch.logsumexp(z, -1)
            c, s, m = pack(k)
            size = (c.double().unflatten(-1, (-1, 64)) * s.double()[..., None] + m.double().abs()[..., None]).flatten(-2)
            S = scale * (q.abs() @ size.transpose(1, 2)).amax(-1, keepdim=True)
            ds = (dh + 10) * 2 ** -23 * S
            c, s, m = pack(v)
            A = p @ (c.double().unflatten(-1, (-1, 64)) * s.double()[..., None] + m.double().abs()[..., None]).flatten(-2)
            bar = U[self.dtype] * ref.abs() + A * (2 * ds + W[self.dtype] + n * 2 ** -23) + n * 2 ** -29 * s.double().amax((1, 2))[:, None, None]
            bad = (o - ref).abs() > bar
            assert not bad.any(), (b, ln, float(((o - ref).abs() / bar).max()))
            assert ((ls - rl).abs() <= ds[..., 0] + 2 ** -20 + n * 2 ** -23 + 2 ** -21 * rl.abs()).all(), b


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dh", [64, 128, 256])
@pytest.mark.parametrize("step", [False, True])
def test_lengths(dtype, dh, step):
    lens = [1, 2, 7, 15, 16, 17, 31, 32, 33, 127, 128, 129, 300, 0 if not step else 1, 1000]
    c = Case(lens, 8, 2, dh=dh, dtype=dtype, step=step, seed=dh)
    c.check(c.run())


@pytest.mark.parametrize("G", [1, 2, 3, 5, 7, 8, 9, 12, 16, 17, 24, 33])
@pytest.mark.parametrize("dh", [64, 128, 256])
def test_head_ratios(G, dh):
    for dtype in DTYPES:
        c = Case([5, 200, 1500], 2 * G, 2, dh=dh, dtype=dtype, step=G % 2 == 0, seed=G)
        c.check(c.run())


@pytest.mark.parametrize("page,token_major", [(16, True), (32, False), (48, True), (64, False), (128, True), (16 * 7, False)])
def test_pages(page, token_major):
    for dh in (64, 128, 256):
        c = Case([3, 333, 64, 2049, 0], 6, 3, dh=dh, page=page, token_major=token_major, seed=page)
        c.check(c.run())


@pytest.mark.parametrize("window", [1, 2, 15, 16, 17, 100, 1000, 5000])
def test_windows(window):
    for dtype in DTYPES:
        c = Case([1, 16, 17, 100, 999, 1000, 1001, 4097, 0], 8, 2, dtype=dtype, seed=window)
        c.check(c.run(window=window), window=window)
    c = Case([1, 16, 300, 2000], 6, 2, dh=64, page=48, step=True, seed=window)
    c.check(c.run(window=window), window=window)


@pytest.mark.parametrize("lens,Hq,Hkv", [([20000], 8, 2), ([131072], 8, 2), ([70001, 3, 0, 12345], 4, 1), ([9000] * 17, 8, 2), ([640] * 64, 2, 2),
                                         ([1300, 1290, 1310, 1281, 1297] * 9, 4, 4), ([100000, 1, 1, 1], 16, 1), ([30000, 29999], 24, 1)])
@pytest.mark.parametrize("dh", [64, 128, 256])
def test_pairs_cut_between_ctas(lens, Hq, Hkv, dh):
    c = Case(lens, Hq, Hkv, dh=dh, page=64, dtype=DTYPES[len(lens) % 2], seed=len(lens))
    first = c.run()
    c.check(first)
    assert all(torch.equal(a, b) for a, b in zip(first, c.run()))  # equal calls, equal bits


@pytest.mark.parametrize("G", [1, 3, 4])
@pytest.mark.parametrize("dh", [64, 128, 256])
def test_granules_without_a_second_one(G, dh):
    """Up to 4 heads take a warp's granules two at a time: odd and even numbers of them, in whole and cut pairs, of
    windows that begin in either one, with the new row in either one."""
    lens = [128 * i + d for i in (0, 1, 2, 3, 7) for d in (1, 16, 17, 33, 127, 128)]
    for case, window in ((lens, 0), (lens, 150), ([20011, 9001, 4999], 0), ([33333], 0), ([33333], 7001)):
        for step in (False, True):
            c = Case(case, 2 * G, 2, dh=dh, step=step, seed=G + dh)
            c.check(c.run(window=window), window=window)


def test_lengths_around_a_cut():
    """One pair just below and above the lengths at which it is cut, and where cuts move to its ends."""
    for ln in list(range(16 * 79, 16 * 84, 16)) + [16 * 127 + 1, 16 * 128, 16 * 161, 16 * 200]:
        c = Case([ln], 4, 1, page=16, seed=ln)
        c.check(c.run())
    for B in (2, 3, 5, 37):
        c = Case([1500 + 97 * i for i in range(B)], 4, 2, page=32, seed=B)
        c.check(c.run())


def test_many_requests():
    lens = [(i * 37) % 90 for i in range(1500)]  # more than are kept in shared memory, empty ones among them
    c = Case(lens, 4, 2, dh=64, seed=1)
    c.check(c.run(), rows=list(range(0, 1500, 13)) + [1023, 1024, 1025, 1499])
    lens = [0] * 1400 + [5000, 0, 3000]
    c = Case(lens, 4, 2, dh=64, seed=2)
    c.check(c.run(), rows=[0, 1399, 1400, 1401, 1402])


def test_new_rows_and_active():
    for dh, G in ((64, 2), (128, 4), (256, 1), (128, 20)):
        lens = [1, 16, 17, 250, 2000]
        c = Case(lens, 2 * G, 2, dh=dh, page=32, step=True, seed=dh + G)
        before = c.pool.clone()
        active = torch.tensor([True, False, True, True, False], device=DEV)
        ref = Case(lens, 2 * G, 2, dh=dh, page=32, step=False, seed=dh + G)
        for b in range(5):
            if not active[b]:
                c.k[b], c.v[b] = ref.k[b], ref.v[b]
        c.check(c.run(active=active))
        pos = [(ln - 1) for ln in lens]
        slots = torch.tensor([int(c.table[b, p // 32]) * 32 + p % 32 if active[b] else -1 for b, p in enumerate(pos)], device=DEV)
        want = _expected(before, c.new["k_new"][:, :, 0], c.new["v_new"][:, :, 0], slots)
        assert torch.equal(c.pool, want)  # the rows an append would write, and nothing else


def test_same_as_append_then_attend():
    c = Case([5, 77, 1030], 8, 2, page=16, step=True, seed=4)
    slots = torch.tensor([int(c.table[b, (n - 1) // 16]) * 16 + (n - 1) % 16 for b, n in enumerate(c.host)], device=DEV)
    pool = c.pool.clone()
    bb.paged_append_int4(c.new["k_new"][:, :, 0], c.new["v_new"][:, :, 0], pool, slots)
    want = bb.paged_decode_attention_int4(c.q, pool, c.table, c.lens, return_lse=True)
    got = c.run()
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and torch.equal(pool, c.pool)


def test_page_numbers_outside_the_pool_read_as_zeros():
    c = Case([100, 500], 4, 2, page=16, seed=6)
    for b, col, bad in ((0, 2, -1), (0, 6, 10 ** 6), (1, 0, 2 ** 31 - 1), (1, 31, -2 ** 31)):
        c.table[b, col] = bad
        c.k[b][:, col * 16:(col + 1) * 16] = 0
        c.v[b][:, col * 16:(col + 1) * 16] = 0
    c.check(c.run())


def test_lengths_are_cut_to_the_table():
    c = Case([64, 48], 4, 2, page=16, seed=6)
    c.table = c.table[:, :4].contiguous()
    c.lens = torch.tensor([1000, -5], dtype=torch.int32, device=DEV)
    c.host[1] = 0
    c.check(c.run())


def test_scale_and_layouts():
    c = Case([100, 333], 8, 2, seed=2)
    c.check(c.run(scale=0.5), scale=0.5)
    c.check(c.run(scale=1e-3), scale=1e-3)
    qs = torch.empty(2, 1, 8, 136, dtype=c.dtype, device=DEV)[..., :128].transpose(1, 2)  # strides of a projection's output
    qs.copy_(c.q)
    want = c.run()
    c.q = qs
    wide = torch.full((2, c.table.shape[1] + 5), -1, dtype=torch.int32, device=DEV)
    wide[:, :c.table.shape[1]] = c.table
    c.table = wide[:, :c.table.shape[1]]
    assert all(torch.equal(a, b) for a, b in zip(want, c.run()))


@pytest.mark.parametrize("dtype", DTYPES)
def test_magnitudes(dtype):
    """Queries, keys and values far from 1, and scales that differ widely between keys."""
    lim = 1e4 if dtype == torch.float16 else 1e20
    for qs, ks, vs in ((1e-3, 1.0, 1e-3), (30.0, 0.3, 50.0), (1e-4, lim ** 0.5, lim / 8), (1.0, 1.0, 2.0 ** -12)):
        g = torch.Generator(device=DEV).manual_seed(8)
        c = Case([700, 40], 8, 2, dtype=dtype, q_scale=qs, k=lambda b, n: _rows(g, 2, n, 128, dtype=dtype, scale=ks),
                 v=lambda b, n: _rows(g, 2, n, 128, dtype=dtype, scale=vs))
        c.check(c.run())

    def varied(b, n):
        x = torch.randn(2, n, 128, generator=g, device=DEV) * torch.exp2(torch.randint(-9, 6, (2, n, 1), generator=g, device=DEV).float())
        return x.to(dtype)

    c = Case([900, 17, 5000], 8, 2, dtype=dtype, v=varied, q_scale=0.5)
    c.check(c.run())
    c = Case([900, 5000], 8, 2, dtype=dtype, v=lambda b, n: (varied(b, n).float() * 0.01 + 7).to(dtype))  # minima far from zero
    c.check(c.run())


def test_a_tail_below_a_dominant_key_keeps_its_weight():
    """One key 14 nats above 60,000 equal ones, which together weigh 5% of it."""
    n = 60000
    for dtype in DTYPES:
        def k(b, ln):
            x = torch.zeros(1, ln, 128, device=DEV)
            x[0, 31, :] = 1.0
            return x.to(dtype)

        def v(b, ln):
            x = torch.ones(1, ln, 128, device=DEV)
            x[0, 31] = 0.0
            x[0, 31, ::2] = 0.25
            x[0, 0] = torch.linspace(0, 2, 128)
            return x.to(dtype)

        c = Case([n], 4, 1, page=128, dtype=dtype, k=k, v=v)
        c.q = torch.full_like(c.q, 14 / 128 * math.sqrt(128))
        c.check(c.run())


def test_queries_far_apart_in_one_head():
    c = Case([300], 4, 1, dtype=torch.bfloat16, seed=3)
    c.q *= torch.exp2(torch.randint(-30, 3, c.q.shape, device=DEV).float()).to(c.dtype)
    c.q[:, 2] = 0
    c.check(c.run())


def test_nan_stays_in_its_head_and_request():
    c = Case([50, 60, 70], 4, 2, seed=5)
    rows = list(range(3))
    c.pool[int(c.table[1, 0]), 1, 0, 8 * 128:8 * 128 + 2] = 255  # a key scale of request 1, head 1
    out, lse = c.run()
    assert torch.isnan(out[1, 2:]).all() and torch.isnan(lse[1, 2:]).all()
    assert torch.isfinite(out[1, :2].float()).all() and torch.isfinite(lse[1, :2]).all()
    del rows[1]
    c.check((out, lse), rows=rows)
    q = c.q.clone()
    c.q[0, 0, 0, 5] = math.nan
    out, lse = c.run()
    assert torch.isnan(out[0, 0]).all() and torch.isnan(lse[0, 0]) and torch.isfinite(out[0, 1:].float()).all()
    c.q = q


# ------------------------------------------------------------------------------ streams, capture, refusals
def test_other_streams_and_shared_workspace():
    a, b = Case([20000, 5], 8, 2, page=64, seed=1), Case([500] * 40, 8, 2, page=64, seed=2)
    want_a, want_b = a.run(), b.run()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    got = []
    for _ in range(20):
        with torch.cuda.stream(s):
            got.append((a.run(), want_a))
        got.append((b.run(), want_b))
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for r, w in got for x, y in zip(r, w))
    ws = paged.decode_workspace()
    for c, w in ((a, want_a), (b, want_b), (a, want_a)):
        assert all(torch.equal(x, y) for x, y in zip(c.run(workspace=ws), w))
    assert (ws[:4096] == 0).all()  # as the 16-bit kernel needs them


def test_captured_calls():
    a, b = Case([20000, 5], 8, 2, page=64, seed=1), Case([20000, 5], 8, 2, page=64, seed=9)
    want_a = [x.clone() for x in a.run()]
    want_b = [x.clone() for x in b.run()]
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(a.run())
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for g, s in zip(graphs, streams):  # side by side
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            for _ in range(5):
                g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for o in outs for x, y in zip(o, want_a))
    a.q.copy_(b.q)
    a.table.copy_(b.table)
    a.pool.copy_(b.pool)
    graphs[1].replay()
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(outs[1], want_b))


def test_refusals():
    c = Case([5, 20], 4, 2)
    ok = dict(q=c.q, kv_pages=c.pool, block_table=c.table, lens=c.lens)

    def call(**kw):
        return bb.paged_decode_attention_int4(**{**ok, **kw})

    call()
    bad = [dict(q=c.q.float()), dict(q=c.q[:, :3]), dict(q=c.q[..., :64]), dict(q=c.q.expand(2, 4, 2, 128)), dict(kv_pages=c.pool.short()),
           dict(kv_pages=c.pool[..., :-16]), dict(kv_pages=c.pool[..., 0]), dict(lens=c.lens.long()), dict(lens=c.lens[:1]),
           dict(block_table=c.table.long()), dict(block_table=c.table[:1]), dict(window=-1), dict(scale=0.0), dict(scale=math.nan),
           dict(k_new=c.q[:, :2]), dict(active=torch.ones(2, dtype=torch.bool, device=DEV)), dict(k_new=c.q, v_new=c.q),
           dict(k_new=c.q[:, :2].half(), v_new=c.q[:, :2].half()), dict(workspace=torch.empty(10, device=DEV)),
           dict(kv_pages=c.pool.cpu()), dict(lens=c.lens.cpu())]
    for kw in bad:
        with pytest.raises(ValueError):
            call(**kw)
    with pytest.raises(RuntimeError):
        call(workspace=torch.empty(4096, dtype=torch.uint8, device=DEV))
    rows = torch.zeros(3, 2, 128, dtype=torch.bfloat16, device=DEV)
    slots = torch.zeros(3, dtype=torch.long, device=DEV)
    for args in ((rows, rows[:2], c.pool, slots), (rows, rows.half(), c.pool, slots), (rows.float(), rows.float(), c.pool, slots),
                 (rows, rows, c.pool, slots.int()), (rows, rows, c.pool, slots[:2]), (rows[:, :1], rows[:, :1], c.pool, slots),
                 (rows[..., :64], rows[..., :64], c.pool, slots), (rows, rows, c.pool[:, :, :, ::2], slots), (rows, rows, c.pool.cpu(), slots)):
        with pytest.raises(ValueError):
            bb.paged_append_int4(*args)
    for kw in (dict(dtype=torch.float32), dict(slot_map=slots.int()), dict(kv_pages=c.pool[..., :100])):
        with pytest.raises(ValueError):
            bb.paged_read_int4(**{**dict(kv_pages=c.pool, slot_map=slots, dtype=torch.bfloat16), **kw})
    torch.cuda.synchronize()


def test_empty_batch():
    c = Case([5], 4, 2)
    out, lse = bb.paged_decode_attention_int4(c.q[:0], c.pool, c.table[:0], c.lens[:0], return_lse=True)
    assert out.shape == (0, 4, 1, 128) and lse.shape == (0, 4, 1)
    c = Case([0, 0], 4, 2)
    c.check(c.run())
