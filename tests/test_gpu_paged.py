"""The paged key/value cache on the GPU: reservation, append and one-token attention.

Whole numbers (tables, slots, the free stack) must equal a restatement with Python lists;
appended rows must be bit-equal.  Attention is compared with float64 arithmetic on the same
16-bit inputs.  Its bars, per element, with u the unit roundoff of the 16-bit type (2^-8 bf16,
2^-11 fp16), n the keys attended to, A = sum_j p_j |v_j| and S = scale * max_j sum_i |q_i k_ji|:
  * a score is an fp32 sum of dh exact products (tensor cores truncate: 2^-23 a step), so it is
    off by ds <= (dh + 4) 2^-23 S;
  * a probability is off by a factor of 1 +- (ds + 2^-21), carried in two 16-bit parts at best:
    u^2 relative, or 2^-25 absolute where the second part is subnormal in fp16; sums over n keys
    add n 2^-23; the result is rounded once:
      |out - ref| <= u |ref| + A (2 ds + 2^-15 + n 2^-23) + n 2^-25 max|v|
  * |lse - ref| <= ds + 2^-20 + n 2^-23 + 2^-21 |ref|
"""
import math

import numpy as np
import pytest
import torch

import butterfly_b200 as bb
from butterfly_b200 import paged

pytestmark = pytest.mark.gpu
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
DEV = "cuda"


# ------------------------------------------------------------------------------ attention
class Case:
    """Requests with the given lengths over a shuffled pool whose unused rows are NaN."""

    def __init__(self, lens, Hq, Hkv, dh=128, page=16, dtype=torch.bfloat16, nhd=False, step=False, seed=0, spare=2,
                 q_scale=1.0):
        g = torch.Generator(device=DEV).manual_seed(seed)
        self.lens_host, self.page, self.dh, self.Hq, self.Hkv = list(lens), page, dh, Hq, Hkv
        B = len(lens)
        n = [-(-x // page) for x in lens]
        P = sum(n) + spare
        ids = torch.randperm(P, generator=g, device=DEV).int()
        width = max(n + [1]) + 1
        self.table = torch.full((B, width), -1, dtype=torch.int32, device=DEV)
        shape = (P, page, Hkv, dh) if nhd else (P, Hkv, page, dh)
        self.kp, self.vp = (torch.full(shape, math.nan, dtype=dtype, device=DEV) for _ in range(2))
        if nhd:
            self.kp, self.vp = self.kp.permute(0, 2, 1, 3), self.vp.permute(0, 2, 1, 3)
        self.k, self.v = [], []
        at = 0
        for b, ln in enumerate(lens):
            rows = ids[at:at + n[b]]
            at += n[b]
            self.table[b, :n[b]] = rows
            k, v = (torch.randn(Hkv, ln, dh, generator=g, device=DEV).to(dtype) for _ in range(2))
            for x, pool in ((k, self.kp), (v, self.vp)):
                for i in range(n[b]):
                    part = x[:, i * page:(i + 1) * page]
                    pool[rows[i], :, :part.shape[1]] = part
            self.k.append(k)
            self.v.append(v)
        self.lens = torch.tensor(lens, dtype=torch.int32, device=DEV)
        self.q = (torch.randn(B, Hq, 1, dh, generator=g, device=DEV) * q_scale).to(dtype)
        self.kn = self.vn = None
        if step:  # the last token of every request is the new one: its pool row is still NaN
            self.kn, self.vn = (torch.randn(B, Hkv, 1, dh, generator=g, device=DEV).to(dtype) for _ in range(2))
            for b, ln in enumerate(lens):
                if ln:
                    self.kp[self.table[b, (ln - 1) // page], :, (ln - 1) % page] = math.nan
                    self.vp[self.table[b, (ln - 1) // page], :, (ln - 1) % page] = math.nan
                    self.k[b][:, -1], self.v[b][:, -1] = self.kn[b, :, 0], self.vn[b, :, 0]

    def run(self, **kw):
        if self.kn is not None:
            kw = dict(k_new=self.kn, v_new=self.vn, **kw)
        return bb.paged_decode_attention(self.q, self.kp, self.vp, self.table, self.lens, return_lse=True, **kw)

    def check(self, out, lse, window=0, scale=None):
        scale = 1 / math.sqrt(self.dh) if scale is None else scale
        u, G = U[self.q.dtype], self.Hq // self.Hkv
        assert out.shape == self.q.shape and out.dtype == self.q.dtype and lse.shape == self.q.shape[:3]
        for b, ln in enumerate(self.lens_host):
            o, l = out[b, :, 0].double(), lse[b, :, 0].double()
            lo = max(0, ln - window) if window else 0
            if ln == lo:
                assert bool((o == 0).all()) and bool((l == -math.inf).all())
                continue
            q = self.q[b, :, 0].double().view(self.Hkv, G, self.dh)
            k, v = self.k[b][:, lo:].double(), self.v[b][:, lo:].double()
            s = q @ k.transpose(1, 2) * scale
            p = torch.softmax(s, -1)
            ref, rl = (p @ v).reshape(self.Hq, self.dh), torch.logsumexp(s, -1).reshape(-1)
            n = ln - lo
            ds = (self.dh + 4) * 2.0 ** -23 * scale * (q.abs() @ k.abs().transpose(1, 2)).amax(-1).reshape(-1, 1)
            A = (p @ v.abs()).reshape(self.Hq, self.dh)
            bar = u * ref.abs() + A * (2 * ds + 2.0 ** -15 + n * 2.0 ** -23) + n * 2.0 ** -25 * float(v.abs().max())
            assert bool(((o - ref).abs() <= bar).all()), (b, ln, float(((o - ref).abs() / bar).max()))
            lbar = ds[:, 0] + 2.0 ** -20 + n * 2.0 ** -23 + 2.0 ** -21 * rl.abs()
            assert bool(((l - rl).abs() <= lbar).all()), (b, ln, float(((l - rl).abs() / lbar).max()))


LENS = [0, 1, 2, 15, 16, 17, 31, 33, 47, 48, 49, 127, 128, 129, 255, 256, 257, 300, 513, 1000]


@pytest.mark.parametrize("Hq,Hkv,dh,page,dtype,nhd", [
    (8, 2, 128, 16, torch.bfloat16, False),
    (16, 4, 128, 128, torch.float16, True),
    (3, 3, 64, 48, torch.float16, False),
    (15, 3, 64, 16, torch.bfloat16, True),
    (4, 2, 256, 32, torch.bfloat16, False),
    (8, 1, 256, 16, torch.float16, True),
])
@pytest.mark.parametrize("step", [False, True])
def test_lengths(Hq, Hkv, dh, page, dtype, nhd, step):
    c = Case(LENS, Hq, Hkv, dh, page, dtype, nhd, step, seed=Hq + dh)
    c.check(*c.run())


@pytest.mark.parametrize("G", [1, 2, 3, 4, 5, 7, 8, 9, 12, 15, 16, 17, 20, 24, 33])
def test_query_heads_per_kv_head(G):
    for dh in (64, 128, 256):
        c = Case([5, 0, 129, 700], 2 * G, 2, dh, 32, seed=G)
        c.check(*c.run())


@pytest.mark.parametrize("window", [1, 2, 15, 16, 17, 64, 100, 255, 256, 1000, 5000])
def test_window(window):
    for step, dtype in ((False, torch.bfloat16), (True, torch.float16)):
        c = Case(LENS + [3001], 8, 2, 128, 48, dtype, seed=window, step=step)
        # pages wholly before the window may have gone: their entries and rows must not matter
        for b, ln in enumerate(c.lens_host):
            gone = max(0, ln - window) // 48
            rows = c.table[b, :gone].long()
            c.kp[rows], c.vp[rows] = math.nan, math.nan
            c.table[b, :gone] = -1
        c.check(*c.run(window=window), window=window)


def test_long_requests_are_split_and_joined():
    for lens, Hq, Hkv, dh in (([40000], 8, 2, 128), ([1, 30011, 0, 513, 9000], 16, 4, 128), ([50001], 2, 1, 64),
                              ([20017, 20], 6, 2, 256), ([12345], 40, 2, 128)):
        c = Case(lens, Hq, Hkv, dh, 64, seed=len(lens))
        first = c.run()
        c.check(*first)
        again = c.run()  # the same call gives the same bits, whatever order the parts arrive in
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


@pytest.mark.parametrize("Hq,Hkv,dh,page,step", [(4, 4, 256, 16, True), (8, 2, 128, 16, False), (12, 6, 64, 48, True)])
def test_many_requests_cut_between_ctas(Hq, Hkv, dh, page, step):
    # adjacent requests that each cross a boundary between CTAs, in different orders
    for seed in range(4):
        lens = np.random.default_rng(seed).permutation(np.geomspace(301, 8191, 24).astype(int)).tolist()
        c = Case(lens, Hq, Hkv, dh, page, seed=seed, step=step)
        for _ in range(2):
            c.check(*c.run())


def test_many_short_requests():
    rng = np.random.default_rng(5)
    lens = rng.integers(0, 90, 1500).tolist()
    c = Case(lens, 4, 1, 128, 16, seed=11, step=True)
    c.check(*c.run())


@pytest.mark.parametrize("q_scale", [0.0, 30.0])
def test_flat_and_peaked_scores(q_scale):
    c = Case([1, 40, 2000], 8, 2, seed=3, q_scale=q_scale)
    c.check(*c.run())


def test_scale_argument_and_lse_optional():
    c = Case([100, 7], 8, 2, seed=4)
    out, lse = c.run(scale=0.03)
    c.check(out, lse, scale=0.03)
    assert torch.equal(out, bb.paged_decode_attention(c.q, c.kp, c.vp, c.table, c.lens, scale=0.03))


def test_row_without_finite_score_and_infinite_values():
    c = Case([40, 40, 40], 4, 2, dtype=torch.float16, seed=5)
    c.q.fill_(1.0)
    c.kp[c.table[0, :3].long()] = -math.inf  # every score of request 0 is -inf
    c.vp[c.table[1, 0].long(), 0, 3, 5] = math.inf  # one value of request 1
    c.kp[c.table[2, 1].long(), 1, 2, 7] = math.nan  # one key of request 2, KV head 1
    out, lse = c.run()
    assert bool((out[0] == 0).all()) and bool((lse[0] == -math.inf).all())
    # (two-part probabilities may turn an infinite value into NaN: not finite is what is promised)
    assert not bool(out[1, :2, 0, 5].isfinite().any()) and bool(out[1, :2, 0, :5].isfinite().all())
    assert bool(out[1, 2:].isfinite().all())
    assert bool(out[2, :2].isfinite().all()) and bool(out[2, 2:].isnan().all()) and bool(lse[2, 2:].isnan().all())


def test_step_writes_the_new_rows_and_nothing_else():
    for nhd in (False, True):
        c = Case([0, 1, 16, 17, 300, 48], 10, 2, 128, 16, nhd=nhd, step=True, seed=6)
        kp, vp = c.kp.clone(), c.vp.clone()
        active = torch.tensor([True, True, False, True, True, False], device=DEV)
        for b in (2, 5):  # requests without a new row attend to what their page holds
            ln = c.lens_host[b]
            old = torch.randn(2, 2, 128, device=DEV).to(c.q.dtype)
            for pool, x, keep in ((kp, old[0], c.k), (vp, old[1], c.v)):
                pool[c.table[b, (ln - 1) // 16], :, (ln - 1) % 16] = x
                keep[b][:, -1] = x
        c.kp.copy_(kp), c.vp.copy_(vp)
        out, lse = c.run(active=active)
        c.check(out, lse)
        for b in (1, 3, 4):
            ln = c.lens_host[b]
            kp[c.table[b, (ln - 1) // 16], :, (ln - 1) % 16] = c.kn[b, :, 0]
            vp[c.table[b, (ln - 1) // 16], :, (ln - 1) % 16] = c.vn[b, :, 0]
        assert torch.equal(c.kp.view(torch.int16), kp.view(torch.int16))
        assert torch.equal(c.vp.view(torch.int16), vp.view(torch.int16))


def test_strides_shared_pages_and_other_streams():
    c = Case([200, 33, 64], 8, 2, 128, 16, seed=7)
    ref = c.run()
    c.check(*ref)
    # q inside a merged projection, keys and values interleaved in one allocation, a wider table
    wide = torch.randn(3, 1, 8, 3 * 128, device=DEV).to(c.q.dtype)
    q = wide[..., 128:256].transpose(1, 2)
    q.copy_(c.q)
    both = torch.empty(c.kp.shape[0], 16, 2, 2, 128, device=DEV, dtype=c.q.dtype)
    kp, vp = both[:, :, 0].transpose(1, 2), both[:, :, 1].transpose(1, 2)
    kp.copy_(c.kp), vp.copy_(c.vp)
    table = torch.full((3, 100), 12345678, dtype=torch.int32, device=DEV)[:, 3:90]
    table[:, :c.table.shape[1]] = c.table
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = bb.paged_decode_attention(q, kp, vp, table, c.lens, return_lse=True)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got[0], ref[0]) and torch.equal(got[1], ref[1])
    # a prefix shared by two requests: same pages, same answers
    c.table[1, :2], c.lens[1] = c.table[0, :2], 32
    q = c.q[:1].expand(3, 8, 1, 128).contiguous()
    out = bb.paged_decode_attention(q, c.kp, c.vp, c.table, torch.tensor([32, 32, 64], dtype=torch.int32, device=DEV))
    assert torch.equal(out[0], out[1])


def test_overlong_lengths_and_page_numbers_outside_the_pool_stay_inside():
    c = Case([40, 33], 4, 2, seed=8)
    c.vp.nan_to_num_(0), c.kp.nan_to_num_(0)
    width = c.table.shape[1]  # 4 entries: the fourth is -1 and reads as zeros
    c.table[1, 1] = 1 << 20
    lens = torch.tensor([10 ** 9, 33], dtype=torch.int32, device=DEV)
    out, lse = bb.paged_decode_attention(c.q, c.kp, c.vp, c.table, lens, return_lse=True)
    zeros = lambda x: torch.nn.functional.pad(x, (0, 0, 0, 64 - x.shape[1]))  # noqa: E731
    assert width == 4
    c.k[0], c.v[0] = zeros(c.k[0]), zeros(c.v[0])
    c.k[1][:, 16:32], c.v[1][:, 16:32] = 0, 0
    c.lens_host = [64, 33]
    c.check(out, lse)


def test_pool_past_32_bit_offsets():
    # 2.2e9 elements (4.4 GB) a pool: byte and element offsets of the last pages pass 32 bits
    page, Hkv, dh = 128, 2, 128
    P = (2 ** 31 + 2 ** 26) // (page * Hkv * dh)
    kp, vp = (torch.empty(P, Hkv, page, dh, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    c = Case([300, 128], 8, Hkv, dh, page, seed=9, spare=0)
    far = torch.arange(P - c.kp.shape[0], P, device=DEV)
    k = torch.cat([c.k[0], c.k[1]], 1).transpose(0, 1)
    v = torch.cat([c.v[0], c.v[1]], 1).transpose(0, 1)
    c.table = torch.where(c.table >= 0, far[c.table.clamp(min=0).long()].int(), -1)
    pos = torch.cat([torch.arange(300), torch.arange(128)]).to(DEV)
    row = torch.cat([torch.zeros(300, dtype=torch.long), torch.ones(128, dtype=torch.long)]).to(DEV)
    slots = c.table[row, pos // page].long() * page + pos % page
    assert int(slots.max()) * Hkv * dh > 2 ** 31
    bb.paged_append(k, v, kp, vp, slots)
    c.kp, c.vp = kp, vp
    c.check(*c.run())


def test_graph_capture_replays():
    c = Case([70, 1000, 16], 8, 2, seed=10, step=True)
    want = c.run()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = c.run()
    for _ in range(3):
        g.replay()
    torch.cuda.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_cache_step_in_a_graph():
    # reservation and both layers' attention captured; each replay starts from the captured lengths
    cache = bb.PagedKVCache(num_layers=2, num_pages=40, page_size=16, num_kv_heads=2, head_dim=128, max_requests=3,
                            max_tokens_per_request=256)
    g = torch.Generator(device=DEV).manual_seed(2)
    rnd = lambda *s: torch.randn(*s, generator=g, device=DEV).bfloat16()  # noqa: E731
    r = cache.reserve([30, 200, 16])
    for layer in range(2):
        cache.append(layer, rnd(246, 2, 128), rnd(246, 2, 128), r.slot_map)
    q, kn, vn, add = rnd(3, 8, 1, 128), rnd(3, 2, 1, 128), rnd(3, 2, 1, 128), torch.ones(3, dtype=torch.int32, device=DEV)
    lens, num_free = cache.lens, cache.num_free

    def step():
        cache.lens, cache.num_free = lens, num_free
        r = cache.reserve(add, 3)
        return [cache.attend(layer, q, k_new=kn, v_new=vn, active=r.granted) for layer in range(2)] + [r.lens, r.slot_map]

    want = [x.clone() for x in step()]
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        got = step()
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and got[2].tolist() == [31, 201, 17]


def test_empty_batch():
    c = Case([5], 8, 2, seed=1)
    out, lse = bb.paged_decode_attention(c.q[:0], c.kp, c.vp, c.table[:0], c.lens[:0], return_lse=True)
    assert out.shape == (0, 8, 1, 128) and lse.shape == (0, 8, 1)


# ------------------------------------------------------------------------------ append
@pytest.mark.parametrize("T,Hkv,dh,page,dtype,nhd", [
    (1, 2, 128, 16, torch.bfloat16, False), (7, 1, 64, 48, torch.float16, True), (1000, 3, 256, 32, torch.bfloat16, True),
    (4099, 2, 128, 128, torch.float16, False), (64, 8, 64, 16, torch.bfloat16, False),
])
def test_append(T, Hkv, dh, page, dtype, nhd):
    g = torch.Generator(device=DEV).manual_seed(T)
    P = -(-T // page) + 2
    shape = (P, page, Hkv, dh) if nhd else (P, Hkv, page, dh)
    kp, vp = (torch.randn(shape, generator=g, device=DEV).to(dtype) for _ in range(2))
    if nhd:
        kp, vp = kp.permute(0, 2, 1, 3), vp.permute(0, 2, 1, 3)
    merged = torch.randn(T, 2 * Hkv + 1, dh, generator=g, device=DEV).to(dtype)
    k, v = merged[:, :Hkv], merged[:, Hkv + 1:]
    slots = torch.randperm(P * page, generator=g, device=DEV)[:T]
    slots[torch.rand(T, generator=g, device=DEV) < 0.2] = -1
    if T > 5:
        slots[3], slots[4] = P * page, 2 ** 40  # outside the pool: skipped
    rk, rv = kp.clone(), vp.clone()
    ok = (slots >= 0) & (slots < P * page)
    rk[slots[ok] // page, :, slots[ok] % page] = k[ok]
    rv[slots[ok] // page, :, slots[ok] % page] = v[ok]
    bb.paged_append(k, v, kp, vp, slots)
    assert torch.equal(kp, rk) and torch.equal(vp, rv)
    # head-major rows [Hkv, T, dh], as an attention layer holds them
    kp.zero_(), vp.zero_()
    rk.zero_(), rv.zero_()
    rk[slots[ok] // page, :, slots[ok] % page] = v[ok]
    rv[slots[ok] // page, :, slots[ok] % page] = k[ok]
    hm = [x.transpose(0, 1).contiguous().transpose(0, 1) for x in (v, k)]
    bb.paged_append(hm[0], hm[1], kp, vp, slots)
    assert torch.equal(kp, rk) and torch.equal(vp, rv)


def test_append_nothing():
    kp = torch.zeros(2, 2, 16, 128, dtype=torch.bfloat16, device=DEV)
    x = torch.ones(0, 2, 128, dtype=torch.bfloat16, device=DEV)
    bb.paged_append(x, x, kp, kp.clone(), torch.empty(0, dtype=torch.int64, device=DEV))
    assert float(kp.abs().max()) == 0


# ------------------------------------------------------------------------------ reserve
def _pages(n, page):
    return -(-n // page)


class Model:
    """The cache's bookkeeping with Python lists."""

    def __init__(self, B, pages, width, page):
        self.page, self.width = page, width
        self.lens, self.rows, self.stack = [0] * B, [[] for _ in range(B)], list(range(pages - 1, -1, -1))

    def reserve(self, add):
        page, back = self.page, []
        for b, a in enumerate(add):
            if a < 0:
                keep = _pages(max(0, self.lens[b] + a), page)
                back += self.rows[b][keep:]
                self.rows[b] = self.rows[b][:keep]
                self.lens[b] = max(0, self.lens[b] + a)
        self.stack += back[::-1]
        room, asked, slots, positions, granted = len(self.stack), 0, [], [], []
        for b, a in enumerate(add):
            if a <= 0:
                granted.append(False)
                continue
            need = _pages(self.lens[b] + a, page) - _pages(self.lens[b], page)
            ok = _pages(self.lens[b] + a, page) <= self.width
            if ok and need:
                asked += need
                ok = asked <= room
            granted.append(ok)
            pos = range(self.lens[b], self.lens[b] + a)
            if ok:
                self.rows[b] += [self.stack.pop() for _ in range(need)]
                self.lens[b] += a
            slots += [self.rows[b][p // page] * page + p % page if ok else -1 for p in pos]
            positions += [p if ok else -1 for p in pos]
        return slots, positions, granted


def _same(cache, model, r, want, extra):
    slots, positions, granted = want
    assert r.slot_map.tolist() == slots + [-1] * extra
    assert r.positions.tolist() == positions + [-1] * extra
    assert r.granted.tolist() == granted
    assert cache.lens.tolist() == model.lens
    n = int(cache.num_free)
    assert n == len(model.stack) and cache.free_pages[:n].tolist() == model.stack
    table = cache.block_table.tolist()
    for b, row in enumerate(model.rows):
        assert table[b][:len(row)] == row, b


@pytest.mark.parametrize("B,pages,page,width", [(1, 9, 16, 7), (5, 40, 16, 12), (64, 300, 32, 9), (300, 700, 48, 5),
                                                (4096, 5000, 16, 4)])
def test_reserve_follows_the_model(B, pages, page, width):
    rng = np.random.default_rng(B)
    cache = bb.PagedKVCache(num_layers=1, num_pages=pages, page_size=page, num_kv_heads=1, head_dim=64, max_requests=B,
                            max_tokens_per_request=width * page)
    model = Model(B, pages, width, page)
    for step in range(12):
        kind = rng.random(B)
        add = np.where(kind < 0.3, 1, np.where(kind < 0.6, rng.integers(0, 2 * page, B), 0))
        add = np.where((kind > 0.8) & (step % 3 == 2), rng.integers(-3 * page, 1, B), add)
        add = np.where(kind > 0.95, paged.RELEASE, add).tolist()
        if step == 7:
            add[-1] = width * page + 1  # can never fit
        extra = int(rng.integers(0, 5))
        want = model.reserve(add)
        total = sum(max(a, 0) for a in add)
        r = cache.reserve(torch.tensor(add, dtype=torch.int32, device=DEV), total + extra)
        _same(cache, model, r, want, extra)
    owned = [p for row in model.rows for p in row] + model.stack
    assert sorted(owned) == list(range(pages))  # no page lost, none owned twice


def test_reserve_many_tokens():
    # prompts of all lengths, some ending inside a page, and more tokens than entries of one CTA
    rng = np.random.default_rng(3)
    for B, extra, start in ((70, 0, 0), (3, 5, 37), (2000, 3, 1)):
        add = rng.integers(0, 160000 // B, B).tolist()
        add[1] = 0
        pages = sum(_pages(a + start, 16) for a in add) - 2
        cache = bb.PagedKVCache(num_layers=1, num_pages=pages + B, page_size=16, num_kv_heads=1, head_dim=64, max_requests=B,
                                max_tokens_per_request=max(add) + 64)
        model = Model(B, pages + B, -(-(max(add) + 64) // 16), 16)
        if start:
            first = [start] * B
            _same(cache, model, cache.reserve(first), model.reserve(first), 0)
        want = model.reserve(add)
        r = cache.reserve(torch.tensor(add, dtype=torch.int32, device=DEV), sum(add) + extra)
        _same(cache, model, r, want, extra)


def test_reserve_then_rollback_is_the_identity():
    cache = bb.PagedKVCache(num_layers=1, num_pages=64, page_size=16, num_kv_heads=1, head_dim=64, max_requests=4,
                            max_tokens_per_request=512)
    cache.reserve([100, 0, 37, 16])
    before = (cache.lens.clone(), cache.num_free.clone(), cache.free_pages.clone())
    cache.reserve([29, 300, 1, 16])
    cache.reserve([-29, -300, -1, -16])
    assert all(torch.equal(a, b) for a, b in zip(before, (cache.lens, cache.num_free, cache.free_pages)))


def test_reserve_without_requests():
    none = torch.empty(0, dtype=torch.int32, device=DEV)
    free = torch.arange(5, dtype=torch.int32, device=DEV)
    r = bb.paged_reserve(none, none, torch.empty(0, 3, dtype=torch.int32, device=DEV), free, free[4:], page_size=16, num_tokens=0)
    assert r.num_free.tolist() == [4] and all(x.numel() == 0 for x in (r.lens, r.slot_map, r.positions, r.granted))


def test_reserve_does_not_change_its_inputs_and_repeats():
    lens = torch.tensor([5, 20], dtype=torch.int32, device=DEV)
    add = torch.tensor([40, -20], dtype=torch.int32, device=DEV)
    table = torch.tensor([[3, -1, -1], [0, 2, -1]], dtype=torch.int32, device=DEV)
    free = torch.tensor([1, 4, -1, -1, -1], dtype=torch.int32, device=DEV)
    num = torch.tensor([2], dtype=torch.int32, device=DEV)
    one = bb.paged_reserve(lens, add, table, free, num, page_size=16, num_tokens=40)
    two = bb.paged_reserve(lens, add, table, free, num, page_size=16, num_tokens=40)
    assert lens.tolist() == [5, 20] and num.tolist() == [2]
    assert all(torch.equal(a, b) for a, b in zip(one, two))
    # pages 0 and 2 go back on the stack, the first of them on top, and are taken again
    assert table[0].tolist() == [3, 0, 2] and one.lens.tolist() == [45, 0] and one.num_free.tolist() == [2]


# ------------------------------------------------------------------------------ the cache
def test_cache_serves_requests_that_come_and_go():
    """Reserve, append and attend over several steps, against attention over each request's rows."""
    page, Hq, Hkv, dh, R = 16, 8, 2, 128, 4
    cache = bb.PagedKVCache(num_layers=2, num_pages=40, page_size=page, num_kv_heads=Hkv, head_dim=dh, max_requests=R,
                            max_tokens_per_request=320)
    g = torch.Generator(device=DEV).manual_seed(1)
    rnd = lambda *s: torch.randn(*s, generator=g, device=DEV).bfloat16()  # noqa: E731
    hist = [[(rnd(Hkv, 0, dh), rnd(Hkv, 0, dh)) for _ in range(R)] for _ in range(2)]
    for step, prompts in enumerate([[37, 0, 5, 0], [0, 200, 0, 1], [0, 0, 0, 0], [0, 0, 64, 0], [0, 0, 0, 0]]):
        if step == 3:
            cache.release([2])
            for layer in range(2):
                hist[layer][2] = (rnd(Hkv, 0, dh), rnd(Hkv, 0, dh))
        r = cache.reserve(prompts)
        if sum(prompts):
            for layer in range(2):
                k, v = rnd(sum(prompts), Hkv, dh), rnd(sum(prompts), Hkv, dh)
                cache.append(layer, k, v, r.slot_map)
                at = 0
                for b, n in enumerate(prompts):
                    hist[layer][b] = tuple(torch.cat([h, x[at:at + n].transpose(0, 1)], 1) for h, x in zip(hist[layer][b], (k, v)))
                    at += n
        live = [int(h[0].shape[1] > 0) for h in hist[0]]
        r = cache.reserve(live)
        assert r.granted.tolist() == [bool(x) for x in live]
        for layer in range(2):
            q, kn, vn = rnd(R, Hq, 1, dh), rnd(R, Hkv, 1, dh), rnd(R, Hkv, 1, dh)
            out, lse = cache.attend(layer, q, k_new=kn, v_new=vn, active=r.granted, return_lse=True)
            c = Case([0] * R, Hq, Hkv, dh, page)
            for b in range(R):
                if live[b]:
                    hist[layer][b] = tuple(torch.cat([h, x[b]], 1) for h, x in zip(hist[layer][b], (kn, vn)))
            c.q, c.k, c.v = q, [h[0] for h in hist[layer]], [h[1] for h in hist[layer]]
            c.lens_host = [int(k.shape[1]) for k in c.k]
            assert cache.lens.tolist() == c.lens_host
            c.check(out, lse)
