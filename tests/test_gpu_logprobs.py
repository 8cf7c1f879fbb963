"""Token log probabilities, entropies and likeliest alternatives on the GPU, against float64 on the same logits.

Bars, per row of V entries, M their maximum, p their softmax, A = sum p |x - M| and n = V / 512 + 24 additions in a
row of fp32 sums (512 threads or more share a row; 24 covers the trees after them):
  * a term e^(x - ref) is off by a factor of 1 +- (2^-22 (the exponential) + 2^-23 |x - ref|), and the reference
    lies 8 below M at most, so Z is off by dz <= 2^-22 + 2^-23 (A + 8) + n 2^-24 relative
  * |logprob - its value| <= dz + 2^-22 (|x - M| + 8 + log V)
  * W = sum (x - ref) e^(x - ref) is off by 2 dz (A + 8) Z at most, so
    |entropy - its value| <= 3 dz (A + 9) + 2^-22 log V
Ids must be equal: largest first, of equal ones the lowest index.
"""
import math

import pytest
import torch

import butterfly_b200 as bb

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def _rand(*shape, dtype="bf16", seed=0, scale=3.0, pad=0, offset=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    V = shape[-1]
    x = (torch.randn(*shape[:-1], V + pad + offset, generator=g, device=DEV) * scale).to(TYPES[dtype])
    return x[..., offset:offset + V]


def check(x, tokens=None, k=0, got=None):
    V = x.shape[-1]
    r = bb.token_logprobs(x, tokens, top_k=k) if got is None else got
    assert r.entropy.shape == x.shape[:-1] and r.top_ids.shape == (*x.shape[:-1], k) == r.top_logprobs.shape
    d = x.double().reshape(-1, V)
    logp = torch.log_softmax(d, -1)
    logp = torch.where(logp < -torch.finfo(torch.float32).max, -math.inf, logp)  # (what fp32 results can hold)
    p = logp.exp()
    M = d.max(-1, keepdim=True).values
    A = torch.where(p > 0, p * (d - M).abs(), 0).sum(-1)
    dz = 2 ** -22 + 2 ** -23 * (A + 8) + (V / 512 + 24) * 2 ** -24
    ent = -torch.where(p > 0, p * logp, 0).sum(-1)
    assert ((r.entropy.reshape(-1) - ent).abs() <= 3 * dz * (A + 9) + 2 ** -22 * math.log(V)).all()

    def bar(v):  # for the log probability of an entry of value v
        return dz[:, None] + 2 ** -22 * ((v - M).abs() + 8 + math.log(V))

    if tokens is None:
        assert r.logprobs is None
    else:
        assert r.logprobs.shape == tokens.shape
        t = tokens.long().reshape(-1, 1)
        at = t.clamp(0, V - 1)
        want = logp.gather(1, at)
        lp = r.logprobs.double().reshape(-1, 1)
        inside = (t >= 0) & (t < V) & (want > -math.inf)
        assert torch.where(inside, (lp - want).abs() <= bar(d.gather(1, at)), True).all()
        assert (lp[t < 0] == 0).all() and (lp[(t >= V) | ((t >= 0) & (want == -math.inf))] == -math.inf).all()
    if k:
        ids = torch.sort(d, dim=-1, descending=True, stable=True).indices[:, :k]
        assert torch.equal(r.top_ids.reshape(-1, k), ids)
        want = logp.gather(1, ids)
        lp = r.top_logprobs.double().reshape(-1, k)
        assert torch.where(want > -math.inf, (lp - want).abs() <= bar(d.gather(1, ids)), lp == want).all()
    return r


def _tokens(x, seed=1, dtype=torch.int64):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randint(0, x.shape[-1], x.shape[:-1], generator=g, device=DEV, dtype=dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [1, 2, 7, 8, 33, 1000, 4097, 32003, 151936])
def test_sizes(V, dtype):
    for rows in (1, 3, 40, 170):
        x = _rand(rows, V, dtype=dtype, seed=V + rows)
        check(x, _tokens(x), min(V, 20))


@pytest.mark.parametrize("rows,V", [(149, 5000), (900, 1000), (3000, 77), (1200, 20011)])
def test_many_rows(rows, V):
    for dtype in TYPES:
        x = _rand(rows, V, dtype=dtype, seed=rows)
        check(x, _tokens(x), 20)


@pytest.mark.parametrize("dtype", TYPES)
def test_row_starts_and_strides(dtype):
    for pad in range(9):
        for offset in (0, 1, 3):
            for V in (257, 9001):
                x = _rand(5, V, dtype=dtype, pad=pad, offset=offset, seed=pad)
                check(x, _tokens(x), 5)


@pytest.mark.parametrize("k", [0, 1, 2, 31, 32, 33, 63, 64])
def test_numbers_of_alternatives(k):
    for rows, V in ((2, 5000), (300, 700), (1, 64)):
        x = _rand(rows, V, seed=k)
        check(x, _tokens(x), k)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [1, 30, 200])
def test_ties_and_orders(rows, dtype):
    t = TYPES[dtype]
    V = 20011
    up = torch.linspace(-9, 9, V, device=DEV).to(t)
    few = (_rand(V, dtype="f32", seed=4) * 0.4).round().to(t)  # a handful of values
    for row in (torch.zeros(V, device=DEV, dtype=t), up, up.flip(0), few, -few.abs(), torch.full((V,), -50.0, device=DEV, dtype=t)):
        x = row.repeat(rows, 1)
        check(x, _tokens(x), 64)
    signed = torch.zeros(rows, 999, device=DEV, dtype=t)
    signed[:, ::3] = -0.0  # ties with 0
    check(signed, _tokens(signed), 64)


def test_more_entries_above_the_bound_than_the_list_holds():
    """512 threads in 64 groups: one thread of each group but the last holds only large entries, so
    that the least of the groups' largest lets all of those through."""
    for rows in (1, 160):
        V = 151936
        x = _rand(rows, V, seed=9) * 0.1
        thread = torch.arange(V, device=DEV) // 8 % 512
        big = (thread % 8 == 3) & (thread < 504)
        x[:, big] = _rand(rows, int(big.sum()), seed=10).abs() + 5
        check(x, _tokens(x), 64)


@pytest.mark.parametrize("dtype", TYPES)
def test_masked_entries(dtype):
    for V in (100, 30000):
        x = _rand(160, V, dtype=dtype).clone()
        x[0] = -math.inf  # no distribution
        x[1] = -math.inf
        x[1, V // 2] = -3.0  # one entry
        x[2, 1:] = -math.inf
        x[3, V // 3:] = -math.inf
        x[4] = torch.finfo(x.dtype).min  # the type's lowest value is a value
        x[5, ::2] = torch.finfo(x.dtype).min
        tok = _tokens(x)
        check(x[1:], tok[1:], min(V, 64))
        for rows in (1, 160):
            r = bb.token_logprobs(x[:rows], tok[:rows], top_k=4)
            assert r.logprobs[0] == -math.inf and r.entropy[0] == 0
            assert (r.top_logprobs[0] == -math.inf).all() and r.top_ids[0].tolist() == [0, 1, 2, 3]


@pytest.mark.parametrize("value", [math.nan, math.inf])
def test_nan_and_infinity_stay_in_their_row(value):
    for rows in (3, 400):
        x = _rand(rows, 5003)
        clean = x.clone()
        x = x.clone()
        x[1, 77] = value
        r = bb.token_logprobs(x, _tokens(x), top_k=10)
        assert torch.isnan(r.logprobs[1]) and torch.isnan(r.entropy[1])
        assert sorted(set(r.top_ids[1].tolist())) == sorted(r.top_ids[1].tolist()) and int(r.top_ids[1].max()) < 5003
        if math.isnan(value):
            masked = clean[1].clone()
            masked[77] = -math.inf
            assert torch.equal(r.top_ids[1], torch.sort(masked.double(), descending=True, stable=True).indices[:10])
        keep = [i for i in range(rows) if i != 1]
        check(clean[keep], _tokens(x)[keep], 10, got=bb.TokenLogprobs(*(y[keep] for y in r)))


def test_large_and_small_logits():
    for scale, shift in ((300.0, 0.0), (1e-3, 0.0), (5.0, 2000.0), (5.0, -2000.0)):
        x = _rand(7, 12345, dtype="f32", scale=scale) + shift
        check(x, _tokens(x), 20)


@pytest.mark.parametrize("dtype", TYPES)
def test_entries_at_the_ends_of_the_range(dtype):
    fi = torch.finfo(TYPES[dtype])
    for rows in (1, 200):
        x = _rand(rows, 9001, dtype=dtype).clone()
        x[:, ::7] = -math.inf
        x[:, 1::7] = fi.min
        x[:, 2::7] = fi.min / 2
        check(x, _tokens(x), 20)
        x[:, 40] = fi.max  # beside masked entries and the lowest ones
        x[:, 51] = fi.max
        check(x, _tokens(x), 20)
        low = torch.full_like(x, fi.min)
        low[:, 5::9] = -math.inf
        low[:, 17] = fi.min * (1 - 2 * fi.eps)
        check(low, _tokens(low), 20)
        check((low.double() / 2).to(x.dtype), _tokens(low), 20)


def test_tokens():
    x = _rand(50, 3001)
    tok = _tokens(x)
    tok[::7] = -100
    tok[3], tok[4] = 3001, 2 ** 40
    check(x, tok, 3)
    tok[4] = 5
    check(x, tok.int(), 0)
    check(x, None, 5)
    assert bb.token_logprobs(x, tok[:, None].expand(50, 2)[:, 1]).logprobs.shape == (50,)  # any strides


def test_leading_shapes():
    x = _rand(4, 9, 777)
    ids = _tokens(x)
    check(x, ids, 5)
    check(x[:, :-1], ids[:, 1:], 5)        # a prompt's tokens: the rows of each sequence but its last
    check(x.transpose(0, 1), ids.T, 5)
    check(x[:, 2], ids[:, 2], 5)
    check(x[1, 2], ids[1, 2], 5)           # one row
    check(x[:1].expand(3, 9, 777), ids[:3], 2)
    y = _rand(2, 3, 2, 5, 40)
    check(y, _tokens(y), 2)
    check(y[:, :, :, 1:], _tokens(y)[:, :, :, 1:], 2)
    for shape in ((0, 77), (3, 0, 77)):
        r = bb.token_logprobs(torch.empty(shape, device=DEV), torch.empty(shape[:-1], device=DEV, dtype=torch.long), top_k=2)
        assert r.logprobs.shape == shape[:-1] and r.top_ids.shape == (*shape[:-1], 2)


def test_rows_further_apart_than_32_bits():
    buf = torch.empty(2 ** 31 + 5000, dtype=torch.bfloat16, device=DEV)
    x = buf.as_strided((2, 4099), (2 ** 31 + 8, 1))
    x.copy_(_rand(2, 4099))
    check(x, _tokens(x), 8)


def test_refusals():
    x = _rand(6, 100)
    tok = _tokens(x)
    with pytest.raises(ValueError, match="CUDA"):
        bb.token_logprobs(x.cpu(), tok.cpu())
    with pytest.raises(ValueError):
        bb.token_logprobs(x, tok.cpu())
    for bad in (x.double(), x.long(), x.t()):
        with pytest.raises(ValueError):
            bb.token_logprobs(bad)
    for t in (tok[:5], tok[:, None], tok.float()):
        with pytest.raises(ValueError):
            bb.token_logprobs(x, t)
    for k in (-1, 65, 101):
        with pytest.raises(ValueError):
            bb.token_logprobs(x, top_k=k)
    with pytest.raises(ValueError):
        bb.token_logprobs(x[:, :10], top_k=11)
    with pytest.raises(ValueError):
        bb.token_logprobs(x[:, :0])
    with pytest.raises(ValueError, match="strided"):
        bb.token_logprobs(_rand(4, 5, 6, 50)[:, ::2, ::2])
    with pytest.raises(TypeError):
        bb.token_logprobs([1.0])


def test_streams_capture_and_equal_bits():
    x, y = _rand(8, 151936, seed=1), _rand(8, 151936, seed=2)
    tok = _tokens(x)
    want_x, want_y = check(x, tok, 20), check(y, tok, 20)
    other = torch.cuda.Stream()
    other.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(other):
        on_other = [bb.token_logprobs(x, tok, top_k=20) for _ in range(20)]
    here = [bb.token_logprobs(y, tok, top_k=20) for _ in range(20)]
    torch.cuda.synchronize()
    for got, want in [(r, want_x) for r in on_other] + [(r, want_y) for r in here]:
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    buf = x.clone()
    graphs, results = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            results.append(bb.token_logprobs(buf, tok, top_k=20))
        graphs.append(g)
    buf.copy_(y)
    for g in graphs:
        g.replay()
    torch.cuda.synchronize()
    for got in results:
        assert all(torch.equal(a, b) for a, b in zip(got, want_y))


def test_under_grad_and_inference_mode():
    x = _rand(3, 500, dtype="f32").requires_grad_()
    r = bb.token_logprobs(x * 1.0, _tokens(x), top_k=3)
    assert not r.logprobs.requires_grad and not r.entropy.requires_grad
    with torch.inference_mode():
        i = bb.token_logprobs(x.detach(), _tokens(x), top_k=3)
    assert torch.equal(r.logprobs, i.logprobs) and torch.equal(r.top_ids, i.top_ids)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V,k", [(1, 1), (2, 2), (31, 31), (32, 32), (33, 33), (64, 64), (65, 64), (257, 50), (513, 33), (1016, 20), (1017, 64), (1018, 64),
                                 (1021, 1), (1022, 5), (1024, 64), (1030, 64)])
def test_short_rows(V, k, dtype):
    """Rows that a warp holds, up to where they end being short, that begin at every place of a 16-byte vector."""
    for offset in range(0, 8, 3 if V > 100 else 1):
        x = _rand(37, V, dtype=dtype, seed=V + offset, pad=5, offset=offset)
        check(x, _tokens(x), k=k)
    x = _rand(4099, V, dtype=dtype, seed=V)
    check(x, _tokens(x, dtype=torch.int32), k=min(k, 7))
    check(x[:, :], None, k=0)


@pytest.mark.parametrize("dtype", TYPES)
def test_short_rows_with_ties_and_masks(dtype):
    t = TYPES[dtype]
    for V in (40, 64, 200, 1000):
        k = min(V, 64)
        x = _rand(24, V, dtype=dtype, seed=V)
        x[0] = 1.5                                            # all equal
        x[1] = torch.arange(V, device=DEV).to(t)              # ascending
        x[2] = -torch.arange(V, device=DEV).to(t)             # descending
        x[3] = (torch.arange(V, device=DEV) % 3).to(t)        # three values
        x[4, 1::2] = -math.inf                                # masks by either kind of lowest value
        x[5, 3:] = -math.inf
        x[6, ::2] = torch.finfo(t).min
        x[7, :-1] = torch.finfo(t).min
        x[8] = 0.0
        x[8, ::2] = -0.0                                      # zeros of both signs are equal
        x[9, V // 2] = torch.finfo(t).max / 4
        x[10] = torch.finfo(t).tiny * (torch.arange(V, device=DEV) % 5).to(t)
        check(x, _tokens(x), k=k)
    y = _rand(6, 100, dtype=dtype, seed=5)
    y[0] = -math.inf
    y[1, 7] = math.nan
    y[2, 9] = math.inf
    y[3] = math.nan
    r = bb.token_logprobs(y, _tokens(y), top_k=30)
    assert r.logprobs[0] == -math.inf and r.entropy[0] == 0 and (r.top_logprobs[0] == -math.inf).all()
    assert torch.equal(r.top_ids[0], torch.arange(30, device=DEV)) and torch.equal(r.top_ids[3], r.top_ids[0])
    assert r.logprobs[1:4].isnan().all() and r.entropy[1:4].isnan().all() and r.top_logprobs[1:4].isnan().all()
    assert r.top_ids[2, 0] == 9 and not (r.top_ids[1] == 7).any()
    check(y[4:], _tokens(y[4:]), k=30)
    assert all(torch.equal(a, b) for a, b in zip((z[4:] for z in bb.token_logprobs(y, _tokens(y), top_k=30)[1:]),
                                                 (z[4:] for z in r[1:])))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V,R", [(1100, 500), (4233, 37), (5000, 3), (30011, 2), (151936, 3), (151936, 200)])
def test_many_entries_that_reach_the_bound(V, R, dtype):
    """Long masked ends, rows in order and rows of few values: whole groups of threads with nothing large, so that far
    more entries than are asked for reach the first bound."""
    t = TYPES[dtype]
    x = _rand(R, V, dtype=dtype, seed=V)
    x[:, V - V // 7:] = -math.inf
    x[0, : V // 3] = torch.finfo(t).min
    x[1] = torch.linspace(-50, 50, V, device=DEV).to(t)
    x[-1] = torch.linspace(9, -9, V, device=DEV).to(t)
    if R > 3:
        x[2, 20:] = -math.inf
        x[3] = 0.25
        x[4] = (torch.arange(V, device=DEV) % 7).to(t)
        x[5, : V - 70] = -math.inf
    for k in (64, 33, 5):
        tokens = _tokens(x)
        r = bb.token_logprobs(x, tokens, top_k=k)
        some = (x > -math.inf).any(-1)  # (a plain log softmax has no value for a row of masks alone)
        check(x[some], tokens[some], k=k, got=type(r)(*(y[some] for y in r)))
        assert (r.logprobs[~some] == -math.inf).all() and (r.entropy[~some] == 0).all() and (r.top_logprobs[~some] == -math.inf).all()
        assert (r.top_ids[~some] == torch.arange(k, device=DEV)).all()
