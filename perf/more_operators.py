"""Measured cases of the 4-bit paged cache (rows into pages and back, one-token attention) and of
token log probabilities.

A serving program that keeps its requests' keys and values in 4 bits writes the new tokens' rows
into pages (quantising them), reads rows back where a prompt's prefix is used again, and lets one
new token of every request attend over that request's pages.  Its answers, and the comparison of
a compressed cache with the full one, need the log probabilities of given tokens, the entropy of
their distributions and the likeliest alternatives.  ``run`` makes one of those calls: in its
plain form (elementary torch operations in 32 bits), or, where ``own`` is set, through
``butterfly_b200.paged`` and ``butterfly_b200.logits``.

The format: a row of ``dh`` columns is cut into groups of 64.  A group holds its minimum m and
the scale s = (maximum - m) / 15, both rounded to the rows' 16-bit type, and codes
c = round((x - m) / s) in 0..15: x is read as s c + m.  A pool ``[pages, Hkv, page_size / 16,
18 dh]`` of bytes holds 16 tokens of a head in a block: key codes [16, dh / 2], key scales and
minima [16, groups, 2], and the same of the values.  Code word (8 codes, the first in the
lowest bits) g * groups + y of a row holds columns 64 y + 8 g .. + 7.

Sizes: the 8/2- and 16/4-head attention layers of head dimension 128, the 131,072- and
262,144-token contexts, the 64 x 65,536 batched decode, the 151,936-entry vocabulary and the 8
requests of the serving example are this repository's; the others are generic.
"""
import math

import numpy as np
import torch

own = False

_DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_GROUP = 64


# ------------------------------------------------------------------------------------ cases
def listed():
    return [
        # the new tokens of 64 decoding requests
        _store("store-64-tokens", T=64, Hkv=2, dh=128, page=16),
        # a whole 128k prompt, in the [token, head, dim] order the projection wrote
        _store("store-prompt-128k", T=131072, Hkv=2, dh=128, page=64),
        # a ragged fp16 step of 4 heads, some tokens refused (no slot), pages of 48
        _store("store-ragged-f16", T=5003, Hkv=4, dh=128, page=48, dtype="f16", skipped=211),
        # a few short requests, their new rows written by the same call: latency
        _decode("decode-short-4", B=4, lo=37, hi=513, Hq=8, Hkv=2, dh=128, page=16, step=True),
        # one long request: split over its length
        _decode("decode-one-128k", B=1, lo=131072, hi=131072, Hq=8, Hkv=2, dh=128, page=16),
        # the batched decode, every request at 65,536 tokens
        _decode("decode-64x65536", B=64, lo=65536, hi=65536, Hq=8, Hkv=2, dh=128, page=64),
        # ragged requests up to 262,144 tokens, 16/4 heads, fp16, two requests still empty
        _decode("decode-ragged-262k-f16", B=13, lo=211, hi=262144, Hq=16, Hkv=4, dh=128, page=32, dtype="f16", empty=2),
        # local layers: a 1,000-token window, 5 query heads per key head of 64, pages of 48
        _decode("decode-window-d64", B=96, lo=17, hi=30000, Hq=15, Hkv=3, dh=64, page=48, window=1000),
        # one request's next token, its 20 likeliest alternatives: latency
        _logprobs("logprobs-one-row", R=1, V=151936, top=20),
        # a step of the 8-request server in fp32 logits
        _logprobs("logprobs-8-rows-f32", R=8, V=151936, dtype="f32", top=5),
        # the tokens of a 4,096-token prompt scored, a padded vocabulary
        _logprobs("logprobs-prompt-4096", R=4096, V=151936, top=1, masked=267),
        # odd sizes, fp16, rows further apart than they are long, some tokens padding
        _logprobs("logprobs-odd-f16", R=333, V=32003, dtype="f16", top=50, pad=13, ignored=29),
    ]


def _named(name, d):
    return {**d, **({"name": name} if name else {})}


def _store(name, **k):
    return _named(name, {"op": "store", "dtype": "bf16", "skipped": 0, **k})


def _decode(name, **k):
    return _named(name, {"op": "decode", "dtype": "bf16", "window": 0, "empty": 0, "step": False, **k})


def _logprobs(name, **k):
    return _named(name, {"op": "logprobs", "dtype": "bf16", "pad": 0, "masked": 0, "ignored": 0, **k})


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["store", "decode", "decode", "logprobs"])
    if op == "logprobs":
        dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
        V = rng.choice([151936, _log(rng, 64, 262144)])
        R = _log(rng, 1, min(65536, 4096 * 151936 * 2 // (V * (4 if dtype == "f32" else 2))))
        return _logprobs("", R=R, V=V, dtype=dtype, top=rng.choice([0, 1, 5, 20, 50, 64]) if V >= 128 else rng.randint(0, 32),
                         pad=rng.choice([0, 0, 1, 8, 13]), masked=rng.choice([0, 0, V // 7]), ignored=rng.randint(0, R // 4))
    page = rng.choice([16, 32, 48, 64, 128])
    dtype = rng.choice(["bf16", "f16"])
    if op == "store":
        Hkv, dh = rng.choice([1, 2, 3, 4, 8]), rng.choice([64, 128, 256])
        T = _log(rng, 1, 131072 * 2 * 128 // (Hkv * dh))
        return _store("", T=T, Hkv=Hkv, dh=dh, page=page, dtype=dtype, skipped=rng.randint(0, T // 8))
    dh, Hkv = rng.choice([64, 128, 128, 256]), rng.choice([1, 2, 3, 4, 8])
    Hq = Hkv * rng.choice([1, 2, 3, 4, 5, 8, 12, 16])
    B = _log(rng, 1, 128)
    hi = _log(rng, 1, min(262144, 64 * 65536 * 8 * 128 // (B * max(Hq, 4 * Hkv) * dh)))
    step = rng.random() < 0.5
    return _decode("", B=B, lo=rng.randint(1, hi), hi=hi, Hq=Hq, Hkv=Hkv, dh=dh, page=page, dtype=dtype, step=step,
                   window=rng.choice([0, 0, 1, _log(rng, 2, 4096)]), empty=0 if step else rng.randint(0, B // 4))


def _lens(c):
    """The requests' lengths: spread evenly over their logarithm from lo to hi, odd ones among them, `empty` zeros."""
    n = c["B"] - c["empty"]
    x = np.exp(np.linspace(math.log(c["hi"]), math.log(c["lo"]), max(n, 1)))[:n]
    return np.concatenate([np.round(x).astype(np.int64), np.zeros(c["B"] - n, np.int64)])


def _pages(tokens, page):
    return -(-tokens // page)


# ------------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    c = dict(case)
    return {"store": _prepare_store, "decode": _prepare_decode, "logprobs": _prepare_logprobs}[c["op"]](c, g)


def _perm(n, g):
    return torch.randperm(n, generator=g, device="cuda")


def _randn(g, *shape, dtype, scale=1.0):
    x = torch.randn(*shape, generator=g, device="cuda", dtype=dtype)
    return x.mul_(scale) if scale != 1.0 else x


def _prepare_store(c, g):
    dt, T, dh = _DT[c["dtype"]], c["T"], c["dh"]
    pages = _pages(T, c["page"]) + 3
    slots = _perm(pages, g)[:, None] * c["page"] + torch.arange(c["page"], device="cuda")[None, :]
    slots = slots.reshape(-1)[:T].clone()
    slots[_perm(T, g)[: c["skipped"]]] = -1
    kv = _randn(g, T, 2 * c["Hkv"], dh, dtype=dt)  # rows of a merged projection output
    kv[:, : c["Hkv"]] += _randn(g, c["Hkv"], dh, dtype=dt, scale=2.0)  # keys have columns far from zero
    # pages hold older requests' bytes where nothing newer was written
    pool = torch.randint(0, 256, (pages, c["Hkv"], c["page"] // 16, 18 * dh), generator=g, device="cuda", dtype=torch.uint8)
    return {"case": c, "k": kv[:, : c["Hkv"]], "v": kv[:, c["Hkv"]:], "pool": pool, "slots": slots}


def _prepare_decode(c, g):
    dt, page = _DT[c["dtype"]], c["page"]
    lens = torch.from_numpy(_lens(c)).cuda()[_perm(c["B"], g)]
    n = _pages(lens, page)
    total, width = int(n.sum()), int(n.max()) + 1
    ids = _perm(total + 3, g).int()
    first, col = torch.cumsum(n, 0) - n, torch.arange(width, device="cuda")[None, :]
    table = torch.where(col < n[:, None], ids[(first[:, None] + col).clamp(max=ids.numel() - 1)], -1).int()
    B, Hq, Hkv, dh = c["B"], c["Hq"], c["Hkv"], c["dh"]
    bias = _randn(g, Hkv, 1, dh, dtype=dt, scale=2.0)
    pool = torch.empty(total + 3, Hkv, page // 16, 18 * dh, device="cuda", dtype=torch.uint8)
    some = max(1, (1 << 25) // (Hkv * page * dh))
    for i in range(0, total + 3, some):
        p = pool[i:i + some]
        for part, b in zip(_halves(p, dh), (bias, 0)):
            x = (_randn(g, p.shape[0], Hkv, page, dh, dtype=dt) + b).unflatten(2, (-1, 16))
            for to, y in zip(part, _pack(x)):
                to.copy_(y)
    s = {"case": c, "lens": lens.int(), "table": table, "pool": pool, "q": _randn(g, B, Hq, 1, dh, dtype=dt, scale=1.5)}
    if c["step"]:
        s["kn"], s["vn"] = _randn(g, B, Hkv, 1, dh, dtype=dt) + bias, _randn(g, B, Hkv, 1, dh, dtype=dt)
        at = lens - 1
        s["slots"] = table.long().gather(1, (at // page)[:, None])[:, 0] * page + at % page
    return s


def _prepare_logprobs(c, g):
    R, V = c["R"], c["V"]
    x = torch.empty(R, V + c["pad"], device="cuda", dtype=_DT[c["dtype"]]).normal_(generator=g).mul_(2.5)
    x[:, V - c["masked"]: V] = -math.inf
    tokens = torch.randint(0, V - c["masked"], (R,), generator=g, device="cuda")
    x.scatter_add_(1, tokens[:, None], torch.rand(R, 1, generator=g, device="cuda").mul_(12).to(x.dtype))  # answers are likely
    tokens[_perm(R, g)[: c["ignored"]]] = -1
    return {"case": c, "logits": x[:, :V], "tokens": tokens}


# ------------------------------------------------------------------------------------ one pass
def run(s):
    return {"store": _run_store, "decode": _run_decode, "logprobs": _run_logprobs}[s["case"]["op"]](s)


def _halves(blocks, dh):
    """Views (codes [.., 16, dh / 2], scales and minima [.., 16, dh / 16] in bytes) of the keys' and the values' half of blocks."""
    at = lambda o: (blocks[..., o:o + 8 * dh].unflatten(-1, (16, dh // 2)), blocks[..., o + 8 * dh:o + 9 * dh].unflatten(-1, (16, dh // 16)))  # noqa: E731
    return at(0), at(9 * dh)


def _pack(x):
    """Rows [.., dh] -> their codes [.., dh / 2] and their scales and minima [.., dh / 16], in bytes."""
    f = x.float().unflatten(-1, (-1, _GROUP))
    low, high = f.amin(-1), f.amax(-1)
    s = ((high - low) / torch.full_like(low, 15.0)).to(x.dtype)  # (a tensor of 15s: torch multiplies by 1 / 15 for a number)
    step = torch.where(s == 0, 1.0, s.float())[..., None]
    n = torch.round((f - low[..., None]) / step).clamp(0, 15)
    n = torch.where(s[..., None] == 0, 0.0, n).to(torch.uint8)
    n = n.unflatten(-1, (8, 8)).transpose(-3, -2)  # [.., 8 chunks, groups, 8 codes]
    codes = (n[..., 0::2] | (n[..., 1::2] << 4)).flatten(-3)
    return codes, torch.stack([s, low.to(x.dtype)], -1).flatten(-2).contiguous().view(torch.uint8)


def _unpack(codes, params, dtype):
    """What rows stand for, in 32 bits: codes [.., dh / 2], scales and minima [.., dh / 16] -> [.., dh]."""
    p = params.contiguous().view(dtype).float().unflatten(-1, (-1, 2))
    n = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).unflatten(-1, (8, -1, 8)).transpose(-3, -2).flatten(-2)
    return (n.float() * p[..., 0:1] + p[..., 1:2]).flatten(-2)


def _plain_append(k, v, pool, slots):
    ok = slots >= 0
    slot, page = slots[ok], 16 * pool.shape[2]
    p, off = slot // page, slot % page
    for part, x in zip(_halves(pool, k.shape[-1]), (k[ok], v[ok])):
        for to, y in zip(part, _pack(x)):
            to[p, :, off // 16, off % 16] = y


def _plain_read(pool, slots, dtype):
    page, dh = 16 * pool.shape[2], pool.shape[3] // 18
    p, off = slots.clamp(min=0) // page, slots.clamp(min=0) % page
    rows = (_unpack(*(x[p, :, off // 16, off % 16] for x in part), dtype) for part in _halves(pool, dh))
    return [torch.where((slots >= 0)[:, None, None], x, 0.0).to(dtype) for x in rows]


def _run_store(s):
    dt = s["k"].dtype
    if own:
        from butterfly_b200.paged import paged_append_int4, paged_read_int4
        paged_append_int4(s["k"], s["v"], s["pool"], s["slots"])
        k, v = paged_read_int4(s["pool"], s["slots"], dtype=dt)
    else:
        _plain_append(s["k"], s["v"], s["pool"], s["slots"])
        k, v = _plain_read(s["pool"], s["slots"], dt)
    return {"k": k, "v": v}


def _run_decode(s):
    c = s["case"]
    if own:
        from butterfly_b200.paged import paged_decode_attention_int4, paged_read_int4
        new = {"k_new": s["kn"], "v_new": s["vn"]} if c["step"] else {}
        out, lse = paged_decode_attention_int4(s["q"], s["pool"], s["table"], s["lens"], window=c["window"], return_lse=True, **new)
        rows = paged_read_int4(s["pool"], s["slots"], dtype=s["q"].dtype) if c["step"] else None
    else:
        if c["step"]:
            _plain_append(s["kn"][:, :, 0], s["vn"][:, :, 0], s["pool"], s["slots"])
        out, lse = _plain_decode(s["q"], s["pool"], s["table"], s["lens"], c["window"])
        rows = _plain_read(s["pool"], s["slots"], s["q"].dtype) if c["step"] else None
    r = {"out": out, "lse": lse}
    return {**r, "k_rows": rows[0], "v_rows": rows[1]} if c["step"] else r


def _plain_decode(q, pool, table, lens, window):
    B, Hq, _, dh = q.shape
    Hkv, ln = pool.shape[1], lens.long()
    blocks = pool[table.long().clamp(min=0)].transpose(1, 2).flatten(2, 3)  # [B, Hkv, blocks, 18 dh]
    keys, values = _halves(blocks, dh)
    k = _unpack(*keys, q.dtype).flatten(2, 3)
    x = torch.arange(k.shape[2], device=q.device)[None, :]
    seen = (x < ln[:, None]) & (x >= (ln[:, None] - window if window else 0))
    k = torch.where(seen[:, None, :, None], k, 0.0)  # (what pages hold beyond is anything)
    s = q.reshape(B, Hkv, Hq // Hkv, dh).float() @ k.transpose(-1, -2) / math.sqrt(dh)
    del k
    s = s.masked_fill(~seen[:, None, None], -math.inf)
    m = s.amax(-1, keepdim=True)
    e = torch.exp(s - torch.where(m == -math.inf, 0.0, m))
    v = _unpack(*values, q.dtype).flatten(2, 3)
    v = torch.where(seen[:, None, :, None], v, 0.0)
    total = e.sum(-1, keepdim=True)
    out = (e @ v) / torch.where(total == 0, 1.0, total)
    return out.reshape(B, Hq, 1, dh).to(q.dtype), (m + torch.log(total)).reshape(B, Hq, 1)


def _run_logprobs(s):
    k = s["case"]["top"]
    if own:
        from butterfly_b200.logits import token_logprobs
        r = token_logprobs(s["logits"], s["tokens"], top_k=k)
        out = {"logprobs": r.logprobs, "entropy": r.entropy}
        return {**out, "top_ids": r.top_ids, "top_logprobs": r.top_logprobs} if k else out
    return _plain_logprobs(s["logits"], s["tokens"], k)


def _plain_logprobs(logits, tokens, k):
    x = logits.float() + 0.0  # (-0 becomes 0: equal values tie)
    m = x.amax(-1, keepdim=True)
    t = x - m
    e = torch.exp(t)
    z = e.sum(-1)
    entropy = torch.log(z) - torch.where(e > 0, e * t, 0.0).sum(-1) / z
    del e
    lse = m[:, 0] + torch.log(z)
    picked = t.gather(1, tokens.clamp(min=0)[:, None])[:, 0] - torch.log(z)
    out = {"logprobs": torch.where(tokens >= 0, picked, 0.0), "entropy": entropy}
    del t
    if not k:
        return out
    # the k largest, of equal ones the lowest index: whole numbers in the same order as (value, -index)
    bits = x.view(torch.int32)
    key = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long() * 2 ** 32
    key += torch.arange(x.shape[1] - 1, -1, -1, device=x.device)
    ids = x.shape[1] - 1 - (torch.topk(key, k, dim=-1).values & 0xFFFFFFFF)
    return {**out, "top_ids": ids, "top_logprobs": x.gather(1, ids) - lse[:, None]}


# ------------------------------------------------------------------------------------ the least work
def work(case):
    c = case
    if c["op"] == "logprobs":
        n = c["R"] * c["V"]
        # logits and tokens in; log probability and entropy, ids and log probabilities of the top out
        return {"bytes": n * (4 if c["dtype"] == "f32" else 2) + c["R"] * (8 + 8 + 12 * c["top"]), "flops": 6 * n}
    wide, packed = c["Hkv"] * c["dh"] * 2 * 2, c["Hkv"] * c["dh"] // 64 * 36 * 2  # one token's rows in 16 and in 4 bits
    if c["op"] == "store":
        n = c["T"] - c["skipped"]
        return {"bytes": n * (wide + packed) + c["T"] * (wide + 8), "flops": 8 * n * c["Hkv"] * c["dh"]}
    ln = _lens(c)
    keys = int((np.minimum(ln, c["window"]) if c["window"] else ln).sum())
    b = keys * packed + 2 * c["B"] * c["Hq"] * c["dh"] * 2 + c["B"] * c["Hq"] * 4 + c["B"] * 4 + 4 * _pages(keys, c["page"])
    return {"bytes": int(b + (c["B"] * 2 * wide if c["step"] else 0)), "flops": 4 * keys * c["Hq"] * c["dh"]}


# ------------------------------------------------------------------------------------ 64 bits
def exact(case, seed):
    """From the definitions: a code word's columns by their formula, the softmax in float64, request by request or some rows at a time."""
    s = prepare(case, seed)
    return {"store": _exact_store, "decode": _exact_decode, "logprobs": _exact_logprobs}[s["case"]["op"]](s)


def _exact_row(x):
    """What rows [.., dh] are read as."""
    out = torch.empty(x.shape, dtype=torch.float64, device=x.device)
    for y in range(0, x.shape[-1], _GROUP):
        f = x[..., y:y + _GROUP].double()
        m = f.min(-1, keepdim=True).values
        s = ((f.max(-1, keepdim=True).values - m) / 15).to(x.dtype).double()
        c = ((f - m) / torch.where(s > 0, s, 1)).round().clamp(0, 15)
        out[..., y:y + _GROUP] = torch.where(s > 0, c * s, 0) + m
    return out


def _exact_block(raw, dh, dtype, first):
    """Keys (first 0) or values (first 9 dh) of one head's blocks [n, 18 dh] as [16 n, dh]."""
    raw = raw[:, first:first + 9 * dh]
    word = raw[:, :8 * dh].contiguous().view(torch.int32).view(-1, 16, dh // 8)
    p = raw[:, 8 * dh:].contiguous().view(dtype).view(-1, 16, dh // _GROUP, 2).double()
    out = torch.empty(word.shape[0], 16, dh, dtype=torch.float64, device=raw.device)
    shifts = 4 * torch.arange(8, dtype=torch.int32, device=raw.device)
    for col in range(0, dh, 8):
        y, g = col // 64, col % 64 // 8
        c = (word[..., g * (dh // 64) + y, None] >> shifts) & 15
        out[..., col:col + 8] = c * p[:, :, y, :1] + p[:, :, y, 1:]
    return out.view(-1, dh)


def _exact_store(s):
    ok = (s["slots"] >= 0)[:, None, None]
    return {x: torch.where(ok, _exact_row(s[x]), 0.0) for x in ("k", "v")}


def _exact_decode(s):
    c = s["case"]
    q = s["q"][:, :, 0].double()
    B, Hq, dh = q.shape
    G, page, dt = Hq // c["Hkv"], c["page"], s["q"].dtype
    out = torch.zeros(B, Hq, 1, dh, dtype=torch.float64, device="cuda")
    lse = torch.full((B, Hq, 1), -math.inf, dtype=torch.float64, device="cuda")
    for b, ln in enumerate(s["lens"].tolist()):
        if ln == 0:
            continue
        first = max(0, ln - c["window"]) if c["window"] else 0
        p0 = first // page
        rows = s["table"][b, p0: _pages(ln, page)].long()
        for h in range(c["Hkv"]):
            raw = s["pool"][rows, h].flatten(0, 1)
            k, v = (_exact_block(raw, dh, dt, o)[first - p0 * page: ln - p0 * page] for o in (0, 9 * dh))
            if c["step"]:
                k[-1], v[-1] = _exact_row(s["kn"][b, h, 0]), _exact_row(s["vn"][b, h, 0])
            z = q[b, h * G:(h + 1) * G] @ k.T / math.sqrt(dh)
            lse[b, h * G:(h + 1) * G, 0] = torch.logsumexp(z, -1)
            out[b, h * G:(h + 1) * G, 0] = torch.softmax(z, -1) @ v
    r = {"out": out, "lse": lse}
    return {**r, "k_rows": _exact_row(s["kn"][:, :, 0]), "v_rows": _exact_row(s["vn"][:, :, 0])} if c["step"] else r


def _exact_logprobs(s):
    x, tokens, k = s["logits"], s["tokens"], s["case"]["top"]
    R, V = x.shape
    out = {"logprobs": torch.zeros(R, dtype=torch.float64, device="cuda"), "entropy": torch.zeros(R, dtype=torch.float64, device="cuda")}
    if k:
        out["top_ids"] = torch.zeros(R, k, dtype=torch.int64, device="cuda")
        out["top_logprobs"] = torch.zeros(R, k, dtype=torch.float64, device="cuda")
    some = max(1, (1 << 26) // V)
    for i in range(0, R, some):
        d = x[i:i + some].double()
        logp = d - torch.logsumexp(d, -1, keepdim=True)
        at = tokens[i:i + some]
        out["logprobs"][i:i + some] = torch.where(at >= 0, logp.gather(1, at.clamp(min=0)[:, None])[:, 0], 0)
        out["entropy"][i:i + some] = -torch.special.xlogy(logp.exp(), logp.exp()).sum(-1)
        for j in range(k):  # the largest, the first of equal ones, k times
            best = d.max(-1, keepdim=True).values
            first = (d == best).to(torch.uint8).argmax(-1, keepdim=True)
            out["top_ids"][i:i + some, j] = first[:, 0]
            out["top_logprobs"][i:i + some, j] = logp.gather(1, first)[:, 0]
            d.scatter_(1, first, -math.inf)
    return out
