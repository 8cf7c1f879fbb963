"""Measured cases of the paged key/value cache: reservation, append, one-token attention.

A serving program keeps the keys and values of many requests in pages of ``page_size`` tokens
taken from one pool.  Each step it reserves room for the step's tokens (block tables and slot
maps from the requests' lengths), writes the new keys and values into their slots, and lets one
new token of every request attend over that request's pages.  ``run`` makes one of those three
calls: in its plain form (elementary torch operations in 32 bits), or, where ``own`` is set,
through ``butterfly_b200.paged``.

Sizes: the 8/2- and 16/4-head attention layers of head dimension 128, the 131,072- and
262,144-token contexts and the 64 x 65,536 batched decode that this repository's benchmark and
tests use; head dimensions 64 and 256, other head ratios and page sizes are generic.
"""
import math

import numpy as np
import torch

own = False

_DT = {"bf16": torch.bfloat16, "f16": torch.float16}


# ------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one request decodes: one token, its page already there
        _reserve("reserve-one-request", B=1, lo=32767, hi=32767, page=16),
        # a server's step: decoding requests, one 512-token prompt chunk in eight, two requests done
        _reserve("reserve-mixed-64", B=64, lo=100, hi=65536, page=16, prompts=8, prompt=512, done=2),
        # many requests and 131,072 prompt tokens admitted at once
        _reserve("reserve-admit-1000", B=1000, lo=1, hi=4096, page=64, prompts=64, prompt=2048, done=37),
        # the new tokens of 64 decoding requests
        _append("append-64-tokens", T=64, Hkv=2, dh=128, page=16),
        # a whole 128k prompt, keys and values in the [token, head, dim] order the projection wrote
        _append("append-prompt-128k", T=131072, Hkv=2, dh=128, page=128),
        # a ragged fp16 step of 4 heads, some tokens refused (no slot), token-major pages
        _append("append-ragged-f16", T=5003, Hkv=4, dh=128, page=48, dtype="f16", nhd=True, skipped=211),
        # a few short requests: latency
        _decode("decode-short-4", B=4, lo=37, hi=513, Hq=8, Hkv=2, dh=128, page=16, step=True),
        # one long request: split over its length
        _decode("decode-one-128k", B=1, lo=131072, hi=131072, Hq=8, Hkv=2, dh=128, page=16, step=True),
        # the batched decode, every request at 65,536 tokens
        _decode("decode-64x65536", B=64, lo=65536, hi=65536, Hq=8, Hkv=2, dh=128, page=64),
        # ragged requests up to 262,144 tokens, 16/4 heads, fp16, two requests still empty
        _decode("decode-ragged-262k-f16", B=13, lo=211, hi=262144, Hq=16, Hkv=4, dh=128, page=32, dtype="f16", empty=2),
        # local layers: a 1,000-token window, 5 query heads per key head, token-major pages of 48
        _decode("decode-window-d64", B=96, lo=17, hi=30000, Hq=15, Hkv=3, dh=64, page=48, nhd=True, window=1000),
        # head dimension 256, one query head per key head
        _decode("decode-d256", B=24, lo=301, hi=8191, Hq=4, Hkv=4, dh=256, page=16, step=True),
    ]


def _reserve(name, **k):
    return dict({"op": "reserve", "prompts": 0, "prompt": 0, "done": 0, "page": 16}, **({"name": name} if name else {}), **k)


def _append(name, **k):
    d = {"op": "append", "dtype": "bf16", "nhd": False, "skipped": 0}
    return {**d, **({"name": name} if name else {}), **k}


def _decode(name, **k):
    d = {"op": "decode", "dtype": "bf16", "nhd": False, "window": 0, "empty": 0, "step": False}
    return {**d, **({"name": name} if name else {}), **k}


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["reserve", "append", "decode", "decode"])
    page = rng.choice([16, 32, 48, 64, 128])
    if op == "reserve":
        B = _log(rng, 1, 1000)
        hi = _log(rng, 1, 65536 if B <= 64 else 4096)
        prompts = rng.randint(0, min(B, 64))
        done = rng.randint(0, (B - prompts) // 4)
        return _reserve("", B=B, lo=rng.randint(1, hi), hi=hi, page=page, prompts=prompts, prompt=_log(rng, 1, 2048), done=done)
    dtype, nhd = rng.choice(["bf16", "f16"]), rng.random() < 0.4
    if op == "append":
        Hkv, dh = rng.choice([1, 2, 3, 4, 8]), rng.choice([64, 128, 256])
        T = _log(rng, 1, 131072 * 2 * 128 // (Hkv * dh))
        return _append("", T=T, Hkv=Hkv, dh=dh, page=page, dtype=dtype, nhd=nhd, skipped=rng.randint(0, T // 8))
    dh, Hkv = rng.choice([64, 128, 128, 256]), rng.choice([1, 2, 3, 4, 8])
    Hq = Hkv * rng.choice([1, 2, 3, 4, 5, 8, 12, 16])
    B = _log(rng, 1, 128)
    hi = _log(rng, 1, min(262144, 64 * 65536 * 8 * 128 // (B * max(Hq, 4 * Hkv) * dh)))
    step = rng.random() < 0.5
    return _decode("", B=B, lo=rng.randint(1, hi), hi=hi, Hq=Hq, Hkv=Hkv, dh=dh, page=page, dtype=dtype, nhd=nhd, step=step,
                   window=rng.choice([0, 0, 1, _log(rng, 2, 4096)]), empty=0 if step else rng.randint(0, B // 4))


def _lens(c):
    """The requests' lengths: spread evenly over their logarithm from lo to hi, odd ones among them, `empty` zeros."""
    n = c["B"] - c.get("empty", 0)
    x = np.exp(np.linspace(math.log(c["hi"]), math.log(c["lo"]), max(n, 1)))[:n]
    return np.concatenate([np.round(x).astype(np.int64), np.zeros(c["B"] - n, np.int64)])


def _adds(c):
    """Tokens added per request: one each, `prompt` for the shortest `prompts`, all taken back for the `done` longest."""
    a = np.ones(c["B"], np.int64)
    if c["prompts"]:
        a[-c["prompts"]:] = c["prompt"]
    a[: c["done"]] = -(2 ** 31)
    return a


def _pages(tokens, page):
    return -(-tokens // page)


# ------------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    c = dict(case)
    return {"reserve": _prepare_reserve, "append": _prepare_append, "decode": _prepare_decode}[c["op"]](c, g)


def _perm(n, g):
    return torch.randperm(n, generator=g, device="cuda")


def _table(lens, width, page, ids):
    """Block table [B, width] int32 whose requests own consecutive runs of `ids`, -1 elsewhere."""
    n = _pages(lens, page)
    first = torch.cumsum(n, 0) - n
    col = torch.arange(width, device="cuda")[None, :]
    t = ids[(first[:, None] + col).clamp(max=ids.numel() - 1)]
    return torch.where(col < n[:, None], t, -1).int()


def _prepare_reserve(c, g):
    order = _perm(c["B"], g)
    lens = torch.from_numpy(_lens(c)).cuda()[order]
    add = torch.from_numpy(_adds(c)).cuda()[order]
    page = c["page"]
    used = int(_pages(lens, page).sum())
    width = int(_pages((lens + add.clamp(min=0)).max(), page)) + 1
    need = int((_pages(lens + add.clamp(min=0), page) - _pages(lens, page)).sum())
    ids = _perm(used + need + 7, g).int()
    free = torch.full((ids.numel(),), -1, dtype=torch.int32, device="cuda")
    n = ids.numel() - used
    free[:n] = ids[used:]
    tokens = int(np.maximum(_adds(c), 0).sum())
    return {"case": c, "lens": lens.int(), "add": add.int(), "table": _table(lens, width, page, ids), "free": free,
            "num_free": torch.tensor([n], dtype=torch.int32, device="cuda"), "tokens": tokens}


def _randn(g, *shape, dtype, scale=1.0):
    x = torch.randn(*shape, generator=g, device="cuda", dtype=dtype)
    return x.mul_(scale) if scale != 1.0 else x


def _pool(c, pages, g, dt):
    """A pool view [pages, Hkv, page, dh]: pages hold older requests' rows where nothing newer was written."""
    if c["nhd"]:
        return _randn(g, pages, c["page"], c["Hkv"], c["dh"], dtype=dt).permute(0, 2, 1, 3)
    return _randn(g, pages, c["Hkv"], c["page"], c["dh"], dtype=dt)


def _prepare_append(c, g):
    dt, T = _DT[c["dtype"]], c["T"]
    pages = _pages(T, c["page"]) + 3
    slots = _perm(pages, g)[:, None] * c["page"] + torch.arange(c["page"], device="cuda")[None, :]
    slots = slots.reshape(-1)[:T].clone()
    slots[_perm(T, g)[: c["skipped"]]] = -1
    kv = _randn(g, T, 2 * c["Hkv"], c["dh"], dtype=dt)  # rows of a merged projection output
    return {"case": c, "k": kv[:, : c["Hkv"]], "v": kv[:, c["Hkv"]:], "kp": _pool(c, pages, g, dt), "vp": _pool(c, pages, g, dt),
            "slots": slots}


def _prepare_decode(c, g):
    dt, page = _DT[c["dtype"]], c["page"]
    lens = torch.from_numpy(_lens(c)).cuda()[_perm(c["B"], g)]
    total = int(_pages(lens, page).sum())
    width = int(_pages(lens.max(), page)) + 1
    ids = _perm(total + 3, g).int()
    B, Hq, Hkv, dh = c["B"], c["Hq"], c["Hkv"], c["dh"]
    s = {"case": c, "lens": lens.int(), "table": _table(lens, width, page, ids), "kp": _pool(c, total + 3, g, dt),
         "vp": _pool(c, total + 3, g, dt), "q": _randn(g, B, Hq, 1, dh, dtype=dt, scale=1.5)}
    if c["step"]:
        s["kn"], s["vn"] = (_randn(g, B, Hkv, 1, dh, dtype=dt) for _ in range(2))
    return s


# ------------------------------------------------------------------------------------ one pass
def run(s):
    return {"reserve": _run_reserve, "append": _run_append, "decode": _run_decode}[s["case"]["op"]](s)


def _run_reserve(s):
    c = s["case"]
    if own:
        from butterfly_b200.paged import paged_reserve
        r = paged_reserve(s["lens"], s["add"], s["table"], s["free"], s["num_free"], page_size=c["page"], num_tokens=s["tokens"])
    else:
        r = _plain_reserve(s["lens"], s["add"], s["table"], s["free"], s["num_free"], c["page"], s["tokens"])
    lens, num_free, slots, positions, granted = r
    return {"lens": lens, "num_free": num_free, "slots": slots, "positions": positions, "granted": granted, "table": s["table"],
            "free": s["free"]}


def _plain_reserve(lens, add, table, free, num_free, page, tokens):
    """Pages for lens + add: a shrinking request's last pages go back on the free stack, a growing one takes pages from its top, requests in order
    as long as the pages last.  The j-th page given back lies j below the new top, the i-th taken comes from i below it."""
    B, width = table.shape
    dev = lens.device
    ln, ad, tab = lens.long(), add.long(), table.long()
    want = (ln + ad).clamp(min=0)
    old_p, new_p = _pages(ln, page), _pages(want, page)
    fits = new_p <= width
    need = torch.where((ad > 0) & fits, new_p - old_p, 0)
    back = torch.where(ad < 0, old_p - new_p, 0)
    n = num_free.long()[0]
    cum_need, cum_back = need.cumsum(0), back.cumsum(0)
    top = n + cum_back[-1]
    granted = (ad > 0) & fits & ((need == 0) | (cum_need <= top))
    kept = (ad > 0) & ~granted
    take = torch.where(granted, need, 0).cumsum(0)
    out_len = torch.where(kept, ln, want)
    # the stack with the pages given back, read from the top: entry x below the top
    P = free.numel()
    x = torch.arange(P + 1, device=dev)
    rb = torch.searchsorted(cum_back, x, right=True).clamp(max=B - 1)
    given = tab[rb, (new_p[rb] + x - (cum_back[rb] - back[rb])).clamp(0, width - 1)]
    from_top = torch.where(x < cum_back[-1], given, free.long()[(top - 1 - x).clamp(0, P - 1)])
    # table entries of the pages taken
    col = torch.arange(width, device=dev)[None, :]
    fresh = (col >= old_p[:, None]) & (col < new_p[:, None]) & granted[:, None]
    which = (take - torch.where(granted, need, 0))[:, None] + col - old_p[:, None]
    tab = torch.where(fresh, from_top[which.clamp(0, P)], tab)
    # the stack afterwards: pages given back and not taken again
    left = top - take[-1]
    y = torch.arange(P, device=dev)
    free.copy_(torch.where((y >= n) & (y < left), from_top[(top - 1 - y).clamp(0, P)], free.long()))
    table.copy_(tab)
    # slots and positions of the step's tokens, packed request by request
    cum = ad.clamp(min=0).cumsum(0)
    t = torch.arange(tokens, device=dev)
    b = torch.searchsorted(cum, t, right=True).clamp(max=B - 1)
    pos = ln[b] + t - (cum[b] - ad.clamp(min=0)[b])
    ok = (t < cum[-1]) & granted[b]
    slot = tab[b, (pos // page).clamp(0, width - 1)] * page + pos % page
    return out_len.int(), left.int().reshape(1), torch.where(ok, slot, -1), torch.where(ok, pos, -1).int(), granted


def _run_append(s):
    if own:
        from butterfly_b200.paged import paged_append
        paged_append(s["k"], s["v"], s["kp"], s["vp"], s["slots"])
    else:
        page = s["case"]["page"]
        ok = s["slots"] >= 0
        slot = s["slots"][ok]
        s["kp"][slot // page, :, slot % page] = s["k"][ok]
        s["vp"][slot // page, :, slot % page] = s["v"][ok]
    return {"k_pages": s["kp"], "v_pages": s["vp"]}


def _run_decode(s):
    c = s["case"]
    new = (s["kn"], s["vn"]) if c["step"] else (None, None)
    if own:
        from butterfly_b200.paged import paged_decode_attention
        out, lse = paged_decode_attention(s["q"], s["kp"], s["vp"], s["table"], s["lens"], k_new=new[0], v_new=new[1],
                                          window=c["window"], return_lse=True)
    else:
        out, lse = _plain_decode(s["q"], s["kp"], s["vp"], s["table"], s["lens"], new[0], new[1], c["window"])
    r = {"out": out, "lse": lse}
    return {**r, "k_pages": s["kp"], "v_pages": s["vp"]} if c["step"] else r


def _plain_decode(q, kp, vp, table, lens, k_new, v_new, window):
    B, Hq, _, dh = q.shape
    Hkv, page = kp.shape[1], kp.shape[2]
    tab, ln = table.long().clamp(min=0), lens.long()
    if k_new is not None:  # the new token's row, at position len - 1
        pos = ln - 1
        p = tab.gather(1, (pos // page)[:, None])[:, 0]
        kp[p, :, pos % page] = k_new[:, :, 0]
        vp[p, :, pos % page] = v_new[:, :, 0]
    k = kp[tab].transpose(1, 2).reshape(B, Hkv, -1, dh).float()
    x = torch.arange(k.shape[2], device=q.device)[None, :]
    seen = (x < ln[:, None]) & (x >= (ln[:, None] - window if window else 0))
    s = q.reshape(B, Hkv, Hq // Hkv, dh).float() @ k.transpose(-1, -2) / math.sqrt(dh)
    del k
    s = s.masked_fill(~seen[:, None, None], -math.inf)
    m = s.amax(-1, keepdim=True)
    e = torch.exp(s - torch.where(m == -math.inf, 0.0, m))
    v = vp[tab].transpose(1, 2).reshape(B, Hkv, -1, dh).float()
    l = e.sum(-1, keepdim=True)
    out = (e @ v) / torch.where(l == 0, 1.0, l)
    return out.reshape(B, Hq, 1, dh).to(q.dtype), (m + torch.log(l)).reshape(B, Hq, 1)


# ------------------------------------------------------------------------------------ the least work
def work(case):
    c = case
    if c["op"] == "reserve":
        ln, ad = _lens(c), _adds(c)
        tokens = int(np.maximum(ad, 0).sum())
        want = np.maximum(ln + ad, 0)
        moved = int(np.abs(_pages(want, c["page"]) - _pages(ln, c["page"])).sum())
        # lengths, additions and grants; slots (8) and positions (4); page numbers read and written
        return {"bytes": c["B"] * (4 + 4 + 4 + 1) + tokens * 12 + moved * 8 + c["B"] * 4 + 8, "flops": 8 * c["B"] + 4 * tokens}
    row = c["Hkv"] * c["dh"] * 2 * 2  # one token's key and value rows
    if c["op"] == "append":
        n = c["T"] - c["skipped"]
        return {"bytes": 2 * n * row + 8 * c["T"], "flops": n}
    ln = _lens(c)
    keys = int((np.minimum(ln, c["window"]) if c["window"] else ln).sum())
    b = keys * row + 2 * c["B"] * c["Hq"] * c["dh"] * 2 + c["B"] * c["Hq"] * 4 + c["B"] * 4 + 4 * _pages(keys, c["page"])
    return {"bytes": int(b + (c["B"] * row if c["step"] else 0)), "flops": 4 * keys * c["Hq"] * c["dh"]}


# ------------------------------------------------------------------------------------ 64 bits
def exact(case, seed):
    """From the definitions, request by request: the stack as a Python list, the softmax in float64."""
    s = prepare(case, seed)
    c = s["case"]
    if c["op"] == "append":
        return None  # copies
    lens = s["lens"].tolist()
    page = c["page"]
    if c["op"] == "reserve":
        add, table = s["add"].tolist(), s["table"].cpu().numpy().copy()
        n = int(s["num_free"])
        disk = s["free"].tolist()
        stack, back = disk[:n], []
        for b, (ln, ad) in enumerate(zip(lens, add)):
            if ad < 0:
                back += table[b, _pages(max(0, ln + ad), page):_pages(ln, page)].tolist()
        stack += back[::-1]
        new, slots, positions, granted, asked, room = [], [], [], [], 0, len(stack)
        for b, (ln, ad) in enumerate(zip(lens, add)):
            ok = ad > 0
            if ad > 0:
                need = _pages(ln + ad, page) - _pages(ln, page)
                ok = _pages(ln + ad, page) <= table.shape[1]
                if ok and need:
                    asked += need
                    ok = asked <= room
                if ok:
                    for i in range(need):
                        table[b, _pages(ln, page) + i] = stack.pop()
                for p in range(ln, ln + ad):
                    slots.append(int(table[b, p // page]) * page + p % page if ok else -1)
                    positions.append(p if ok else -1)
            new.append(ln if ad > 0 and not ok else max(0, ln + ad))
            granted.append(ok)
        disk[n:len(stack)] = stack[n:]
        return {"lens": np.array(new), "num_free": np.array([len(stack)]), "slots": np.array(slots), "positions": np.array(positions),
                "granted": np.array(granted), "table": table, "free": np.array(disk)}
    q = s["q"][:, :, 0].double()
    B, Hq, dh = q.shape
    G = Hq // c["Hkv"]
    out = torch.zeros(B, Hq, 1, dh, dtype=torch.float64, device="cuda")
    lse = torch.full((B, Hq, 1), -math.inf, dtype=torch.float64, device="cuda")
    for b, ln in enumerate(lens):
        if ln == 0:
            continue
        rows = s["table"][b, : _pages(ln, page)].long()
        first = max(0, ln - c["window"]) if c["window"] else 0
        for h in range(c["Hkv"]):
            k, v = (s[x][rows, h].reshape(-1, dh)[first:ln].double() for x in ("kp", "vp"))
            if c["step"]:
                k[-1], v[-1] = s["kn"][b, h, 0].double(), s["vn"][b, h, 0].double()
            z = q[b, h * G:(h + 1) * G] @ k.T / math.sqrt(dh)
            lse[b, h * G:(h + 1) * G, 0] = torch.logsumexp(z, -1)
            out[b, h * G:(h + 1) * G, 0] = torch.softmax(z, -1) @ v
    r = {"out": out, "lse": lse}
    return {**r, "k_pages": None, "v_pages": None} if c["step"] else r
