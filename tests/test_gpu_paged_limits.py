"""The paged cache at its limits: request counts around the shared-memory bounds, additions that no
request can hold, probabilities far below their row's maximum.

Bars as in tests/test_gpu_paged.py, where the second part of an fp16 probability that is subnormal
counts in steps of 2^-39 of the row's largest (rounding: 2^-40), probabilities being held times 2^15;
an fp16 result that is subnormal is off by 2^-25."""
import math
import os
import subprocess
import sys

import pytest
import torch

import butterfly_b200 as bb

pytestmark = pytest.mark.gpu
DEV = "cuda"
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


# ------------------------------------------------------------------------------ attention
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("Hq,Hkv,dh,lens", [(8, 2, 128, [6000, 33]), (24, 2, 128, [5000, 700]), (6, 2, 64, [5000, 129]),
                                            (4, 2, 256, [4096, 65]), (8, 2, 128, [120000])])
@pytest.mark.parametrize("gap", [10.0, 14.0, 18.0, 22.0])
def test_tail_below_a_dominant_key(dtype, Hq, Hkv, dh, lens, gap):
    # the first key lies `gap` nats above the others and its value is zero (an attention sink): the
    # output is the others' share, however small each is
    g = torch.Generator(device=DEV).manual_seed(int(gap) + dh)
    page, u, scale = 32, 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -11, 1 / math.sqrt(dh)
    n = [-(-x // page) for x in lens]
    table = torch.full((len(lens), max(n)), -1, dtype=torch.int32, device=DEV)
    ids, at = torch.randperm(sum(n), generator=g, device=DEV).int(), 0
    kp, vp = (torch.randn(sum(n), Hkv, page, dh, generator=g, device=DEV) * 0.05 for _ in range(2))
    kp[..., 0], vp = 0.0, vp + 1.0
    for b, m in enumerate(n):
        table[b, :m] = ids[at:at + m]
        at += m
        kp[table[b, 0].long(), :, 0] = 0.0
        kp[table[b, 0].long(), :, 0, 0] = gap * math.sqrt(dh) / 8.0
        vp[table[b, 0].long(), :, 0] = 0.0
    q = torch.randn(len(lens), Hq, 1, dh, generator=g, device=DEV) * 0.05
    q[..., 0] = 8.0
    q, kp, vp = q.to(dtype), kp.to(dtype), vp.to(dtype)
    out, lse = bb.paged_decode_attention(q, kp, vp, table, torch.tensor(lens, dtype=torch.int32, device=DEV), return_lse=True)
    for b, ln in enumerate(lens):
        rows = table[b, :n[b]].long()
        k, v = (x[rows].transpose(0, 1).reshape(Hkv, -1, dh)[:, :ln].double() for x in (kp, vp))
        qb = q[b, :, 0].double().view(Hkv, Hq // Hkv, dh)
        s = qb @ k.transpose(1, 2) * scale
        p = torch.softmax(s, -1)
        ref, rl = (p @ v).reshape(Hq, dh), torch.logsumexp(s, -1).reshape(-1)
        ds = (dh + 4) * 2.0 ** -23 * scale * (qb.abs() @ k.abs().transpose(1, 2)).amax(-1).reshape(-1, 1)
        A = (p @ v.abs()).reshape(Hq, dh)
        bar = u * ref.abs() + A * (2 * ds + 2.0 ** -15 + ln * 2.0 ** -23)
        if dtype == torch.float16:
            bar = bar + ln * 2.0 ** -40 * float(v.abs().max()) + 2.0 ** -25
        err = (out[b, :, 0].double() - ref).abs()
        assert bool((err <= bar).all()), (b, float((err / bar).max()), float((err / ref.abs()).max()))
        lbar = ds[:, 0] + 2.0 ** -20 + ln * 2.0 ** -23 + 2.0 ** -21 * rl.abs()
        assert bool(((lse[b, :, 0].double() - rl).abs() <= lbar).all())


# ------------------------------------------------------------------------------ reserve
_ONE_CALL = """
import sys
import torch
import butterfly_b200 as bb
B, tokens = int(sys.argv[1]), int(sys.argv[2])
z = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")
free = torch.arange(B, dtype=torch.int32, device="cuda")
table = torch.full((B, 1), -1, dtype=torch.int32, device="cuda")
r = bb.paged_reserve(z(B), z(B) + 1, table, free, z(1) + B, page_size=16, num_tokens=tokens)
want = (B - 1 - torch.arange(B, device="cuda"))
assert bool((table[:, 0] == want).all()) and bool(r.granted.all()) and int(r.num_free) == 0
assert bool((r.slot_map[:B] == want * 16).all()) and bool((r.slot_map[B:] == -1).all())
"""


@pytest.mark.parametrize("B", [2048, 2560, 2816, 3024, 3025, 3048, 3072, 3073, 4096])
@pytest.mark.parametrize("tokens", [0, 50000])  # (one token a thread, or four)
def test_reserve_first_call_at_every_request_count(B, tokens):
    # in a process of its own: an earlier, larger call would have raised the shared-memory limit
    r = subprocess.run([sys.executable, "-c", _ONE_CALL, str(B), str(max(tokens, B))], cwd=ROOT, capture_output=True, text=True,
                       timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]


def _i(*x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("add", [(2 ** 31 - 1, 5), (2 ** 31 - 3, 5), (2 ** 30, 2 ** 30, 2 ** 30, 5), (2 ** 31 - 1,) * 40 + (5,),
                                 (7, 2 ** 31 - 1, 5, 2 ** 31 - 1, 70, 20)])
def test_oversized_additions_are_refused_and_take_nothing(add):
    # the sum of the additions passes 32 bits; those that fit are served all the same
    B, page, width, pages, tokens = len(add), 16, 4, 9, 10
    table, free = torch.full((B, width), -1, dtype=torch.int32, device=DEV), _i(*range(pages))
    r = bb.paged_reserve(_i(*[0] * B), _i(*add), table, free, _i(pages), page_size=page, num_tokens=tokens)
    stack, slots, positions = list(range(pages)), [], []
    for b, n in enumerate(add):
        ok = n <= width * page
        rows = [stack.pop() for _ in range(-(-n // page))] if ok else []
        assert table[b].tolist() == rows + [-1] * (width - len(rows)), b
        assert r.granted[b].item() == ok and r.lens[b].item() == (n if ok else 0), b
        for p in range(min(n, tokens - len(slots))):
            slots.append(rows[p // page] * page + p % page if ok else -1)
            positions.append(p if ok else -1)
    assert int(r.num_free) == len(stack)
    assert r.slot_map.tolist() == slots and r.positions.tolist() == positions


@pytest.mark.parametrize("tokens", [0, 1, 30, 47, 48, 49, 119, 120, 500])
def test_table_entries_past_the_slot_map(tokens):
    # the pages of granted tokens that slot_map has no entry for are in the table all the same
    lens, add, page = [5, 16, 0, 31], [40, 0, 70, 10], 16
    table = torch.full((4, 6), -1, dtype=torch.int32, device=DEV)
    table[0, 0], table[1, 0], table[3, :2] = 20, 21, _i(22, 23)
    r = bb.paged_reserve(_i(*lens), _i(*add), table, _i(*range(20)), _i(20), page_size=page, num_tokens=tokens)
    assert table.tolist() == [[20, 19, 18, -1, -1, -1], [21, -1, -1, -1, -1, -1], [17, 16, 15, 14, 13, -1], [22, 23, 12, -1, -1, -1]]
    assert int(r.num_free) == 12 and r.lens.tolist() == [45, 16, 70, 41]
    want = [int(table[b, p // page]) * page + p % page for b in range(4) for p in range(lens[b], lens[b] + add[b])]
    assert r.slot_map.tolist() == (want + [-1] * tokens)[:tokens]


def test_pages_asked_for_past_32_bits():
    # four requests of 2^30 pages each over a stack of ten: all are refused, and a later one too
    table = torch.empty(5, 2 ** 30, dtype=torch.int32, device=DEV)
    table[:, :3] = -1
    r = bb.paged_reserve(_i(0, 0, 0, 0, 0), _i(*[2 ** 30] * 4, 3), table, _i(*range(10)), _i(10), page_size=1, num_tokens=7)
    assert r.granted.tolist() == [False] * 5 and r.lens.tolist() == [0] * 5 and int(r.num_free) == 10
    assert r.slot_map.tolist() == [-1] * 7 and bool((table[:, :3] == -1).all())
