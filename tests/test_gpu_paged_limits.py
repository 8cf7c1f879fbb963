"""The paged cache at its limits: request counts around the shared-memory bounds, probabilities far below their row's maximum.

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
