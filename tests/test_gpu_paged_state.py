"""What the paged cache keeps between calls: workspaces."""
import pytest
import torch

import butterfly_b200 as bb
from butterfly_b200 import paged

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _rnd(seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return lambda *s: torch.randn(*s, generator=g, device=DEV).bfloat16()


def _cache(**kw):
    a = dict(num_layers=1, num_pages=400, page_size=16, num_kv_heads=2, head_dim=128, max_requests=3, max_tokens_per_request=4096)
    a.update(kw)
    return bb.PagedKVCache(**a)


# ------------------------------------------------------------------------------ workspaces
@pytest.mark.parametrize("how", ["reset", "error"])
def test_counters_of_a_call_that_gave_up_are_zeroed(how, monkeypatch):
    rnd, cache = _rnd(1), _cache()
    lens = [4000, 17, 600]
    cache.append(0, rnd(sum(lens), 2, 128), rnd(sum(lens), 2, 128), cache.reserve(lens).slot_map)
    q, own = rnd(3, 8, 1, 128), paged.decode_workspace()
    calls = [lambda: cache.attend(0, q, return_lse=True),
             lambda: bb.paged_decode_attention(q, cache.k_pages[0], cache.v_pages[0], cache.block_table, cache.lens, return_lse=True),
             lambda: bb.paged_decode_attention(q, cache.k_pages[0], cache.v_pages[0], cache.block_table, cache.lens, return_lse=True,
                                               workspace=own)]
    want = [f() for f in calls]
    kept = paged._workspaces[(torch.cuda.current_device(), torch.cuda.current_stream().cuda_stream)]
    for ws in (cache.workspace, kept, own):  # as a call that ended early may leave them
        assert not bool(ws[:4096].any())
        ws[:4096].view(torch.int32)[::3] = 5
    if how == "reset":
        paged.reset_workspaces()
    else:
        monkeypatch.setattr(paged, "_read_device_error", lambda device: 0x1041)
        assert paged.take_device_error(DEV) == 0x1041
    for ws in (cache.workspace, kept, own):
        assert not bool(ws[:4096].any())
    for f, (out, lse) in zip(calls, want):
        got = f()
        assert torch.equal(got[0], out) and torch.equal(got[1], lse)


def test_no_error_and_no_reset_without_a_failure():
    ws = paged.decode_workspace()
    ws[4095] = 1
    assert paged.take_device_error() == 0
    assert int(ws[4095]) == 1
    key = id(ws)
    assert key in paged._made
    del ws
    assert key not in paged._made
