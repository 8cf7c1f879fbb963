"""What the paged cache keeps between calls: workspaces, and the state that captured calls go on from."""
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


# ------------------------------------------------------------------------------ captured steps
def _filled(seed, lens, layers=2):
    rnd, cache = _rnd(seed), _cache(num_layers=layers)
    r = cache.reserve(lens)
    for layer in range(layers):
        cache.append(layer, rnd(sum(lens), 2, 128), rnd(sum(lens), 2, 128), r.slot_map)
    return rnd, cache


def _step(cache, add, q, kn, vn):
    r = cache.reserve(add, q.shape[0])
    outs = [cache.attend(layer, q, k_new=kn, v_new=vn, active=r.granted) for layer in range(2)]
    return outs + [r.lens, r.num_free, r.slot_map, r.positions, r.granted]


def test_replayed_steps_advance_like_eager_ones():
    lens = [30, 200, 0]
    rnd, eager = _filled(3, lens)
    _, cache = _filled(3, lens)
    q, kn, vn = rnd(3, 8, 1, 128), rnd(3, 2, 1, 128), rnd(3, 2, 1, 128)
    add = torch.tensor([1, 1, 0], dtype=torch.int32, device=DEV)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        got = _step(cache, add, q, kn, vn)
    assert cache.lens.tolist() == lens  # a capture runs nothing
    for i in range(40):  # (through several pages)
        if i == 20:  # requests come and go between replays
            for c in (eager, cache):
                c.release([1])
                r = c.reserve([0, 33, 70])
                for layer in range(2):
                    rows = _rnd(9)(2, 103, 2, 128)
                    c.append(layer, rows[0], rows[1], r.slot_map)
        for x in (q, kn, vn):
            x.copy_(rnd(*x.shape))
        want = _step(eager, add, q, kn, vn)
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), i
        for name in ("lens", "num_free", "block_table", "free_pages"):
            assert torch.equal(getattr(cache, name), getattr(eager, name)), (i, name)
    assert cache.lens.tolist() == [70, 53, 70]


def test_captured_attention_reads_the_lengths_of_its_replay():
    rnd, cache = _filled(4, [30, 200, 5])
    q = rnd(3, 8, 1, 128)
    cache.attend(0, q)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        got = cache.attend(0, q, return_lse=True)
    for add in ([100, 1, 0], [0, 0, 900], [-60, 300, -905]):
        r = cache.reserve(add)
        n = sum(max(x, 0) for x in add)
        cache.append(0, rnd(n, 2, 128), rnd(n, 2, 128), r.slot_map)
        junk = [torch.full((4,), 10 ** 6, dtype=torch.int32, device=DEV) for _ in range(64)]  # over what the call let go of
        graph.replay()
        want = cache.attend(0, q, return_lse=True)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        del junk


def test_lengths_handed_out_are_of_their_time():
    _, cache = _filled(5, [3, 0, 40])
    before, free = cache.lens, cache.num_free
    r = cache.reserve([1, 50, -40])
    assert before.tolist() == [3, 0, 40] and cache.lens.tolist() == [4, 50, 0] == r.lens.tolist()
    cache.reserve([1, 1, 1])
    assert r.lens.tolist() == [4, 50, 0] and cache.lens.tolist() == [5, 51, 1]
    cache.lens, cache.num_free = before, free
    assert cache.lens.tolist() == [3, 0, 40] and torch.equal(cache.num_free, free)


@pytest.mark.parametrize("inside", ["make", "use", "both"])
def test_inference_mode(inside):
    with torch.inference_mode(inside != "use"):
        rnd, cache = _filled(6, [30, 0, 5])
    with torch.inference_mode(inside != "make"):
        q, kn, vn = rnd(3, 8, 1, 128), rnd(3, 2, 1, 128), rnd(3, 2, 1, 128)
        add = torch.tensor([1, 0, 1], dtype=torch.int32, device=DEV)
        for i in range(2):
            out = _step(cache, add, q, kn, vn)
            assert cache.lens.tolist() == [31 + i, 0, 6 + i] == out[2].tolist()
        cache.lens = cache.lens - 1
        assert cache.lens.tolist() == [31, -1, 6]
        paged.reset_workspaces()
