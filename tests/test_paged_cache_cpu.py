"""Refusals of PagedKVCache that need no device."""
import pytest

import butterfly_b200 as bb


def _cache(**kw):
    a = dict(num_layers=1, num_pages=4, page_size=16, num_kv_heads=1, head_dim=64, max_requests=3, max_tokens_per_request=64,
             device="cpu")
    a.update(kw)
    return bb.PagedKVCache(**a)


@pytest.mark.parametrize("requests", [0, -1, 4097, 10000])
def test_request_counts_that_no_reservation_takes(requests):
    with pytest.raises(ValueError, match="max_requests"):
        _cache(max_requests=requests)


def test_the_most_requests():
    assert _cache(max_requests=4096).max_requests == 4096


@pytest.mark.parametrize("rows", [[-1], [3], [0, 7]])
def test_release_of_rows_that_are_not_there(rows):
    with pytest.raises(ValueError, match="row"):
        _cache().release(rows)


@pytest.mark.parametrize("add,tokens", [([3, 0, 2], 4), ([1, 1, 1], 0), ([-5, 40, 0], 39)])
def test_slot_maps_shorter_than_the_tokens_of_a_host_list(add, tokens):
    with pytest.raises(ValueError, match="num_tokens"):
        _cache().reserve(add, tokens)


def test_host_lists_of_another_length():
    with pytest.raises(ValueError, match="one entry per row"):
        _cache().reserve([1, 1])


def test_capture_is_looked_up_on_the_tensors_device(monkeypatch):
    # a call on device 1, whose stream captures, while device 0 is current (the devices are stand-ins)
    from types import SimpleNamespace

    import torch

    from butterfly_b200 import paged
    current = [0]

    class Device:
        def __init__(self, index):
            self.index = index

        def __enter__(self):
            self.before, current[0] = current[0], self.index

        def __exit__(self, *a):
            current[0] = self.before

    x = SimpleNamespace(is_cuda=True, get_device=lambda: 1, device=1)
    monkeypatch.setattr(torch.cuda, "device", Device)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: current[0], raising=False)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: current[0] == 1)
    monkeypatch.setattr(paged, "decode_workspace", lambda device: object())
    monkeypatch.setattr(paged, "_workspaces", {})
    assert paged._workspace_for(x, 7) is not paged._workspace_for(x, 7) and not paged._workspaces
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    assert paged._workspace_for(x, 7) is paged._workspace_for(x, 7) and current == [0]
