"""Paged key/value cache: requests of different lengths, and decode over their whole context.

``CompressedKVCache`` keeps one offset for a whole batch and a bounded window per sequence.  The
layers that keep ordinary (dense) attention, served to requests that come and go, need the
other kind: keys and values in pages of ``page_size`` tokens from one pool, a block table per
request, and attention that reads through the table.

  paged_reserve            pages, slots and positions for a step's tokens, from the requests'
                           lengths (block tables and the free-page stack stay on the GPU)
  paged_append             the tokens' key / value rows into their slots
  paged_decode_attention   one new token per request over its pages, optionally writing that
                           token's rows in the same launch
  PagedKVCache             the three of them over per-layer pools

Pools are ``[pages, Hkv, page_size, dh]`` views (``page_size`` a multiple of 16, ``dh`` 64, 128
or 256; rows of ``dh`` contiguous), so token-major pages are a transposed view.  Everything is
enqueued on the current stream and nothing waits for the host.
"""
from __future__ import annotations

import ctypes
import math
import weakref
from typing import NamedTuple, Optional, Sequence

import torch

from . import _lib

MAX_REQUESTS = 4096  # requests of one reservation call
RELEASE = -2 ** 31  # an ``add`` entry that gives all of a request's pages back


class PagedReservation(NamedTuple):
    """What ``paged_reserve`` returns, all on the device."""
    lens: torch.Tensor        # [B] int32 lengths after the call
    num_free: torch.Tensor    # [1] int32 pages left on the stack
    slot_map: torch.Tensor    # [num_tokens] int64, -1 for refused and unused entries
    positions: torch.Tensor   # [num_tokens] int32, -1 likewise
    granted: torch.Tensor     # [B] bool: this request's added tokens have slots


_raw_stream = torch._C._cuda_getCurrentRawStream  # the current stream's handle, without a Stream object
_native = None


def _binding():
    """The compiled binding (csrc/binding.cpp), given the C entry points of the loaded library."""
    global _native
    if _native is None:
        try:
            from . import _native as mod
        except ImportError as e:
            raise ImportError(f"butterfly_b200/_native.so is missing or stale: build it with "
                              f"`python -m butterfly_b200.build` ({e})") from e
        L = _lib.lib()
        mod.init(*(ctypes.cast(f, ctypes.c_void_p).value for f in (L.bna_paged_reserve, L.bna_paged_append,
                                                                  L.bna_paged_decode)))
        _native = mod
    return _native


def _stream(x: torch.Tensor) -> int:
    return _raw_stream(x.get_device()) if x.is_cuda else 0  # (a CPU tensor is refused further on)


def paged_reserve(lens: torch.Tensor, add: torch.Tensor, block_table: torch.Tensor, free_pages: torch.Tensor,
                  num_free: torch.Tensor, *, page_size: int, num_tokens: int) -> PagedReservation:
    """Room for ``add[b]`` more tokens of every request (``lens``, ``add`` [B] int32).

    ``add > 0`` takes the pages the request's ``block_table`` row [B, width] lacks from the top
    of the stack ``free_pages[:num_free]``; ``add < 0`` takes tokens back (a rollback; ``RELEASE``
    for a request that is done) and returns pages emptied by it.  Requests are served in order
    while pages last; one that is refused (``add > 0`` and not ``granted``) keeps its length.  The added
    tokens of request 0, then 1, ... are entries 0, 1, ... of ``slot_map`` and ``positions``
    (``num_tokens`` of them: at least the sum of the positive ``add``).  ``block_table`` and
    ``free_pages`` are updated in place, the lengths and the stack height are returned.  A page
    belongs to one row: one that two rows name would come back on the stack twice."""
    r = (_native or _binding()).reserve(lens, add, block_table, free_pages, num_free, page_size, num_tokens, _stream(lens),
                                        None)
    if r.__class__ is int:
        _lib.check(r)
    return PagedReservation(*r)


def paged_append(k: torch.Tensor, v: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                 slot_map: torch.Tensor) -> None:
    """Write token t's rows ``k[t]`` / ``v[t]`` ([tokens, Hkv, dh], any token and head strides)
    into slot ``slot_map[t]`` (int64) of the pools; negative slots are skipped."""
    _lib.check((_native or _binding()).append(k, v, k_pages, v_pages, slot_map, _stream(k)))


_workspaces: dict = {}  # (device, stream) -> the workspace kept for it
_made: dict = {}  # id -> weak reference to every workspace there is, for reset_workspaces


def decode_workspace(device: torch.device | str | int = "cuda") -> torch.Tensor:
    """A workspace for ``paged_decode_attention`` calls that follow one another on a stream."""
    with torch.inference_mode(False):  # (an inference tensor could not be zeroed again outside that mode)
        ws = torch.empty(_lib.lib().bna_paged_decode_workspace_bytes(), dtype=torch.uint8, device=device)
        ws[:4096].zero_()  # the arrival counters; every call leaves them zero
    key = id(ws)
    _made[key] = weakref.ref(ws, lambda _: _made.pop(key, None))
    return ws


def reset_workspaces(device: torch.device | str | int = "cuda") -> None:
    """Zero the counters of every ``decode_workspace`` of a device (those kept per stream and the caches'
    own among them), after its kernels have ended.  Needed where a call did not run to its end (see
    ``take_device_error``) or its lengths were changed while it ran: counts left by such a call
    would make later ones leave out work."""
    device = torch.empty(0, device=device).device
    torch.cuda.synchronize(device)
    for ref in list(_made.values()):
        ws = ref()
        if ws is not None and ws.device == device:
            ws[:4096].zero_()
    torch.cuda.synchronize(device)


def _read_device_error(device: int) -> int:
    code = ctypes.c_int32()
    _lib.check(_lib.lib().bna_take_device_error(device, ctypes.byref(code)))
    return code.value


def take_device_error(device: torch.device | str | int = "cuda") -> int:
    """Read and clear a device's error word, once its kernels have ended: 0, or the site of the first wait
    that a kernel gave up since the last call.  What kernels wrote since then is not to be used;
    the workspaces are made usable again (``reset_workspaces``)."""
    device = torch.empty(0, device=device).device
    torch.cuda.synchronize(device)
    code = _read_device_error(device.index)
    if code:
        reset_workspaces(device)
    return code


def _workspace_for(x: torch.Tensor, stream: int) -> torch.Tensor:
    """The workspace kept for a stream.  A call under capture gets its own (zeroed inside the graph;
    pass one to share it): its replays may run beside later calls on the stream."""
    if not x.is_cuda:
        raise ValueError("butterfly_b200 kernels run on CUDA tensors only (no CPU path)")
    if torch._C._cuda_getDevice() == x.get_device():
        capturing = torch.cuda.is_current_stream_capturing()
    else:
        with torch.cuda.device(x.device):  # (the question is about the current device's stream)
            capturing = torch.cuda.is_current_stream_capturing()
    if capturing:
        return decode_workspace(x.device)
    ws = _workspaces.get((x.get_device(), stream))
    if ws is None:
        ws = _workspaces[(x.get_device(), stream)] = decode_workspace(x.device)
    return ws


def paged_decode_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, block_table: torch.Tensor,
                           lens: torch.Tensor, *, k_new: Optional[torch.Tensor] = None,
                           v_new: Optional[torch.Tensor] = None, active: Optional[torch.Tensor] = None,
                           window: int = 0, scale: Optional[float] = None, return_lse: bool = False,
                           workspace: Optional[torch.Tensor] = None):
    """Attention of one new token per request: q [B,Hq,1,dh] over the first ``lens[b]`` tokens of
    request b (the last ``window`` of them where ``window`` > 0).  ``lens`` counts the new token.

    With ``k_new`` / ``v_new`` [B,Hkv,1,dh] the new token's rows are read from there and written
    into their slot by the same launch (in place of ``paged_append``) for the requests that
    ``active`` [B] bool names (default: all; pass ``PagedReservation.granted`` where some
    requests got no room, or rest).  Returns [B,Hq,1,dh] in q's dtype, contiguous (so that
    ``transpose(1, 2)`` is [B,1,Hq,dh] storage); with ``return_lse`` also the fp32 natural-log sums
    [B,Hq,1].  A request of length 0 gives zeros and -inf; an infinite value attended to gives an
    infinity or NaN in its column.  ``workspace`` (``decode_workspace``)
    defaults to one kept per stream; calls that may overlap need one each.  Lengths and tables
    must not change while the call runs; ``take_device_error`` tells whether a kernel gave up."""
    stream = _stream(q)
    r = (_native or _binding()).decode(
        q, k_pages, v_pages, block_table, lens, k_new, v_new, active, window,
        1.0 / math.sqrt(q.shape[-1] or 1) if scale is None else scale, return_lse,
        _workspace_for(q, stream) if workspace is None else workspace, stream)
    if r.__class__ is int:
        _lib.check(r)
    return r


class PagedKVCache:
    """Pools of ``num_layers`` layers under one set of block tables, lengths and free pages.

    The requests are the ``max_requests`` rows of the tables; a row of length 0 is vacant.  The
    cache's state (lengths, stack height, tables, the attention's workspace) stays at one address
    and moves on in stream order, so calls may be captured: a replayed ``reserve`` (with a device
    tensor) advances the requests from wherever they are then, a replayed ``attend`` reads their
    lengths of then.  Calls on one cache, and replays of graphs that hold them, follow one another."""

    def __init__(self, *, num_layers: int, num_pages: int, page_size: int, num_kv_heads: int, head_dim: int,
                 max_requests: int, max_tokens_per_request: int, dtype: torch.dtype = torch.bfloat16,
                 device: torch.device | str = "cuda") -> None:
        if not 0 < int(max_requests) <= MAX_REQUESTS:
            raise ValueError(f"max_requests must be in [1, {MAX_REQUESTS}], what one reservation serves")
        self.page_size = int(page_size)
        shape = (int(num_pages), int(num_kv_heads), self.page_size, int(head_dim))
        # every read goes through a row written before, so the pools need no clearing
        self.k_pages = [torch.empty(shape, dtype=dtype, device=device) for _ in range(int(num_layers))]
        self.v_pages = [torch.empty(shape, dtype=dtype, device=device) for _ in range(int(num_layers))]
        width = -(-int(max_tokens_per_request) // self.page_size)
        self.block_table = torch.full((int(max_requests), width), -1, dtype=torch.int32, device=device)
        with torch.inference_mode(False):  # (updated in place, in whichever mode the caller is then)
            self._state = torch.zeros(int(max_requests) + 1, dtype=torch.int32, device=device)
            self._lens, self._num_free = self._state[:-1], self._state[-1:]
            self._num_free.fill_(int(num_pages))
        self.free_pages = torch.arange(int(num_pages) - 1, -1, -1, dtype=torch.int32, device=device)
        self.workspace = decode_workspace(device)

    @property
    def max_requests(self) -> int:
        return int(self._lens.shape[0])

    @property
    def lens(self) -> torch.Tensor:
        """The requests' lengths [max_requests] int32, as of now (a copy; assign to set them)."""
        return self._lens.clone()

    @lens.setter
    def lens(self, value: torch.Tensor) -> None:
        self._lens.copy_(value)

    @property
    def num_free(self) -> torch.Tensor:
        """The free pages' number [1] int32, as of now (a copy; assign to set it)."""
        return self._num_free.clone()

    @num_free.setter
    def num_free(self, value: torch.Tensor) -> None:
        self._num_free.copy_(value)

    @property
    def nbytes(self) -> int:
        """Bytes of all pools (what the cache holds on the device, used or not)."""
        return sum(x.numel() * x.element_size() for x in self.k_pages + self.v_pages)

    def reserve(self, add: torch.Tensor | Sequence[int], num_tokens: Optional[int] = None) -> PagedReservation:
        """Advance every request by ``add`` tokens (see ``paged_reserve``); done once per step, for
        all layers.  ``num_tokens`` may be left out when ``add`` is a host sequence."""
        if not isinstance(add, torch.Tensor):
            add = [int(x) for x in add]
            if len(add) != self.max_requests:
                raise ValueError("add must have one entry per row")
            added = sum(max(x, 0) for x in add)
            if num_tokens is None:
                num_tokens = added
            elif num_tokens < added:
                raise ValueError(f"num_tokens is {num_tokens}, but add has {added} tokens to give slots to")
            add = torch.tensor(add, dtype=torch.int32).to(self._state.device, non_blocking=True)
        if num_tokens is None:
            raise ValueError("num_tokens is needed when add is a device tensor")
        r = (_native or _binding()).reserve(self._lens, add, self.block_table, self.free_pages, self._num_free, self.page_size,
                                            num_tokens, _stream(self._state), self._state)
        if r.__class__ is int:
            _lib.check(r)
        return PagedReservation(*r)

    def release(self, rows: Sequence[int]) -> None:
        """Give back all pages of the requests in ``rows``."""
        add = [0] * self.max_requests
        for b in rows:
            if not 0 <= int(b) < self.max_requests:
                raise ValueError(f"there is no row {int(b)}: the cache has {self.max_requests}")
            add[int(b)] = RELEASE
        self.reserve(add)

    def append(self, layer: int, k: torch.Tensor, v: torch.Tensor, slot_map: torch.Tensor) -> None:
        """The reserved tokens' rows [tokens, Hkv, dh] of one layer into their slots."""
        paged_append(k, v, self.k_pages[layer], self.v_pages[layer], slot_map)

    def attend(self, layer: int, q: torch.Tensor, *, k_new: Optional[torch.Tensor] = None,
               v_new: Optional[torch.Tensor] = None, active: Optional[torch.Tensor] = None, window: int = 0,
               scale: Optional[float] = None, return_lse: bool = False):
        """One new token per request, q [max_requests,Hq,1,dh], over its cached context (see
        ``paged_decode_attention``)."""
        return paged_decode_attention(q, self.k_pages[layer], self.v_pages[layer], self.block_table, self._lens,
                                      k_new=k_new, v_new=v_new, active=active, window=window, scale=scale,
                                      return_lse=return_lse, workspace=self.workspace)


__all__ = ["PagedKVCache", "PagedReservation", "RELEASE", "decode_workspace", "paged_append", "paged_decode_attention", "paged_reserve",
           "reset_workspaces", "take_device_error"]
