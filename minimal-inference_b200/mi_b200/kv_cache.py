"""Paged KV cache with a device-side page pool (kernel 4).

``PagedKVCache`` keeps the reference's interface and layout
(scheduler.py:168-221): per-layer ``kv_data[P, 2, ps, Hkv, D]`` (NHD, K at
index 0), ``P = max_batch * ceil(max_seq/ps)``, page ``P-1`` reserved as the
scratch page, FIFO allocation, zero-on-release. The free list lives on the
GPU (``free_ring`` + ``pool_ctrl``) and is driven by the library's pool
kernels, so page tables come out identical to the reference's while the
decode step's page growth can run inside a CUDA graph.

Two ways to use it:

* the reference's list API -- ``allocate_pages(n) -> list[int]`` and
  ``release_pages(pages)`` (one launch for all pages and layers). These read
  the popped ids back to the host, i.e. they synchronise.
* the slot API the graph-captured scheduler uses -- each request owns a
  slot row of ``page_table`` on the device; ``slot_alloc`` (admission),
  ``step_prepare`` (page growth + CSR for a step) and ``slot_release``
  (retire) never synchronise.

``track_scores`` adds one fp32 score per cached token, KV head and layer
(``score_data``), which the attention calls accumulate and ``evict`` ranks by:
a slot longer than a budget is cut to it and its freed pages return to the
pool. Scores of free pages are zero, as their K and V are.

The host keeps an exact mirror of the free-page count (``num_free_pages``),
so admission control and the out-of-pages error (scheduler.py:208-214) need
no device read.
"""
from __future__ import annotations

import math

import torch

from . import capi
from ._tensor import dtype_code, need_i32, on_device_of, ptr, stream_of


class _FreeCount:
    """``len()``-able stand-in for the reference's ``free_pages`` deque."""

    def __init__(self, cache: "PagedKVCache"):
        self._c = cache

    def __len__(self) -> int:
        return self._c.num_free_pages


class PagedKVCache:
    def __init__(self, config, max_batch_size: int, max_seq_len: int, page_size: int,
                 device, dtype: torch.dtype, num_layers: int | None = None,
                 num_kv_heads: int | None = None, track_scores: bool = False):
        device = torch.device(device)
        if device.type != "cuda":
            raise capi.MiError("PagedKVCache lives on a CUDA device (no CPU fallback)")
        self.page_size = page_size
        self.num_layers = config.num_hidden_layers if num_layers is None else num_layers
        self.num_kv_heads = config.num_key_value_heads if num_kv_heads is None else num_kv_heads
        self.head_dim = config.head_dim
        self.device, self.dtype = device, dtype
        self.max_batch_size = max_batch_size
        self.max_pages_per_seq = math.ceil(max_seq_len / page_size)
        self.max_num_pages = max_batch_size * self.max_pages_per_seq
        self.kv_data: list[torch.Tensor] = [
            torch.zeros(self.max_num_pages, 2, page_size, self.num_kv_heads, self.head_dim,
                        device=device, dtype=dtype)
            for _ in range(self.num_layers)
        ]
        self.scratch_page = self.max_num_pages - 1
        self.page_bytes = 2 * page_size * self.num_kv_heads * self.head_dim * \
            torch.empty((), dtype=dtype).element_size()
        self.layer_ptrs = torch.tensor([t.data_ptr() for t in self.kv_data], dtype=torch.int64,
                                       device=device)
        i32 = dict(dtype=torch.int32, device=device)
        self.free_ring = torch.empty(self.max_num_pages, **i32)
        self.pool_ctrl = torch.zeros(4, **i32)
        self.page_table = torch.full((max_batch_size, self.max_pages_per_seq), -1, **i32)
        self.slot_num_pages = torch.zeros(max_batch_size, **i32)
        self.status = torch.zeros(1, **i32)
        self._call("mi_page_pool_init", self.free_ring.data_ptr(), self.pool_ctrl.data_ptr(),
                   self.max_num_pages, stream_of(self.free_ring))
        # accumulated attention weights [layers, P, Hkv, ps], or None
        self.score_data = (torch.zeros(self.num_layers, self.max_num_pages, self.num_kv_heads,
                                       page_size, device=device) if track_scores else None)
        self.num_free_pages = self.max_num_pages - 1
        self.free_pages = _FreeCount(self)

    def _call(self, name: str, *args) -> None:
        """An entry point, launched on the cache's device whichever is current."""
        with on_device_of(self.page_table):
            capi.call(name, *args)

    # ---- reference list API ---------------------------------------------
    def allocate_pages(self, num_pages: int) -> list[int]:
        """Pop ``num_pages`` pages FIFO (scheduler.py:208-214); synchronises."""
        if self.num_free_pages < num_pages:
            raise RuntimeError(
                f"Cannot allocate {num_pages} pages, only {self.num_free_pages} free")
        if num_pages == 0:
            return []
        counts = torch.tensor([num_pages], dtype=torch.int32, device=self.device)
        out = torch.empty(num_pages, dtype=torch.int32, device=self.device)
        self._call("mi_page_alloc", self.free_ring.data_ptr(), self.pool_ctrl.data_ptr(),
                   self.max_num_pages, counts.data_ptr(), 1, out.data_ptr(),
                   self.status.data_ptr(), stream_of(out))
        self.num_free_pages -= num_pages
        return out.tolist()

    def release_pages(self, page_indices) -> None:
        """Zero the pages in every layer, then free them (scheduler.py:216-221)."""
        pages = [int(p) for p in page_indices]
        if not pages:
            return
        t = torch.tensor(pages, dtype=torch.int32, device=self.device)
        if self.score_data is not None:
            own = [p for p in pages if 0 <= p < self.max_num_pages]  # others are flagged below
            self.score_data.index_fill_(
                1, torch.tensor(own, dtype=torch.int64, device=self.device), 0.0)
        self._call("mi_page_release", self.free_ring.data_ptr(), self.pool_ctrl.data_ptr(),
                   self.max_num_pages, t.data_ptr(), len(pages), self.layer_ptrs.data_ptr(),
                   self.num_layers, self.page_bytes, self.status.data_ptr(), stream_of(t))
        self.num_free_pages += len(pages)

    # ---- slot API (no host synchronisation) --------------------------------
    def slot_alloc(self, slots: torch.Tensor, counts: torch.Tensor, total: int) -> None:
        """Admission: pop ``counts[i]`` pages into slot ``slots[i]`` (device int32)."""
        if self.num_free_pages < total:
            raise RuntimeError(
                f"Cannot allocate {total} pages, only {self.num_free_pages} free")
        self._call("mi_slot_alloc", self.free_ring.data_ptr(), self.pool_ctrl.data_ptr(),
                   self.max_num_pages, self.page_table.data_ptr(), self.slot_num_pages.data_ptr(),
                   self.max_batch_size, self.max_pages_per_seq, slots.data_ptr(),
                   counts.data_ptr(), slots.numel(), self.status.data_ptr(), stream_of(slots))
        self.num_free_pages -= total

    def slot_release(self, slots: torch.Tensor, total_pages: int) -> None:
        """Retire: zero every page of ``slots`` in every layer and free them."""
        if self.score_data is not None:
            self._trim(slots, 0, total_pages)
            return
        self._call("mi_slot_release", self.free_ring.data_ptr(), self.pool_ctrl.data_ptr(),
                   self.max_num_pages, self.page_table.data_ptr(), self.slot_num_pages.data_ptr(),
                   self.max_batch_size, self.max_pages_per_seq, slots.data_ptr(), slots.numel(),
                   self.layer_ptrs.data_ptr(), self.num_layers, self.page_bytes,
                   self.status.data_ptr(), stream_of(slots))
        self.num_free_pages += total_pages

    def _trim(self, slots: torch.Tensor, keep_pages: int, freed_pages: int) -> None:
        """Free the pages of ``slots`` from the ``keep_pages``-th on, zeroed."""
        sc = self.score_data
        self._call("mi_slot_trim", self.free_ring.data_ptr(), self.pool_ctrl.data_ptr(),
                   self.max_num_pages, self.page_table.data_ptr(), self.slot_num_pages.data_ptr(),
                   self.max_batch_size, self.max_pages_per_seq, slots.data_ptr(), slots.numel(),
                   keep_pages, self.layer_ptrs.data_ptr(), self.num_layers, self.page_bytes,
                   ptr(sc), self.num_kv_heads * self.page_size, self.status.data_ptr(),
                   stream_of(slots))
        self.num_free_pages += freed_pages

    def evict(self, slots: torch.Tensor, lengths: torch.Tensor, budget: int,
              freed_pages: int, *, recent: int = 0, sinks: int = 0) -> None:
        """Cut each of ``slots`` (holding ``lengths`` tokens, both device int32)
        to at most ``budget`` tokens by accumulated score, in every layer and KV
        head (``page.evict_paged_kv_cache``), and free the pages past the
        budget. ``slots`` must be distinct. ``freed_pages``: how many that is
        over all slots (the caller knows the lengths). A slot's next token goes
        to position ``min(length, budget)`` of its pages. Does not
        synchronise."""
        if self.score_data is None:
            raise RuntimeError("evict() needs PagedKVCache(track_scores=True)")
        if budget < 1 or recent < 0 or sinks < 0 or recent + sinks > budget:
            raise ValueError(f"need 0 <= recent + sinks <= budget, got {recent} + {sinks}, "
                             f"{budget}")
        n = slots.numel()
        need_i32("slots", slots, self.page_table.device)
        need_i32("lengths", lengths, self.page_table.device)
        if lengths.numel() != n:
            raise ValueError("slots and lengths differ in length")
        if n == 0:
            return
        i32 = dict(dtype=torch.int32, device=self.device)
        indptr, last, unused = (torch.empty(n + 1, **i32), torch.empty(n, **i32),
                                torch.empty(n, **i32))
        indices = torch.empty(n * self.max_pages_per_seq, **i32)
        lanes = torch.where(lengths > 0, slots, -1)  # an empty slot: a padding lane
        self.step_prepare(lanes, lengths - 1, indptr, indices, last, unused, grow=False)
        self._call("mi_kv_evict", self.layer_ptrs.data_ptr(), None, 0, self.score_data.data_ptr(),
                   self.num_layers, self.max_num_pages, self.page_size, self.num_kv_heads,
                   self.head_dim, dtype_code(self.dtype), indptr.data_ptr(), indices.data_ptr(),
                   last.data_ptr(), n, self.max_pages_per_seq * self.page_size, budget, recent,
                   sinks, None, self.status.data_ptr(), stream_of(slots))
        self._trim(slots, math.ceil(budget / self.page_size), freed_pages)

    def step_prepare(self, lane_slots: torch.Tensor, lane_positions: torch.Tensor,
                     kv_indptr: torch.Tensor, kv_indices: torch.Tensor,
                     kv_last_page_len: torch.Tensor, append_positions: torch.Tensor,
                     grow: bool = True) -> None:
        """Page growth + CSR metadata of one step, all on the device.

        Graph-capturable. The caller accounts for grown pages in
        ``num_free_pages`` (it knows positions on the host).
        """
        self._call("mi_step_prepare", self.free_ring.data_ptr(), self.pool_ctrl.data_ptr(),
                   self.max_num_pages, self.page_table.data_ptr(), self.slot_num_pages.data_ptr(),
                   self.max_batch_size, self.max_pages_per_seq, lane_slots.data_ptr(),
                   lane_positions.data_ptr(), lane_slots.numel(), self.page_size, int(grow),
                   kv_indptr.data_ptr(), kv_indices.data_ptr(), kv_indices.numel(),
                   kv_last_page_len.data_ptr(), append_positions.data_ptr(),
                   self.status.data_ptr(), stream_of(lane_slots))

    def slot_pages(self, slot: int) -> list[int]:
        """Pages held by ``slot`` (reads the device table; synchronises)."""
        n = int(self.slot_num_pages[slot].item())
        return self.page_table[slot, :n].tolist()

    def check_status(self) -> None:
        w = int(self.status.item())
        if w:
            self.status.zero_()
            if w == 1:
                raise RuntimeError("page pool exhausted on the device (OUT_OF_PAGES)")
            raise capi.MiError(f"page pool device status: {capi.status_names(w)}")
