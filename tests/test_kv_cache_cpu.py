"""PagedKVCache's host side, without a GPU: the calls it makes, recorded in
place of the library."""
import pytest

torch = pytest.importorskip("torch")

from mi_b200 import kv_cache  # noqa: E402


@pytest.fixture
def cache(monkeypatch):
    """(a cache of 2 layers x 8 pages with scores, the entry points it called)."""
    calls = []
    monkeypatch.setattr(kv_cache.capi, "call", lambda name, *a: calls.append(name))
    monkeypatch.setattr(kv_cache, "stream_of", lambda t: 0)
    c = kv_cache.PagedKVCache.__new__(kv_cache.PagedKVCache)
    c.device, c.dtype = torch.device("cpu"), torch.bfloat16
    c.page_size, c.num_layers, c.num_kv_heads, c.head_dim = 16, 2, 2, 64
    c.max_batch_size, c.max_pages_per_seq, c.max_num_pages = 2, 4, 8
    c.page_bytes = 2 * 16 * 2 * 64 * 2
    i32 = dict(dtype=torch.int32)
    c.layer_ptrs = torch.zeros(2, dtype=torch.int64)
    c.free_ring, c.pool_ctrl = torch.zeros(8, **i32), torch.zeros(4, **i32)
    c.page_table, c.slot_num_pages = torch.zeros(2, 4, **i32), torch.zeros(2, **i32)
    c.status = torch.zeros(1, **i32)
    c.score_data = torch.ones(2, 8, 2, 16)
    c.num_free_pages = 3
    return c, calls


@pytest.mark.parametrize("pages,cleared", [([9], []), ([-1, 8, 100], []), ([9, 5], [5]),
                                           ([2, 3], [2, 3])])
def test_release_with_scores_reaches_the_pool(cache, pages, cleared):
    """Pages outside the pool are the device's to flag, also when all are."""
    c, calls = cache
    c.release_pages(pages)
    assert calls == ["mi_page_release"]
    assert c.num_free_pages == 3 + len(pages)
    own = [p for p in range(8) if not c.score_data[:, p].any()]
    assert own == cleared


def test_every_launch_is_made_on_the_caches_device(cache, monkeypatch):
    """A stream handle does not name its device (every device's default stream is
    handle 0), so the cache's device has to be the current one at each launch,
    whichever is current at the call."""
    c, _ = cache
    current, calls = [], []

    class On:
        def __init__(self, t):
            self.t = t

        def __enter__(self):
            current.append(self.t.device)

        def __exit__(self, *a):
            current.pop()

    monkeypatch.setattr(kv_cache, "on_device_of", On)
    monkeypatch.setattr(kv_cache.capi, "call",
                        lambda name, *a: calls.append((name, bool(current))))
    i32 = lambda x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    c.evict(i32([0, 1]), i32([40, 20]), 16, 3, recent=4)
    c.slot_release(i32([0]), 1)
    c.release_pages([3])
    assert calls == [(n, True) for n in ("mi_step_prepare", "mi_kv_evict", "mi_slot_trim",
                                         "mi_slot_trim", "mi_page_release")]


def test_evict_passes_an_empty_slot_over(cache, monkeypatch):
    """A slot without tokens has no newest one: it goes in as a padding lane, not
    as position -1, which the device would flag."""
    c, _ = cache
    seen = []
    monkeypatch.setattr(c, "step_prepare", lambda slots, pos, *a, **k: seen.append(
        (slots.tolist(), pos.tolist())))
    i32 = lambda x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    c.evict(i32([1, 0]), i32([0, 40]), 16, 2)
    (slots, pos), = seen
    assert slots[0] == -1 and slots[1] == 0 and pos[1] == 39
