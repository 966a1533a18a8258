"""Refusals of the score, eviction and sampling calls that need no GPU, and the
eviction oracle on cases written out by hand."""
import numpy as np
import pytest

from oracle import scores_oracle as so

torch = pytest.importorskip("torch")

from mi_b200 import capi  # noqa: E402
from mi_b200.page import evict_paged_kv_cache  # noqa: E402


def test_evict_oracle_by_hand():
    s = [0.1, 0.9, 0.2, 0.8, 0.3, 0.7, 0.4, 0.6]
    # 4 of 8, the last 1 and the first 1 stay: of 1..6 the best two are 1 and 3;
    # 1 stays, 3 fills slot 2
    assert so.evict_slots(s, 4, 1, 1) == [0, 1, 3, 7]
    # of 0..7 the best two are 1 and 3: 1 stays, 3 fills slot 0
    assert so.evict_slots(s, 2, 0, 0) == [3, 1]
    assert so.evict_slots(s, 3, 3, 0) == [5, 6, 7]
    assert so.evict_slots(s, 3, 0, 3) == [0, 1, 2]
    assert so.evict_slots([1.0] * 6, 3, 1, 0) == [0, 1, 5]           # ties: lowest slots
    assert so.evict_slots([np.nan, 0.0, np.nan, -np.inf], 2, 0, 0) == [3, 1]
    assert so.evict_slots(s[:3], 5, 1, 1) == [0, 1, 2, -1, -1]


def _args(layers=0):
    lead = (layers,) if layers else ()
    i32 = lambda x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    return dict(paged_kv_cache=torch.zeros(*lead, 4, 2, 16, 2, 64, dtype=torch.bfloat16),
                scores=torch.zeros(*lead, 4, 2, 16), kv_indices=i32([0, 1, 2]),
                kv_indptr=i32([0, 2, 3]), kv_last_page_len=i32([16, 3]), budget=8)


@pytest.mark.parametrize("layers", [0, 3])
@pytest.mark.parametrize("change,err", [
    (dict(budget=0), ValueError), (dict(recent=5, sinks=4), ValueError),
    (dict(recent=-1), ValueError), (dict(sinks=-1), ValueError), (dict(max_len=0), ValueError),
    (dict(scores=torch.zeros(4, 16, 2)), ValueError),
    (dict(scores=torch.zeros(4, 2, 16).double()), ValueError),
    (dict(kv_indices=torch.zeros(3)), TypeError),
    (dict(kv_last_page_len=torch.zeros(1, dtype=torch.int32)), ValueError),
    (dict(kv_indptr=torch.zeros(6, dtype=torch.int32)[::2]), ValueError),
    (dict(status=torch.zeros(1)), TypeError),
    ({}, capi.MiError),  # no CPU fallback
])
def test_evict_refusals(layers, change, err):
    with pytest.raises(err):
        evict_paged_kv_cache(**{**_args(layers), **change})


def test_evict_refuses_strided_layers():
    a = _args(4)
    a["paged_kv_cache"], a["scores"] = a["paged_kv_cache"][::2], a["scores"][:2]
    with pytest.raises(ValueError):
        evict_paged_kv_cache(**a)


def test_c_entries_refuse():
    lib = capi.lib()
    evict = lambda **k: lib.mi_kv_evict(  # noqa: E731
        None, k.get("kv", 256), 0, 256, 1, 4, 16, 2, k.get("d", 64), k.get("dt", capi.DTYPE_BF16),
        256, 256, 256, 1, k.get("max_len", 64), k.get("budget", 8), k.get("recent", 0),
        k.get("sinks", 0), None, None, None)
    for bad in (dict(kv=None), dict(budget=0), dict(recent=9), dict(recent=5, sinks=4),
                dict(recent=-1), dict(sinks=-1), dict(max_len=0), dict(dt=5), dict(d=0)):
        assert evict(**bad) == capi.ERR_INVALID, bad
    assert lib.mi_slot_trim(None, None, 4, None, None, 1, 1, None, 1, 0, None, 0, 0, None, 0,
                            None, None) == capi.ERR_INVALID
    assert lib.mi_paged_prefill_scores(None, 0, 0, None, 4, None, 4, 16, 2, 64, 2, None, None,
                                       None, 1, 4, 1, 0, 0.1, None, None, None, 0, None,
                                       None) == capi.ERR_INVALID
    n = lib.mi_paged_decode_scores_scratch_size(3, 8, 16, 5)
    assert n >= 5 * 16 * 8 * 4 + 3 * 8 * 4
    assert lib.mi_paged_decode_scores_scratch_size(0, 8, 16, 5) == 0
    dec = lambda scratch, hq: lib.mi_paged_decode_scores(  # noqa: E731
        256, 8, 8, None, 0, 0, None, 0, 0, None, None, 0, None, 256, 4, 16, 2, 64,
        capi.DTYPE_BF16, 256, 256, 5, 256, 3, hq, 0.1, 256, None, 256, 256, scratch, 256, 1 << 20,
        None, None)
    assert dec(n - 1, 8) == capi.ERR_WORKSPACE
    assert dec(n, 7) == capi.ERR_INVALID


def test_scheduler_request_defaults_are_plain():
    from mi_b200.scheduler import Request
    assert Request("a", [1], 4, 0.7).plain_sampling
    for kw in (dict(top_k=3), dict(top_p=0.9), dict(min_p=0.1), dict(seed=0), dict(logprobs=True)):
        assert not Request("a", [1], 4, 0.7, **kw).plain_sampling
    a, b = Request("a", [1], 4, 0.7, seed=5), Request("b", [1], 4, 0.7, seed=5)
    draws = [a.next_uniform() for _ in range(5)]
    assert draws == [b.next_uniform() for _ in range(5)]
    assert all(0 <= u < 1 and np.float32(u) == u for u in draws)
