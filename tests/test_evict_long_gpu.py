"""Eviction of long requests: past what a CTA keeps of the scores in shared memory
(10360 tokens where max_len allows it, else 6504), at the lengths around both, and
with page tables whose requests add up to far more than the longest."""
import numpy as np
import pytest

from oracle import scores_oracle as so

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from mi_b200 import capi  # noqa: E402
from mi_b200.page import evict_paged_kv_cache  # noqa: E402
from tests.test_scores_gpu import DEV, _case, _t  # noqa: E402


def _check(c, budget, recent, sinks, scores, **kw):
    kv, sc = c["pool"].copy(), scores.copy()
    t_kv, t_sc = _t(kv, c["dtype"]), torch.from_numpy(sc.copy()).to(DEV)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    got = evict_paged_kv_cache(t_kv, t_sc, c["t_indices"], c["t_indptr"], c["t_last"], budget,
                               recent=recent, sinks=sinks, return_kept=True, status=status, **kw)
    kept = so.evict(kv, sc, c["indptr"], c["indices"], c["last"], budget, recent, sinks)
    assert int(status.item()) == 0
    assert np.array_equal(got.cpu().numpy(), kept)
    assert np.array_equal(t_kv.float().cpu().numpy(), kv)
    assert np.array_equal(t_sc.cpu().numpy(), sc, equal_nan=True)


@pytest.mark.parametrize("max_len", [None, "longest"])
@pytest.mark.parametrize("lens,budget,recent,sinks", [
    ([4112, 4097, 100, 4096], 4096, 1024, 4),    # decoding at a budget
    ([9000, 24000, 3], 4096, 1024, 4),           # long prompts
    ([10359, 10360, 10361, 10400], 2000, 100, 1), ([10360, 10329], 2000, 100, 1),
    ([6503, 6504, 6505, 6529], 2000, 100, 1),
    ([24000], 23000, 0, 0), ([12000], 11000, 10998, 2), ([15000, 11000], 1, 0, 0)])
def test_long_requests(lens, budget, recent, sinks, max_len):
    c = _case(len(lens) + budget, lens, 2, 2, 64, 16, "bfloat16")
    _check(c, budget, recent, sinks, c["prior"],
           **({} if max_len is None else {"max_len": max(lens)}))


@pytest.mark.parametrize("kind", ["equal", "few", "special"])
def test_long_requests_with_ties(kind):
    """Ties at the threshold across the warps' segments, NaN and infinities."""
    c = _case(5, [13000, 10500, 9999], 2, 2, 16, 16, "float16")
    s = c["prior"].copy()
    if kind == "equal":
        s[:] = 0.5
    elif kind == "few":
        s = np.round(s * 3).astype(np.float32)
    else:
        r = np.random.default_rng(0).integers(0, 6, s.shape)
        s[r == 0], s[r == 1], s[r == 2] = np.inf, -np.inf, np.nan
        s[r == 3] = -0.0
    for budget, recent, sinks in ((9000, 300, 2), (300, 0, 0)):
        _check(c, budget, recent, sinks, s)


@pytest.mark.parametrize("dtype,d", [("float32", 9), ("bfloat16", 5)])
def test_long_requests_of_odd_rows(dtype, d):
    c = _case(8, [11111, 4000], 1, 1, d, 7, dtype)
    _check(c, 3999, 777, 3, c["prior"])


def test_many_requests_by_the_tables_bound():
    """64 requests of 8192 slots: without max_len the bound is all of them."""
    rng = np.random.default_rng(2)
    c = _case(6, rng.integers(8100, 8193, 64).tolist(), 1, 1, 16, 16, "float16")
    _check(c, 8000, 512, 4, c["prior"])


def test_a_request_past_the_bound_is_left():
    c = _case(9, [12000, 20000], 1, 1, 16, 16, "float16")
    kv, sc = c["t_pool"].clone(), c["t_scores"].clone()
    st = torch.zeros(1, dtype=torch.int32, device=DEV)
    kept = evict_paged_kv_cache(kv, sc, c["t_indices"], c["t_indptr"], c["t_last"], 500, status=st,
                                return_kept=True, max_len=12000)
    assert capi.status_names(int(st.item())) == ["BAD_POSITION"]
    assert (kept[1] == -1).all() and (kept[0] >= 0).all()
    own = torch.as_tensor(c["indices"][c["indptr"][1]:], device=DEV).long()
    assert torch.equal(kv[own], c["t_pool"][own]) and torch.equal(sc[own], c["t_scores"][own])
