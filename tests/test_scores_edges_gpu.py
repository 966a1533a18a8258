"""Score and eviction calls at the edges of what they take."""
import numpy as np
import pytest

from oracle import scores_oracle as so

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from mi_b200.page import evict_paged_kv_cache  # noqa: E402
from mi_b200.prefill import BatchPrefillWithPagedKVCacheWrapper  # noqa: E402
from tests.test_scores_gpu import (DEV, TDT, _case, _check_scores, _decode_wrapper,  # noqa: E402
                                   _expected, _i32, _mag, _prompt_check)


@pytest.mark.parametrize("hq,hkv,d,ps,dtype", [(32, 8, 128, 16, "bfloat16"), (12, 3, 64, 16, "bfloat16"),
                                               (14, 2, 64, 16, "float32"), (4, 2, 80, 16, "bfloat16"),
                                               (16, 1, 64, 16, "bfloat16")])
def test_decode_scores_of_rows_without_a_weight(hq, hkv, d, ps, dtype):
    """Products that overflow to -inf for every token: such a head's output is 0
    and its log-sum-exp -inf, and it gives no token a weight (NaN would stay in
    the token's score for good)."""
    c = _case(3, [40, 33], hq, hkv, d, ps, dtype)
    c["t_pool"][:, 0, ..., 0] = torch.finfo(TDT[dtype]).max
    q = torch.zeros(2, hq, d, dtype=TDT[dtype], device=DEV)
    q[0, :, 0] = torch.finfo(TDT[dtype]).min    # request 0: every head
    q[1, 1::2, 0] = torch.finfo(TDT[dtype]).min  # request 1: every other head
    w = _decode_wrapper(c)
    out, lse = w.run(q, c["t_pool"], return_lse=True, scores=c["t_scores"])
    w.check_status()
    dead = torch.zeros(2, hq, dtype=torch.bool, device=DEV)
    dead[0], dead[1, 1::2] = True, True
    assert torch.equal(lse == -np.inf, dead) and not out[dead].any()
    got = c["t_scores"].double().cpu().numpy() - c["prior"]
    group = hq // hkv
    for b, n in enumerate((40, 33)):
        pages = c["indices"][c["indptr"][b]:c["indptr"][b + 1]]
        rows = got[pages].transpose(0, 2, 1).reshape(-1, hkv)[:n]
        # q = 0: each live head gives each token 1 / n
        live = [sum(not dead[b, h * group + g] for g in range(group)) for h in range(hkv)]
        assert np.abs(rows - np.array([int(x) for x in live]) / n).max() <= 1e-6


def test_evict_without_pages():
    """Requests that hold nothing at all: nothing to cut, nothing kept."""
    kv = torch.ones(4, 2, 16, 2, 64, device=DEV, dtype=torch.bfloat16)
    sc = torch.ones(4, 2, 16, device=DEV)
    kept = evict_paged_kv_cache(kv, sc, _i32([]), _i32([0, 0, 0]), _i32([0, 0]), 8,
                                return_kept=True)
    assert kept.shape == (2, 2, 8) and (kept == -1).all()
    assert (kv == 1).all() and (sc == 1).all()


def test_pages_past_32_bits():
    """Pages whose rows lie past 2^32 bytes and 2^31 elements of the pool: the same
    bits as in a small pool."""
    hq, hkv, d, ps = 32, 8, 128, 16
    c = _case(21, [300, 77], hq, hkv, d, ps, "bfloat16")
    far = 140_000
    kv = torch.empty(far + c["P"], 2, ps, hkv, d, dtype=torch.bfloat16, device=DEV)
    assert far * 2 * ps * hkv * d > 2 ** 32
    kv[far:] = c["t_pool"]
    sc = torch.zeros(far + c["P"], hkv, ps, device=DEV)
    sc[far:] = c["t_scores"]
    q = torch.randn(2, hq, d, device=DEV, generator=torch.Generator(DEV).manual_seed(1)).bfloat16()
    near = _decode_wrapper(c)
    want = near.run(q, c["t_pool"], scores=c["t_scores"])
    kept = evict_paged_kv_cache(c["t_pool"], c["t_scores"], c["t_indices"], c["t_indptr"],
                                c["t_last"], 64, recent=9, sinks=2, return_kept=True)
    c["t_indices"] = c["t_indices"] + far
    got = _decode_wrapper(c).run(q, kv, scores=sc)
    far_kept = evict_paged_kv_cache(kv, sc, c["t_indices"], c["t_indptr"], c["t_last"], 64,
                                    recent=9, sinks=2, return_kept=True)
    assert torch.equal(got, want) and torch.equal(far_kept, kept)
    assert torch.equal(sc[far:], c["t_scores"]) and torch.equal(kv[far:], c["t_pool"])
    assert not sc[:far].any()


def test_prompt_scores_of_pages_past_32_bits():
    hq, hkv, d, ps = 8, 8, 128, 16
    for dtype in ("bfloat16", "float32"):
        c = _case(22, [150], hq, hkv, d, ps, dtype)
        far = 140_000 if dtype == "bfloat16" else 70_000
        kv = torch.empty(far + c["P"], 2, ps, hkv, d, dtype=TDT[dtype], device=DEV)
        kv[far:] = c["t_pool"]
        sc = torch.zeros(far + c["P"], hkv, ps, device=DEV)
        sc[far:] = c["t_scores"]
        q = torch.randn(150, hq, d, device=DEV, generator=torch.Generator(DEV).manual_seed(1))
        q, lse = q.to(TDT[dtype]), torch.full((150, hq), 2.0, device=DEV)
        w = BatchPrefillWithPagedKVCacheWrapper(torch.zeros(1 << 20, dtype=torch.uint8, device=DEV))
        for pool, scores, base in ((c["t_pool"], c["t_scores"], 0), (kv, sc, far)):
            w.plan(_i32([0, 150]), c["t_indptr"], c["t_indices"] + base, c["t_last"], hq, hkv, d,
                   ps, causal=True)
            w.accumulate_scores(q, pool, lse, scores, window=70)
            w.check_status()
        assert torch.equal(sc[far:], c["t_scores"]) and not sc[:far].any()
        del kv, sc


@pytest.mark.parametrize("hq,hkv,d,dtype", [(28, 4, 128, "bfloat16"), (14, 2, 64, "float32"),
                                            (32, 32, 64, "float16")])
def test_decode_scores_of_long_requests(hq, hkv, d, dtype):
    lens = [20000, 1, 9001]
    c = _case(40, lens, hq, hkv, d, 16, dtype)
    q = torch.from_numpy(c["q"]).to(TDT[dtype]).to(DEV)
    w = _decode_wrapper(c)
    w.run(q, c["t_pool"], scores=c["t_scores"])
    w.check_status()
    add = _expected(c, lambda b, k: so.decode_weights(c["q"][b], k, d ** -0.5))
    _check_scores(c, add, c["t_scores"], hq // hkv + max(lens) / 16, _mag(c["q"], c))


@pytest.mark.parametrize("hq,hkv,d,dtype", [(28, 4, 128, "bfloat16"), (14, 2, 64, "float32")])
def test_prompt_scores_of_a_long_prompts_end(hq, hkv, d, dtype):
    lens = [12000, 3, 5000]
    _prompt_check(_case(41, lens, hq, hkv, d, 16, dtype), lens, [100, 3, 64], 64, True)
