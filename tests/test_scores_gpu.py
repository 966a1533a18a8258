"""Accumulated attention weights (decode and prompt) against 64-bit softmax.

Tolerance of a weight, derived: a logit's dot product of d terms accumulated
in fp32 is off by at most (d + 8) 2^-23 of the sum of its terms' magnitudes
(tensor-core accumulation truncates, hence 2^-23 a step), and the exponent's
argument, the row's log-sum-exp and the exponential add at most 64 * 2^-23
(arguments below 32 in size, a few roundings each). Weights are positive, so
their sums keep that relative error, plus 2^-24 per addition.
"""
import math

import numpy as np
import pytest

from oracle import scores_oracle as so
from tests.gpu_cases import paged_case

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from mi_b200 import capi  # noqa: E402
from mi_b200.decode import BatchDecodeWithPagedKVCacheWrapper  # noqa: E402
from mi_b200.page import append_paged_kv_cache, evict_paged_kv_cache  # noqa: E402
from mi_b200.prefill import BatchPrefillWithPagedKVCacheWrapper  # noqa: E402

DEV = "cuda"
TDT = {"bfloat16": torch.bfloat16, "float16": torch.float16, "float32": torch.float32}


def _i32(x):
    return torch.as_tensor(np.asarray(x, np.int32), device=DEV)


def _t(x, dtype):
    return torch.from_numpy(np.ascontiguousarray(x)).to(TDT[dtype]).to(DEV)


def _case(seed, lens, hq, hkv, d, ps, dtype):
    c = paged_case(seed, lens, hq, hkv, d, page_size=ps, dtype=dtype)
    c["t_pool"] = _t(c["pool"], dtype)
    for k in ("indptr", "indices", "last"):
        c["t_" + k] = _i32(c[k])
    c["prior"] = np.random.default_rng(seed + 1).random((c["P"], hkv, ps)).astype(np.float32)
    c["t_scores"] = torch.from_numpy(c["prior"].copy()).to(DEV)
    return c


def _decode_wrapper(c):
    w = BatchDecodeWithPagedKVCacheWrapper(torch.zeros(64 << 20, dtype=torch.uint8, device=DEV))
    w.plan(c["t_indptr"], c["t_indices"], c["t_last"], c["hq"], c["hkv"], c["d"], c["ps"])
    return w


def _check_scores(c, want_add, got, terms, mag):
    """got == prior + want_add within the bound; untouched slots are untouched."""
    got = got.double().cpu().numpy()
    prior = c["prior"].astype(np.float64)
    rel = (c["d"] + 8) * 2.0 ** -23 * mag + 64 * 2.0 ** -23 + terms * 2.0 ** -24
    tol = want_add * rel + 2.0 ** -24 * (prior + want_add) + 1e-38
    bad = np.abs(got - prior - want_add) > tol
    assert not bad.any(), (np.argwhere(bad)[:5], np.abs(got - prior - want_add).max(), rel)
    assert (got[want_add == 0] == prior[want_add == 0]).all()


def _expected(c, weights_of):
    """[P, Hkv, ps] additions; weights_of(b, k) -> [n, Hkv]."""
    add = np.zeros((c["P"], c["hkv"], c["ps"]))
    for b in range(len(c["lens"])):
        pages, n = so.request_tokens(c["indptr"], c["indices"], c["last"], b, c["ps"])
        if n == 0:
            continue
        k = c["pool"][pages, 0].reshape(-1, c["hkv"], c["d"])[:n]
        w = np.zeros((len(pages) * c["ps"], c["hkv"]))
        w[:n] = weights_of(b, k)
        add[pages] += w.reshape(len(pages), c["ps"], -1).transpose(0, 2, 1)
    return add


def _mag(q, c):
    """Bound of sum |q_i k_i| * scale over the rows (Cauchy-Schwarz on magnitudes)."""
    qn = np.sqrt((q.astype(np.float64) ** 2).sum(-1)).max()
    kn = np.sqrt((c["pool"][:, 0].astype(np.float64) ** 2).sum(-1)).max()
    return qn * kn / math.sqrt(c["d"])


SHAPES = [  # hq, hkv, d, ps, dtype
    (32, 8, 128, 16, "bfloat16"), (28, 4, 128, 16, "float16"), (14, 2, 64, 16, "bfloat16"),
    (14, 2, 64, 16, "float32"), (16, 1, 128, 32, "bfloat16"), (8, 8, 64, 16, "float16"),
    (16, 2, 128, 48, "bfloat16"), (12, 3, 128, 16, "bfloat16"), (6, 3, 80, 7, "float32"),
    (32, 32, 64, 16, "bfloat16"), (40, 2, 128, 16, "bfloat16"), (4, 2, 256, 5, "float16"),
]


@pytest.mark.parametrize("hq,hkv,d,ps,dtype", SHAPES)
@pytest.mark.parametrize("lens", [[1], [16], [17, 1, 500, 33], [3000, 5, 0, 64, 1200, 15]])
def test_decode_scores(hq, hkv, d, ps, dtype, lens):
    c = _case(hq + d + len(lens), lens, hq, hkv, d, ps, dtype)
    q = _t(c["q"], dtype)
    w = _decode_wrapper(c)
    want, want_lse = w.run(q, c["t_pool"], return_lse=True)
    out, lse = w.run(q, c["t_pool"], return_lse=True, scores=c["t_scores"])
    w.check_status()
    if dtype != "float32" and d in (64, 128) and hq // hkv <= 16:
        assert torch.equal(out, want) and torch.equal(lse, want_lse)
    else:  # other kernels than run()'s: both within a few fp32 roundings and the output's own
        half = torch.finfo(out.dtype).eps / 2
        gap = (out.double() - want.double()).abs()
        assert (gap <= 2 * half * want.double().abs() + 1e-4).all(), gap.max()
        fin = torch.isfinite(want_lse)
        assert torch.equal(fin, torch.isfinite(lse))
        assert (lse[fin] - want_lse[fin]).abs().max() <= 1e-4
    scale = 1 / math.sqrt(d)
    add = _expected(c, lambda b, k: so.decode_weights(c["q"][b], k, scale))
    _check_scores(c, add, c["t_scores"], hq // hkv + max(lens) / 16, _mag(c["q"], c))


def test_decode_scores_accumulate_and_repeat():
    """Two steps add up; the same step on the same state gives the same bits;
    captured and replayed it follows its inputs."""
    c = _case(5, [700, 90, 2500], 32, 8, 128, 16, "bfloat16")
    q = _t(c["q"], "bfloat16")
    w = _decode_wrapper(c)
    a, b = c["t_scores"].clone(), c["t_scores"].clone()
    w.run(q, c["t_pool"], scores=a)
    w.run(q, c["t_pool"], scores=b)
    assert torch.equal(a, b)
    once = a.clone()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    out = torch.empty_like(q)
    with torch.cuda.stream(s):
        w.run(q, c["t_pool"], out=out, scores=b)
    s.synchronize()
    with torch.cuda.graph(g):
        w.run(q, c["t_pool"], out=out, scores=a)
    a.copy_(c["t_scores"])
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(a, once)
    q.copy_(q.flip(0))
    a.copy_(c["t_scores"])
    g.replay()
    c["q"] = c["q"][::-1]
    add = _expected(c, lambda i, k: so.decode_weights(c["q"][i], k, 1 / math.sqrt(128)))
    _check_scores(c, add, a, 4 + 2500 / 16, _mag(c["q"], c))


def test_decode_scores_bad_page_and_extreme_logits():
    """A bad page's tokens are left out and flagged; huge logits give one-hot weights."""
    c = _case(9, [200, 64], 32, 8, 128, 16, "bfloat16")
    idx = c["t_indices"].clone()
    idx[3] = c["P"] + 7
    c["t_indices"] = idx
    w = _decode_wrapper(c)
    q = _t(c["q"] * 40, "bfloat16")
    w.run(q, c["t_pool"], scores=c["t_scores"])
    with pytest.raises(capi.MiError, match="BAD_PAGE"):
        w.check_status()
    got = c["t_scores"].double().cpu().numpy() - c["prior"]
    assert np.isfinite(got).all()
    pages = c["indices"]
    hole = pages[3]
    assert (got[hole] == 0).all()
    # every query head gives a weight of 1 in all (fp32 sums over 4 heads' tokens)
    for b, n in ((0, 200), (1, 64)):
        own = pages[c["indptr"][b]:c["indptr"][b + 1]]
        total = got[own].sum((0, 2))
        assert np.abs(total - 4).max() < 1e-4, total


@pytest.mark.parametrize("hq,hkv,d,ps,dtype", [(32, 8, 128, 16, "bfloat16"),
                                               (14, 2, 64, 16, "float16"),
                                               (14, 2, 64, 16, "float32"),
                                               (12, 3, 128, 16, "bfloat16")])
def test_decode_scores_with_append_and_positions(hq, hkv, d, ps, dtype):
    """run_with_append(scores, rope_positions) is the append at those positions
    followed by run(scores): pages, output and scores bit for bit."""
    lens = [40, 1, 129, 1000]
    c = _case(21, lens, hq, hkv, d, ps, dtype)
    g = torch.Generator(device=DEV).manual_seed(1)
    mk = lambda h: torch.randn(4, h, d, device=DEV, generator=g).to(TDT[dtype])  # noqa: E731
    q, k, v = mk(hq), mk(hkv), mk(hkv)
    ang = torch.rand(4096, d, device=DEV, generator=g) * 6
    cos, sin = ang.cos().to(TDT[dtype]), ang.sin().to(TDT[dtype])
    rope_pos = _i32([3000, 17, 129, 2222])
    w = _decode_wrapper(c)
    pool_a, sc_a = c["t_pool"].clone(), c["t_scores"].clone()
    q_rot = torch.empty_like(q)
    append_paged_kv_cache(k, v, torch.arange(4, dtype=torch.int32, device=DEV),
                          _i32([n - 1 for n in lens]), pool_a, c["t_indices"], c["t_indptr"],
                          c["t_last"], rope_cos=cos, rope_sin=sin, rope_positions=rope_pos, q=q,
                          q_out=q_rot)
    want = w.run(q_rot, pool_a, scores=sc_a)
    pool_b, sc_b = c["t_pool"].clone(), c["t_scores"].clone()
    out = w.run_with_append(q, pool_b, k, v, cos, sin, scores=sc_b, rope_positions=rope_pos)
    w.check_status()
    assert torch.equal(pool_a, pool_b) and torch.equal(out, want) and torch.equal(sc_a, sc_b)
    # without rope_positions: the same as run_with_append alone
    pool_c, pool_d = c["t_pool"].clone(), c["t_pool"].clone()
    a = w.run_with_append(q, pool_c, k, v, cos, sin)
    b = w.run_with_append(q, pool_d, k, v, cos, sin, scores=c["t_scores"].clone())
    assert torch.equal(pool_c, pool_d)
    assert torch.equal(a, b) or (dtype == "float32" and (a - b).abs().max() <= 1e-4)


@pytest.mark.parametrize("hq,hkv,d,ps,dtype", SHAPES)
@pytest.mark.parametrize("lens,window", [([1], 0), ([77], 0), ([77], 1), ([130, 1, 300], 0),
                                         ([700, 40, 0, 129], 32), ([257, 128], 64),
                                         ([500], 1000)])
def test_prompt_scores(hq, hkv, d, ps, dtype, lens, window):
    c = _case(hq + d + len(lens) + window, lens, hq, hkv, d, ps, dtype)
    _prompt_check(c, lens, lens, window, True)


def _prompt_check(c, lens, nq, window, causal, strides=False):
    dtype, d, hq, hkv = c["dtype"], c["d"], c["hq"], c["hkv"]
    rng = np.random.default_rng(3)
    q = _t(rng.standard_normal((sum(nq), hq, d), dtype=np.float32), dtype)
    qh = q.float().cpu().numpy()
    if strides:  # heads of a fused projection's output
        big = torch.zeros(sum(nq), hq + 2 * hkv, d, dtype=q.dtype, device=DEV)
        big[:, :hq] = q
        q = big[:, :hq]
    qo = np.concatenate([[0], np.cumsum(nq)])
    w = BatchPrefillWithPagedKVCacheWrapper(torch.zeros(1 << 20, dtype=torch.uint8, device=DEV))
    w.plan(_i32(qo), c["t_indptr"], c["t_indices"], c["t_last"], hq, hkv, d, c["ps"],
           causal=causal)
    scale = 1 / math.sqrt(d)
    # the rows' log-sum-exp in 64 bits, rounded once
    lse = np.full((sum(nq), hq), -np.inf, np.float32)
    for b in range(len(lens)):
        pages, n = so.request_tokens(c["indptr"], c["indices"], c["last"], b, c["ps"])
        if not n or not nq[b]:
            continue
        k = c["pool"][pages, 0].reshape(-1, hkv, d)[:n].astype(np.float64)
        for h in range(hq):
            z = qh[qo[b]:qo[b + 1], h].astype(np.float64) @ k[:, h // (hq // hkv)].T * scale
            if causal:
                z = np.where(np.arange(n)[None] <= (n - nq[b] + np.arange(nq[b]))[:, None], z,
                             -np.inf)
            m = z.max(-1)
            ok = np.isfinite(m)
            lse[qo[b]:qo[b + 1], h][ok] = (
                m[ok] + np.log(np.exp(z[ok] - m[ok, None]).sum(-1))).astype(np.float32)
    t_lse = torch.from_numpy(lse).to(DEV)
    w.accumulate_scores(q, c["t_pool"], t_lse, c["t_scores"], window=window)
    w.check_status()
    add = _expected(c, lambda b, k: so.prompt_weights(qh[qo[b]:qo[b + 1]], k, scale, window,
                                                      causal, lse[qo[b]:qo[b + 1]]))
    rows = (min(max(nq), window) if window else max(nq)) * hq // hkv
    _check_scores(c, add, c["t_scores"], rows, _mag(qh, c))


@pytest.mark.parametrize("dtype,d", [("bfloat16", 128), ("float16", 64), ("float32", 64)])
@pytest.mark.parametrize("nq,lens,causal", [([5, 40], [200, 40], True), ([30, 7], [20, 7], True),
                                            ([5, 40], [200, 41], False), ([0, 9], [50, 100], True),
                                            ([150, 3], [400, 0], True)])
def test_prompt_scores_chunks(dtype, d, nq, lens, causal):
    """Queries that are only the prompt's end (chunked prefill), more queries than
    keys (rows that see nothing), no mask, no queries, no keys."""
    c = _case(31, lens, 8, 2, d, 16, dtype)
    _prompt_check(c, lens, nq, 0, causal, strides=True)


def test_prompt_scores_follow_prefill():
    """With the log-sum-exp that run() returns, a prompt's weights add up to one
    per query and head."""
    lens = [300, 45]
    c = _case(8, lens, 32, 8, 128, 16, "bfloat16")
    g = torch.Generator(device=DEV).manual_seed(2)
    q = torch.randn(345, 32, 128, device=DEV, generator=g).bfloat16()
    w = BatchPrefillWithPagedKVCacheWrapper(torch.zeros(1 << 20, dtype=torch.uint8, device=DEV))
    w.plan(_i32([0, 300, 345]), c["t_indptr"], c["t_indices"], c["t_last"], 32, 8, 128, 16,
           causal=True)
    _, lse = w.run(q, c["t_pool"], return_lse=True)
    scores = torch.zeros(c["P"], 8, 16, device=DEV)
    w.accumulate_scores(q, c["t_pool"], lse, scores)
    w.check_status()
    for b, n in enumerate(lens):
        own = torch.as_tensor(c["indices"][c["indptr"][b]:c["indptr"][b + 1]], device=DEV).long()
        total = scores[own].double().sum((0, 2)).cpu()
        assert ((total / (4 * n) - 1).abs() < 1e-5).all(), total


def test_prompt_scores_bad_page():
    c = _case(9, [200], 32, 8, 128, 16, "bfloat16")
    c["t_indices"][3] = -4
    w = BatchPrefillWithPagedKVCacheWrapper(torch.zeros(1 << 20, dtype=torch.uint8, device=DEV))
    w.plan(_i32([0, 200]), c["t_indptr"], c["t_indices"], c["t_last"], 32, 8, 128, 16, causal=True)
    q = torch.zeros(200, 32, 128, device=DEV, dtype=torch.bfloat16)
    w.accumulate_scores(q, c["t_pool"], torch.zeros(200, 32, device=DEV), c["t_scores"])
    with pytest.raises(capi.MiError, match="BAD_PAGE"):
        w.check_status()
    got = c["t_scores"].double().cpu().numpy() - c["prior"]
    assert (got[c["indices"][3]] == 0).all()
    # q = 0, lse = 0: each query and head gives 1 to each token it sees
    assert got[c["indices"][0], :, 0] == pytest.approx(800.0, rel=1e-5)


# ---- eviction ----------------------------------------------------------------
def _evict_check(c, budget, recent, sinks, scores, layers=0):
    kv, sc = c["pool"].copy(), scores.copy()
    t_kv, t_sc = _t(kv, c["dtype"]), torch.from_numpy(sc.copy()).to(DEV)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    got = evict_paged_kv_cache(t_kv, t_sc, c["t_indices"], c["t_indptr"], c["t_last"], budget,
                               recent=recent, sinks=sinks, return_kept=True, status=status)
    kept = so.evict(kv, sc, c["indptr"], c["indices"], c["last"], budget, recent, sinks)
    assert int(status.item()) == 0
    assert np.array_equal(got.cpu().numpy(), kept)
    assert np.array_equal(t_kv.float().cpu().numpy(), kv)
    assert np.array_equal(t_sc.cpu().numpy(), sc, equal_nan=True)


@pytest.mark.parametrize("hq,hkv,d,ps,dtype", [(4, 4, 128, 16, "bfloat16"), (2, 2, 64, 16, "float32"),
                                               (3, 3, 80, 7, "float16"), (1, 1, 256, 32, "float32"),
                                               (2, 2, 5, 3, "bfloat16"), (2, 2, 9, 16, "float32")])
@pytest.mark.parametrize("lens,budget,recent,sinks", [
    ([100, 64, 65, 0, 30], 64, 16, 4), ([500], 1, 0, 0), ([500], 1, 1, 0), ([90, 33], 32, 32, 0),
    ([90, 33], 32, 0, 32), ([90, 700], 32, 20, 12), ([1000, 41, 333], 40, 0, 0),
    ([300], 290, 250, 3), ([2000, 1999], 1024, 128, 4)])
def test_evict(hq, hkv, d, ps, dtype, lens, budget, recent, sinks):
    c = _case(len(lens) + budget, lens, hq, hkv, d, ps, dtype)
    _evict_check(c, budget, recent, sinks, c["prior"])


@pytest.mark.parametrize("kind", ["equal", "few", "special", "negative"])
def test_evict_ties_and_special_scores(kind):
    c = _case(3, [400, 150, 77], 4, 4, 64, 16, "bfloat16")
    s = c["prior"].copy()
    if kind == "equal":
        s[:] = 0.5
    elif kind == "few":
        s = np.round(s * 3).astype(np.float32)
    elif kind == "negative":
        s = np.round((s - 0.5) * 8).astype(np.float32) / 8
        s[s == 0] = -0.0
        s[::2][s[::2] == 0] = 0.0
    else:
        r = np.random.default_rng(0).integers(0, 6, s.shape)
        s[r == 0], s[r == 1], s[r == 2] = np.inf, -np.inf, np.nan
        s[r == 3] = np.finfo(np.float32).tiny / 4
    for budget, recent, sinks in ((64, 10, 2), (100, 0, 0), (20, 20, 0)):
        _evict_check(c, budget, recent, sinks, s)


def test_evict_layers_and_repeat():
    """Layers in one tensor choose by themselves; a second call with the new
    length changes nothing; two streams' calls do not meet."""
    c = _case(17, [260, 40, 900], 2, 2, 64, 16, "bfloat16")
    layers = 3
    rng = np.random.default_rng(5)
    kv = np.stack([np.roll(c["pool"], i, axis=-1) for i in range(layers)])
    sc = rng.random((layers, c["P"], 2, 16)).astype(np.float32)
    t_kv, t_sc = _t(kv, "bfloat16"), torch.from_numpy(sc.copy()).to(DEV)
    got = evict_paged_kv_cache(t_kv, t_sc, c["t_indices"], c["t_indptr"], c["t_last"], 200,
                               recent=33, sinks=1, return_kept=True)
    for l in range(layers):
        kept = so.evict(kv[l], sc[l], c["indptr"], c["indices"], c["last"], 200, 33, 1)
        assert np.array_equal(got[l].cpu().numpy(), kept)
    assert np.array_equal(t_kv.float().cpu().numpy(), kv)
    assert np.array_equal(t_sc.cpu().numpy(), sc)
    # cut to 200 tokens: 13 pages each now
    indptr, last = _i32([0, 13, 16, 29]), _i32([8, 8, 8])
    first = c["indptr"]
    idx = np.concatenate([c["indices"][first[0]:first[0] + 13], c["indices"][first[1]:first[1] + 3],
                          c["indices"][first[2]:first[2] + 13]])
    before = t_kv.clone()
    evict_paged_kv_cache(t_kv, t_sc, _i32(idx), indptr, last, 200, recent=33, sinks=1)
    assert torch.equal(before, t_kv) and np.array_equal(t_sc.cpu().numpy(), sc)


def test_evict_leaves_bad_requests():
    c = _case(2, [100, 100], 2, 2, 64, 16, "bfloat16")
    c["t_indices"][2] = 999
    kv, sc = c["t_pool"].clone(), c["t_scores"].clone()
    st = torch.zeros(1, dtype=torch.int32, device=DEV)
    kept = evict_paged_kv_cache(kv, sc, c["t_indices"], c["t_indptr"], c["t_last"], 50, status=st,
                                return_kept=True)
    assert capi.status_names(int(st.item())) == ["BAD_PAGE"]
    own = torch.as_tensor(c["indices"][:7], device=DEV).long()
    assert torch.equal(kv[own], c["t_pool"][own]) and torch.equal(sc[own], c["t_scores"][own])
    assert (kept[0] == -1).all() and (kept[1] >= 0).all()
    st.zero_()
    kept = evict_paged_kv_cache(kv, sc, c["t_indices"], c["t_indptr"], c["t_last"], 50, status=st,
                                return_kept=True, max_len=99)
    assert "BAD_POSITION" in capi.status_names(int(st.item()))
    assert (kept == -1).all()
