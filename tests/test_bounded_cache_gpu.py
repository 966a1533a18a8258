"""The operators together, as the scheduler uses them: prompt scores, eviction,
decode steps over the cut cache, sampling -- at the level of the cache against
64-bit attention over the kept tokens, and through the scheduler.
"""
import dataclasses
import math

import numpy as np
import pytest

from oracle import scores_oracle as so

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from mi_b200.decode import BatchDecodeWithPagedKVCacheWrapper  # noqa: E402
from mi_b200.kv_cache import PagedKVCache  # noqa: E402
from mi_b200.page import append_paged_kv_cache  # noqa: E402
from mi_b200.prefill import BatchPrefillWithPagedKVCacheWrapper  # noqa: E402

DEV = "cuda"


def _i32(x):
    return torch.as_tensor(np.asarray(x, np.int32), device=DEV)


def _all_free_and_zero(kv):
    kv.check_status()
    P = kv.max_num_pages
    assert int(kv.pool_ctrl[1].item()) == P - 1 == kv.num_free_pages
    head, ring = int(kv.pool_ctrl[0].item()), kv.free_ring.cpu().numpy()
    assert sorted(int(ring[(head + i) % P]) for i in range(P - 1)) == list(range(P - 1))
    if kv.score_data is not None:
        assert not kv.score_data[:, :P - 1].any()
    for t in kv.kv_data:
        assert not t[:P - 1].any()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_prompt_evict_decode_against_dense_attention(dtype):
    hq, hkv, d, ps = 8, 2, 64, 16
    lens, budget, recent, sinks, window = [150, 40, 97], 64, 16, 3, 24

    class Cfg:
        num_hidden_layers, num_key_value_heads, head_dim = 1, hkv, d

    kv = PagedKVCache(Cfg, 4, 256, ps, DEV, dtype, track_scores=True)
    slots = _i32([3, 0, 2])
    kv.slot_alloc(slots, _i32([math.ceil(n / ps) for n in lens]),
                  sum(math.ceil(n / ps) for n in lens))
    csr = lambda: (torch.empty(4, dtype=torch.int32, device=DEV),  # noqa: E731
                   torch.empty(3 * kv.max_pages_per_seq, dtype=torch.int32, device=DEV),
                   torch.empty(3, dtype=torch.int32, device=DEV),
                   torch.empty(3, dtype=torch.int32, device=DEV))
    indptr, indices, last, apos = csr()
    kv.step_prepare(slots, _i32([n - 1 for n in lens]), indptr, indices, last, apos, grow=False)
    g = torch.Generator(device=DEV).manual_seed(4)
    rnd = lambda *s: torch.randn(*s, device=DEV, generator=g).to(dtype)  # noqa: E731
    total = sum(lens)
    q, k, v = rnd(total, hq, d) * 1.5, rnd(total, hkv, d), rnd(total, hkv, d)
    qo = np.concatenate([[0], np.cumsum(lens)])
    append_paged_kv_cache(k, v, _i32(np.repeat(np.arange(3), lens)),
                          _i32(np.concatenate([np.arange(n) for n in lens])), kv.kv_data[0],
                          indices, indptr, last)
    pre = BatchPrefillWithPagedKVCacheWrapper(torch.zeros(1 << 16, dtype=torch.uint8, device=DEV))
    pre.plan(_i32(qo), indptr, indices, last, hq, hkv, d, ps, causal=True)
    _, lse = pre.run(q, kv.kv_data[0], return_lse=True)
    pre.accumulate_scores(q, kv.kv_data[0], lse, kv.score_data[0], window=window)
    scale = 1 / math.sqrt(d)
    host = lambda t: t.double().cpu().numpy()  # noqa: E731
    scores = host(kv.score_data[0])
    dense = []  # per request and head: kept K, V rows and their scores
    for b, n in enumerate(lens):
        pages = kv.slot_pages(int(slots[b]))
        got = scores[pages].transpose(0, 2, 1).reshape(-1, hkv)[:n]
        rows = slice(qo[b], qo[b + 1])
        want = so.prompt_weights(host(q[rows]), host(k[rows]), scale, window)
        # a logit is off by (d + 8) 2^-23 of the sum of its terms' sizes (below 30 here), the
        # row's log-sum-exp likewise
        assert np.abs(got - want).max() <= 2 * (d + 8) * 2.0 ** -23 * 30 * want.max()
        heads = []
        for h in range(hkv):
            src = [s for s in so.evict_slots(got[:, h], budget, recent, sinks) if s >= 0]
            heads.append((host(k[rows])[src, h], host(v[rows])[src, h], got[src, h]))
        dense.append(heads)
    freed = sum(math.ceil(n / ps) - math.ceil(min(n, budget) / ps) for n in lens)
    free_before = kv.num_free_pages
    kv.evict(slots, _i32(lens), budget, freed, recent=recent, sinks=sinks)
    kv.check_status()
    assert kv.num_free_pages == free_before + freed == int(kv.pool_ctrl[1].item())
    # two decode steps over what is left: new tokens at the cut slots, rotated by their position
    cached = [min(n, budget) for n in lens]
    ang = torch.rand(512, d, device=DEV, generator=g) * 6
    cos, sin = torch.cos(ang).to(dtype), torch.sin(ang).to(dtype)
    dec = BatchDecodeWithPagedKVCacheWrapper(torch.zeros(8 << 20, dtype=torch.uint8, device=DEV))
    for step in range(2):
        indptr, indices, last, apos = csr()
        kv.step_prepare(slots, _i32(cached), indptr, indices, last, apos, grow=True)
        dec.plan(indptr, indices, last, hq, hkv, d, ps)
        qd, kd, vd = rnd(3, hq, d), rnd(3, hkv, d), rnd(3, hkv, d)
        pos = [n + step for n in lens]
        out = dec.run_with_append(qd, kv.kv_data[0], kd, vd, cos, sin, positions=apos,
                                  scores=kv.score_data[0], rope_positions=_i32(pos))
        dec.check_status()

        def rot(x):
            x = x.float()
            half = torch.cat([-x[..., d // 2:], x[..., :d // 2]], -1)
            c, s = cos[pos].float()[:, None], sin[pos].float()[:, None]
            return ((x * c).to(dtype).float() + (half * s).to(dtype).float()).to(dtype)

        qr, kr = host(rot(qd)), host(rot(kd))
        for b in range(3):
            pages = kv.slot_pages(int(slots[b]))
            flat = host(kv.score_data[0])[pages].transpose(0, 2, 1).reshape(-1, hkv)
            for h in range(hkv):
                kk, vv, ss = dense[b][h]
                kk = np.concatenate([kk, kr[b, h][None]])
                vv = np.concatenate([vv, host(vd)[b, h][None]])
                z = qr[b, h * 4:h * 4 + 4] @ kk.T * scale
                w = np.exp(z - z.max(-1, keepdims=True))
                w /= w.sum(-1, keepdims=True)
                assert np.abs(host(out)[b, h * 4:h * 4 + 4] - w @ vv).max() <= 2e-2
                ss = np.concatenate([ss, [0.0]]) + w.sum(0)
                n = len(ss)
                assert np.abs(flat[:n, h] - ss).max() <= 2 * (d + 8) * 2.0 ** -23 * 30 * 4 + 2e-6
                assert (flat[n:, h] == 0).all()
                dense[b][h] = (kk, vv, ss)
        cached = [n + 1 for n in cached]
    kv.slot_release(slots, sum(math.ceil(n / ps) for n in cached))
    kv.num_free_pages = int(kv.pool_ctrl[1].item())  # pages the steps grew
    _all_free_and_zero(kv)


def _model(layers=2, seed=9):
    from mi_b200.model import PRESETS, Model
    cfg = dataclasses.replace(PRESETS["qwen2.5-0.5b"], num_hidden_layers=layers)
    return cfg, Model.create(cfg, torch.device(DEV, 0), torch.bfloat16, seed=seed)


def _serve(cfg, model, prompts, new=40, **kw):
    from mi_b200.scheduler import Request, Scheduler
    reqkw = kw.pop("requests", [{}] * len(prompts))
    sched = Scheduler(model, cfg, torch.device(DEV, 0), torch.bfloat16, max_batch_size=4,
                      max_seq_len=512, page_size=16, eos_token_ids=set(), **kw)
    reqs = [Request(f"r{i}", p, new, rk.pop("temperature", 0.0), **rk)
            for i, (p, rk) in enumerate(zip(prompts, [dict(r) for r in reqkw]))]
    for r in reqs:
        sched.submit_request(r)
    peak = 0
    for _ in range(400):
        if not (sched.active_requests or sched.waiting_queue):
            break
        sched.step()
        peak = max([peak] + [r.cached_len for r in sched.active_requests])
    assert not sched.active_requests
    torch.cuda.synchronize()
    _all_free_and_zero(sched.kv_cache)
    out = [list(r.generated_tokens) for r in reqs]
    sched.close()
    return out, reqs, peak


def _prompts(lens, vocab, seed=12):
    rng = np.random.default_rng(seed)
    return [rng.integers(0, vocab, n).tolist() for n in lens]


def test_scheduler_with_room_for_everything_matches_the_plain_one():
    """A budget no request reaches: the same tokens as without one."""
    cfg, model = _model()
    prompts = _prompts([5, 130, 61, 200, 17], cfg.vocab_size)
    a, _, _ = _serve(cfg, model, prompts)
    b, reqs, _ = _serve(cfg, model, prompts, kv_budget=400)
    assert a == b
    assert all(r.cached_len == r.current_position for r in reqs)


@pytest.mark.parametrize("graph", [True, False])
def test_scheduler_bounds_the_cache(graph):
    cfg, model = _model()
    prompts = _prompts([5, 130, 61, 200, 17], cfg.vocab_size)
    out, reqs, peak = _serve(cfg, model, prompts, new=60, kv_budget=64, kv_recent=16, kv_sinks=2,
                             kv_score_window=8, use_cuda_graph=graph)
    assert [len(o) for o in out] == [60] * 5
    assert peak <= 64 + 16
    assert [r.current_position for r in reqs] == [len(p) + 59 for p in prompts]
    if graph:
        again, _, _ = _serve(cfg, model, prompts, new=60, kv_budget=64, kv_recent=16, kv_sinks=2,
                             kv_score_window=8, use_cuda_graph=False)
        # until a request is cut, its steps are those of the plain scheduler
        plain, _, _ = _serve(cfg, model, prompts, new=60)
        assert out[0][:60] == again[0][:60] == plain[0][:60]  # 5 + 60 tokens: never cut


def test_scheduler_sampling():
    """Filters, seeds and log-probabilities through the scheduler: top_k = 1 is
    greedy whatever the temperature; a seeded request repeats itself in other
    company; log-probabilities come one per token."""
    cfg, model = _model()
    prompts = _prompts([5, 30, 61], cfg.vocab_size)
    greedy, _, _ = _serve(cfg, model, prompts, new=12)
    out, reqs, _ = _serve(cfg, model, prompts, new=12, requests=[
        dict(temperature=1.5, top_k=1), dict(temperature=0.9, top_p=0.8, seed=7, logprobs=True),
        dict(temperature=1.1, min_p=0.2, seed=3)])
    assert out[0] == greedy[0]
    assert len(reqs[1].token_logprobs) == 12 and all(lp <= 0 for lp in reqs[1].token_logprobs)
    assert not reqs[0].token_logprobs
    alone, _, _ = _serve(cfg, model, prompts[:1], new=12, requests=[dict(temperature=1.5, top_k=1)])
    assert alone[0] == greedy[0]
    same, _, _ = _serve(cfg, model, prompts, new=12, requests=[
        dict(), dict(temperature=0.9, top_p=0.8, seed=7, logprobs=True), dict(temperature=1.0)])
    assert same[1] == out[1] and same[0] == greedy[0]


def test_scheduler_ends_a_request_without_a_token():
    cfg, model = _model()
    with torch.no_grad():
        model.norm.weight.fill_(float("nan"))
    out, reqs, _ = _serve(cfg, model, _prompts([9], cfg.vocab_size), new=5,
                          requests=[dict(temperature=1.0, top_k=5)])
    assert out == [[]] and reqs[0].finish_reason == "error"
