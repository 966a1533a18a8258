"""Measured cases of the operators around a decode step: choosing the next token
(``sample``), decode attention that accumulates the weight each cached token
receives (``decode_scores``), the same for a prompt's last queries
(``prompt_scores``) and eviction from the paged cache by those scores
(``evict``).

``run`` makes the library's calls where ``own`` is true and computes the same in
elementary torch operations where it is false; ``exact`` is the definition in 64
bits, written apart from both.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

_DEV = "cuda"
_DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_NEG = float("-inf")


def _library():
    """The package's modules (it lives in a folder of its own under the root)."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    path = os.path.join(root, "minimal-inference_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    from mi_b200 import decode, page, prefill, sampling
    return decode, page, prefill, sampling


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # one user, a chat request's usual settings, the smaller vocabulary: latency
        dict(name="sample-1x32768", op="sample", rows=1, vocab=32768, dtype="bf16", style="peaked",
             temperature=0.8, top_k=50, top_p=0.95, min_p=0.0, mixed=False, logprobs=False),
        # a full decode batch of the larger vocabulary, nucleus sampling
        dict(name="sample-64x152064-nucleus", op="sample", rows=64, vocab=152064, dtype="bf16",
             style="peaked", temperature=1.0, top_k=0, top_p=0.9, min_p=0.0, mixed=False,
             logprobs=False),
        # many requests, each with its own settings (some greedy), logits in 32 bits, with logprobs
        dict(name="sample-200x152064-mixed", op="sample", rows=200, vocab=152064, dtype="fp32",
             style="peaked", temperature=0.7, top_k=40, top_p=0.9, min_p=0.05, mixed=True,
             logprobs=True),
        # an odd vocabulary, near-flat logits, temperature alone: every token counts
        dict(name="sample-9x50257-flat", op="sample", rows=9, vocab=50257, dtype="fp16",
             style="flat", temperature=1.3, top_k=0, top_p=1.0, min_p=0.0, mixed=False,
             logprobs=True),
        # the decode batch of the repository's benchmark (32 requests, 256-4096 tokens)
        dict(name="decode-scores-32x4096", op="decode_scores", batch=32, lo=256, hi=4096, hq=32,
             hkv=8, d=128, ps=16, dtype="bf16"),
        # one long document, grouped heads of 7
        dict(name="decode-scores-1x32000", op="decode_scores", batch=1, lo=32000, hi=32000, hq=28,
             hkv=4, d=128, ps=16, dtype="bf16"),
        # the small 32-bit model: short prompts, seven heads per KV head, head size 64
        dict(name="decode-scores-4x500-fp32", op="decode_scores", batch=4, lo=37, hi=500, hq=14,
             hkv=2, d=64, ps=16, dtype="fp32"),
        # whole prompts of a prefill batch: every query counts
        dict(name="prompt-scores-16x1500", op="prompt_scores", batch=16, lo=100, hi=1500, hq=32,
             hkv=8, d=128, ps=16, window=0, dtype="bf16"),
        # long prompts judged by their last queries
        dict(name="prompt-scores-4x24000-w64", op="prompt_scores", batch=4, lo=9000, hi=24000,
             hq=28, hkv=4, d=128, ps=16, window=64, dtype="bf16"),
        # a short odd prompt
        dict(name="prompt-scores-1x77-fp16", op="prompt_scores", batch=1, lo=77, hi=77, hq=14,
             hkv=2, d=64, ps=16, window=0, dtype="fp16"),
        # prompts cut to the cache's budget after prefill
        dict(name="evict-8x4096-to-1024", op="evict", layers=4, batch=8, lo=1100, hi=4096, hkv=8,
             d=128, ps=16, budget=1024, recent=128, sinks=4, dtype="bf16"),
        # decoding at the budget: every 16 tokens one page is freed again
        dict(name="evict-32x1040-to-1024", op="evict", layers=8, batch=32, lo=1025, hi=1040, hkv=8,
             d=128, ps=16, budget=1024, recent=128, sinks=4, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["sample", "sample", "decode_scores", "prompt_scores", "evict"])
    if op == "sample":
        case = dict(op=op, rows=_log(rng, 1, 128), vocab=_log(rng, 1000, 160000),
                    dtype=rng.choice(["bf16", "fp16", "fp32"]),
                    style=rng.choice(["peaked", "flat"]),
                    temperature=round(rng.uniform(0.3, 1.6), 3),
                    top_k=rng.choice([0, 0, 1, 5, 40, 50, 1000]),
                    top_p=rng.choice([1.0, 1.0, round(rng.uniform(0.3, 0.99), 3)]),
                    min_p=rng.choice([0.0, 0.0, round(rng.uniform(0.01, 0.2), 3)]),
                    mixed=rng.random() < 0.4, logprobs=rng.random() < 0.5)
        return case
    heads = rng.choice([(32, 8, 128), (28, 4, 128), (14, 2, 64), (16, 2, 128), (64, 8, 128),
                        (8, 8, 128), (8, 1, 64)])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    if op == "decode_scores":
        batch = _log(rng, 1, 48)
        hi = _log(rng, 20, min(16000, 60000 // batch))
        return dict(op=op, batch=batch, lo=rng.randint(1, hi), hi=hi, hq=heads[0], hkv=heads[1],
                    d=heads[2], ps=rng.choice([16, 16, 32]), dtype=dtype)
    if op == "prompt_scores":
        window = rng.choice([0, 1, 16, 32, 64])
        batch = _log(rng, 1, 12)
        hi = _log(rng, 20, min(1400, 12000 // batch) if window == 0 else min(12000, 40000 // batch))
        return dict(op=op, batch=batch, lo=rng.randint(1, hi), hi=hi, hq=heads[0], hkv=heads[1],
                    d=heads[2], ps=rng.choice([16, 16, 32]), window=window, dtype=dtype)
    budget = _log(rng, 40, 1000)
    hi = _log(rng, budget + 1, 3500)
    batch = _log(rng, 1, min(16, 16000 // hi))
    recent = rng.randint(0, budget // 2)
    return dict(op=op, layers=rng.randint(1, 4), batch=batch, lo=rng.randint(budget // 2, hi),
                hi=hi, hkv=heads[1], d=heads[2], ps=rng.choice([16, 16, 32]), budget=budget,
                recent=recent, sinks=rng.choice([0, 1, 4]), dtype=dtype)


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _lens(case, seed):
    """The case's sequence lengths; work() counts the same ones, so they do not go by the seed."""
    rng = np.random.default_rng([case["batch"], case["lo"], case["hi"]])
    lens = rng.integers(case["lo"], case["hi"] + 1, size=case["batch"])
    lens[-1] = case["hi"]
    return lens.tolist()


def _tables(lens, ps, seed):
    """Disjoint page lists scattered over the pool, as a CSR page table."""
    rng = np.random.default_rng(seed)
    need = [-(-n // ps) for n in lens]
    pages = rng.permutation(sum(need) + 5)[:sum(need)]
    i32 = dict(dtype=torch.int32, device=_DEV)
    return dict(pages=sum(need) + 6, indices=torch.tensor(pages, **i32),
                indptr=torch.tensor(np.concatenate([[0], np.cumsum(need)]), **i32),
                last=torch.tensor([n - (m - 1) * ps for n, m in zip(lens, need)], **i32))


def prepare(case, seed):
    g = torch.Generator(device=_DEV).manual_seed(seed * 7919 + 13)
    dt = _DT[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, device=_DEV, generator=g)

    def uniform(*shape):
        return torch.rand(*shape, device=_DEV, generator=g)

    if case["op"] == "sample":
        rows, vocab = case["rows"], case["vocab"]
        x = normal(rows, vocab) * (2.0 if case["style"] == "peaked" else 0.3)
        if case["style"] == "peaked":  # some likely tokens stand out, as a language model's do
            at = torch.randint(0, vocab, (rows, 48), device=_DEV, generator=g)
            x.scatter_add_(1, at, 6 + 8 * uniform(rows, 48))
        st = dict(case=case, logits=x.to(dt), u=uniform(rows))
        full = dict(device=_DEV)
        T = torch.full((rows,), case["temperature"], **full)
        k = torch.full((rows,), case["top_k"], dtype=torch.int32, **full)
        p = torch.full((rows,), case["top_p"], **full)
        m = torch.full((rows,), case["min_p"], **full)
        if case["mixed"]:  # settings differ from request to request; every fifth is greedy
            r = torch.arange(rows, device=_DEV)
            T = torch.where(r % 5 == 4, 0.0, T * (0.6 + 0.8 * uniform(rows)))
            k = torch.where(r % 3 == 1, 0, k)
            p = torch.where(r % 4 == 2, 1.0, p)
            m = torch.where(r % 2 == 1, 0.0, m)
        st.update(temperature=T, top_k=k, top_p=p, min_p=m)
        return st

    lens, ps, hkv, d = _lens(case, seed), case["ps"], case["hkv"], case["d"]
    st = dict(case=case, lens=lens, **_tables(lens, ps, seed))
    if case["op"] == "evict":
        L = case["layers"]
        st["kv"] = torch.empty(L, st["pages"], 2, ps, hkv, d, device=_DEV, dtype=dt)
        st["kv"].normal_(generator=g)
        # accumulated weights: few tokens hold most of it
        st["given"] = torch.exp(2.5 * normal(L, st["pages"], hkv, ps) - 4)
        st["scores"] = st["given"].clone()
        return st
    st["kv"] = torch.empty(st["pages"], 2, ps, hkv, d, device=_DEV, dtype=dt)
    st["kv"].normal_(generator=g)
    hq = case["hq"]
    if case["op"] == "decode_scores":
        st["q"] = (1.5 * normal(case["batch"], hq, d)).to(dt)
        st["scores"] = torch.exp(normal(st["pages"], hkv, ps) - 5)
        return st
    total = sum(lens)  # every prompt token was a query of the prefill
    st["q"] = (1.5 * normal(total, hq, d)).to(dt)
    st["qo"] = torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int32, device=_DEV)
    st["scores"] = torch.zeros(st["pages"], hkv, ps, device=_DEV)
    # log-sum-exp of the rows, as the prefill attention returned it: the last
    # `window` queries' rows are read, the others' are left at zero
    lse = torch.zeros(total, hq, device=_DEV)
    row, _, _, visible, s = _prompt_logits(st, torch.float32)
    real = row >= 0
    lse[row[real]] = torch.logsumexp(s.masked_fill_(~visible[:, None], _NEG), -1).permute(
        0, 2, 1)[real]
    st["lse"] = lse
    return st


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------
def _slots(st):
    """For padded tokens [batch, longest]: page, slot in it, and whether the token exists."""
    ps = st["case"]["ps"]
    indptr, indices, last = st["indptr"].long(), st["indices"].long(), st["last"].long()
    npages = indptr[1:] - indptr[:-1]
    length = torch.where(npages > 0, (npages - 1) * ps + last, 0)
    t = torch.arange(max(st["lens"]), device=_DEV)
    at = (indptr[:-1, None] + t // ps).clamp(max=indices.numel() - 1)
    return indices[at], (t % ps).expand_as(at), t < length[:, None], length


def _plain_sample(st):
    x = st["logits"].double()
    x = torch.where(x.isnan(), _NEG, x)
    top = x.amax(-1, keepdim=True)
    T, k, p, m = (st[n].double().unsqueeze(1) for n in ("temperature", "top_k", "top_p", "min_p"))
    d = torch.where(x == top, 0.0, x - top)
    w = torch.exp(d / torch.where(T > 0, T, 1.0))
    order = torch.argsort(x, dim=-1, descending=True, stable=True)
    ws = w.gather(1, order)
    rank = torch.arange(x.shape[1], device=x.device)
    keep = (rank < k) | (k <= 0)
    ws = ws * keep
    upto = ws.cumsum(-1)
    before = torch.nn.functional.pad(upto[:, :-1], (1, 0))
    keep &= (before < p * upto[:, -1:]) | (p >= 1) | (rank == 0)
    keep &= ws >= m.clamp(max=1.0)
    kept = torch.zeros_like(w).scatter_(1, order, ws * keep)
    c = kept.cumsum(-1)
    token = (c <= st["u"].double().unsqueeze(1) * c[:, -1:]).sum(-1)
    token = torch.where(T.squeeze(1) > 0, token, order[:, 0])
    out = [token.int()]
    if st["case"]["logprobs"]:
        out.append((x.gather(1, token.unsqueeze(1)) - torch.logsumexp(x, -1, True)).squeeze(1).float())
    return out


def _plain_decode(st):
    case = st["case"]
    hq, hkv, d, ps = case["hq"], case["hkv"], case["d"], case["ps"]
    page, slot, there, _ = _slots(st)
    kv = st["kv"]
    k, v = kv[page, 0, slot].float(), kv[page, 1, slot].float()  # [b, t, hkv, d]
    q = st["q"].float().view(-1, hkv, hq // hkv, d)
    s = torch.matmul(q, k.permute(0, 2, 3, 1)) / math.sqrt(d)  # [b, hkv, g, t]
    s = s.masked_fill(~there[:, None, None], _NEG)
    e = torch.exp(s - s.amax(-1, keepdim=True))
    w = e / e.sum(-1, keepdim=True)
    out = torch.matmul(w, v.permute(0, 2, 1, 3)).reshape(-1, hq, d).to(kv.dtype)
    at = (page[:, None] * hkv + torch.arange(hkv, device=_DEV)[:, None]) * ps + slot[:, None]
    there = there[:, None].expand_as(at)
    st["scores"].view(-1)[at[there]] += w.sum(2)[there]
    return [out, st["scores"]]


def _prompt_logits(st, dt):
    """Padded window queries against padded keys: query rows (-1: none), keys' pages and slots,
    visible pairs [b, queries, keys] and logits [b, heads, queries, keys] in `dt`."""
    case = st["case"]
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    page, slot, there, length = _slots(st)
    qo = st["qo"].long()
    rows = min(max(st["lens"]), case["window"]) if case["window"] else max(st["lens"])
    i = torch.arange(rows, device=_DEV) - rows  # from the last query backwards
    nq = qo[1:] - qo[:-1]
    row = torch.where(i >= -nq[:, None], qo[1:, None] + i, -1)
    pos = length[:, None] + i  # a query's place among the keys
    t = torch.arange(page.shape[1], device=_DEV)
    visible = (row >= 0)[:, :, None] & there[:, None] & (t <= pos[:, :, None])
    k = st["kv"][page, 0, slot].to(dt).permute(0, 2, 3, 1)  # [b, hkv, d, t]
    q = st["q"][row.clamp(min=0)].to(dt)  # [b, i, hq, d]
    q = q.view(q.shape[0], rows, hkv, hq // hkv, d).permute(0, 2, 3, 1, 4).flatten(2, 3)
    s = torch.matmul(q, k).view(q.shape[0], hq, rows, -1) / math.sqrt(d)
    return row, (page, slot, there), rows, visible, s


def _plain_prompt(st):
    case = st["case"]
    hq, hkv, ps = case["hq"], case["hkv"], case["ps"]
    row, (page, slot, there), rows, visible, s = _prompt_logits(st, torch.float32)
    lse = st["lse"][row.clamp(min=0)].permute(0, 2, 1)  # [b, hq, i]
    s = s.sub_(lse.unsqueeze(-1)).masked_fill_(~visible[:, None], _NEG).exp_()
    w = s.sum(2).view(s.shape[0], hkv, hq // hkv, -1).sum(2)  # [b, hkv, t]
    at = (page[:, None] * hkv + torch.arange(hkv, device=_DEV)[:, None]) * ps + slot[:, None]
    there = there[:, None].expand_as(at)
    st["scores"].view(-1)[at[there]] += w[there]
    return [st["scores"]]


def _plain_evict(st):
    case = st["case"]
    L, hkv, ps = case["layers"], case["hkv"], case["ps"]
    budget, recent, sinks = case["budget"], case["recent"], case["sinks"]
    kv, scores = st["kv"], st["scores"]
    scores.copy_(st["given"])
    page, slot, there, length = _slots(st)
    B, n = page.shape
    t = torch.arange(n, device=_DEV)
    s = scores[:, page, :, slot]  # [b, t, L, hkv]
    s = s.permute(2, 0, 3, 1)  # [L, b, hkv, t]
    cut = length > budget
    middle = (t >= sinks) & (t < (length - recent)[:, None])  # [b, t]
    order = torch.argsort(s.masked_fill(~middle[None, :, None], _NEG), dim=-1, descending=True,
                          stable=True)
    rank = torch.empty_like(order).scatter_(-1, order, t.expand_as(order))
    low = budget - recent  # middle tokens end up below this slot
    keep = middle[None, :, None] & (rank < low - sinks)
    hole = ~keep & (t >= sinks) & (t < low)
    mover = keep & (t >= low)
    # the i-th mover goes to the i-th hole
    width = min(budget, n)
    src = torch.where(t[:width] < low, t[:width], t[:width] + (length - budget)[:, None])
    src = src[None, :, None].expand(L, B, hkv, width).contiguous()
    nth = torch.where(mover, mover.cumsum(-1) - 1, n)
    by_rank = torch.zeros(L, B, hkv, n + 1, dtype=torch.long, device=_DEV)
    by_rank.scatter_(-1, nth, t.expand_as(nth))
    fill = by_rank.gather(-1, (hole.cumsum(-1) - 1).clamp(min=0))[..., :width]
    src = torch.where(hole[..., :width], fill, src)
    alive = t[:width] < length[:, None]
    src = torch.where(cut[:, None, None], src, torch.where(alive, t[:width], 0)[:, None])
    # move the rows of K and V and the scores
    l = torch.arange(L, device=_DEV)[:, None, None, None]
    b = torch.arange(B, device=_DEV)[:, None, None]
    h = torch.arange(hkv, device=_DEV)[:, None]
    rows = kv[l, page[b, src], :, slot[b, src], h]  # [L, b, hkv, width, 2, d]
    vals = scores[l, page[b, src], h, slot[b, src]]
    put = (cut[:, None, None] & alive[:, None]).expand(L, B, hkv, width)
    dl, db, dh, dj = torch.nonzero(put, as_tuple=True)
    kv[dl, page[db, dj], :, slot[db, dj], dh] = rows[dl, db, dh, dj]
    scores[dl, page[db, dj], dh, slot[db, dj]] = vals[dl, db, dh, dj]
    # the slots behind what is kept, to the end of the request's pages, have no score
    npages = (st["indptr"][1:] - st["indptr"][:-1]).long()
    end = torch.arange(int(max(-(-x // ps) for x in st["lens"])) * ps, device=_DEV)
    behind = (end >= budget) & (end < (npages * ps)[:, None]) & cut[:, None]
    rb, rt = torch.nonzero(behind, as_tuple=True)
    rp = st["indices"].long()[st["indptr"].long()[rb] + rt // ps]
    scores[:, rp, :, rt % ps] = 0.0
    kept = torch.where(alive[:, None], src, -1)
    if width < budget:
        kept = torch.nn.functional.pad(kept, (0, budget - width), value=-1)
    return [kv, scores, kept.int()]


# ---------------------------------------------------------------------------
# the library's calls
# ---------------------------------------------------------------------------
def _own_sample(st):
    _, _, _, sampling = _library()
    out = sampling.sample_tokens(st["logits"], st["u"], st["temperature"], st["top_k"],
                                 st["top_p"], st["min_p"],
                                 return_logprobs=st["case"]["logprobs"])
    return list(out) if st["case"]["logprobs"] else [out]


def _own_decode(st):
    if "wrapper" not in st:  # kept from step to step, as the scheduler keeps it
        case = st["case"]
        decode, _, _, _ = _library()
        w = decode.BatchDecodeWithPagedKVCacheWrapper(
            torch.zeros(64 << 20, dtype=torch.uint8, device=_DEV))
        w.plan(st["indptr"], st["indices"], st["last"], case["hq"], case["hkv"], case["d"],
               case["ps"])
        st["wrapper"] = w
    return [st["wrapper"].run(st["q"], st["kv"], scores=st["scores"]), st["scores"]]


def _own_prompt(st):
    if "wrapper" not in st:
        case = st["case"]
        _, _, prefill, _ = _library()
        w = prefill.BatchPrefillWithPagedKVCacheWrapper(
            torch.zeros(1 << 20, dtype=torch.uint8, device=_DEV))
        w.plan(st["qo"], st["indptr"], st["indices"], st["last"], case["hq"], case["hkv"],
               case["d"], case["ps"], causal=True)
        st["wrapper"] = w
    st["wrapper"].accumulate_scores(st["q"], st["kv"], st["lse"], st["scores"],
                                    window=st["case"]["window"])
    return [st["scores"]]


def _own_evict(st):
    _, page, _, _ = _library()
    case = st["case"]
    st["scores"].copy_(st["given"])  # a pass evicts by the same scores each time
    kept = page.evict_paged_kv_cache(st["kv"], st["scores"], st["indices"], st["indptr"],
                                     st["last"], case["budget"], recent=case["recent"],
                                     sinks=case["sinks"], return_kept=True)
    return [st["kv"], st["scores"], kept]


def run(state):
    op = state["case"]["op"]
    if own:
        return dict(sample=_own_sample, decode_scores=_own_decode, prompt_scores=_own_prompt,
                    evict=_own_evict)[op](state)
    return dict(sample=_plain_sample, decode_scores=_plain_decode, prompt_scores=_plain_prompt,
                evict=_plain_evict)[op](state)


# ---------------------------------------------------------------------------
# work and exact values
# ---------------------------------------------------------------------------
def work(case):
    es = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "sample":
        n = case["rows"] * case["vocab"]
        return dict(bytes=n * es + case["rows"] * 24, flops=4 * n)
    lens = _lens(case, 0)
    tokens, row = sum(lens), case["hkv"] * case["d"] * es
    if case["op"] == "decode_scores":
        q = case["batch"] * case["hq"] * case["d"] * es
        return dict(bytes=2 * tokens * row + 8 * tokens * case["hkv"] + 2 * q,
                    flops=4 * tokens * case["hq"] * case["d"])
    if case["op"] == "prompt_scores":
        w = case["window"]
        nq = [min(n, w) if w else n for n in lens]
        pairs = sum(q * n - q * (q - 1) // 2 for q, n in zip(nq, lens))
        return dict(bytes=tokens * row + 8 * tokens * case["hkv"]
                    + sum(nq) * case["hq"] * (case["d"] * es + 4),
                    flops=pairs * case["hq"] * (2 * case["d"] + 4))
    # scores are read once; a token that is kept and moves is read and written
    budget, moved = case["budget"], 0
    for n in lens:
        if n > budget:  # the recent ones move, and as many others as the cut leaves holes for
            gone = n - budget
            old = max(0, n - case["recent"] - case["sinks"])
            room = max(0, budget - case["recent"] - case["sinks"])
            moved += case["recent"] + (gone * room // old if old else 0)
    heads = case["layers"] * case["hkv"]
    return dict(bytes=heads * (4 * tokens + 8 * min(budget, max(lens)) * len(lens)
                               + moved * 4 * case["d"] * es),
                flops=heads * tokens * 4)


def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    if op == "sample":
        return _exact_sample(st)
    if op == "evict":
        return _exact_evict(st)
    group, scale = case["hq"] // case["hkv"], case["d"] ** -0.5
    indptr, indices, ps = st["indptr"].tolist(), st["indices"].long(), case["ps"]
    scores = st["scores"].double()
    outs = []
    start = 0
    for b, n in enumerate(st["lens"]):
        pages = indices[indptr[b]:indptr[b + 1]]
        keys = st["kv"][pages, 0].double().flatten(0, 1)[:n]  # [n, hkv, d]
        add = torch.zeros(len(pages) * ps, case["hkv"], dtype=torch.float64, device=_DEV)
        if op == "decode_scores":
            values = st["kv"][pages, 1].double().flatten(0, 1)[:n]
            q = st["q"][b].double().view(case["hkv"], group, -1)
            w = torch.softmax(torch.einsum("hgd,nhd->hgn", q, keys) * scale, -1)
            outs.append(torch.einsum("hgn,nhd->hgd", w, values).reshape(case["hq"], -1))
            add[:n] = w.sum(1).t()
        else:
            m = min(n, case["window"]) if case["window"] else n
            q = st["q"][start + n - m:start + n].double()
            lse = st["lse"][start + n - m:start + n].double()
            seen = (torch.arange(n, device=_DEV)[None]
                    <= torch.arange(n - m, n, device=_DEV)[:, None])
            for h in range(case["hq"]):  # one head at a time: the logits are large
                z = q[:, h] @ keys[:, h // group].t() * scale - lse[:, h, None]
                add[:n, h // group] += torch.where(seen, z, _NEG).exp().sum(0)
            start += n
        scores[pages] += add.view(len(pages), ps, -1).permute(0, 2, 1)
    return [torch.stack(outs), scores] if op == "decode_scores" else [scores]


def _exact_sample(st):
    x = st["logits"].double().cpu().numpy()
    u = st["u"].double().tolist()
    T, k, p, m = (st[n].double().tolist() for n in ("temperature", "top_k", "top_p", "min_p"))
    tokens, logprobs = [], []
    for r in range(x.shape[0]):
        row = x[r]
        if T[r] <= 0:
            token = int(np.argmax(row))
        else:
            # the likeliest tokens first; equal ones by index
            order = np.argsort(-row, kind="stable")
            if k[r] > 0:
                order = order[:int(k[r])]
            w = np.exp((row[order] - row[order[0]]) / T[r])
            if p[r] < 1:
                mass = np.cumsum(w)
                order = order[:max(1, 1 + int(np.count_nonzero(mass[:-1] < p[r] * mass[-1])))]
                w = w[:len(order)]
            order = np.sort(order[w >= m[r]])
            w = np.exp((row[order] - row.max()) / T[r])
            c = np.cumsum(w)
            token = int(order[np.searchsorted(c, u[r] * c[-1], side="right")])
        tokens.append(token)
        logprobs.append(row[token] - row.max() - math.log(np.exp(row - row.max()).sum()))
    out = [torch.tensor(tokens, dtype=torch.int32)]
    return out + [torch.tensor(logprobs, dtype=torch.float64)] if st["case"]["logprobs"] else out


def _exact_evict(st):
    case = st["case"]
    ps, budget, recent, sinks = (case[n] for n in ("ps", "budget", "recent", "sinks"))
    L, hkv = case["layers"], case["hkv"]
    indptr, indices = st["indptr"].tolist(), st["indices"].cpu().numpy()
    given = st["given"].cpu().numpy()
    scores = given.astype(np.float64)
    kv = st["kv"].double()
    kept = np.full((L, len(st["lens"]), hkv, budget), -1, np.int32)
    for b, n in enumerate(st["lens"]):
        pages = indices[indptr[b]:indptr[b + 1]].astype(np.int64)
        kept[:, b, :, :min(n, budget)] = np.arange(min(n, budget))
        if n <= budget:
            continue
        old = given[:, pages].transpose(0, 2, 1, 3).reshape(L, hkv, -1)  # [L, hkv, slots]
        for l in range(L):
            for h in range(hkv):
                s = old[l, h]
                mid = np.arange(sinks, n - recent)
                best = mid[np.argsort(-s[mid], kind="stable")[:budget - recent - sinks]]
                stay = set(best[best < budget - recent].tolist())
                come = np.sort(best[best >= budget - recent])
                src = np.arange(budget)
                holes = [j for j in range(sinks, budget - recent) if j not in stay]
                src[holes] = come
                src[budget - recent:] = np.arange(n - recent, n)
                kept[l, b, h] = src
                new = np.zeros(len(pages) * ps)
                new[:budget] = s[src]
                scores[l, pages, h] = new.reshape(-1, ps)
        src = torch.tensor(kept[:, b].astype(np.int64), device=_DEV)  # [L, hkv, budget]
        pg = torch.tensor(pages, device=_DEV)
        rows = kv[:, pg].permute(0, 4, 1, 3, 2, 5).flatten(2, 3)  # [L, hkv, slots, 2, d]
        moved = rows.clone()
        moved[:, :, :budget] = rows.gather(2, src[..., None, None].expand(
            -1, -1, -1, 2, case["d"]))
        kv[:, pg] = moved.unflatten(2, (len(pages), ps)).permute(0, 2, 4, 3, 1, 5)
    return [kv, torch.tensor(scores), torch.tensor(kept)]
