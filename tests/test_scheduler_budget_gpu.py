"""Requests that the scheduler cuts back to its budget, step by step beside the
same requests without one: what is written to the cache, what the scores gain,
what each eviction leaves, and the count of free pages."""
import dataclasses

import numpy as np
import pytest

from oracle import scores_oracle as so

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from mi_b200.scheduler import Request, RequestStatus, Scheduler  # noqa: E402

DEV, PS = "cuda", 16
BUDGET, RECENT, SINKS, WINDOW = 64, 16, 2, 8


def _model(layers=2):
    from mi_b200.model import PRESETS, Model
    cfg = dataclasses.replace(PRESETS["qwen2.5-0.5b"], num_hidden_layers=layers)
    return cfg, Model.create(cfg, torch.device(DEV, 0), torch.bfloat16, seed=9)


class Watched:
    """A scheduler whose evictions are checked against the definition."""

    def __init__(self, cfg, model, prompts, teacher, graph, **kw):
        self.s = Scheduler(model, cfg, torch.device(DEV, 0), torch.bfloat16, max_batch_size=4,
                           max_seq_len=512, page_size=PS, eos_token_ids=set(),
                           use_cuda_graph=graph, teacher_tokens=teacher, **kw)
        self.kv = self.s.kv_cache
        self.reqs = [Request(f"r{i}", p, len(teacher[f"r{i}"]), 0.0)
                     for i, p in enumerate(prompts)]
        for r in self.reqs:
            self.s.submit_request(r)
        self.cuts = 0
        self.totals = {}  # slot -> scores per layer and head before its eviction in this step
        self._evict, self.kv.evict = self.kv.evict, self.evict

    def slot_scores(self, slot):
        """[layers, heads, slots of its pages] on the host."""
        pages = self.kv.slot_pages(slot)
        sc = self.kv.score_data[:, pages].cpu().numpy()
        return sc.transpose(0, 2, 1, 3).reshape(sc.shape[0], sc.shape[2], -1)

    def rows(self, slot, layer):
        """K and V [slots of its pages, 2, heads, d], exact in fp32."""
        kv = self.kv.kv_data[layer][self.kv.slot_pages(slot)].float().cpu().numpy()
        return kv.transpose(0, 2, 1, 3, 4).reshape(-1, *kv.shape[1:2], *kv.shape[3:])

    def evict(self, slots, lengths, budget, freed, **kw):
        assert (budget, kw) == (BUDGET, dict(recent=RECENT, sinks=SINKS))
        layers = self.kv.num_layers
        before = {s: (n, self.slot_scores(s), [self.rows(s, l) for l in range(layers)])
                  for s, n in zip(slots.tolist(), lengths.tolist())}
        self._evict(slots, lengths, budget, freed, **kw)
        for s, (n, sc, rows) in before.items():
            self.totals[s] = sc.sum(-1, dtype=np.float64)
            assert n > BUDGET and len(self.kv.slot_pages(s)) == BUDGET // PS
            assert (sc[:, :, n:] == 0).all()
            after = self.slot_scores(s)
            for l in range(layers):
                got = self.rows(s, l)
                for h in range(sc.shape[1]):
                    src = so.evict_slots(sc[l, h, :n], BUDGET, RECENT, SINKS)
                    assert np.array_equal(after[l, h], sc[l, h, src])
                    assert np.array_equal(got[:, :, h], rows[l][src][:, :, h])
            self.cuts += 1

    def step(self):
        self.totals = {}
        self.s.step()
        self.kv.check_status()
        assert self.kv.num_free_pages == int(self.kv.pool_ctrl[1].item())

    def newest(self, req):
        """The row of layer 0 that holds the request's last cached token."""
        return self.rows(req.batch_slot, 0)[req.cached_len - 1]


@pytest.mark.parametrize("graph", [True, False])
def test_cut_requests_step_by_step(graph):
    cfg, model = _model()
    rng = np.random.default_rng(12)
    prompts = [rng.integers(0, cfg.vocab_size, n).tolist() for n in (130, 61, 200, 17)]
    steps = 70
    teacher = {f"r{i}": rng.integers(0, cfg.vocab_size, steps).tolist() for i in range(4)}
    plain = Watched(cfg, model, prompts, teacher, graph)
    cut = Watched(cfg, model, prompts, teacher, graph, kv_budget=BUDGET, kv_recent=RECENT,
                  kv_sinks=SINKS, kv_score_window=WINDOW)
    group = cfg.num_attention_heads // cfg.num_key_value_heads
    sums = {}
    for step in range(steps - 1):
        plain.step()
        cut.step()
        for a, b in zip(plain.reqs, cut.reqs):
            if step == 0 and b.status == RequestStatus.DECODING:
                # prefill (the prompt's last queries) and the first decode step
                sums[b.request_id] = np.zeros(())
            assert a.generated_tokens == b.generated_tokens
            assert a.current_position == b.current_position == len(a.input_ids) + step + 1
            assert a.cached_len == a.current_position
            assert b.cached_len <= min(b.current_position, BUDGET + PS)
            if b.status != RequestStatus.DECODING:
                continue
            # layer 0's K and V of a token depend on the token and its position
            # alone: with the slot for the position K would be rotated elsewhere
            assert np.array_equal(plain.newest(a), cut.newest(b)), (step, b.request_id)
            # each query head's weights add up to one, in every layer and KV head:
            # exact logits' weights but for the argument's and exp2's rounding (64
            # 2^-23) and the sum of 128 tokens, and each score's own addition
            kept = cut.slot_scores(b.batch_slot).sum(-1, dtype=np.float64)
            total = cut.totals.get(b.batch_slot, kept)
            if step > 0:
                gain = total - sums[b.request_id]
                assert np.abs(gain - group).max() <= group * 128 * 2.0 ** -23 + total.max() * 2.0 ** -23
            sums[b.request_id] = kept
    assert cut.cuts >= 10 and all(r.cached_len < r.current_position for r in cut.reqs)
    for w in (plain, cut):
        for _ in range(3):
            w.s.step()
        assert not w.s.active_requests
        assert w.kv.num_free_pages == int(w.kv.pool_ctrl[1].item()) == w.kv.max_num_pages - 1
        w.s.close()


def test_prompts_scores_are_those_of_its_last_queries():
    cfg, model = _model()
    rng = np.random.default_rng(3)
    prompts = [rng.integers(0, cfg.vocab_size, n).tolist() for n in (5, 40, 200)]
    teacher = {f"r{i}": [1, 2, 3] for i in range(3)}
    w = Watched(cfg, model, prompts, teacher, True, kv_budget=256, kv_score_window=WINDOW)
    w.s._admit_new_requests()
    w.s._prefill_new_requests()
    group = cfg.num_attention_heads // cfg.num_key_value_heads
    for r in w.reqs:
        n = len(r.input_ids)
        sc = w.slot_scores(r.batch_slot)
        assert (sc[:, :, n:] == 0).all() and (sc >= 0).all()
        want = min(n, WINDOW) * group
        # a logit and its row's log-sum-exp are each off by at most (d + 8) 2^-23 of the
        # sizes of a product's terms (below 6 here)
        assert np.abs(sc.sum(-1, dtype=np.float64) / want - 1).max() <= 1e-4
    for _ in range(4):
        w.s.step()
    assert not w.s.active_requests
    w.s.close()
