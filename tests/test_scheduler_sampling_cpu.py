"""How the scheduler samples a batch, without a GPU: sample_tokens is stood in for
by the 64-bit definition."""
import math

import pytest

from oracle.sampling_oracle import sample_row

torch = pytest.importorskip("torch")

from mi_b200 import scheduler as sched_mod  # noqa: E402
from mi_b200.scheduler import Request, Scheduler, sample_rows  # noqa: E402


def sample_tokens_by_definition(logits, uniform, temperature, top_k, top_p, min_p,
                                return_logprobs=False):
    rows = [sample_row(x.numpy(), float(u), float(t), int(k), float(p), float(m))
            for x, u, t, k, p, m in zip(logits.double(), uniform, temperature, top_k, top_p, min_p)]
    tokens = torch.tensor([r[0] for r in rows], dtype=torch.int32)
    return (tokens, torch.tensor([r[1] for r in rows])) if return_logprobs else tokens


@pytest.fixture
def sched(monkeypatch):
    monkeypatch.setattr(sched_mod, "sample_tokens", sample_tokens_by_definition)
    s = Scheduler.__new__(Scheduler)
    s.device = torch.device("cpu")
    s.model = None
    return s


def _req(name, temperature=0.0, **kw):
    return Request(name, [1], 8, temperature, **kw)


def test_plain_requests_are_sampled_as_they_are_alone(sched):
    """A request with temperature alone goes through sample_rows whoever else is
    in its batch: its draws are multinomial's."""
    g = torch.Generator().manual_seed(3)
    rows = torch.randn(5, 50, generator=g)
    reqs = [_req("greedy"), _req("filtered", 0.9, top_k=5, seed=4), _req("warm", 1.2),
            _req("scored", 0.0, logprobs=True), _req("warm2", 0.7)]
    plain = [0, 2, 4]
    for seed in range(8):
        torch.manual_seed(seed)
        want = sample_rows(rows[plain], [reqs[i].temperature for i in plain]).tolist()
        torch.manual_seed(seed)
        got = sched._sample(rows, reqs)
        assert [got[i] for i in plain] == want
        assert got[3] == int(rows[3].argmax())
    assert len(reqs[3].token_logprobs) == 8 and not reqs[1].token_logprobs
    u = _req("copy", seed=4)
    last = [u.next_uniform() for _ in range(8)][-1]
    assert got[1] == sample_row(rows[1].double().numpy(), last, 0.9, 5)[0]


def test_a_mate_does_not_change_how_nan_ranks(sched):
    rows = torch.zeros(2, 50)
    rows[0, 7] = math.nan  # to argmax the largest, to sample_tokens -inf
    assert sched._sample(rows[:1], [_req("greedy")]) == [7]
    assert sched._sample(rows, [_req("greedy"), _req("filtered", 0.9, top_k=1)]) == [7, 0]


def test_unseeded_draws_repeat_with_torchs_generator(sched):
    rows = torch.zeros(3, 1000)
    draw = lambda: sched._sample(rows, [_req("a", 1.0, top_p=0.99), _req("b", 1.0, top_k=900),  # noqa: E731
                                        _req("c", 1.0, seed=5)])
    torch.manual_seed(5)
    a = draw()
    torch.manual_seed(5)
    b = draw()
    assert a[:2] == b[:2] and draw()[:2] != a[:2]
    assert a[2] == b[2]  # a seeded request's own numbers


def test_a_request_that_ends_without_a_token_has_no_log_probability_of_it(sched):
    rows = torch.full((2, 20), -math.inf)
    rows[1, 3] = 0.0
    reqs = [_req("nothing", 1.0, logprobs=True), _req("one", 1.0, logprobs=True)]
    assert sched._sample(rows, reqs) == [-1, 3]
    assert reqs[0].token_logprobs == [] and reqs[1].token_logprobs == [0.0]
