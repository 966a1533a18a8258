"""Sampling under tensor parallelism, as two gloo ranks: every rank runs its own
scheduler on the same requests, so all must go on with the same tokens whatever
their generators hold."""
import multiprocessing as mp
from types import SimpleNamespace

import pytest

torch = pytest.importorskip("torch")


def _rank(rank, init_file, out_q):
    import torch.distributed as dist

    from mi_b200 import scheduler as sched_mod
    from mi_b200.scheduler import Request, Scheduler
    from tests.test_scheduler_sampling_cpu import sample_tokens_by_definition

    dist.init_process_group("gloo", init_method=f"file://{init_file}", rank=rank, world_size=2)
    try:
        sched_mod.sample_tokens = sample_tokens_by_definition
        s = Scheduler.__new__(Scheduler)
        s.device = torch.device("cpu")
        s.model = SimpleNamespace(tp_size=2, tp_rank=rank, tp_group=dist.group.WORLD)
        torch.manual_seed(100 + rank)  # fresh processes: unlike seeds
        rows = torch.randn(4, 5000, generator=torch.Generator().manual_seed(1))
        req = lambda t, **kw: Request("r", [1], 4, t, **kw)  # noqa: E731
        got = {}
        for name, make in dict(
                warm=lambda: [req(1.0), req(0.0), req(1.4), req(0.8)],
                filtered=lambda: [req(1.0, top_p=0.99), req(1.0, min_p=1e-4),
                                  req(1.2, top_k=4000), req(1.0, seed=3)],
                mixed=lambda: [req(1.0), req(1.0, top_p=0.99, logprobs=True), req(0.0),
                               req(0.0, logprobs=True)],
                greedy=lambda: [req(0.0)] * 4).items():
            reqs = make()
            got[name] = [s._sample(rows, reqs) for _ in range(3)], [r.token_logprobs for r in reqs]
        out_q.put((rank, got))
    finally:
        dist.destroy_process_group()


def test_ranks_go_on_with_the_same_tokens(tmp_path):
    ctx = mp.get_context("spawn")
    q = ctx.Queue()
    procs = [ctx.Process(target=_rank, args=(r, str(tmp_path / "rendezvous"), q))
             for r in range(2)]
    for p in procs:
        p.start()
    got = dict(q.get(timeout=240) for _ in procs)
    for p in procs:
        p.join(timeout=60)
        assert p.exitcode == 0
    assert got[0] == got[1]
    tokens, logprobs = got[0]["mixed"]
    assert len({t[1] for t in tokens}) > 1  # (drawn anew each time)
    assert [len(lp) for lp in logprobs] == [0, 3, 0, 3]
