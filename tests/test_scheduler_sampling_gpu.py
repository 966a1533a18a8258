"""The scheduler's sampling of a batch on the GPU."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from mi_b200.scheduler import Request, Scheduler, sample_rows  # noqa: E402


def _sched():
    s = Scheduler.__new__(Scheduler)
    s.device = torch.device("cuda", 0)
    s.model = None
    return s


def test_draws_repeat_with_the_devices_seed():
    """One seed of the device's generator repeats a batch with any settings, and
    requests with temperature alone draw what they draw without company."""
    s = _sched()
    rows = torch.randn(6, 32000, device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    req = lambda i, **kw: Request(f"r{i}", [1], 4, 1.0, **kw)  # noqa: E731
    batch = lambda: [req(0), req(1, top_p=0.99), req(2, top_k=5000), req(3), req(4, min_p=0.001),  # noqa: E731
                     req(5, logprobs=True)]
    torch.cuda.manual_seed(77)
    a = s._sample(rows, batch())
    torch.cuda.manual_seed(77)
    assert s._sample(rows, batch()) == a
    assert s._sample(rows, batch()) != a
    torch.cuda.manual_seed(77)
    assert sample_rows(rows[[0, 3]], [1.0, 1.0]).tolist() == [a[0], a[3]]
