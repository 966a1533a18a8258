"""Top-p edges in a tail of tied tokens just below 2^-8 of the largest weight:
the mass there is first summed with the hardware's exp2, so what its error bound
leaves uncertain has to be decided in 64 bits."""
import numpy as np
import pytest

from oracle.sampling_oracle import sample_row

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from mi_b200.sampling import sample_tokens  # noqa: E402


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("tail,below", [(300, 5.5625), (12000, 5.5625), (40000, 5.5625),
                                        (40000, 6.25), (40000, 11.1875)])
def test_top_p_in_a_tied_tail(dtype, tail, below):
    """p is the fp32 number nearest to the share of the largest token and n tied
    ones: p times the mass lies within 2^-25 of an edge. With u next to 1 the
    last kept token is drawn, which tells on which side it was put."""
    rows = 24
    rng = np.random.default_rng(tail)
    x = np.full((rows, tail + 7), -np.inf)
    x[:, :tail] = -below
    x[:, 0] = 0.0
    temperature = 1.0  # 5.5625 is 2^-8.025, 6.25 is 2^-9.02, 11.1875 is 2^-16.1
    w = float(np.exp(-below))
    n = np.sort(rng.integers(1, tail - 1, rows))
    p = ((1 + n * w) / (1 + (tail - 1) * w)).astype(np.float32)
    t = torch.from_numpy(x).to(dtype).cuda()
    assert (t.double().cpu().numpy() == x).all()
    u = torch.full((rows,), 1.0, device="cuda")
    got = sample_tokens(t, u, temperature, 0, torch.from_numpy(p).cuda()).tolist()
    want = [sample_row(x[r], 1 - 2.0 ** -24, temperature, 0, float(p[r]))[0] for r in range(rows)]
    assert got == want
    assert {b - a for a, b in zip(n.tolist(), want)} <= {0, 1}
