"""sample_tokens refuses what it cannot take before any launch, and the oracle
it is tested against agrees with a draw written out by hand."""
import math

import pytest

torch = pytest.importorskip("torch")

from mi_b200 import capi  # noqa: E402
from mi_b200.sampling import MAX_VOCAB, sample_tokens  # noqa: E402
from oracle.sampling_oracle import sample_row  # noqa: E402

X = torch.zeros(2, 10)
U = torch.zeros(2)


@pytest.mark.parametrize("args,kw,err", [
    ((X[0], U), {}, ValueError),                                # one row without its dimension
    ((X.double(), U), {}, TypeError),
    ((X.t(), torch.zeros(10)), {}, ValueError),                 # vocabulary not contiguous
    ((X[:1].expand(2, 10), U), {}, ValueError),                 # rows overlap
    ((X, torch.zeros(3)), {}, ValueError),
    ((X, U.double()), {}, ValueError),
    ((torch.empty(2, 0), U), {}, ValueError),
    ((torch.empty(1, 1).expand(1, MAX_VOCAB + 1), torch.zeros(1)), {}, ValueError),
    ((X, U, torch.ones(3)), {}, ValueError),
    ((X, U, torch.ones(2).double()), {}, TypeError),
    ((X, U, 1.0, torch.ones(2)), {}, TypeError),                # top_k is int32
    ((X, U, 1.0, 0, torch.ones(4)[::2]), {}, ValueError),
    ((X, U), dict(out=torch.zeros(2)), ValueError),
    ((X, U), dict(out=torch.zeros(3, dtype=torch.int32)), ValueError),
    ((X, U), dict(logprobs=torch.zeros(2).half()), ValueError),
    ((X, U), dict(status=torch.zeros(1)), ValueError),
    ((X, U), {}, capi.MiError),                                 # no CPU fallback
])
def test_refusals(args, kw, err):
    with pytest.raises(err):
        sample_tokens(*args, **kw)


def test_c_entry_refuses(built=None):
    lib = capi.lib()
    call = lambda rows, vocab, dt, ptr=None: lib.mi_sample_tokens(  # noqa: E731
        ptr, vocab, rows, vocab, dt, ptr, None, 1.0, None, 0, None, 1.0, None, 0.0, ptr, None,
        None, None)
    assert call(0, 100, capi.DTYPE_BF16) == 0
    assert call(1, 100, capi.DTYPE_BF16) == capi.ERR_INVALID
    assert call(1, 0, capi.DTYPE_BF16) == capi.ERR_INVALID
    assert call(1, MAX_VOCAB + 1, capi.DTYPE_F32) == capi.ERR_INVALID
    assert call(-1, 100, capi.DTYPE_F32) == capi.ERR_INVALID
    assert call(1, 100, 9, 64) == capi.ERR_INVALID


def test_oracle_by_hand():
    x = [0.0, math.log(3.0), math.log(4.0), -math.inf]
    # weights 1/4, 3/4, 1: running masses 1/8, 1/2, 1
    assert [sample_row(x, u, 1.0)[0] for u in (0.0, 0.124, 0.126, 0.49, 0.51)] == [0, 0, 1, 1, 2]
    assert sample_row(x, 0.9, 1.0, top_k=1)[2] == [2]
    assert sample_row(x, 0.9, 1.0, top_p=0.4)[2] == [2]
    assert sample_row(x, 0.9, 1.0, top_p=0.51)[2] == [1, 2]
    assert sample_row(x, 0.9, 1.0, min_p=0.5)[2] == [1, 2]
    assert sample_row(x, 0.9, 0.0)[0] == 2
    assert sample_row([math.nan, -math.inf], 0.9, 1.0)[0] == -1
    assert abs(sample_row(x, 0.0, 1.0)[1] - math.log(1 / 8)) < 1e-12
