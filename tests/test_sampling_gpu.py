"""sample_tokens against the 64-bit definition (oracle/sampling_oracle.py).

Tokens are compared for equality: the kernel's weights are 2^-44-step fixed
point from 64-bit exponentials, so a different token needs u (or a filter's
border) within ~2^-40 of a boundary of the running mass, which seeded inputs
do not hit. Log-probabilities: fp32 sum of fp32 exponentials, at most a few
2^-23 relative in the sum, so an absolute 2e-6 in its logarithm, plus half a
step of the fp32 result.
"""
import math

import numpy as np
import pytest

from oracle.sampling_oracle import sample_row

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from mi_b200 import capi  # noqa: E402
from mi_b200.sampling import sample_tokens  # noqa: E402

DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def _check(logits, u, t, k, p, m, tokens, logprobs=None):
    rows = logits.shape[0]
    x = logits.double().cpu().numpy()
    per = lambda v: v.double().tolist() if isinstance(v, torch.Tensor) else [v] * rows  # noqa: E731
    T, K, P, M, U = per(t), per(k), per(p), per(m), u.double().tolist()
    P, M = ([float(np.float32(a)) for a in v] for v in (P, M))
    T = [float(np.float32(a)) for a in T]
    got = tokens.tolist()
    lp = None if logprobs is None else logprobs.double().tolist()
    for r in range(rows):
        want, want_lp, kept = sample_row(x[r], U[r], T[r], int(K[r]), P[r], M[r])
        assert got[r] == want, (r, got[r], want, len(kept), T[r], K[r], P[r], M[r], U[r])
        if lp is not None:
            if math.isinf(want_lp):
                assert lp[r] == want_lp
            else:
                assert abs(lp[r] - want_lp) <= 2e-6 + abs(want_lp) * 2.0 ** -24, (r, lp[r], want_lp)


def _logits(rows, vocab, dtype, style, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(rows, vocab, device="cuda", generator=g) * (0.3 if style == "flat" else 2.5)
    if style == "equal":
        x.fill_(1.25)
    u = torch.rand(rows, device="cuda", generator=g)
    return x.to(dtype), u


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 2), (2, 7), (5, 100), (4, 1023), (1, 32768),
                                        (9, 50257), (3, 152064), (150, 5001)])
@pytest.mark.parametrize("t,k,p,m", [
    (1.0, 0, 1.0, 0.0), (0.0, 5, 0.5, 0.1), (0.7, 50, 1.0, 0.0), (1.0, 0, 0.9, 0.0),
    (1.3, 0, 1.0, 0.08), (0.9, 200, 0.8, 0.02), (1.0, 1, 0.3, 0.0), (2.0, 1000, 0.95, 0.0)])
def test_sample_matches_the_definition(dtype, rows, vocab, t, k, p, m):
    x, u = _logits(rows, vocab, dtype, "normal", rows * 7 + vocab + k)
    tok, lp = sample_tokens(x, u, t, k, p, m, return_logprobs=True)
    _check(x, u, t, k, p, m, tok, lp)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("style", ["flat", "equal"])
@pytest.mark.parametrize("vocab", [3000, 152064, 262144])
@pytest.mark.parametrize("k,p", [(0, 0.5), (20000, 1.0), (20000, 0.37), (700, 0.999), (0, 1.0),
                                 (262143, 0.9999)])
def test_wide_sets_and_ties(dtype, style, vocab, k, p):
    """Thresholds among thousands of near or exact ties: the range divisions."""
    x, u = _logits(3, vocab, dtype, style, vocab + k)
    u[0] = 0.0
    u[1] = 1 - 2.0 ** -24
    tok = sample_tokens(x, u, 1.0, k, p)
    _check(x, u, 1.0, k, p, 0.0, tok)


def test_exact_borders():
    """Masses that meet the border exactly: a token starting at p is left out,
    u on a border takes the next token."""
    x = torch.full((4, 64), -math.inf, device="cuda")
    x[:, [3, 10, 20, 40]] = 0.5
    u = torch.tensor([0.0, 0.5, 0.25, 0.75], device="cuda")
    assert sample_tokens(x, u, 1.0, 0, 1.0).tolist() == [3, 20, 10, 40]
    assert sample_tokens(x, u, 1.0, 0, 0.5).tolist() == [3, 10, 3, 10]
    assert sample_tokens(x, u, 1.0, 0, 0.51).tolist() == [3, 10, 3, 20]
    assert sample_tokens(x, u, 1.0, 2, 1.0).tolist() == [3, 10, 3, 10]
    assert sample_tokens(x, u, 1.0, 0, 0.0).tolist() == [3, 3, 3, 3]
    assert sample_tokens(x, u, 1.0, 0, 1.0, 1.0).tolist() == [3, 20, 10, 40]
    assert sample_tokens(x, u, 1.0, 0, 1.0, 7.0).tolist() == [3, 20, 10, 40]


@pytest.mark.parametrize("dtype", DTYPES)
def test_special_logits(dtype):
    """-inf and the type's lowest value, +inf, NaN, rows with nothing, -0 against 0."""
    low = torch.finfo(dtype).min
    inf, nan = math.inf, math.nan
    rows = [
        [-inf] * 5, [nan] * 5, [nan, -inf, 2.0, -inf, nan], [low] * 5, [low, low, 0.0, low, -inf],
        [inf, 1.0, inf, 2.0, -inf], [-0.0, 0.0, -0.0, -1.0, nan], [low, -inf, low, nan, low],
    ]
    x = torch.tensor(rows, device="cuda").to(dtype)
    for uu in (0.0, 0.4, 0.9):
        u = torch.full((len(rows),), uu, device="cuda")
        for t, k, p, m in ((1.0, 0, 1.0, 0.0), (0.0, 0, 1.0, 0.0), (0.5, 2, 1.0, 0.0),
                           (1.0, 0, 0.6, 0.0), (3.0, 4, 0.9, 0.5)):
            status = torch.zeros(1, dtype=torch.int32, device="cuda")
            tok, lp = sample_tokens(x, u, t, k, p, m, return_logprobs=True, status=status)
            _check(x, u, t, k, p, m, tok, lp)
            assert capi.status_names(int(status.item())) == ["NO_TOKEN"]


def test_settings_out_of_range():
    x, _ = _logits(6, 500, torch.float32, "normal", 4)
    nan, inf = math.nan, math.inf
    u = torch.tensor([nan, -1.0, 1.0, 5.0, -inf, inf], device="cuda")
    for t, k, p, m in ((nan, 0, 1.0, 0.0), (-1.0, 0, 1.0, 0.0), (1.0, -7, nan, nan),
                       (1.0, 500, 2.0, -3.0), (1.0, 2 ** 31 - 1, 1.0, 0.0), (1e-30, 0, 0.9, 0.1),
                       (1e30, 0, 0.9, 0.1), (1e-42, 3, 1.0, 0.0), (1.0, 3, -2.0, 0.0)):
        tok = sample_tokens(x, u, t, k, p, m)
        _check(x, u, t, k, p, m, tok)
    # infinite temperature: every token above -inf weighs the same
    x[:, ::2] = -inf
    tok = sample_tokens(x, torch.full((6,), 0.5, device="cuda"), inf)
    assert tok.tolist() == [251] * 6


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab,stride,offset", [(1001, 1003, 1), (4099, 5000, 3), (640, 640, 0),
                                                 (33, 35, 5)])
def test_strided_unaligned_rows_and_mixed_settings(dtype, vocab, stride, offset):
    rows = 11
    g = torch.Generator(device="cuda").manual_seed(vocab)
    flat = (3 * torch.randn(rows * stride + offset, device="cuda", generator=g)).to(dtype)
    x = flat[offset:].as_strided((rows, vocab), (stride, 1))
    u = torch.rand(rows, device="cuda", generator=g)
    t = torch.rand(rows, device="cuda", generator=g) * 1.5
    t[::4] = 0
    k = torch.randint(-1, 60, (rows,), device="cuda", generator=g, dtype=torch.int32)
    p = torch.rand(rows, device="cuda", generator=g) + 0.3
    m = torch.rand(rows, device="cuda", generator=g) * 0.2 - 0.05
    before = flat.clone()
    out = torch.full((rows,), -9, dtype=torch.int32, device="cuda")
    got, lp = sample_tokens(x, u, t, k, p, m, out=out, return_logprobs=True)
    assert got.data_ptr() == out.data_ptr()
    _check(x, u, t, k, p, m, got, lp)
    assert torch.equal(flat.view(torch.uint8), before.view(torch.uint8))


def test_frequencies_follow_the_distribution():
    """65536 draws on an even grid of u: each token's count is its mass times
    the number of draws within one (the grid meets each border once)."""
    n = 1 << 16
    x = torch.tensor([[1.0, -0.5, 2.0, 0.25, -3.0]], device="cuda").expand(n, 5).contiguous()
    u = (torch.arange(n, device="cuda", dtype=torch.float64) / n).float()
    tok = sample_tokens(x, u, 0.8)
    counts = torch.bincount(tok, minlength=5).double().cpu()
    want = torch.softmax(x[0].double() / np.float32(0.8), 0).cpu() * n
    assert (counts - want).abs().max() <= 1.0


def test_repeatable_and_captured():
    """The same call twice gives the same bits, and a captured one follows its inputs."""
    x, u = _logits(16, 32768, torch.bfloat16, "flat", 3)
    a, la = sample_tokens(x, u, 0.9, 0, 0.9, return_logprobs=True)
    b, lb = sample_tokens(x, u, 0.9, 0, 0.9, return_logprobs=True)
    assert torch.equal(a, b) and torch.equal(la, lb)
    out = torch.empty(16, dtype=torch.int32, device="cuda")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        sample_tokens(x, u, 0.9, 0, 0.9, out=out)
    s.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        sample_tokens(x, u, 0.9, 0, 0.9, out=out)
    x2, u2 = _logits(16, 32768, torch.bfloat16, "flat", 8)
    x.copy_(x2)
    u.copy_(u2)
    out.fill_(-5)
    g.replay()
    torch.cuda.synchronize()
    _check(x, u, 0.9, 0, 0.9, 0.0, out)


def test_no_rows():
    x = torch.empty(0, 100, device="cuda", dtype=torch.bfloat16)
    assert sample_tokens(x, torch.empty(0, device="cuda")).shape == (0,)


@pytest.mark.parametrize("style,temperature", [("wide", 1.518), ("wide", 0.9), ("list", 1.0),
                                               ("list", 0.77)])
def test_top_p_next_to_a_tokens_edge(style, temperature):
    """p is the fp32 number nearest to the share of a prefix, so p times the
    mass lies within 2^-25 of a token's edge, and the token after the prefix is
    the vocabulary's last: with u next to 1 it is drawn exactly when it is kept."""
    rows, vocab = 48, 30011
    rng = np.random.default_rng(int(temperature * 1000))
    x = rng.normal(size=(rows, vocab)).astype(np.float32) * np.float32(1 if style == "list" else 2.5)
    if style == "list":  # some hundred tokens above 2^-8, the others near 2^-13
        x = (x * 0.1 - 9.0 * temperature).astype(np.float32)
        x[:, :300] = -np.abs(rng.normal(size=(rows, 300))) * 2 * temperature
    p = np.zeros(rows, np.float32)
    want = []
    for r in range(rows):
        n = 40 + 4 * r if style == "list" else 2000 + 300 * r
        order = np.argsort(-x[r], kind="stable")
        at = order[n]  # the token after the prefix trades places with the last one
        x[r, at], x[r, -1] = x[r, -1], x[r, at]
        d = x[r].astype(np.float64)
        w = np.exp((d - d.max()) / float(np.float32(temperature)))
        mass = np.cumsum(np.sort(w)[::-1])
        p[r] = mass[n - 1] / mass[-1]
        want.append(sample_row(x[r], 1 - 2.0 ** -24, float(np.float32(temperature)), 0,
                               float(p[r]), 0.0)[0])
    u = torch.full((rows,), 1.0, device="cuda")
    got = sample_tokens(torch.from_numpy(x).cuda(), u, temperature, 0, torch.from_numpy(p).cuda())
    assert got.tolist() == want
    assert 8 < sum(t == vocab - 1 for t in want) < rows - 8  # both sides of the edge occur
