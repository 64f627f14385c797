"""Router, token log probabilities and divergence of logits against their definitions in 64 bits.

Where tolerances come from.  A single-precision step rounds by 2^-24 of its result.  The library's
exponential of d rounds d log2(e) and takes 2^x within 2 units of the last place: off by at most
(|d| + 4) 2^-24 of the value.  Terms that matter have |d| below 40 (e^-40 of a row of 2^18 is 1e-12 of its
sum), and a thread adds fewer than 80 of them before the tree of the warp: a sum of exponentials
is off by at most 130 2^-24 = 8e-6 of itself.
"""

import math

import pytest
import torch

import cfm_b200  # noqa: F401
from cfm_b200.runtime.fidelity import compare_logits, token_logprobs
from cfm_b200.runtime.routing import route_tokens

pytestmark = pytest.mark.gpu

SUM = 8e-6  # of a sum of exponentials
STEP = 2.0**-24
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def logits(rows, columns, dtype, seed, scale=2.5, peak=True):
    generator = torch.Generator(device="cuda").manual_seed(seed)
    x = scale * torch.randn((rows, columns), device="cuda", generator=generator)
    if peak:
        at = torch.randint(0, columns, (rows, 1), device="cuda", generator=generator)
        lift = 25.0 * torch.rand((rows, 1), device="cuda", generator=generator)
        lift[::2] = 0.0
        x.scatter_add_(1, at, lift)
    return x.to(dtype)


def inside(x, offset, spare):
    """The same rows in a wider buffer, `offset` elements from its aligned start."""
    wide = torch.full((x.shape[0], x.shape[1] + offset + spare), 100.0, device="cuda", dtype=x.dtype)
    wide[:, offset:offset + x.shape[1]] = x
    return wide[:, offset:offset + x.shape[1]]


def ranked(x, count):
    """Places of the largest, NaN above all, equal ones by the lowest place."""
    return torch.sort(x.float(), dim=-1, descending=True, stable=True).indices[:, :count]


# -- router ----------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,experts,top_k", [
    (1, 1, 1), (1, 128, 8), (3, 31, 4), (5, 32, 32), (2, 33, 7), (64, 64, 6), (17, 129, 8),
    (1000, 256, 8), (6, 257, 10), (9, 1024, 32),
])
@pytest.mark.parametrize("renormalize", [True, False])
def test_router(dtype, rows, experts, top_k, renormalize):
    x = logits(rows, experts, dtype, rows + experts, 1.5, peak=False)
    weights, ids = route_tokens(x, top_k, renormalize=renormalize)
    want_ids = ranked(x, top_k)
    assert ids.dtype == torch.int32 and torch.equal(ids.long(), want_ids)
    p = torch.softmax(x.double(), dim=-1).gather(1, want_ids)
    if renormalize:
        p = p / p.sum(-1, keepdim=True)
    # Exponentials of |d| < 16, a sum of 32 steps and two trees, one division.
    torch.testing.assert_close(weights.double(), p, rtol=64 * STEP, atol=0)
    wide, ids64 = route_tokens(inside(x, 3, 5), top_k, renormalize=renormalize,
                               weights_dtype=torch.bfloat16, ids_dtype=torch.int64)
    assert torch.equal(ids64, want_ids) and torch.equal(wide, weights.bfloat16())


def test_router_ties_and_rows_without_a_distribution():
    inf, nan = math.inf, math.nan
    x = torch.tensor([
        [0.0, -0.0, 0.0, 1.0, 1.0, -1.0],   # ties, 0 and -0 among them
        [-inf, 2.0, -inf, -inf, 2.0, -inf],  # fewer experts than are picked
        [-inf] * 6,
        [1.0, nan, 3.0, nan, 2.0, 0.0],
        [1.0, inf, 3.0, 0.0, 2.0, inf],
    ], device="cuda")
    weights, ids = route_tokens(x, 4)
    assert ids.tolist() == [[3, 4, 0, 1], [1, 4, 0, 2], [0, 1, 2, 3], [1, 3, 2, 4], [1, 5, 2, 4]]
    torch.testing.assert_close(weights[1].cpu(), torch.tensor([0.5, 0.5, 0.0, 0.0]), rtol=0, atol=0)
    assert weights[2].isnan().all() and weights[3].isnan().all()
    assert weights[4].isnan().any()
    assert not route_tokens(x, 4, renormalize=False)[0][:2].isnan().any()


# -- log probabilities -----------------------------------------------------------------------
def check_scores(x, tokens, top):
    got = token_logprobs(x, tokens, top)
    wide = x.double()
    largest = wide.amax(-1)
    shifted = wide - largest[:, None]
    log_z = shifted.exp().sum(-1).log()
    log_p = shifted - log_z[:, None]
    log_p[~largest.isfinite()] = math.nan  # no distribution
    p = log_p.exp()
    rest = 1.0 - (-log_z).exp()  # what the largest does not have
    ok = (tokens >= 0) & (tokens < x.shape[1])
    want = log_p.gather(1, tokens.clamp(0, x.shape[1] - 1).long()[:, None])[:, 0]
    assert got.logprobs[~ok].isnan().all()

    def near(found, value, allowed):
        same = (found.double() == value) | (found.isnan() & value.isnan())
        off = torch.where(same, 0.0, (found.double() - value).abs())
        assert (off <= allowed.nan_to_num(0.0, 0.0, 0.0)).all(), (off - allowed).max().item()

    # The difference to the largest, the logarithm's sum, the result.
    allowed = SUM * rest + 4 * STEP * (want.abs() + (want + log_z).abs())
    near(got.logprobs[ok], want[ok], allowed[ok])
    entropy = -torch.where(log_p > -math.inf, p * log_p, 0.0).sum(-1)
    spread = torch.where(p > 0, p * (largest[:, None] - wide), 0.0).sum(-1)
    entropy = torch.where(largest.isfinite(), entropy, math.nan)
    near(got.entropy, entropy, SUM * (rest + 2 * spread) + 4 * STEP * entropy)
    if top:
        ids = ranked(x, top)
        assert got.top_ids.dtype == torch.int32 and torch.equal(got.top_ids.long(), ids)
        want = log_p.gather(1, ids)
        below = (largest[:, None] - wide.gather(1, ids)).abs()
        near(got.top_logprobs, want, SUM * rest[:, None] + 4 * STEP * (want.abs() + below))
    else:
        assert got.top_ids is None and got.top_logprobs is None


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,vocabulary,top", [
    (1, 1, 1), (1, 2, 2), (2, 7, 0), (3, 8, 8), (3, 9, 3), (2, 32, 32), (4, 100, 32), (1, 1000, 1),
    (2, 4095, 5), (2, 4097, 5), (33, 8192, 20), (1, 32003, 20), (7, 50257, 5), (1, 151936, 20),
    (3, 262144, 32), (600, 3001, 4), (700, 1030, 0),
])
def test_scores(dtype, rows, vocabulary, top):
    x = logits(rows, vocabulary, dtype, rows * vocabulary)
    tokens = torch.randint(0, vocabulary, (rows,), device="cuda")
    tokens[::2] = x[::2].argmax(-1)
    check_scores(x, tokens, top)
    check_scores(inside(x, 1, 0), tokens.int(), top)
    check_scores(inside(x, 3, 6), tokens, top)


def test_scores_of_tokens_that_have_nearly_all_probability():
    """The log probability of such a token is the small sum of the others, which 1 + sum would lose."""
    x = torch.randn((4, 3000), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    tokens = torch.tensor([0, 17, 1500, 2999], device="cuda")
    x[torch.arange(4, device="cuda"), tokens] = 22.0
    check_scores(x, tokens, 4)
    assert (token_logprobs(x, tokens).logprobs > -1e-5).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("order", ["rising", "falling", "flat", "steps", "one thread"])
def test_scores_of_rows_in_order(dtype, order):
    """Rows whose largest elements lie together, or are all equal."""
    v = 40000
    places = torch.arange(v, device="cuda")
    row = {"rising": places / 5000.0, "falling": -places / 5000.0, "flat": 0 * places + 1.5,
           "steps": (places // 9000) / 2.0,
           "one thread": torch.where(places // 8 % 512 == 7, 3.0 + places / 20000.0, 0.0)}[order]
    x = row.to(dtype).expand(3, v).contiguous()
    check_scores(x, torch.tensor([0, 5, v - 1], device="cuda"), 32)


def test_scores_of_rows_with_banned_tokens_and_without_a_distribution():
    x = logits(8, 20000, torch.float32, 5)
    x[0, 1:] = -math.inf         # one token left
    x[1] = -math.inf
    x[2, 777] = math.nan
    x[3, 19999] = math.inf
    x[4, ::2] = -math.inf
    x[5, 10:] = -math.inf        # fewer than are asked for
    x[6, 100:12000] = -math.inf  # whole warps' worth
    x[7, :12000] = -math.inf
    tokens = torch.tensor([0, 1, 2, 3, 4, 9, 500, 15000], device="cuda")
    check_scores(x, tokens, 20)
    check_scores(x.bfloat16(), tokens, 20)
    got = token_logprobs(x, tokens, 20)
    assert got.logprobs[0] == 0 and got.entropy[0] == 0
    for row in (1, 2, 3):
        assert got.logprobs[row].isnan() and got.entropy[row].isnan() and got.top_logprobs[row].isnan().all()
    assert got.logprobs[4] == -math.inf and got.entropy[4].isfinite()


def test_tokens_outside_of_the_vocabulary_have_no_log_probability():
    x = logits(5, 300, torch.bfloat16, 9)
    tokens = torch.tensor([-1, 300, 2**31 - 1, -2**31, 299], device="cuda")
    check_scores(x, tokens, 2)
    check_scores(x, torch.tensor([-100, 2**40, -2**62, 1, 0], device="cuda"), 2)


# -- divergence ------------------------------------------------------------------------------
def check_divergence(a, b):
    divergence, agreement = compare_logits(a, b)
    assert torch.equal(agreement, ranked(a, 1)[:, 0] == ranked(b, 1)[:, 0])
    x, y = a.double(), b.double()
    log_p, log_q = torch.log_softmax(x, -1), torch.log_softmax(y, -1)
    p = log_p.exp()
    gap = log_p - log_q
    # With p - q added to each term, whose sum is zero: no cancellation.
    want = torch.where(log_p == -math.inf, log_q.exp(), p * (gap + torch.expm1(-gap))).sum(-1)
    # What the sums round: t = d - shift with the shift at the largest a; its error, times its size.
    # Where rows are far apart nothing is small, and the sums' errors are of the values themselves.
    there = ranked(a, 1)
    d = x - y
    t = (d - d.gather(1, there)).nan_to_num(0.0, 0.0, 0.0)
    size = torch.where(t.abs() < 0.5, t.square(), t.abs() + 1.0)
    moved = STEP * torch.where(t.abs() < 0.5, t.abs(), 2.0) * (d.abs().nan_to_num(0.0, 0.0, 0.0) + t.abs())
    allowed = (p.nan_to_num(0.0) * (2 * SUM * size + 4 * moved)).sum(-1) + 4 * SUM * want
    same = (divergence.double() == want) | (divergence.isnan() & want.isnan())
    off = torch.where(same, 0.0, (divergence.double() - want).abs())
    assert (off <= allowed.nan_to_num(0.0, 0.0, 0.0)).all(), (off / want).max().item()
    return divergence


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,vocabulary", [
    (1, 1), (2, 2), (3, 7), (2, 8), (3, 9), (5, 100), (2, 4097), (33, 8192), (1, 32003), (7, 50257),
    (1, 151936), (2, 262144), (600, 3001),
])
@pytest.mark.parametrize("noise", [0.001, 0.05, 1.0, 30.0])
def test_divergence(dtype, rows, vocabulary, noise):
    a = logits(rows, vocabulary, torch.float32, rows + vocabulary)
    generator = torch.Generator(device="cuda").manual_seed(vocabulary)
    b = a + noise * torch.randn(a.shape, device="cuda", generator=generator)
    a, b = a.to(dtype), b.to(dtype)
    check_divergence(a, b)
    if noise == 0.05:
        check_divergence(inside(a, 1, 2), inside(b, 1, 2))
        check_divergence(inside(a, 3, 0), inside(b, 2, 5))  # of different alignment


@pytest.mark.parametrize("dtype", TYPES)
def test_divergence_of_a_row_from_itself_and_from_a_shifted_one(dtype):
    a = logits(6, 30000, dtype, 3)
    divergence, agreement = compare_logits(a, a)
    assert not divergence.any() and agreement.all()
    whole = logits(4, 5000, torch.float32, 4).round()
    assert check_divergence(whole, whole + 64.0).abs().max() == 0.0


def test_divergence_of_rows_with_banned_tokens_and_without_a_distribution():
    a = logits(9, 20000, torch.float32, 6)
    b = a + 0.1 * torch.randn(a.shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(2))
    a[0, ::3] = b[0, ::3] = -math.inf  # the same ones
    a[1, ::3] = -math.inf              # those of the reference only: finite
    b[2, 5] = -math.inf                # of the other only: infinite
    a[3] = -math.inf
    b[4] = -math.inf
    a[5, 7] = math.nan
    b[6, 8] = math.inf
    b[7] = -math.inf
    b[7, 3] = 0.0
    a[8], b[8] = -math.inf, -math.inf
    a[8, 11], b[8, 11] = 2.0, 5.0      # the same certain token
    divergence = check_divergence(a, b)
    assert divergence[[0, 1]].isfinite().all() and divergence[1] > 0.1
    assert divergence[2] == math.inf and divergence[7] == math.inf and divergence[8] == 0
    assert divergence[3:7].isnan().all()


def test_divergence_of_rows_too_far_apart_for_one_shift():
    a = torch.zeros((3, 1000), device="cuda")
    b = torch.zeros((3, 1000), device="cuda")
    a[0, 3], b[0, 900] = 40.0, 200.0
    a[1, 3], b[1, 900] = 1.0, 300.0
    b[2, 10] = 61.0
    check_divergence(a, b)


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_beyond_32_bits_of_elements(dtype):
    buffer = torch.empty(2**31 + 5000, device="cuda", dtype=dtype)
    x, y = buffer[:5000 + 2**31].as_strided((3, 1000), (2**30, 1)), logits(3, 1000, dtype, 5)
    x.copy_(logits(3, 1000, dtype, 4))
    tokens = torch.tensor([0, 999, 5], device="cuda")
    check_scores(x, tokens, 7)
    check_divergence(x, y)
    weights, ids = route_tokens(x, 6)
    assert torch.equal(ids.long(), ranked(x, 6)) and torch.equal(weights, route_tokens(x.contiguous(), 6)[0])


@pytest.mark.parametrize("dtype", TYPES)
def test_huge_values(dtype):
    """Values whose multiples of log2 e are not finite, and the largest of their type."""
    most = torch.finfo(dtype).max
    x = logits(6, 3000, dtype, 8)
    x[0, 5], x[1, 7], x[2] = most, most / 2, -most
    x[2, 11], x[3, 4], x[4, 100:200] = -most / 2, -most, most
    tokens = torch.tensor([5, 7, 11, 4, 150, 0], device="cuda")
    check_scores(x, tokens, 9)
    check_divergence(x, x)
    divergence, agreement = compare_logits(x, x)
    assert not divergence.any() and agreement.all()


@pytest.mark.parametrize("vocabulary,top", [(300000, 32), (1 << 21, 20)])
def test_many_equal_rows_of_a_large_vocabulary(vocabulary, top):
    """More elements as large as the threads' maxima than are sorted at a time."""
    x = (torch.arange(vocabulary, device="cuda") % 7).bfloat16().expand(2, vocabulary).contiguous()
    x[1] = torch.sort(logits(1, vocabulary, torch.bfloat16, 3)[0]).values
    check_scores(x, torch.tensor([6, vocabulary - 1], device="cuda"), top)


# -- calls -----------------------------------------------------------------------------------
def test_no_rows():
    x = torch.empty((0, 128), device="cuda")
    weights, ids = route_tokens(x, 8)
    assert weights.shape == ids.shape == (0, 8)
    scores = token_logprobs(x, torch.empty(0, device="cuda", dtype=torch.int64), 5)
    assert scores.logprobs.shape == (0,) and scores.top_ids.shape == (0, 5)
    assert compare_logits(x, x)[0].shape == (0,)


def test_captured_and_on_another_stream():
    x, y = logits(5, 30000, torch.bfloat16, 1), logits(5, 30000, torch.bfloat16, 2)
    tokens = torch.tensor([1, 2, 3, 4, 5], device="cuda")

    def call():
        return [*route_tokens(x[:, :128], 8), *token_logprobs(x, tokens, 20), *compare_logits(x, y)]

    want = call()
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        got = call()
    stream.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    x.copy_(logits(5, 30000, torch.bfloat16, 7))
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(call(), out))


def test_refusals():
    x = logits(2, 64, torch.float32, 1)
    tokens = torch.zeros(2, device="cuda", dtype=torch.int64)
    for bad in (x.double(), x[0], x.cpu(), x.t(), x[:, ::2], x[:, :0], x[:1].expand(2, 64)):
        with pytest.raises(ValueError):
            route_tokens(bad, 1)
        with pytest.raises(ValueError):
            token_logprobs(bad, tokens)
        with pytest.raises(ValueError):
            compare_logits(bad, bad)
    for top_k in (0, -1, 33, 65):
        with pytest.raises(ValueError):
            route_tokens(x, top_k)
    with pytest.raises(ValueError):
        route_tokens(torch.zeros((1, 1025), device="cuda"), 2)
    with pytest.raises(ValueError):
        route_tokens(x, 2, weights_dtype=torch.float16)
    with pytest.raises(ValueError):
        route_tokens(x, 2, ids_dtype=torch.int16)
    for top in (-1, 33, 65):
        with pytest.raises(ValueError):
            token_logprobs(x, tokens, top)
    for bad in (tokens[:1], tokens.float(), tokens.cpu(), tokens.repeat(2)[::2]):
        with pytest.raises(ValueError):
            token_logprobs(x, bad)
    for bad in (x[:1], x[:, :63], x.bfloat16()):
        with pytest.raises(ValueError):
            compare_logits(x, bad)
    wants = x.clone().requires_grad_()
    for call in (lambda t: route_tokens(t, 2), lambda t: token_logprobs(t, tokens), lambda t: compare_logits(t, x),
                 lambda t: compare_logits(x, t)):
        with pytest.raises(ValueError, match="grad"):
            call(wants)
        with torch.no_grad():
            call(wants)
