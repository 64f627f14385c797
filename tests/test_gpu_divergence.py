"""Divergence of logits where rows are masked, far apart or of unusual size, against 64 bits.

Where tolerances come from, with SUM and STEP as in test_gpu_logits.py.  t is the difference of a pair of logits less
that at the reference's largest, and is off by a few steps of the numbers that it is made of: x, y as they stand where
the rows are at most 60 apart there, else x and y less their values there.  A psi(t) = e^-t - 1 + t is off by 2^-22 of t^2
or of |t| + 1 and by what t is off, a sum by SUM of its terms' sizes, and where KL is E[t] + log E[e^-t] the logarithm
by SUM / E[e^-t] of them, E[e^-t] 1/64 at least (else it has a sum of its own).
"""

import math

import pytest
import torch

import cfm_b200  # noqa: F401
from cfm_b200.runtime.fidelity import compare_logits
from test_gpu_logits import STEP, SUM, TYPES, logits, ranked

pytestmark = pytest.mark.gpu

INF, NAN = math.inf, math.nan


def in_64_bits(a, b):
    """KL(softmax(a) || softmax(b)), and how far from it the library may be."""
    x, y = a.double(), b.double()
    top = x.amax(-1, keepdim=True)
    none = ~(top.isfinite() & y.amax(-1, keepdim=True).isfinite())
    log_p, log_q = torch.log_softmax(x, -1), torch.log_softmax(y, -1)
    p, q = log_p.exp(), log_q.exp()
    gap = torch.where(p > 0, log_p - log_q, 0.0)
    # With q - p added to each term, whose sum is zero.
    near = gap.abs() < 1
    terms = torch.where(near, p * (gap + torch.expm1(-gap.clamp(-1, 1))), p * gap - p + q)
    want = torch.where(none, NAN, torch.where(p > 0, terms, q).sum(-1, keepdim=True))[:, 0]
    at = ranked(a, 1)
    u, v = x - top, y - y.gather(1, at)
    apart = (top - y.gather(1, at)).abs()
    t = u - v
    own = torch.minimum((x - y).abs(), torch.full_like(apart, 120.0))
    off = STEP * torch.where(t.abs() < 0.5, t.abs(), 2.0) * (own + u.abs() + v.abs() + t.abs())
    size = torch.where(t.abs() < 0.5, t.square(), t.abs() + 1.0)
    live = (p > 0) & t.isfinite()
    allowed = torch.where(live, p * (2 * SUM * size + 4 * off), 0.0).sum(-1)
    far = (torch.where(live, p * size, 0.0).sum(-1) > 0.25) | ((p == 0) & (q > 0)).any(-1)
    return want, allowed + 4 * SUM * want + torch.where(far & (want > 0.1), 2 * SUM, 0.0)


def check(a, b):
    divergence, agreement = compare_logits(a, b)
    assert torch.equal(agreement, ranked(a, 1)[:, 0] == ranked(b, 1)[:, 0])
    want, allowed = in_64_bits(a, b)
    # Beyond FP32's numbers, as rounded to it: infinite.
    same = (divergence == want.float()) | (divergence.isnan() & want.isnan())
    off = torch.where(same, 0.0, (divergence.double() - want).abs())
    assert (off <= allowed.nan_to_num(0.0, 0.0, 0.0)).all(), (divergence, want, allowed)
    return divergence


def pair(rows, vocabulary, dtype, noise=0.1, seed=None):
    a = logits(rows, vocabulary, torch.float32, rows + vocabulary if seed is None else seed)
    generator = torch.Generator(device="cuda").manual_seed(vocabulary)
    b = a + noise * torch.randn(a.shape, device="cuda", generator=generator)
    return a.to(dtype), b.to(dtype)


# -- rows banned altogether ------------------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocabulary", [8, 1000, 8192, 32768, 131072, 262144])
@pytest.mark.parametrize("rows", [1, 32, 256])
def test_rows_banned_altogether(dtype, vocabulary, rows):
    """A vocabulary that fills every chunk, or not."""
    a, b = pair(rows, vocabulary, dtype)
    banned = torch.full_like(a, -INF)
    for x, y in ((a, banned), (banned, b), (banned, banned)):
        assert check(x, y).isnan().all()


# -- tokens that the reference alone bans ------------------------------------------------------
BANS = [(1024, 512, 1024), (1024, 510, 1024), (512, 0, 256), (8192, 4096, 8192), (8192, 2048, 6144), (20000, 0, 10000),
        (131072, 0, 65536), (131072, 65536, 131072), (50257, 4096, 50257), (50257, 0, 50000), (3000, 128, 256)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocabulary,start,end", BANS)
@pytest.mark.parametrize("rows", [1, 9, 64])
def test_blocks_that_the_reference_alone_bans(dtype, vocabulary, start, end, rows):
    a, b = pair(rows, vocabulary, dtype)
    a[:, start:end] = -INF
    assert check(a, b).isfinite().all()
    flat = torch.zeros_like(a)
    check(torch.where(a == -INF, a, flat), flat)
    b[0, start + (end - start) // 2] = INF
    assert check(a, b)[0].isnan()
    b[0, start + (end - start) // 2] = NAN
    assert check(a, b)[0].isnan()
    b[:, start:end] = -INF  # both do
    assert check(a, b).isfinite().all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocabulary", [8, 1000, 32768, 262144])
def test_rows_with_one_token_left(dtype, vocabulary):
    a, b = pair(9, vocabulary, dtype)
    banned = torch.full_like(a, -INF)
    banned[:, 3] = 1.0
    assert (check(a, banned) == INF).all() and check(banned, b).isfinite().all()


# -- finite values of any size -----------------------------------------------------------------
LARGE = [-1e4, -1e7, -1e8, -1e9, -3e9, -1e10, -1e11, -1e12, -1e15, -1e20, -1e25, -1e28, -3e29, -1e31]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("fill", LARGE)
def test_rows_masked_by_a_finite_value(dtype, fill):
    for rows, vocabulary, start, end in ((3, 8192, 0, 6000), (260, 8192, 0, 6000), (2, 50257, 0, 40000), (2, 1024, 0, 512), (5, 70000, 30000, 70000)):
        a, b = pair(rows, vocabulary, dtype)
        a[:, start:end] = b[:, start:end] = fill
        assert check(a, b).isfinite().all()
    a[:, :] = b[:, :] = fill  # nothing else
    assert not check(a, b).any()
    a[:, 77] = b[:, 77] = -fill
    assert not check(a, b).any()
    a, b = pair(4, 5000, dtype)
    a[:, 100], b[:, 100] = -fill, -fill
    assert not check(a, b).any()
    a, b = pair(4, 5000, dtype)
    a[:, 2000:] = fill
    b[:, 2000:] = 2 * fill
    check(a, b)


# -- steps of the shift ------------------------------------------------------------------------
def test_shifts_that_add_up():
    """Chunks whose differences are 59 apart from the next one's."""
    for far in (30.0, 45.0, 59.0):
        a = torch.zeros((256, 4096), device="cuda")
        b = torch.zeros_like(a)
        b[:, :2048] = far
        for i in range(2):
            a[:, 2048 * i:2048 * (i + 1):128] = 3.0 * i + 1
            b[:, 2048 * i:2048 * (i + 1):128] = 3.0 * i + 1 - far * i
        check(a, b)
        check(a[:5], b[:5])
        check(a.flip(-1), b.flip(-1))


# -- a flat reference and a token that the other is sure of ------------------------------------
@pytest.mark.parametrize("vocabulary", [64, 1000, 8192, 50257])
@pytest.mark.parametrize("rise", [2.0, 5.0, 12.0, 30.0, 50.0, 59.0, 80.0])
def test_flat_reference_and_a_sure_row(vocabulary, rise):
    generator = torch.Generator(device="cuda").manual_seed(vocabulary)
    a = 0.01 * torch.randn((40, vocabulary), device="cuda", generator=generator)
    b = a + 0.01 * torch.randn(a.shape, device="cuda", generator=generator)
    places = torch.randint(0, vocabulary, (40, 1), device="cuda", generator=generator)
    places[::2] = a[::2].argmax(-1, keepdim=True)
    for many in (1, 20):
        b.scatter_(1, (places + torch.arange(many, device="cuda") * 37) % vocabulary, rise)
        check(a, b)
        check(b, a)
        check(a, -b)


# -- rows a constant apart ---------------------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("offset", [50.0, 100.0, 1e3, 2e4, 1e6, 1e8])
def test_rows_a_constant_apart(dtype, offset):
    if dtype == torch.float16 and offset > 6e4:
        offset = 6e4
    for sign in (1.0, -1.0):
        a, b = pair(5, 9000, torch.float32, 0.5)
        b = (b + sign * offset).to(dtype)
        check(a.to(dtype), b)
        check(b, a.to(dtype))
        check(a.to(dtype), torch.full_like(b, sign * offset))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("fill", LARGE)
def test_a_reference_masked_by_a_finite_value_in_part_and_altogether(dtype, fill):
    a, b = pair(4, 5000, dtype)
    a[:, 2000:] = fill
    check(a, b)
    a[:, :2000] = fill
    check(a, b)


# -- distances of any size ----------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("fill", [-1e4, -1e7, -1e10, -1e15, -1e20])
def test_what_only_the_other_row_masks(dtype, fill):
    """A divergence of the mask's size."""
    for rows, vocabulary, start, end in ((3, 8192, 0, 6000), (260, 8192, 2000, 8192), (2, 50257, 5000, 5001)):
        a, b = pair(rows, vocabulary, dtype)
        b[:, start:end] = fill
        check(a, b)
        check(torch.zeros_like(a), torch.where(b == fill, b, torch.zeros_like(b)))


# -- weights that are none ---------------------------------------------------------------------
@pytest.mark.parametrize("vocabulary", [16, 4096, 20000])
def test_a_banned_token_of_no_weight(vocabulary):
    """A reference that masks by a finite value what the other bans: no weight that 64 bits hold is lost."""
    for dtype in TYPES:
        a, b = pair(6, vocabulary, dtype)
        a[:, 5:12] = torch.finfo(dtype).min
        b[:, 5:12] = -INF
        divergence = check(a, b)
        assert divergence.isfinite().all()
        a[3, 5], a[4, 7] = -800.0, -700.0
        divergence = check(a, b)
        assert divergence[3].isfinite() and divergence[4] == INF


# -- the largest numbers -----------------------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocabulary", [9, 4096, 20000])
def test_the_other_row_masks_by_its_types_lowest_value(dtype, vocabulary):
    """Divergences as large as the type's numbers, of which some sum to more, and of next to no weight."""
    most = torch.finfo(dtype).max
    a, b = pair(5, vocabulary, dtype)
    b[:, 2:9] = -most
    check(a, b)
    check(torch.zeros_like(a), b)
    a[:, 2:9] = -100.0
    check(a, b)
    a[:, 2:9] = -most
    assert check(a, b).isfinite().all()
    a, b = pair(5, vocabulary, dtype)
    b[:, 3], b[:, 4] = most, -most
    a[:, 4] = 9.0
    check(a, b)
    check(b, a)
