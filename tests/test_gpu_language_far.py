"""Log probabilities of rows with logits far out: finite masks, rows of nothing but a mask, maxima of any size,
against the definition in 64 bits.

The kernels sum 2^(by * x - R) with by = scale * log2(e) and R = by * m rounded, m the largest x.  What the rounding
leaves, r = by * m - R, is no error, but it is part of every exponent: as long as R is below 2^30 it is at most 32, half
a step there.  Past that only the elements that are equal to m count: neighbouring numbers differ by 64 or more in by * x,
and 2^-64 of an element is nothing next to it.

With F = 32 ln 2 < 23, what r adds to the bounds of test_gpu_language.py: an exponent by * x - R is rounded at a size
of up to |z| log2(e) + 32, which is F u of its power of two (24 u of the sum); the logarithm of the sum is up to F larger
and off by 4 u of that, the product r ln 2 by 2 u of it: 24 u + 6 F u < 164 u of the log sum.  The sum of the products
that the entropy is taken from is larger by r of the sum, off by twice the sum's relative error and 8 u."""
import numpy as np
import pytest

import libgpuarray_amd as ga
from libgpuarray_amd import _lib, gpuarray
from test_gpu_language import HALF_STEP, TINY, U, decode, encode, grad64, logprob_bounds, run_logprobs, softmax64

pytestmark = pytest.mark.gpu

LOG2E = 1.4426950408889634
F = 23
MASKS = {"float32": [-1e4, -1e9, -1e10, -3e10, -1e20, -1e30, float(np.finfo(np.float32).min)],
         "bfloat16": [-1e9, -1e10, -3e10, -1e20, -1e30, float(ga.from_bfloat16(np.array([0xff7f], np.uint16).view(ga.bfloat16))[0])],
         "float16": [-1e4, -65504.0]}
CASES = [(kind, low) for kind in MASKS for low in MASKS[kind]]


def masked_rows(v, low, rng):
    """Rows with `low` in whole lanes, wavefronts and pieces; a running maximum has to leave it in most of them."""
    k = max(v // 16, 1)
    x = np.round(rng.standard_normal((10, v)) * 2, 2)
    x[0] = low
    x[1, :-k] = low
    x[2, : v // 2] = low
    x[3, rng.random(v) < 0.9] = low
    x[4, -1] = low
    x[5] = 0.0
    x[5, v // 2] = -low                                  # one large maximum
    x[6, [0, v // 2, v - 1]] = -low                      # three of them
    x[7] = low
    x[7, : v // 2] = -np.inf
    x[8] = low
    x[8, : v // 2] = low * 0.5                           # half of what was a mask is the maximum
    x[9] = -1000.0
    x[9, : v // 2] = low
    x[9, -k:] = 3.0
    return x


def remainders(x, scale):
    """32 for rows that have R anywhere between 2^8 and 2^30 (below that the bounds of nearer logits hold), else 0; -> F or 0."""
    r = np.abs(np.where(np.isfinite(x), x, 0)) * scale * LOG2E
    return np.where(((r >= 2.0 ** 8) & (r <= 2.0 ** 30 * (1 + 2.0 ** -20))).any(1), F, 0)


def in_float(a):
    """64-bit values with those that no float holds infinite."""
    return np.where(np.abs(a) >= 2.0 ** 128 * (1 - 2.0 ** -25), np.copysign(np.inf, a), a)


def expected(x, scale):
    """(m, log sum, log p, entropy) and bounds of the last three."""
    m, ls, z, p = softmax64(x, scale)
    ls_err, lp_err, h_err = logprob_bounds(x, scale)
    f = remainders(x, scale)
    s_rel = (x.shape[1] / 64 + 32 + 128 + 4 + 24) * U + 3 * U * (p * np.where(p > 0, np.abs(z), 0)).sum(1)
    ls_err = ls_err + np.where(f > 0, 164 * U, 0)
    lp_err = lp_err + np.where(f > 0, 164 * U, 0)[:, None]
    h_err = h_err + f * (2 * s_rel + 8 * U) + np.where(f > 0, 164 * U, 0)
    return m, ls, z - ls[:, None], ls - (p * np.where(p > 0, z, 0)).sum(1), ls_err, lp_err, h_err


def close(got, want, bound):
    want = in_float(want)
    fin = np.isfinite(want)
    assert np.array_equal(got[~fin], want[~fin]), np.argwhere((got != want) & ~fin)[:4]
    off = np.abs(got[fin] - want[fin])
    assert np.all(off <= bound[fin]), (float((off / bound[fin]).max()), got[fin][:8], want[fin][:8])


def check_far(ctx, x, scale, top, rng):
    x64 = decode(x)
    t, v = x64.shape
    ids = rng.integers(0, v, t)
    m, ls, lp, entropy, ls_err, lp_err, h_err = expected(x64, scale)
    logp, h, stats, top_logp, top_ids = run_logprobs(ctx, gpuarray.array(x, context=ctx), gpuarray.array(ids, context=ctx), v,
                                                     scale, top)
    assert np.array_equal(stats[:, 0], m.astype(np.float32))
    close(stats[:, 1], ls, ls_err)
    close(logp, lp[np.arange(t), ids], lp_err[np.arange(t), ids])
    close(h, entropy, h_err)
    order = np.argsort(-x64, axis=1, kind="stable")[:, :top]
    assert np.array_equal(top_ids, order)
    close(top_logp, np.take_along_axis(lp, order, 1), np.take_along_axis(lp_err, order, 1))


@pytest.mark.parametrize("kind,low", CASES)
@pytest.mark.parametrize("v", [20, 1000, 60000])
def test_finite_masks(ctx, kind, low, v):
    rng = np.random.default_rng(v)
    x = encode(masked_rows(v, low, rng), kind)
    for scale, top in ((0.5, 5), (1.0, 20), (float(np.float32(1.4)), 1)):
        check_far(ctx, x, scale, top, rng)


@pytest.mark.parametrize("low", [-1e9, -1e10, -1e20])
@pytest.mark.parametrize("t,v", [(300, 5000), (140, 60000)])
def test_finite_masks_of_rows_that_a_group_shares(ctx, low, t, v):
    rng = np.random.default_rng(t)
    x = masked_rows(v, low, rng)[np.arange(t) % 10].astype(np.float32)
    check_far(ctx, x, 1.0, 5, rng)


def maxima(exponent):
    """Maxima m with by * m on both sides of 2^exponent, positive and negative, and neighbours of them."""
    m = np.array([2.0 ** exponent / LOG2E * f for f in (0.75, 0.97, 0.9999999, 1.0, 1.0000001, 1.03, 1.3)], np.float32)
    m = np.concatenate([m, -m])
    x = np.full((m.size, 700), -np.inf, np.float32)
    x[:, ::3] = m[:, None]
    x[:, 1::3] = np.nextafter(m, np.float32(-np.inf))[:, None]
    x[:, 2::6] = (m - np.abs(m) * np.float32(0.01))[:, None]
    return x


@pytest.mark.parametrize("exponent", [20, 24, 27, 28, 29, 30, 31, 32, 33, 40, 64])
def test_maxima_around_the_limit(ctx, exponent):
    """The two ways of counting meet at 2^30."""
    check_far(ctx, maxima(exponent), 1.0, 5, np.random.default_rng(exponent))


def one_among_neighbours(v, size):
    """Rows of the next lower number, and one maximum that meets them when lanes, wavefronts or pieces are joined."""
    rng = np.random.default_rng(v)
    m = np.concatenate([rng.uniform(size, 2 * size, 12), -rng.uniform(size, 2 * size, 12)]).astype(np.float32)
    x = np.repeat(np.nextafter(m, np.float32(-np.inf))[:, None], v, 1)
    x[np.arange(m.size), rng.integers(0, v, m.size)] = m
    return x


@pytest.mark.parametrize("size", [2.0 ** 22, 2.0 ** 28, 2.0 ** 30, 2.0 ** 31, 1e20, 1e30, 1.6e38])
@pytest.mark.parametrize("v", [20, 700, 60000])
def test_one_maximum_among_its_neighbours(ctx, size, v):
    """What is rounded to the same multiple of log2(e) is not equal for that."""
    check_far(ctx, one_among_neighbours(v, size), 1.0, 5, np.random.default_rng(1))


# ---- the gradient -----------------------------------------------------------------------------------

def check_far_grad(ctx, x, kind, scale, rng):
    """With statistics that are rounded from 64 bits, and with those that the operator leaves."""
    x64 = decode(x)
    t, v = x64.shape
    ids = rng.integers(0, v, t)
    g, gh = (rng.standard_normal(t).astype(np.float32) for _ in range(2))
    want, bound, h, m, ls = grad64(x64, ids, g.astype(np.float64), gh.astype(np.float64), scale)
    _, _, lp, _, ls_err, _, h_err = expected(x64, scale)
    _, _, _, p = softmax64(x64, scale)
    lp, size = np.where(p > 0, lp, 0), np.abs(g) + np.abs(gh)
    # r is part of the exponent, of what is taken from it, and of the difference: three roundings at a size that is up to
    # 32 larger, F u each of p and of log p
    rest = np.where(remainders(x64, scale) > 0, 3 * F * U, 0)[:, None]
    bound = bound + scale * p * rest * (np.abs(g)[:, None] + np.abs(gh)[:, None] * (np.abs(lp) + np.abs(h)[:, None] + 1))
    dev = lambda a: gpuarray.array(a, context=ctx)  # noqa: E731
    own = ga.token_logprobs(dev(x), dev(ids), scale=scale, entropy=True)
    exact = dev(np.stack([m, ls], 1).astype(np.float32)), dev(h.astype(np.float32))
    # what the operator's own statistics may be off by
    joined = scale * p * (ls_err[:, None] * (size[:, None] * 2 + np.abs(gh)[:, None] * (np.abs(lp) + np.abs(h)[:, None])) +
                          (h_err * np.abs(gh))[:, None])
    for stats, entropy, more in ((*exact, 0), (own.stats, own.entropy, joined)):
        limit = (bound + more) * (1 + 2.0 ** -7) + np.abs(want) * HALF_STEP[kind] + TINY[kind]
        got = decode(ga.token_logprobs_grad(dev(x), dev(ids), stats, dev(g), entropy=entropy, dentropy=dev(gh), scale=scale))
        close(got, want, limit)          # (a gradient that no float holds is infinite)
        want_g, bound_g = grad64(x64, ids, g.astype(np.float64), np.zeros(t), scale)[:2]
        limit = (bound_g + scale * p * rest * np.abs(g)[:, None] + (more != 0) * scale * p * ls_err[:, None] * np.abs(g)[:, None])
        limit = limit * (1 + 2.0 ** -7) + np.abs(want_g) * HALF_STEP[kind] + TINY[kind]
        got = decode(ga.token_logprobs_grad(dev(x), dev(ids), stats, dev(g), scale=scale))
        close(got, want_g, limit)


@pytest.mark.parametrize("kind,low", CASES)
@pytest.mark.parametrize("v", [20, 1000, 60000])
def test_gradient_of_finite_masks(ctx, kind, low, v):
    rng = np.random.default_rng(v + 1)
    x = encode(masked_rows(v, low, rng), kind)
    for scale in (0.5, 1.0, float(np.float32(1.4))):
        check_far_grad(ctx, x, kind, scale, rng)


@pytest.mark.parametrize("exponent", [20, 24, 27, 28, 29, 30, 31, 32, 33, 40, 64])
def test_gradient_of_maxima_around_the_limit(ctx, exponent):
    rng = np.random.default_rng(exponent + 1)
    check_far_grad(ctx, maxima(exponent), "float32", 1.0, rng)


@pytest.mark.parametrize("size", [2.0 ** 22, 2.0 ** 28, 2.0 ** 30, 2.0 ** 31, 1e20, 1e30, 1.6e38])
@pytest.mark.parametrize("v", [20, 700])
def test_gradient_of_one_maximum_among_its_neighbours(ctx, size, v):
    check_far_grad(ctx, one_among_neighbours(v, size), "float32", 1.0, np.random.default_rng(2))


# ---- logits that are farther apart than the largest float ---------------------------------------------

@pytest.mark.parametrize("scale", [0.25, 2.0 ** -20, 1.0])
@pytest.mark.parametrize("v", [20, 60000])
def test_logits_farther_apart_than_a_float(ctx, scale, v):
    """x - m is -inf in 32 bits where scale * (x - m) need not be."""
    top = float(np.finfo(np.float32).max)
    x = np.full((4, v), -np.inf, np.float32)
    x[0] = -top
    x[0, 7] = top
    x[1] = -2e38
    x[1, v - 1] = 2.5e38
    x[2, [3, 9]] = -3e38, 3e38
    x[3, ::2] = -1e38
    x[3, 1] = 3e38
    check_far(ctx, x, scale, 3, np.random.default_rng(v))
    ids = gpuarray.array(np.array([0, 0, 3, 0]), context=ctx)
    got = np.asarray(ga.token_logprobs(gpuarray.array(x, context=ctx), ids, scale=scale).logp)
    want = in_float(np.array([-2 * top, -4.5e38, -6e38, -4e38]) * scale)
    fin = np.isfinite(want)
    assert np.array_equal(got[~fin], want[~fin]) and np.all(np.abs(got[fin] - want[fin]) <= 6 * U * np.abs(want[fin]))


# ---- the largest and smallest scales ------------------------------------------------------------------

def test_scales_that_are_too_large_in_powers_of_two_are_refused(ctx):
    z = lambda shape, dt="float32": gpuarray.zeros(shape, dt, context=ctx)  # noqa: E731
    x, ids, t1, t2 = z((4, 16)), z((4,), "int64"), z((4,)), z((4, 2))
    before = ctx.last_launch_hash()
    for scale in (2.4e38, 3.4e38):
        for call in (lambda: ga.token_logprobs(x, ids, scale=scale, out=ga.TokenLogprobs(t1, None, None, None, None)),
                     lambda: ga.token_logprobs_grad(x, ids, t2, t1, scale=scale, out=x)):
            with pytest.raises(ga.GpuArrayException) as e:
                call()
            assert e.value.code == _lib.GA_VALUE_ERROR
    assert ctx.last_launch_hash() == before


@pytest.mark.parametrize("scale,size", [(2.3e38, 1e-38), (2.3e38, 1.0), (2.3e38, 1e30), (1e-30, 1e30), (1e-38, 3e38), (1e-38, 1.0)])
def test_the_largest_and_smallest_scales(ctx, scale, size):
    rng = np.random.default_rng(4)
    scale = float(np.float32(scale))
    x = (rng.uniform(-1, 1, (6, 900)) * size).astype(np.float32)
    x[1, ::2] = x[1, 0]
    x[2, 3] = -np.inf
    x[3] = -size
    check_far(ctx, x, scale, 5, rng)
    check_far_grad(ctx, x, "float32", scale, rng)
