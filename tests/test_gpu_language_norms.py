"""The global norm and clipping at the ends of the range of their types, and norms alone."""
import numpy as np
import pytest

import libgpuarray_amd as ga
from libgpuarray_amd import gpuarray
from test_gpu_language import HALF_STEP, TINY, U, decode, encode

pytestmark = pytest.mark.gpu


def norm_of(hosts):
    """The norm in 64 bits, of values that are brought near 1 by a power of two first."""
    x = np.concatenate([np.zeros(0)] + [np.ravel(decode(h)) for h in hosts])
    big = np.abs(x).max() if x.size else 0.0
    if big == 0 or not np.isfinite(big):
        return float(big)
    e = np.frexp(big)[1]
    with np.errstate(over="ignore"):
        return float(np.ldexp(np.sqrt((np.ldexp(x, -e) ** 2).sum()), e))


DOUBLES = [[1e200], [-1e200, 1.0], [1e308, 1e308, 1e-308], [1e-200], [1e-170, 3e-162, -1e-200], [5e-324], [5e-324, 1e-310],
           [1e-155, 1.0], [2.0 ** 486, 2.0 ** 487, 2.0 ** -511, 2.0 ** -512], [1.0, 2.0, 1e-300], [0.0], [1e154, 1e155]]


@pytest.mark.parametrize("values", DOUBLES, ids=str)
@pytest.mark.parametrize("count", [1, 9, 20001])
def test_norm_of_doubles_of_any_size(ctx, values, count):
    """Squares past 2^1024 and below 2^-1074 are in no double, the norm may be."""
    rng = np.random.default_rng(count)
    host = np.zeros(count * 3 + len(values))
    at = rng.permutation(host.size)[: len(values) * min(count, 100)]
    host[at] = np.resize(values, at.size) * rng.uniform(0.5, 1, at.size)
    host[at[0]] = values[0]
    others = np.full(700, 1.5, np.float32)
    for hosts in ([host], [host, others], [others, host[: host.size // 2], host[host.size // 2:]]):
        devs = [gpuarray.array(h, context=ctx) for h in hosts]
        want = norm_of(hosts)
        out = gpuarray.zeros((1,), "float64", context=ctx)
        for norm in (ga.global_norm(devs, out), ga.GlobalNorm(devs).norm(gpuarray.zeros((1,), "float64", context=ctx))):
            got = float(np.asarray(norm)[0])
            if np.isinf(want):
                assert np.isinf(got)
                continue
            # up to 2^16 squares, each and each addition off by 2^-53, a root, and a product with a power of two
            assert abs(got - want) <= want * 2.0 ** -36 + 5e-324, (got, want)
        with np.errstate(over="ignore"):
            assert np.asarray(ga.global_norm(devs)) == np.float32(float(np.asarray(out)[0]))
        if want == 0 or np.isinf(want):
            continue
        bound = want / 3.7 if want / 3.7 > 1e-290 else want * 2
        by = bound / want if bound < want else 1.0
        ga.clip_by_global_norm(devs, bound)
        for h, d in zip(hosts, devs):
            half = 2 * U if h.dtype == np.float32 else 2.0 ** -34
            assert np.all(np.abs(decode(d) - decode(h) * by) <= np.abs(decode(h)) * by * half + 5e-324)


@pytest.mark.parametrize("bad", [np.nan, np.inf])
def test_doubles_without_a_norm_are_left_alone(ctx, bad):
    host = np.full(3000, 1e-200)
    host[77], host[1234] = 1e300, bad
    a, b = gpuarray.array(host, context=ctx), gpuarray.array(np.ones(5, np.float32), context=ctx)
    norm = np.asarray(ga.clip_by_global_norm([a, b], 1.0, norm=gpuarray.zeros((1,), "float64", context=ctx)))
    assert not np.isfinite(norm[0])
    assert np.array_equal(np.asarray(a), host, equal_nan=True) and np.all(np.asarray(b) == 1)
    over = gpuarray.array(np.full(4, 1.5e308), context=ctx)     # the norm itself is in no double
    assert np.isinf(np.asarray(ga.clip_by_global_norm([over], 1.0)))
    assert np.all(np.asarray(over) == 1.5e308)


@pytest.mark.parametrize("kind,value,bound", [("float32", 3e38, 1.0), ("float32", 3e38, 1e-5), ("float32", 1e38, 1e-9), ("float32", 1e30, 1e-30),
                                              ("bfloat16", 1e38, 1e-3), ("bfloat16", 3e38, 1e-20), ("float16", 6e4, 1e-38),
                                              ("float64", 1e300, 1e-5), ("float64", 1e300, 1e-20), ("float64", 1e307, 1e-200)])
@pytest.mark.parametrize("shift", [0, 1])
def test_clipping_by_a_factor_below_the_smallest_normal_number(ctx, kind, value, bound, shift):
    """max_norm / norm below 2^-126 (2^-1022 for doubles) has few bits left, or none; the product has all of them."""
    rng = np.random.default_rng(3)
    x = rng.uniform(-1, 1, 5000) * value / 64
    x[[0, 4999]] = value, -value / 3
    host = x if kind == "float64" else encode(x, kind)
    want = norm_of([host[shift:]])
    root = gpuarray.array(host, context=ctx)
    into = gpuarray.empty((5000,), host.dtype, context=ctx)
    devs, outs = [root[shift:]], [into[shift:]]
    ga.clip_by_global_norm(devs, bound, out=outs)
    exact = decode(host[shift:]) / want * bound
    half, tiny = HALF_STEP.get(kind, 2.0 ** -36), TINY.get(kind, 5e-324)
    assert np.all(np.abs(decode(outs[0]) - exact) <= np.abs(exact) * (half + 2.0 ** -34) + tiny)
    op = ga.GlobalNorm(devs)                                   # in place, by the operator
    op.clip(bound)
    assert np.array_equal(decode(devs[0]), decode(outs[0]))
    mixed = [gpuarray.array(np.full(3, 1e200), context=ctx), gpuarray.array(np.full(300, 1e30, np.float32), context=ctx)]
    ga.clip_by_global_norm(mixed, 1.0)                         # a double's norm, a float's factor: 1e30 / 1.7e200 is 0 in a float
    assert np.max(np.abs(np.asarray(mixed[0]) * np.sqrt(3) - 1)) < 2.0 ** -48 and not np.any(np.asarray(mixed[1]))


def test_norm_operator_without_results(ctx):
    """out=False: norms alone, for lists that could not be clipped: one array twice, overlapping views, shared weights."""
    x = gpuarray.array(np.arange(1, 2001, dtype=np.float32), context=ctx)
    y = gpuarray.array(np.full((3, 5), 2.0, np.float64), context=ctx)
    for arrays in ([x, x], [x[:100], x[50:150], y], [y], []):
        op = ga.GlobalNorm(arrays, out=False, context=ctx)
        want = norm_of([np.asarray(a) for a in arrays])
        got = float(np.asarray(op.norm(gpuarray.zeros((), "float64", context=ctx))))
        assert abs(got - want) <= want * 2.0 ** -40
        assert op.out is None
        with pytest.raises(ga.GpuArrayException):
            op.clip(1.0)
    assert np.array_equal(np.asarray(x), np.arange(1, 2001))
    with pytest.raises(TypeError):                            # (it is the operator that is for norms alone)
        ga.clip_by_global_norm([y], 1.0, out=False)
    with pytest.raises(ga.GpuArrayException):                 # to be clipped in place, no two may overlap
        ga.GlobalNorm([x, x])


def test_long_lists_with_doubles_of_any_size(ctx):
    """More arrays than travel with one launch, so that the partial sums come from several."""
    rng = np.random.default_rng(5)
    kinds = ["float64", "float32", "bfloat16"]
    for large, small in ((1e250, 1e-250), (1.0, 1e-250), (0.0, 1e-250)):
        hosts = [rng.uniform(0.5, 1, 5 + i % 9) * (large if i % 120 == 3 else small) if i % 3 == 0 else
                 encode(rng.standard_normal(7) * (large == 1.0), kinds[i % 3]) for i in range(300)]
        want = norm_of(hosts)
        devs = [gpuarray.array(h, context=ctx) for h in hosts]
        for norm in (ga.global_norm(devs, gpuarray.zeros((), "float64", context=ctx)),
                     ga.GlobalNorm(devs).norm(gpuarray.zeros((), "float64", context=ctx))):
            assert abs(float(np.asarray(norm)) - want) <= want * 2.0 ** -36
        ga.clip_by_global_norm(devs, want / 8)
        for h, d in zip(hosts, devs):
            exact = decode(h) / 8
            assert np.all(np.abs(decode(d) - exact) <= np.abs(exact) * 2.0 ** (-34 if h.dtype == np.float64 else -7))
