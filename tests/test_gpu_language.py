"""Operators of language models (include/gpuarray/language.h) against their
definitions in 64 bits.  The reference has no counterpart; the conventions are
those of its take1 and maxandargmax tests.

Tolerances count roundings.  u = 2^-24 is half a step of float32; a result is
rounded once more to its own type (half a step: 2^-24, 2^-11 for half, 2^-8 for
bfloat16, relative, plus half the smallest subnormal).  Sums of k values of
float32 in any order are off by at most k u times the sum of their magnitudes."""
import ctypes as C

import numpy as np
import pytest

import libgpuarray_amd as ga
from libgpuarray_amd import _lib, gpuarray
from support import arg, to_gpu_view

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF_STEP = {"float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}
TINY = {"float32": 2.0 ** -150, "float16": 2.0 ** -25, "bfloat16": 2.0 ** -134}
TYPES = ["float32", "float16", "bfloat16"]


def np_type(kind):
    return ga.bfloat16 if kind == "bfloat16" else np.dtype(kind)


def encode(x, kind):
    """float64 values as a host array of the type."""
    return ga.to_bfloat16(np.asarray(x, np.float32)) if kind == "bfloat16" else np.asarray(x).astype(kind)


def decode(a, kind=None):
    a = np.asarray(a)
    return (ga.from_bfloat16(a) if a.dtype == ga.bfloat16 else a).astype(np.float64)


def on_gpu(ctx, host, pitch=0, flip=False, fill=None):
    """The host rows on the device, `pitch` elements wider apart than they are
    long, the first one last in memory with `flip`.  Returns (array, root, view of
    a host root that looks like it)."""
    host = np.asarray(host)
    n, d = host.shape
    root = np.zeros((n, d + pitch), host.dtype) if fill is None else np.full((n, d + pitch), fill, host.dtype)
    view = root[::-1, :d] if flip else root[:, :d]
    view[...] = host
    dev, base = to_gpu_view(view, ctx)
    return dev, base, root


def vec(ctx, host, step=1):
    """A 1-D array whose elements lie `step` apart (0: all the same one; negative: in reverse)."""
    host = np.asarray(host)
    if step == 1:
        return gpuarray.array(host, context=ctx)
    if step == 0:
        return gpuarray.from_strided(gpuarray.array(host[:1], context=ctx), 0, host.shape, (0,))
    root = np.zeros(host.size * abs(step), host.dtype)
    view = root[::step] if step > 0 else root[::step][:host.size]
    view[...] = host
    return to_gpu_view(view, ctx)[0]


# ---- embedding --------------------------------------------------------------------------------------

@pytest.mark.parametrize("n,v,d", [(1, 1, 1), (1, 300, 8), (7, 50, 64), (65, 33, 63), (130, 1000, 257), (33, 5, 1000),
                                   (3, 4, 4099), (300, 7, 16)])
@pytest.mark.parametrize("table,out", [("float32", "float32"), ("bfloat16", "bfloat16"), ("float16", "float32"),
                                       ("float32", "bfloat16"), ("bfloat16", "float16")])
def test_embedding(ctx, n, v, d, table, out):
    rng = np.random.default_rng(n + 31 * d)
    w = encode(rng.standard_normal((v, d)), table)
    ids = rng.integers(-v, v, n)
    ids[n // 2] = 77777
    got = ga.embedding(gpuarray.array(w, context=ctx), gpuarray.array(ids, context=ctx), scale=22.5, ignore=77777,
                       dtype=np_type(out))
    want = 22.5 * decode(w)[np.where(ids == 77777, 0, ids)]
    want[ids == 77777] = 0
    err = np.abs(decode(got) - want)
    assert got.dtype == np_type(out)
    assert np.all(err <= np.abs(want) * (U + HALF_STEP[out]) + TINY[out])


@pytest.mark.parametrize("kind", TYPES)
def test_embedding_with_scale_one_copies_the_rows(ctx, kind):
    rng = np.random.default_rng(3)
    w = encode(rng.standard_normal((40, 37)) * 1e3, kind)
    ids = rng.integers(0, 40, 90)
    got = ga.embedding(gpuarray.array(w, context=ctx), gpuarray.array(ids, context=ctx))
    assert np.array_equal(decode(got), decode(w)[ids])


@pytest.mark.parametrize("id_type", ["int8", "uint8", "int16", "uint16", "int32", "uint32", "int64", "uint64"])
def test_embedding_id_types(ctx, id_type):
    w = np.arange(100 * 3, dtype=np.float32).reshape(100, 3)
    ids = np.array([0, 99, 5, 5], id_type)
    got = np.asarray(ga.embedding(gpuarray.array(w, context=ctx), gpuarray.array(ids, context=ctx)))
    assert np.array_equal(got, w[ids.astype(int)])


def test_unsigned_ids_do_not_count_from_the_end(ctx):
    """2^64 - 1 is out of range, and is not `ignore` = -1 either."""
    w = np.arange(12, dtype=np.float32).reshape(4, 3)
    table, ids = gpuarray.array(w, context=ctx), gpuarray.array(np.array([1, 2 ** 64 - 1], np.uint64), context=ctx)
    for ignore in (None, -1):
        out = gpuarray.array(np.full((2, 3), 7, np.float32), context=ctx)
        with pytest.raises(IndexError):
            ga.embedding(table, ids, out=out, ignore=ignore)
        assert np.array_equal(np.asarray(out), [w[1], [7, 7, 7]])
        with pytest.raises(IndexError):
            ga.token_logprobs(table[:2], ids, ignore=ignore)
        grad = gpuarray.zeros((4, 3), context=ctx)
        with pytest.raises(IndexError):
            ga.embedding_grad(table[:2], ids, grad, ignore=ignore)
        assert np.array_equal(np.asarray(grad), [[0, 0, 0], w[0], [0, 0, 0], [0, 0, 0]])
        stats, one = gpuarray.zeros((2, 2), context=ctx), gpuarray.array(np.ones(2, np.float32), context=ctx)
        with pytest.raises(IndexError):
            ga.token_logprobs_grad(table[:2], ids, stats, one, ignore=ignore)


@pytest.mark.parametrize("pitch,flip,step", [(3, False, 2), (0, True, -1), (13, True, 1), (1, False, 0)])
def test_embedding_layouts(ctx, pitch, flip, step):
    rng = np.random.default_rng(5)
    w = rng.standard_normal((30, 45)).astype(np.float32)
    ids = rng.integers(0, 30, 20)
    if step == 0:
        ids[:] = ids[0]
    table, _, _ = on_gpu(ctx, w, pitch, flip)
    out, base, root = on_gpu(ctx, np.zeros((20, 45), np.float32), pitch, flip, fill=-3)
    ga.embedding(table, vec(ctx, ids, step), scale=2.0, out=out)
    assert np.array_equal(np.asarray(out), 2 * w[ids])
    flat = np.asarray(base)[:root.nbytes].view(np.float32).reshape(root.shape)
    assert np.all(flat[:, 45:] == -3)           # what lies between the rows stays


def test_embedding_bounds(ctx):
    w = np.arange(12, dtype=np.float32).reshape(4, 3)
    table = gpuarray.array(w, context=ctx)
    out = gpuarray.array(np.full((5, 3), -9, np.float32), context=ctx)
    ids = gpuarray.array(np.array([0, 4, 3, -5, -4]), context=ctx)
    with pytest.raises(IndexError):
        ga.embedding(table, ids, out=out)
    want = np.full((5, 3), -9, np.float32)
    want[[0, 2, 4]] = w[[0, 3, 0]]
    assert np.array_equal(np.asarray(out), want)
    ga.embedding(table, ids, out=out, check=False)       # not checked: the flag stays for the next one that is
    good = gpuarray.array(np.array([1]), context=ctx)
    with pytest.raises(IndexError):
        ga.embedding(table, good)
    assert np.array_equal(np.asarray(ga.embedding(table, good)), w[1:2])
    # an id is compared with `ignore` before it counts from the end
    got = ga.embedding(table, gpuarray.array(np.array([-1, 3]), context=ctx), ignore=-1)
    assert np.array_equal(np.asarray(got), [[0, 0, 0], w[3]])


def test_embedding_of_nothing(ctx):
    table = gpuarray.zeros((4, 3), context=ctx)
    assert ga.embedding(table, gpuarray.zeros((0,), "int64", context=ctx)).shape == (0, 3)
    assert ga.embedding(gpuarray.zeros((4, 0), context=ctx), gpuarray.zeros((2,), "int64", context=ctx)).shape == (2, 0)
    with pytest.raises(IndexError):
        ga.embedding(gpuarray.zeros((0, 3), context=ctx), gpuarray.zeros((2,), "int64", context=ctx))


@pytest.mark.parametrize("d", [3, 40])
def test_embedding_of_no_token_in_an_empty_table(ctx, d):
    out = gpuarray.array(np.full((5, d), 7, np.float32), context=ctx)
    ids = gpuarray.array(np.full(5, -100), context=ctx)
    ga.embedding(gpuarray.zeros((0, d), context=ctx), ids, ignore=-100, out=out)
    assert np.all(np.asarray(out) == 0)


# ---- its gradient -----------------------------------------------------------------------------------

def check_embedding_grad(got, dout, ids, v, scale, ignore, grad, base=None):
    """`got` against the sums in 64 bits, row by row."""
    x = decode(dout)
    want = np.zeros((v, x.shape[1]))
    mag = np.zeros_like(want)
    count = np.zeros(v)
    keep = ids != ignore
    at = np.where(ids[keep] < 0, ids[keep] + v, ids[keep])
    np.add.at(want, at, x[keep])
    np.add.at(mag, at, np.abs(x[keep]))
    np.add.at(count, at, 1)
    want *= scale
    # the sum, the product with the scale, the sum with the base, the rounding to the type
    bound = (count[:, None] + 1) * U * scale * mag
    if base is not None:
        total = want + decode(base)
        bound = bound + U * np.abs(total)
        want = total
    bound = bound * (1 + 2.0 ** -7) + np.abs(want) * HALF_STEP[grad] + TINY[grad]
    err = np.abs(decode(got) - want)
    assert np.all(err <= bound), (float((err - bound).max()), np.argwhere(err > bound)[:5])
    untouched = count == 0
    if base is None:
        assert not np.any(decode(got)[untouched])
    else:
        assert np.array_equal(decode(got)[untouched], decode(base)[untouched])


@pytest.mark.parametrize("n,v,d", [(1, 1, 1), (1, 70, 8), (64, 5, 64), (65, 33, 63), (1000, 300, 257), (2500, 3, 100),
                                   (700, 2000, 24), (4097, 999, 40), (3, 4, 4099)])
@pytest.mark.parametrize("dout,grad", [("float32", "float32"), ("bfloat16", "float32"), ("float16", "float16"),
                                       ("float32", "bfloat16")])
@pytest.mark.parametrize("accumulate", [False, True])
def test_embedding_grad(ctx, n, v, d, dout, grad, accumulate):
    rng = np.random.default_rng(n + 7 * d)
    x = encode(rng.standard_normal((n, d)), dout)
    ids = np.minimum(rng.geometric(0.02, n) - 1, v - 1)      # low ids come often
    ids[rng.random(n) < 0.2] = -100
    base = encode(rng.standard_normal((v, d)), grad) if accumulate else None
    g = gpuarray.array(base, context=ctx) if accumulate else gpuarray.array(encode(np.full((v, d), 7.0), grad), context=ctx)
    ga.embedding_grad(gpuarray.array(x, context=ctx), gpuarray.array(ids, context=ctx), g, scale=1.5, ignore=-100,
                      accumulate=accumulate)
    check_embedding_grad(g, x, ids, v, 1.5, -100, grad, base)


@pytest.mark.parametrize("n,v,d", [(1, 5000, 1), (256, 3000, 1), (200, 4100, 7), (3, 5000, 8), (256, 4099, 125), (70, 4500, 983), (9, 4200, 4413),
                                   (250, 2, 3001), (256, 30, 2048)])
@pytest.mark.parametrize("dout,grad", [("float16", "float16"), ("bfloat16", "float32"), ("float32", "bfloat16")])
@pytest.mark.parametrize("accumulate", [False, True])
@pytest.mark.parametrize("shift", [0, 1])
def test_embedding_grad_of_few_tokens(ctx, n, v, d, dout, grad, accumulate, shift):
    """Groups of many rows that share 16-byte chunks at their ends, with tokens on either side of such an end or
    none; the memory before and behind the rows stays."""
    rng = np.random.default_rng(n + v + d)
    x = encode(rng.standard_normal((n, d)), dout)
    ids = rng.integers(0, v, n)
    ids[: n // 3] = np.minimum(v - 1, 8192 // (d * np_type(grad).itemsize) * rng.integers(0, 3, n // 3))
    ids[n // 2] = -100
    base = encode(rng.standard_normal((v, d)), grad)
    root = gpuarray.array(np.concatenate([encode([9.0] * shift, grad), base.ravel(), encode([9.0] * 5, grad)]), context=ctx)
    size = np_type(grad).itemsize
    g = gpuarray.from_strided(root, shift * size, (v, d), (d * size, size))
    ga.embedding_grad(gpuarray.array(x, context=ctx), gpuarray.array(ids, context=ctx), g, scale=1.5, ignore=-100, accumulate=accumulate)
    check_embedding_grad(g, x, ids, v, 1.5, -100, grad, base if accumulate else None)
    around = decode(root)
    assert np.all(around[:shift] == 9) and np.all(around[shift + v * d:] == 9)


@pytest.mark.parametrize("n,v,d,share", [(20000, 50257, 72, 0.4), (40000, 700, 64, 0.0), (70001, 65537, 40, 0.9),
                                         (16384, 16384, 64, 0.0), (16385, 300000, 8, 0.1), (150000, 2, 33, 0.0),
                                         (33000, 1, 16, 0.0)])
@pytest.mark.parametrize("accumulate", [False, True])
def test_embedding_grad_of_many_tokens(ctx, n, v, d, share, accumulate):
    """Many tokens, one of them (the share) at every second place."""
    rng = np.random.default_rng(n)
    x = rng.standard_normal((n, d)).astype(np.float32)
    ids = rng.integers(0, v, n)
    ids[rng.random(n) < share] = v // 2
    ids[5::1013] -= v                                        # counted from the end
    ids[::97] = -100
    base = rng.standard_normal((v, d)).astype(np.float32) if accumulate else None
    g = gpuarray.array(base if accumulate else np.full((v, d), 7, np.float32), context=ctx)
    ga.embedding_grad(gpuarray.array(x, context=ctx), gpuarray.array(ids.astype(np.int32), context=ctx), g, ignore=-100,
                      accumulate=accumulate)
    check_embedding_grad(g, x, ids, v, 1.0, -100, "float32", base)


def test_embedding_grad_gives_the_same_bits(ctx):
    rng = np.random.default_rng(8)
    x = gpuarray.array(rng.standard_normal((30000, 96)).astype(np.float32), context=ctx)
    ids = gpuarray.array(np.minimum(rng.geometric(0.001, 30000), 2000), context=ctx)
    first = None
    for _ in range(4):
        g = gpuarray.empty((3000, 96), context=ctx)
        ga.embedding_grad(x, ids, g)
        first = np.asarray(g) if first is None else first
        assert np.array_equal(first, np.asarray(g))


@pytest.mark.parametrize("pitch,flip,step", [(3, False, 2), (0, True, -1), (13, True, 1), (1, False, 0)])
@pytest.mark.parametrize("accumulate", [False, True])
def test_embedding_grad_layouts(ctx, pitch, flip, step, accumulate):
    rng = np.random.default_rng(6)
    x = rng.standard_normal((200, 45)).astype(np.float32)
    ids = rng.integers(0, 30, 200)
    if step == 0:
        ids[:] = ids[0]
    base = rng.standard_normal((30, 45)).astype(np.float32)
    g, root_dev, root = on_gpu(ctx, base, pitch, flip, fill=-3)
    dout, _, _ = on_gpu(ctx, x, pitch, flip)
    ga.embedding_grad(dout, vec(ctx, ids, step), g, accumulate=accumulate)
    check_embedding_grad(g, x, ids, 30, 1.0, -100, "float32", base if accumulate else None)
    flat = np.asarray(root_dev)[:root.nbytes].view(np.float32).reshape(root.shape)
    assert np.all(flat[:, 45:] == -3)


def test_embedding_grad_bounds_and_nothing(ctx):
    x = np.ones((4, 3), np.float32)
    g = gpuarray.array(np.full((5, 3), 7, np.float32), context=ctx)
    with pytest.raises(IndexError):
        ga.embedding_grad(gpuarray.array(x, context=ctx), gpuarray.array(np.array([0, 5, -6, 0]), context=ctx), g)
    want = np.zeros((5, 3))
    want[0] = 2
    assert np.array_equal(np.asarray(g), want)
    g = gpuarray.array(np.full((5, 3), 7, np.float32), context=ctx)
    none = gpuarray.zeros((0, 3), context=ctx), gpuarray.zeros((0,), "int64", context=ctx)
    ga.embedding_grad(*none, g, accumulate=True)
    assert np.all(np.asarray(g) == 7)
    ga.embedding_grad(*none, g)
    assert np.all(np.asarray(g) == 0)
    with pytest.raises(IndexError):
        ga.embedding_grad(gpuarray.array(x, context=ctx), gpuarray.array(np.arange(4), context=ctx),
                          gpuarray.zeros((0, 3), context=ctx))
    ga.embedding_grad(gpuarray.zeros((4, 0), context=ctx), gpuarray.array(np.arange(4), context=ctx),
                      gpuarray.zeros((5, 0), context=ctx))


def test_embedding_grad_infinities_stay_in_their_row(ctx):
    x = np.ones((6, 5), np.float32)
    x[1, 2], x[4, 0] = np.inf, np.nan
    ids = np.array([3, 1, 3, 0, 2, 3])
    g = gpuarray.empty((4, 5), context=ctx)
    ga.embedding_grad(gpuarray.array(x, context=ctx), gpuarray.array(ids, context=ctx), g)
    got = np.asarray(g)
    want = np.zeros((4, 5), np.float32)
    np.add.at(want, ids, x)
    assert np.array_equal(got, want, equal_nan=True)


# ---- log probabilities ------------------------------------------------------------------------------

def softmax64(x, scale):
    """m, log sum, z = scale (x - m), p of the rows in 64 bits; rows of -inf alone have p = 0."""
    m = x.max(1)
    m0 = np.where(np.isinf(m), 0, m)
    z = scale * (x - m0[:, None])
    e = np.exp(z)
    s = e.sum(1)
    with np.errstate(divide="ignore", invalid="ignore"):
        ls = np.log(s)
        p = np.where(s[:, None] > 0, e / s[:, None], 0)
    return m, ls, z, p


def logprob_bounds(x, scale):
    """Bounds for (log sum, log p of every token, entropy).

    z = scale (x - m) is computed with three roundings (the difference, the
    factor, the product): off by 3u|z|; an exponential has two more units (4u).
    The sum has a depth of at most v/64 + 32 additions (64 lanes at least share a row;
    rescaling a partial sum by a new maximum costs its factor, another 8u at
    most 16 times)."""
    m, ls, z, p = softmax64(x, scale)
    az = np.where(p > 0, np.abs(z), 0)
    depth = x.shape[1] / 64 + 32 + 128
    s_rel = depth * U + 4 * U + 3 * U * (p * az).sum(1)
    ls_fin = np.where(np.isfinite(ls), ls, 0)
    ls_err = s_rel + 4 * U * (1 + np.abs(ls_fin))
    zf = np.where(np.isfinite(z), np.abs(z), 0)
    lp_err = 3 * U * zf + ls_err[:, None] + 2 * U * (zf + np.abs(ls_fin)[:, None])
    w = (p * az).sum(1)
    h_err = 2 * w * s_rel + 3 * U * (p * az * az).sum(1) + 8 * U * w + ls_err
    return ls_err, lp_err, h_err


def run_logprobs(ctx, logits, ids, v_x, scale, top, ignore=-100, top_type="int64"):
    t = logits.shape[0]
    new = lambda shape, dt="float32": gpuarray.array(np.full(shape, -77, dt), context=ctx)  # noqa: E731
    out = ga.TokenLogprobs(new((t,)), new((t,)), new((t, 2)), new((t, top)) if top else None,
                           new((t, top), top_type) if top else None)
    ga.token_logprobs(logits, ids, scale=scale, ignore=ignore, out=out)
    return [None if o is None else np.asarray(o) for o in out]


def check_logprobs(x, ids, scale, top, got, ignore=-100):
    """x: the logits in 64 bits, as their type holds them."""
    logp, entropy, stats, top_logp, top_ids = got
    t, v = x.shape
    m, ls, z, p = softmax64(x, scale)
    ls_err, lp_err, h_err = logprob_bounds(x, scale)
    dead = ~np.isfinite(ls)
    with np.errstate(invalid="ignore"):
        lp = np.where(dead[:, None], -np.inf, z - np.where(dead, 0, ls)[:, None])
        entropy64 = np.where(dead, 0, ls - np.where(p > 0, p * z, 0).sum(1))
    assert np.array_equal(stats[:, 0], m.astype(np.float32))
    assert np.array_equal(np.isinf(stats[:, 1]), dead)
    assert np.all(np.abs(stats[~dead, 1] - ls[~dead]) <= ls_err[~dead])
    at = np.where(ids < 0, ids + v, ids)
    at[ids == ignore] = 0
    rows = np.arange(t)
    want = np.where(ids == ignore, 0, lp[rows, at])
    bound = np.where(ids == ignore, 0, lp_err[rows, at])
    assert np.array_equal(np.isinf(want), np.isinf(logp))
    fin = np.isfinite(want)
    assert np.all(np.abs(logp[fin] - want[fin]) <= bound[fin])
    assert np.all(np.abs(entropy - entropy64) <= h_err), float(np.max(np.abs(entropy - entropy64) - h_err))
    if top:
        order = np.argsort(-x, axis=1, kind="stable")[:, :top]
        assert np.array_equal(top_ids, order)
        want = np.take_along_axis(lp, order, 1)
        bound = np.take_along_axis(lp_err, order, 1)
        assert np.array_equal(np.isinf(want), np.isinf(top_logp))
        fin = np.isfinite(want)
        assert np.all(np.abs(top_logp[fin] - want[fin]) <= bound[fin])


@pytest.mark.parametrize("t,v,top", [(1, 1, 1), (1, 2, 2), (3, 64, 64), (5, 65, 5), (2, 100, 0), (64, 1000, 5),
                                     (9, 1001, 20), (2, 4097, 33), (300, 257, 1), (1, 50257, 20), (4, 50257, 64),
                                     (2, 131075, 50), (17, 8191, 3), (1, 300001, 7)])
@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("scale", [1.0, 0.7])
def test_token_logprobs(ctx, t, v, top, kind, scale):
    rng = np.random.default_rng(t + v)
    x = encode(rng.standard_normal((t, v)) * 3, kind)       # in 16 bits many values are equal
    ids = rng.integers(-v, v, t)
    ids[t // 3] = -100 if v < 100 or t > 1 else ids[t // 3]
    if v >= 100:
        ids[ids == -100] += 1
        if t > 1:
            ids[t // 3] = -100
    got = run_logprobs(ctx, gpuarray.array(x, context=ctx), gpuarray.array(ids, context=ctx), v, scale, top)
    check_logprobs(decode(x), ids, scale, top, got)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("v", [70, 1000, 20000])
def test_token_logprobs_masks(ctx, kind, v):
    """Rows of which nothing, one, a few or all but one are left, by -inf and by the type's lowest value; equal rows;
    a rising and a falling row; values at the ends of the type's range."""
    rng = np.random.default_rng(v)
    low = {"float32": np.finfo(np.float32).min, "float16": -65504.0,
           "bfloat16": float(ga.from_bfloat16(np.array([0xff7f], np.uint16).view(ga.bfloat16))[0])}[kind]
    x = np.round(rng.standard_normal((14, v)) * 2, 2)
    x[0] = -np.inf
    x[1] = low
    x[2] = -np.inf
    x[2, v // 2] = 1.5
    x[3] = low
    x[3, v - 1] = 0.25
    x[4, rng.random(v) < 0.99] = -np.inf
    x[5, 3] = -np.inf
    x[6] = 0.0
    x[6, ::3] = -0.0
    x[7] = np.arange(v) * 0.125 if kind == "float32" else np.arange(v) // 64
    x[8] = -x[7]
    x[9] = low
    x[9, : v // 2] = -np.inf
    x[10, rng.random(v) < 0.5] = low
    x[11] = -low * (rng.random(v) < 0.01)
    x[12] = -np.inf
    x[12, [v - 1, v - 2, 1]] = [1, 2, 2]
    x = encode(x, kind)
    ids = rng.integers(0, v, 14)
    ids[12] = 1
    for top in (1, 5, 60):
        got = run_logprobs(ctx, gpuarray.array(x, context=ctx), gpuarray.array(ids, context=ctx), v, 1.0, top)
        check_logprobs(decode(x), ids, 1.0, top, got)


@pytest.mark.parametrize("bad", [np.nan, np.inf])
@pytest.mark.parametrize("v", [66, 3000, 60000])
def test_token_logprobs_rows_without_a_distribution(ctx, bad, v):
    rng = np.random.default_rng(2)
    x = rng.standard_normal((4, v)).astype(np.float32)
    x[1, v - 2] = bad
    x[3, 0] = bad
    x[3, 1] = -np.inf
    ids = np.array([5, 5, 6, 0])
    got = run_logprobs(ctx, gpuarray.array(x, context=ctx), gpuarray.array(ids, context=ctx), v, 1.0, 7)
    check_logprobs(x[::2].astype(np.float64), ids[::2], 1.0, 7, [g[::2] for g in got])
    logp, entropy, stats, top_logp, top_ids = (g[1::2] for g in got)
    assert np.all(np.isnan(logp)) and np.all(np.isnan(entropy)) and np.all(np.isnan(stats[:, 1])) and np.all(np.isnan(top_logp))
    assert np.array_equal(stats[:, 0], np.fmax.reduce(x[1::2], axis=1))
    assert np.array_equal(top_ids, np.tile(np.arange(7), (2, 1)))


@pytest.mark.parametrize("pitch,flip,step", [(3, False, 2), (0, True, -1), (47, True, 1), (1, False, 0)])
@pytest.mark.parametrize("kind", TYPES)
def test_token_logprobs_layouts(ctx, pitch, flip, step, kind):
    rng = np.random.default_rng(9)
    t, v, top = 12, 777, 6
    x = encode(rng.standard_normal((t, v)), kind)
    ids = rng.integers(0, v, t).astype(np.int32)
    if step == 0:
        ids[:] = ids[0]
    logits, _, _ = on_gpu(ctx, x, pitch, flip)
    # results of other layouts: transposed, stepped
    mk = lambda shape, dt="float32": gpuarray.zeros(shape, dt, context=ctx)  # noqa: E731
    out = ga.TokenLogprobs(mk((t * 2,))[::2], mk((t,))[::-1], mk((2, t)).T, mk((top, t)).T, mk((t, 2 * top), "int32")[:, ::2])
    ga.token_logprobs(logits, vec(ctx, ids, step), out=out)
    check_logprobs(decode(x), ids.astype(int), 1.0, top, [np.asarray(o) for o in out])


def test_token_logprobs_only_what_is_asked_for(ctx):
    rng = np.random.default_rng(10)
    x = rng.standard_normal((6, 500)).astype(np.float32)
    logits, ids = gpuarray.array(x, context=ctx), gpuarray.array(rng.integers(0, 500, 6), context=ctx)
    full = ga.token_logprobs(logits, ids, top=4, entropy=True)
    only = ga.token_logprobs(logits, top=4)
    assert only.logp is None and only.entropy is None
    assert np.array_equal(np.asarray(only.top_ids), np.asarray(full.top_ids))
    plain = ga.token_logprobs(logits, ids)
    assert plain.top_ids is None and np.array_equal(np.asarray(plain.logp), np.asarray(full.logp))
    h = gpuarray.zeros((6,), context=ctx)
    ga.token_logprobs(logits, out=ga.TokenLogprobs(None, h, None, None, None))
    assert np.array_equal(np.asarray(h), np.asarray(full.entropy))
    ga.token_logprobs(logits, out=ga.TokenLogprobs(None, None, None, None, None))
    empty = ga.token_logprobs(gpuarray.zeros((0, 500), context=ctx), gpuarray.zeros((0,), "int64", context=ctx), top=3)
    assert empty.top_ids.shape == (0, 3)


def test_token_logprobs_bounds(ctx):
    x = np.zeros((3, 8), np.float32)
    ids = gpuarray.array(np.array([1, 8, -9]), context=ctx)
    out = ga.TokenLogprobs(gpuarray.zeros((3,), context=ctx), None, None, None, None)
    with pytest.raises(IndexError):
        ga.token_logprobs(gpuarray.array(x, context=ctx), ids, out=out)
    assert np.array_equal(np.isnan(np.asarray(out.logp)), [False, True, True])


# ---- their gradient ---------------------------------------------------------------------------------

def grad64(x, ids, g, gh, scale, ignore=-100):
    """The gradient in 64 bits, and a bound.  p = exp(scale (x - m) - ls) has three
    roundings in z, ls rounded to float32 and one in the difference, an
    exponential of two units: off by (4|z| + 3|ls| + 4) u relative; the rest is four
    operations; scale once more."""
    t, v = x.shape
    m, ls, z, p = softmax64(x, scale)
    dead = ~np.isfinite(ls)
    lsf = np.where(dead, 0, ls)
    with np.errstate(invalid="ignore"):
        lp = np.where(p > 0, z - lsf[:, None], 0)
    h = -(p * lp).sum(1)
    g = np.where(ids == ignore, 0, g)
    hot = np.zeros((t, v))
    hot[np.arange(t), np.where(ids == ignore, 0, ids)] = 1
    d = scale * (g[:, None] * (hot - p) - gh[:, None] * p * (lp + h[:, None]))
    d[dead] = 0
    az = np.where(p > 0, np.abs(z), 0)
    rel = (4 * az + 3 * np.abs(lsf)[:, None] + 16) * U
    # the exponent itself, and log p and the entropy inside the second term
    bound = scale * p * rel * (np.abs(g)[:, None] + np.abs(gh)[:, None] * (np.abs(lp) + np.abs(h)[:, None] + 1))
    bound += 8 * U * scale * np.abs(g)[:, None] * hot
    return d, bound, h, m, ls


@pytest.mark.parametrize("t,v", [(1, 1), (1, 2), (3, 64), (5, 65), (64, 1000), (7, 4099), (2, 50257), (130, 31), (1, 131075)])
@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("which", ["logp", "entropy", "both"])
def test_token_logprobs_grad(ctx, t, v, kind, which):
    rng = np.random.default_rng(t + v)
    x = encode(rng.standard_normal((t, v)) * 3, kind)
    ids = rng.integers(0, v, t)
    ids[t // 2] = -100 if t > 1 else ids[t // 2]
    g = rng.standard_normal(t).astype(np.float32) if which != "entropy" else np.zeros(t, np.float32)
    gh = rng.standard_normal(t).astype(np.float32) if which != "logp" else np.zeros(t, np.float32)
    scale = 0.75
    want, bound, h, m, ls = grad64(decode(x), ids, g.astype(np.float64), gh.astype(np.float64), scale)
    dev = lambda a: gpuarray.array(a, context=ctx)  # noqa: E731
    stats = dev(np.stack([m, ls], 1).astype(np.float32))
    pair = (dev(ids), dev(g)) if which != "entropy" else (None, None)
    ent = dict(entropy=dev(h.astype(np.float32)), dentropy=dev(gh)) if which != "logp" else {}
    got = ga.token_logprobs_grad(dev(x), pair[0], stats, pair[1], scale=scale, ignore=-100, **ent)
    err = np.abs(decode(got) - want)
    limit = bound * (1 + 2.0 ** -7) + np.abs(want) * HALF_STEP[kind] + TINY[kind]
    assert np.all(err <= limit), float((err / limit).max())
    logits = dev(x)                                            # in place
    again = ga.token_logprobs_grad(logits, pair[0], stats, pair[1], scale=scale, ignore=-100, out=logits, **ent)
    assert again is logits and np.array_equal(decode(again), decode(got))


def test_token_logprobs_grad_against_differences(ctx):
    """Differences of the definition in 64 bits, at every logit of a small case."""
    rng = np.random.default_rng(12)
    t, v, scale, step = 3, 11, 1.3, 1e-5
    x = rng.standard_normal((t, v)).astype(np.float32)
    ids, g, gh = np.array([2, 10, 0]), rng.standard_normal(t), rng.standard_normal(t)

    def loss(y):
        m, ls, z, p = softmax64(y, scale)
        lp = z - ls[:, None]
        return (g * lp[np.arange(t), ids]).sum() + (gh * -(p * lp).sum(1)).sum()

    want = np.zeros((t, v))
    for i in range(t):
        for j in range(v):
            y = x.astype(np.float64)
            y[i, j] += step
            up = loss(y)
            y[i, j] -= 2 * step
            want[i, j] = (up - loss(y)) / (2 * step)
    dev = lambda a: gpuarray.array(a, context=ctx)  # noqa: E731
    lp = ga.token_logprobs(dev(x), dev(ids), scale=scale, entropy=True)
    got = ga.token_logprobs_grad(dev(x), dev(ids), lp.stats, dev(g.astype(np.float32)), entropy=lp.entropy,
                                 dentropy=dev(gh.astype(np.float32)), scale=scale)
    # truncation: step^2 / 6 times third derivatives of a few tens; the rest are float32 roundings of values below 8
    assert np.max(np.abs(np.asarray(got) - want)) < 1e-8 + 64 * 8 * U


@pytest.mark.parametrize("kind", TYPES)
def test_token_logprobs_grad_of_masked_rows(ctx, kind):
    rng = np.random.default_rng(13)
    t, v = 5, 900
    x = rng.standard_normal((t, v))
    x[0] = -np.inf
    x[1, rng.random(v) < 0.9] = -np.inf
    x[1, 4] = 1.0
    x[2] = -np.inf
    x[2, 7] = 3.0
    x[3] = {"float32": np.finfo(np.float32).min, "float16": -65504.0,
            "bfloat16": float(ga.from_bfloat16(np.array([0xff7f], np.uint16).view(ga.bfloat16))[0])}[kind]
    x = encode(x, kind)
    ids = np.array([3, 4, 7, 5, 6])
    g, gh = rng.standard_normal(t), rng.standard_normal(t)
    want, bound, _, _, _ = grad64(decode(x), ids, g.astype(np.float32).astype(np.float64), gh.astype(np.float32).astype(np.float64), 1.0)
    dev = lambda a: gpuarray.array(a, context=ctx)  # noqa: E731
    lp = ga.token_logprobs(dev(x), dev(ids), entropy=True)
    got = decode(ga.token_logprobs_grad(dev(x), dev(ids), lp.stats, dev(g.astype(np.float32)), entropy=lp.entropy,
                                        dentropy=dev(gh.astype(np.float32))))
    # the statistics are the operator's own here: their bounds join those of grad64
    ls_err, _, h_err = logprob_bounds(decode(x), 1.0)
    _, ls, _, p = softmax64(decode(x), 1.0)
    joined = p * (ls_err[:, None] * (np.abs(g) + np.abs(gh) * 30)[:, None] + (h_err * np.abs(gh))[:, None])
    limit = (bound + joined) * (1 + 2.0 ** -7) + np.abs(want) * HALF_STEP[kind] + TINY[kind]
    assert not np.any(got[0])
    assert np.all(np.abs(got - want) <= limit)


@pytest.mark.parametrize("in_pitch,out_pitch,flip", [(0, 1, False), (5, 0, True), (3, 3, False), (1, 2, True)])
@pytest.mark.parametrize("kind", TYPES)
def test_token_logprobs_grad_layouts(ctx, in_pitch, out_pitch, flip, kind):
    rng = np.random.default_rng(14)
    t, v = 9, 801
    x = encode(rng.standard_normal((t, v)), kind)
    ids, g = rng.integers(0, v, t), rng.standard_normal(t).astype(np.float32)
    want, bound, h, m, ls = grad64(decode(x), ids, g.astype(np.float64), np.zeros(t), 1.0)
    logits, _, _ = on_gpu(ctx, x, in_pitch, flip)
    mark = encode(np.full((1,), -3.0), kind)[0]
    out, base, root = on_gpu(ctx, np.zeros((t, v), x.dtype), out_pitch, not flip, fill=mark)
    stats = to_gpu_view(np.stack([m, ls]).astype(np.float32).T, ctx)[0]
    ga.token_logprobs_grad(logits, vec(ctx, ids, 3), stats, vec(ctx, g, -1), out=out)
    limit = bound * (1 + 2.0 ** -7) + np.abs(want) * HALF_STEP[kind] + TINY[kind]
    assert np.all(np.abs(decode(out) - want) <= limit)
    flat = np.asarray(base)[:root.nbytes].view(root.dtype).reshape(root.shape)
    assert np.all(decode(flat[:, v:]) == -3)


def test_token_logprobs_grad_bounds(ctx):
    dev = lambda a: gpuarray.array(a, context=ctx)  # noqa: E731
    x = dev(np.zeros((2, 4), np.float32))
    stats = dev(np.array([[0, np.log(4)]] * 2, np.float32))
    out = gpuarray.zeros((2, 4), context=ctx)
    with pytest.raises(IndexError):
        ga.token_logprobs_grad(x, dev(np.array([4, 1])), stats, dev(np.ones(2, np.float32)), out=out)
    got = np.asarray(out)
    assert not np.any(got[0]) and abs(got[1, 1] - 0.75) < 1e-6


# ---- global norm and clipping -----------------------------------------------------------------------

def arrays_of(ctx, sizes, kinds, rng, by=1.0):
    hosts = [encode(rng.standard_normal(s) * by, kinds[i % len(kinds)]) if kinds[i % len(kinds)] != "float64"
             else rng.standard_normal(s) * by for i, s in enumerate(sizes)]
    return hosts, [gpuarray.array(h, context=ctx) for h in hosts]


@pytest.mark.parametrize("sizes", [[1], [7, 1, 100], [(3, 5), (1000,), (257, 33), (0,), (8192,), (8193,), (1 << 17,)],
                                   [11] * 130, [(40, i + 1) for i in range(300)], [100003, 3, 70001]])
@pytest.mark.parametrize("kinds", [["float32"], ["bfloat16"], ["float16", "float32", "bfloat16", "float64"]])
@pytest.mark.parametrize("ratio", [0.5, 3.7])
def test_clip_by_global_norm(ctx, sizes, kinds, ratio):
    rng = np.random.default_rng(len(sizes))
    hosts, devs = arrays_of(ctx, sizes, kinds, rng)
    want = np.sqrt(sum((decode(h) ** 2).sum() for h in hosts))
    norm = np.asarray(ga.global_norm(devs))
    assert abs(norm - want) <= want * 2 * U
    into = [gpuarray.empty(h.shape, h.dtype, context=ctx) for h in hosts]
    got = ga.clip_by_global_norm(devs, want / ratio, out=into)
    assert np.array_equal(np.asarray(got), norm)
    by = 1 / ratio if ratio > 1 else 1.0
    for i, (h, o) in enumerate(zip(hosts, into)):
        kind = kinds[i % len(kinds)]
        x = decode(h)
        half = HALF_STEP.get(kind, 2.0 ** -53)
        # the factor in 32 bits (64 for float64, where the norm's own sum counts: 2^-40 is ample), the product, the type
        limit = np.abs(x) * by * ((2 * U if kind != "float64" else 2.0 ** -40) + half) + TINY.get(kind, 0)
        assert np.all(np.abs(decode(o) - by * x) <= (limit if ratio > 1 else 0))
        assert np.array_equal(decode(devs[i]), x)
    ga.clip_by_global_norm(devs, want / ratio)                  # in place
    for a, o in zip(devs, into):
        assert np.array_equal(decode(a), decode(o))


def test_global_norm_at_the_ends_of_the_range(ctx):
    dev = lambda a: gpuarray.array(a, context=ctx)  # noqa: E731
    out64 = gpuarray.zeros((1,), "float64", context=ctx)
    for value in (1e30, 1e-38, 1e-42):
        x = dev(np.full(1000, value, np.float32))
        want = float(np.float32(value)) * np.sqrt(1000.0)
        assert abs(float(np.asarray(ga.global_norm([x], out64))[0]) - want) <= want * 2.0 ** -40
    assert float(np.asarray(ga.global_norm([], context=ctx))) == 0.0
    assert float(np.asarray(ga.global_norm([dev(np.zeros((0, 3), np.float32))]))) == 0.0
    x = dev(np.full(3, 2.0, np.float32))
    assert abs(float(np.asarray(ga.global_norm([x, x]))) - np.sqrt(24.0)) < 1e-6       # listed twice, counts twice


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_clipping_leaves_non_finite_gradients_alone(ctx, bad):
    host = np.ones(5000, np.float32)
    host[4321] = bad
    a, b = gpuarray.array(host, context=ctx), gpuarray.array(np.full(3, 5, np.float32), context=ctx)
    norm = np.asarray(ga.clip_by_global_norm([a, b], 1.0))
    assert not np.isfinite(norm)
    assert np.array_equal(np.asarray(a), host, equal_nan=True) and np.all(np.asarray(b) == 5)


def test_clipping_special_norms_and_layouts(ctx):
    dev = lambda a: gpuarray.array(a, context=ctx)  # noqa: E731
    f = dev(np.asfortranarray(np.arange(12, dtype=np.float32).reshape(3, 4)))
    assert f.flags.f_contiguous and not f.flags.c_contiguous
    view = dev(np.arange(20, dtype=np.float32))[3:11]           # off the 16-byte boundaries
    want = np.sqrt(506 + sum(i * i for i in range(3, 11)))
    ga.clip_by_global_norm([f, view], np.inf)
    assert np.array_equal(np.asarray(view), np.arange(3, 11))
    ga.clip_by_global_norm([f, view], 0.0)
    assert not np.any(np.asarray(f)) and not np.any(np.asarray(view))
    assert abs(want) > 0


@pytest.mark.parametrize("count", [1, 64, 65, 300, 4097])
def test_global_norm_operator(ctx, count):
    """The operator that holds its arrays against the call that does not, over lists of any length."""
    rng = np.random.default_rng(count)
    kinds = ["bfloat16", "float32", "float16", "float64"]
    sizes = [(i % 7,) if count > 1 else (5,) for i in range(count)]
    sizes[count // 2] = (40003,)
    hosts, devs = arrays_of(ctx, sizes, kinds, rng)
    into = [gpuarray.empty(h.shape, h.dtype, context=ctx) for h in hosts]
    op = ga.GlobalNorm(devs, out=into)
    norm = np.asarray(op.norm())
    want = np.sqrt(sum((decode(h) ** 2).sum() for h in hosts))
    assert abs(norm - want) <= want * 2 * U
    assert np.array_equal(np.asarray(op.clip(want / 2)), norm)
    again = [gpuarray.empty(h.shape, h.dtype, context=ctx) for h in hosts]
    ga.clip_by_global_norm(devs, want / 2, out=again)
    # The two add the squares of fewer than 2^16 elements in orders of their own: sums of 64 bits that are each
    # off by less than 2^16 2^-53, norms by half of that.  Factors of 32 bits are the same here; float64 keeps the difference.
    for a, b, h, d in zip(into, again, hosts, devs):
        limit = np.abs(decode(b)) * 2.0 ** -36 if h.dtype == np.float64 else 0
        assert np.all(np.abs(decode(a) - decode(b)) <= limit) and np.array_equal(decode(d), decode(h))
    big = count // 2
    assert np.max(np.abs(decode(into[big]) - decode(hosts[big]) / 2)) < 0.02
    assert np.array_equal(np.asarray(ga.global_norm(devs)), norm)


def test_global_norm_operator_holds_its_arrays(ctx):
    a = gpuarray.array(np.full(1000, 3, np.float32), context=ctx)
    op = ga.GlobalNorm([a])
    op.arrays = None
    view = a[:2]
    del a
    gpuarray.array(np.zeros(1000, np.float32), context=ctx)      # would take the freed block
    assert abs(float(np.asarray(op.clip(1.0))) - 3 * np.sqrt(1000)) < 1e-3
    assert np.max(np.abs(np.asarray(view) - 1 / np.sqrt(1000))) < 1e-6
    nothing = ga.GlobalNorm([], context=ctx)
    assert float(np.asarray(nothing.norm())) == 0.0 and float(np.asarray(nothing.clip(1.0))) == 0.0


# ---- long offsets, graphs, the whole together -------------------------------------------------------

def test_offsets_past_32_bits(ctx):
    """Rows and tables that lie more than 2^32 bytes (and elements) apart."""
    big = gpuarray.empty((5 << 30,), "uint8", context=ctx)
    rng = np.random.default_rng(20)
    v, step = 1003, 3 << 29
    x = rng.standard_normal((4, v)).astype(np.float16)
    logits = gpuarray.from_strided(big, 64, (4, v), (step, 2), dtype="float16")
    for i in range(4):
        gpuarray.from_strided(big, 64 + i * step, (v,), (2,), dtype="float16").write(x[i])
    ids = np.array([1, 2, 1002, 7])
    got = run_logprobs(ctx, logits, gpuarray.array(ids, context=ctx), v, 1.0, 3)
    check_logprobs(x.astype(np.float64), ids, 1.0, 3, got)
    want, bound, h, m, ls = grad64(x.astype(np.float64), ids, np.ones(4), np.zeros(4), 1.0)
    d = ga.token_logprobs_grad(logits, gpuarray.array(ids, context=ctx),
                               gpuarray.array(np.stack([m, ls], 1).astype(np.float32), context=ctx),
                               gpuarray.array(np.ones(4, np.float32), context=ctx))
    assert np.all(np.abs(decode(d) - want) <= bound * 1.01 + np.abs(want) * HALF_STEP["float16"] + TINY["float16"])
    rows = ga.embedding(logits, gpuarray.array(np.array([3, 0]), context=ctx))
    assert np.array_equal(np.asarray(rows), x[[3, 0]])
    dout = rng.standard_normal((3, v)).astype(np.float32)
    ga.embedding_grad(gpuarray.array(dout, context=ctx), gpuarray.array(np.array([3, 1, 3]), context=ctx), logits)
    check_embedding_grad(logits.copy(), dout, np.array([3, 1, 3]), 4, 1.0, -100, "float16")
    del logits, big
    n = (1 << 31) + 12345                                        # more than 2^31 elements
    long = gpuarray.zeros((n,), "float16", context=ctx)
    gpuarray.from_strided(long, 2 * (n - 2), (2,), (2,)).write(np.array([3, 4], np.float16))
    assert float(np.asarray(ga.clip_by_global_norm([long], 2.5))) == 5.0
    assert np.array_equal(np.asarray(long[n - 3:]), [0, 1.5, 2])


def test_language_operators_replay_from_a_graph(ctx):
    """One training step recorded and replayed on changing inputs, with eager work in between."""
    hip = C.CDLL("libamdhip64.so")
    stream = C.c_void_p(_lib.extension("hip_get_stream", C.c_void_p, [C.c_void_p])(ctx.ctx))
    rng = np.random.default_rng(21)
    v, n = 601, 3000
    table = gpuarray.array(rng.standard_normal((v, v)).astype(np.float32), context=ctx)
    ids, targets = gpuarray.zeros((n,), "int32", context=ctx), gpuarray.zeros((n,), "int32", context=ctx)
    dlogp = gpuarray.array(np.full(n, -1.0 / n, np.float32), context=ctx)
    mk = lambda shape, dt="float32": gpuarray.zeros(shape, dt, context=ctx)  # noqa: E731

    def outputs():
        return dict(h=mk((n, v)), logp=mk((n,)), ent=mk((n,)), stats=mk((n, 2)), topl=mk((n, 3)), topi=mk((n, 3), "int64"),
                    d=mk((n, v)), g=mk((v, v)), clipped=mk((v, v)), norm=mk(()))

    def issue(o):
        ga.embedding(table, ids, out=o["h"], check=False)
        ga.token_logprobs(o["h"], targets, out=ga.TokenLogprobs(o["logp"], o["ent"], o["stats"], o["topl"], o["topi"]), check=False)
        ga.token_logprobs_grad(o["h"], targets, o["stats"], dlogp, out=o["d"], check=False)
        ga.embedding_grad(o["d"], ids, o["g"], check=False)
        ga.clip_by_global_norm([o["g"]], 1e-3, out=[o["clipped"]], norm=o["norm"])

    eager, replayed = outputs(), outputs()
    for o in (eager, replayed):
        o["all"] = gpuarray.zeros((), context=ctx)
    ops = {id(o): ga.GlobalNorm([o["d"], o["g"], o["h"]]) for o in (eager, replayed)}
    step = issue

    def issue(o):
        step(o)
        ops[id(o)].clip(5.0, norm=o["all"])

    issue(eager)
    issue(replayed)
    ctx.sync()
    graph, gexec = C.c_void_p(), C.c_void_p()
    assert hip.hipStreamBeginCapture(stream, 0) == 0
    try:
        issue(replayed)
        with pytest.raises(_lib.UnsupportedException):
            ga.GlobalNorm([eager["d"]])                          # its table cannot be copied now
        for call in (lambda: ga.embedding(table, ids, out=replayed["h"]),        # what waits is refused, and breaks nothing
                     lambda: ga.embedding_grad(replayed["d"], ids, replayed["g"]),
                     lambda: ga.token_logprobs(replayed["h"], targets, out=ga.TokenLogprobs(replayed["logp"], None, None, None, None)),
                     lambda: ga.token_logprobs_grad(replayed["h"], targets, replayed["stats"], dlogp, out=replayed["d"])):
            with pytest.raises(_lib.UnsupportedException):
                call()
    finally:
        rc = hip.hipStreamEndCapture(stream, C.byref(graph))
    assert rc == 0
    assert hip.hipGraphInstantiate(C.byref(gexec), graph, None, None, C.c_size_t(0)) == 0
    try:
        for _ in range(4):
            ids.write(rng.integers(0, v, n).astype(np.int32))
            targets.write(rng.integers(0, v, n).astype(np.int32))
            for o in replayed.values():
                o.write(np.full(o.shape, -7, o.dtype))
            issue(eager)
            ctx.sync()
            assert hip.hipGraphLaunch(gexec, stream) == 0
            ctx.sync()
            for k in eager:
                assert np.array_equal(np.asarray(eager[k]), np.asarray(replayed[k])), k
    finally:
        hip.hipGraphExecDestroy(gexec)
        hip.hipGraphDestroy(graph)


def test_two_graphs_share_the_workspaces(ctx):
    """Single steps and a small batch, recorded apart and replayed in turn: rows in pieces and their counters, few
    tokens added and not, the scratch of the sort."""
    hip = C.CDLL("libamdhip64.so")
    stream = C.c_void_p(_lib.extension("hip_get_stream", C.c_void_p, [C.c_void_p])(ctx.ctx))
    rng = np.random.default_rng(29)
    v, d = 50257, 24
    mk = lambda shape, dt="float32": gpuarray.zeros(shape, dt, context=ctx)  # noqa: E731
    table = gpuarray.array(rng.standard_normal((v, d)).astype(np.float32), context=ctx)

    class Step(object):
        def __init__(self, n, t):
            self.logits = gpuarray.array(rng.standard_normal((t, v)).astype(np.float16), context=ctx)
            self.ids, self.targets = mk((n,), "int32"), mk((t,), "int64")
            self.dlogp = gpuarray.array(np.full(t, -1.0 / t, np.float32), context=ctx)
            self.out = dict(h=mk((n, d)), logp=mk((t,)), ent=mk((t,)), stats=mk((t, 2)), topl=mk((t, 20)),
                            topi=mk((t, 20), "int32"), dl=mk((t, v), "float16"), g=mk((v, d)), norm=mk(()))
            self.sum = mk((v, d))
            self.op = ga.GlobalNorm([self.out["g"], self.out["dl"]])

        def issue(self):
            o = self.out
            ga.embedding(table, self.ids, out=o["h"], check=False)
            ga.token_logprobs(self.logits, self.targets, out=ga.TokenLogprobs(o["logp"], o["ent"], o["stats"], o["topl"], o["topi"]),
                              check=False)
            ga.token_logprobs_grad(self.logits, self.targets, o["stats"], self.dlogp, out=o["dl"], check=False)
            ga.embedding_grad(o["h"], self.ids, o["g"], check=False)
            ga.embedding_grad(o["h"], self.ids, self.sum, accumulate=True, check=False)
            self.op.clip(0.5, norm=o["norm"])

        def values(self):
            return {k: np.asarray(a) for k, a in self.out.items()}

    steps = [Step(8, 3), Step(700, 40)]
    graphs = []
    for s in steps:
        s.issue()
    ctx.sync()
    try:
        for s in steps:
            graph, gexec = C.c_void_p(), C.c_void_p()
            assert hip.hipStreamBeginCapture(stream, 0) == 0
            try:
                s.issue()
            finally:
                rc = hip.hipStreamEndCapture(stream, C.byref(graph))
            assert rc == 0
            assert hip.hipGraphInstantiate(C.byref(gexec), graph, None, None, C.c_size_t(0)) == 0
            graphs.append((graph, gexec))
        for turn in range(4):
            for s in steps:
                s.ids.write(rng.integers(0, v, s.ids.shape[0]).astype(np.int32))
                s.targets.write(rng.integers(0, v, s.targets.shape[0]))
                s.sum.memset(0)
            for s in steps:
                s.issue()
            ctx.sync()
            want, sums = [s.values() for s in steps], [np.asarray(s.sum) for s in steps]
            for s in steps:
                for a in s.out.values():
                    a.write(np.full(a.shape, 3, a.dtype))
                s.sum.memset(0)
            for i in (0, 1, 0, 1)[turn % 2:]:
                assert hip.hipGraphLaunch(graphs[i][1], stream) == 0
            ctx.sync()
            for i, s in enumerate(steps):
                got = s.values()
                for k in got:
                    assert np.array_equal(got[k], want[i][k]), (turn, i, k)
                times = (0, 1, 0, 1)[turn % 2:].count(i)          # every replay adds the same rows once more
                assert np.all(np.abs(np.asarray(s.sum) - times * sums[i]) <= 4 * U * np.abs(times * sums[i]))
    finally:
        for graph, gexec in graphs:
            hip.hipGraphExecDestroy(gexec)
            hip.hipGraphDestroy(graph)


def test_a_bigram_model_is_trained(ctx):
    """Rows of a (v, v) table are the logits of the next token: two steps of these operators and an update through
    GpuElemwise against the same steps in 64 bits."""
    rng = np.random.default_rng(22)
    v, n, rate, limit = 97, 400, 0.5, 0.05
    w = (rng.standard_normal((v, v)) * 0.1).astype(np.float32)
    text = rng.integers(0, v, n + 1)
    text[::13] = -100                                            # the ends of documents
    ids, targets = text[:-1], text[1:]
    table = gpuarray.array(w, context=ctx)
    update = ga.GpuElemwise(ctx, "w = w - r * g", [arg("w", "float32", read=True, write=True),
                                                   arg("r", "float32", scalar=True), arg("g", "float32", read=True)])
    dev_ids, dev_targets = gpuarray.array(ids, context=ctx), gpuarray.array(targets, context=ctx)
    dlogp = gpuarray.array(np.full(n, -1.0 / n, np.float32), context=ctx)
    grad = gpuarray.empty((v, v), context=ctx)
    w64 = w.astype(np.float64)
    for _ in range(2):
        rows = ga.embedding(table, dev_ids, ignore=-100)
        lp = ga.token_logprobs(rows, dev_targets, ignore=-100)
        dlogits = ga.token_logprobs_grad(rows, dev_targets, lp.stats, dlogp, ignore=-100)
        ga.embedding_grad(dlogits, dev_ids, grad, ignore=-100)
        norm = ga.clip_by_global_norm([grad], limit)
        update(table, np.float32(rate), grad)

        x = np.where((ids == -100)[:, None], 0, w64[np.where(ids == -100, 0, ids)])
        d, _, _, _, ls = grad64(x, targets, np.full(n, -1.0 / n), np.zeros(n), 1.0)
        g64 = np.zeros((v, v))
        np.add.at(g64, ids[ids != -100], d[ids != -100])
        norm64 = np.sqrt((g64 ** 2).sum())
        # every float32 operation is off by u of values that stay below 8; sums over at most n tokens of 1/n each
        assert abs(float(np.asarray(norm)) - norm64) <= norm64 * 1000 * U
        w64 = w64 - rate * g64 * min(1.0, limit / norm64)
        assert np.max(np.abs(np.asarray(table) - w64)) <= 64 * U
        want = np.where(targets == -100, 0, x[np.arange(n), np.where(targets == -100, 0, targets)] - x.max(1) - ls)
        assert np.max(np.abs(np.asarray(lp.logp) - want)) <= 256 * U


def test_bfloat16_arrays(ctx):
    """The element type itself: host conversions, copies of any layout, conversions on the device."""
    rng = np.random.default_rng(23)
    x = rng.standard_normal((37, 53)).astype(np.float32)
    a = gpuarray.array(ga.to_bfloat16(x), context=ctx)
    assert a.dtype == ga.bfloat16 and a.itemsize == 2
    assert np.all(np.abs(decode(a) - x) <= np.abs(x) * HALF_STEP["bfloat16"])
    assert np.array_equal(decode(a.T.copy()), decode(a).T)
    assert np.array_equal(decode(a[::2, 3:]), decode(a)[::2, 3:])
    assert np.array_equal(np.asarray(a.astype("float32")), decode(a).astype(np.float32))
    back = gpuarray.array(x, context=ctx).astype(ga.bfloat16)
    assert np.array_equal(decode(back), decode(a))
    special = np.array([np.inf, -np.inf, np.nan, 0.0, -0.0, 3.4e38, 1e-40], np.float32)
    dev = gpuarray.array(special, context=ctx).astype(ga.bfloat16)
    assert np.array_equal(decode(dev), decode(ga.to_bfloat16(special)), equal_nan=True)


def test_numbers_become_bfloat16_and_back(ctx):
    """Lists, scalars and arrays of other types, wherever a host value meets an array of bfloat16."""
    x = [[1.5, -2.25], [3.0, 1e30]]
    a = gpuarray.array(x, dtype=ga.bfloat16, context=ctx)
    want = decode(ga.to_bfloat16(x))
    assert a.shape == (2, 2) and np.array_equal(decode(a), want)
    assert np.array_equal(np.asarray(a, dtype="float64"), want)
    assert np.array_equal(np.asarray(gpuarray.array(ga.to_bfloat16(x), dtype="float32", context=ctx)), want)
    assert gpuarray.array(2.5, dtype=ga.bfloat16, context=ctx).shape == ()
    assert ga.from_bfloat16(ga.to_bfloat16(2.5)).shape == ()
    a[0] = 7
    a[1, 1] = -0.5
    assert np.array_equal(decode(a), [[7, 7], [3, -0.5]])
    assert a[1, 1] and not gpuarray.array(-0.0, dtype=ga.bfloat16, context=ctx)
    from libgpuarray_amd.elemwise import GpuElemwise, arg as e_arg
    from libgpuarray_amd import ndgpuarray
    k = GpuElemwise(ctx, "r = a * s", [e_arg("r", ga.bfloat16, write=True), e_arg("a", ga.bfloat16, read=True),
                                       e_arg("s", ga.bfloat16, scalar=True)])
    r = gpuarray.empty((2, 2), ga.bfloat16, context=ctx)
    k(r, a, 1.5)
    assert np.array_equal(decode(r), [[10.5, 10.5], [4.5, -0.75]])
    b = gpuarray.array(ga.to_bfloat16(x), context=ctx, cls=ndgpuarray)
    assert np.array_equal(decode(b + b), 2 * want)
    assert np.array_equal(np.asarray(b > 2.0), want > 2)
    with pytest.raises(TypeError):
        b + 1.0                                              # no common type: convert one of them
    with pytest.raises(_lib.GpuArrayException):
        b.sum()


def test_refusals_of_python_values(ctx):
    z = lambda shape, dt="float32": gpuarray.zeros(shape, dt, context=ctx)  # noqa: E731
    table, ids = z((9, 8)), z((4,), "int64")
    for call in (lambda: ga.embedding(z((9,)), ids), lambda: ga.embedding(table, z((), "int64")),
                 lambda: ga.embedding(table, ids, ignore=1 << 63), lambda: ga.token_logprobs(z(())),
                 lambda: ga.token_logprobs(table, top=-1), lambda: ga.embedding_grad(z((4, 8)), ids, table, ignore=-(1 << 63) - 1)):
        with pytest.raises(ValueError):
            call()


# ---- refusals: nothing is launched, so these also run without a device -------------------------------

def refusals(ctx):
    """(what, error code, call)"""
    z = lambda shape, dt="float32": gpuarray.zeros(shape, dt, context=ctx)  # noqa: E731
    E = _lib
    table, ids, out = z((9, 8)), z((4,), "int64"), z((4, 8))
    x, t1, t2 = z((4, 16)), z((4,)), z((4, 2))
    T = ga.TokenLogprobs
    wide = z((8, 16))
    buf = z((100,), "uint8")
    odd = gpuarray.from_strided(buf, 1, (4,), (4,), dtype="float32")
    other = z((16, 8)).T
    return [
        ("out has another length", E.GA_INVALID_ERROR, lambda: ga.embedding(table, ids, out=z((5, 8)))),
        ("rows have another length", E.GA_INVALID_ERROR, lambda: ga.embedding(table, ids, out=z((4, 7)))),
        ("ids of two dims", E.GA_INVALID_ERROR, lambda: ga.embedding(table, z((4, 1), "int64"), out=out)),
        ("float ids", E.GA_VALUE_ERROR, lambda: ga.embedding(table, t1, out=out)),
        ("a table of integers", E.GA_UNSUPPORTED_ERROR, lambda: ga.embedding(z((9, 8), "int32"), ids, out=out)),
        ("a double table", E.GA_UNSUPPORTED_ERROR, lambda: ga.embedding(z((9, 8), "float64"), ids, out=out)),
        ("rows with steps", E.GA_INVALID_ERROR, lambda: ga.embedding(z((9, 16))[:, ::2], ids, out=out)),
        ("reversed rows", E.GA_INVALID_ERROR, lambda: ga.embedding(table[:, ::-1], ids, out=out)),
        ("out within the table", E.GA_VALUE_ERROR, lambda: ga.embedding(table, ids, out=table[:4])),
        ("rows of out on each other", E.GA_VALUE_ERROR,
         lambda: ga.embedding(table, ids, out=gpuarray.from_strided(wide, 0, (4, 8), (16, 4)))),
        ("read-only out", E.GA_VALUE_ERROR,
         lambda: ga.embedding(table, ids, out=gpuarray.from_strided(wide, 0, (4, 8), (64, 4), writeable=False))),
        ("infinite scale", E.GA_VALUE_ERROR, lambda: ga.embedding(table, ids, scale=float("inf"), out=out)),
        ("scale that no float holds", E.GA_VALUE_ERROR, lambda: ga.embedding(table, ids, scale=1e39, out=out)),
        ("grad within dout", E.GA_VALUE_ERROR, lambda: ga.embedding_grad(wide[:4, :8], ids, wide[:, :8])),
        ("dout of another length", E.GA_INVALID_ERROR, lambda: ga.embedding_grad(z((5, 8)), ids, table)),
        ("grad of one dim", E.GA_INVALID_ERROR, lambda: ga.embedding_grad(out, ids, t1)),
        ("logp without ids", E.GA_VALUE_ERROR, lambda: ga.token_logprobs(x, out=T(t1, None, None, None, None))),
        ("ids without logp", E.GA_VALUE_ERROR, lambda: ga.token_logprobs(x, ids, out=T(None, t1, None, None, None))),
        ("one half of the alternatives", E.GA_VALUE_ERROR, lambda: ga.token_logprobs(x, out=T(None, None, None, t2, None))),
        ("alternatives of two shapes", E.GA_INVALID_ERROR,
         lambda: ga.token_logprobs(x, out=T(None, None, None, t2, z((4, 3), "int64")))),
        ("short ids of alternatives", E.GA_VALUE_ERROR,
         lambda: ga.token_logprobs(x, out=T(None, None, None, t2, z((4, 2), "int16")))),
        ("more alternatives than tokens", E.GA_VALUE_ERROR, lambda: ga.token_logprobs(x, top=17)),
        ("more alternatives than the limit", E.GA_VALUE_ERROR, lambda: ga.token_logprobs(z((2, 100)), top=65)),
        ("logits of one dim", E.GA_INVALID_ERROR, lambda: ga.token_logprobs(t1, out=T(None, t1, None, None, None))),
        ("transposed logits", E.GA_INVALID_ERROR, lambda: ga.token_logprobs(other, out=T(None, z((8,)), None, None, None))),
        ("scale of 0", E.GA_VALUE_ERROR, lambda: ga.token_logprobs(x, ids, scale=0.0)),
        ("negative scale", E.GA_VALUE_ERROR, lambda: ga.token_logprobs(x, ids, scale=-1.0)),
        ("scale that is 0 in 32 bits", E.GA_VALUE_ERROR, lambda: ga.token_logprobs(x, ids, scale=1e-60)),
        ("NaN scale", E.GA_VALUE_ERROR, lambda: ga.token_logprobs(x, ids, scale=float("nan"))),
        ("no vocabulary", E.GA_VALUE_ERROR, lambda: ga.token_logprobs(z((4, 0)), out=T(None, t1, None, None, None))),
        ("two results in one place", E.GA_VALUE_ERROR, lambda: ga.token_logprobs(x, ids, out=T(t1, t1, None, None, None))),
        ("a result within the logits", E.GA_VALUE_ERROR, lambda: ga.token_logprobs(x, ids, out=T(x[0, :4], None, None, None, None))),
        ("half results", E.GA_VALUE_ERROR, lambda: ga.token_logprobs(x, ids, out=T(z((4,), "float16"), None, None, None, None))),
        ("unaligned results", E.GA_UNALIGNED_ERROR, lambda: ga.token_logprobs(x, ids, out=T(odd, None, None, None, None))),
        ("gradient of another type", E.GA_VALUE_ERROR, lambda: ga.token_logprobs_grad(x, ids, t2, t1, out=z((4, 16), "float16"))),
        ("gradient shifted within the logits", E.GA_VALUE_ERROR,
         lambda: ga.token_logprobs_grad(wide[:4], ids, t2, t1, out=wide[1:5])),
        ("gradient in the logits' place with other strides", E.GA_VALUE_ERROR,
         lambda: ga.token_logprobs_grad(wide[:4], ids, t2, t1, out=gpuarray.from_strided(wide, 0, (4, 16), (128, 4)))),
        ("entropy without its gradient", E.GA_VALUE_ERROR, lambda: ga.token_logprobs_grad(x, ids, t2, t1, entropy=t1)),
        ("dlogp without ids", E.GA_VALUE_ERROR, lambda: ga.token_logprobs_grad(x, None, t2, t1)),
        ("statistics of another shape", E.GA_INVALID_ERROR, lambda: ga.token_logprobs_grad(x, ids, z((4, 3)), t1)),
        ("norm of integers", E.GA_UNSUPPORTED_ERROR, lambda: ga.global_norm([ids])),
        ("norm of an array with gaps", E.GA_INVALID_ERROR, lambda: ga.global_norm([wide[:, :3]])),
        ("norm into two elements", E.GA_INVALID_ERROR, lambda: ga.global_norm([x], norm=z((2,)))),
        ("norm into an operand", E.GA_VALUE_ERROR, lambda: ga.global_norm([t1], norm=t1[:1])),
        ("negative bound", E.GA_VALUE_ERROR, lambda: ga.clip_by_global_norm([x], -1.0)),
        ("NaN bound", E.GA_VALUE_ERROR, lambda: ga.clip_by_global_norm([x], float("nan"))),
        ("the same array clipped twice", E.GA_VALUE_ERROR, lambda: ga.clip_by_global_norm([x, t1, x], 1.0)),
        ("results on each other", E.GA_VALUE_ERROR, lambda: ga.clip_by_global_norm([x, z((4, 16))], 1.0, out=[wide[:4], wide[3:7]])),
        ("a result on another operand", E.GA_VALUE_ERROR, lambda: ga.clip_by_global_norm([wide[:4], x], 1.0, out=[z((4, 16)), wide[:4]])),
        ("a result shifted on its operand", E.GA_VALUE_ERROR, lambda: ga.clip_by_global_norm([wide[:4]], 1.0, out=[wide[1:5]])),
        ("a result of another type", E.GA_INVALID_ERROR, lambda: ga.clip_by_global_norm([x], 1.0, out=[z((4, 16), "float16")])),
        ("a result of another shape", E.GA_INVALID_ERROR, lambda: ga.clip_by_global_norm([x], 1.0, out=[z((16, 4))])),
        ("a result of another order", E.GA_INVALID_ERROR, lambda: ga.clip_by_global_norm([x], 1.0, out=[z((16, 4)).T])),
    ]


def test_refusals(ctx):
    for what, code, call in refusals(ctx):
        before = ctx.last_launch_hash()
        with pytest.raises(_lib.GpuArrayException) as e:
            call()
        assert e.value.code == code, (what, e.value.code, str(e.value))
        # zeros() fills with a kernel of its own only beyond a size that is not reached here
        assert ctx.last_launch_hash() == before, what


def test_refusals_of_more_lanes_than_a_launch_has(ctx):
    """2^26 rows of one column each have a wavefront."""
    t = 1 << 26
    logits = gpuarray.from_strided(gpuarray.zeros((1,), "float16", context=ctx), 0, (t, 1), (0, 2))
    stats = gpuarray.from_strided(gpuarray.zeros((2,), context=ctx), 0, (t, 2), (0, 4))
    ids = gpuarray.from_strided(gpuarray.zeros((1,), "int32", context=ctx), 0, (t,), (0,))
    dlogp = gpuarray.from_strided(gpuarray.zeros((1,), context=ctx), 0, (t,), (0,))
    logp, dlogits = gpuarray.empty((t,), context=ctx), gpuarray.empty((t, 1), "float16", context=ctx)
    before = ctx.last_launch_hash()
    for call in (lambda: ga.token_logprobs(logits, ids, out=ga.TokenLogprobs(logp, None, None, None, None)),
                 lambda: ga.token_logprobs_grad(logits, ids, stats, dlogp, out=dlogits)):
        with pytest.raises(_lib.GpuArrayException) as e:
            call()
        assert e.value.code == _lib.GA_XLARGE_ERROR
        assert ctx.last_launch_hash() == before


def test_refusal_of_arrays_of_two_contexts(ctx):
    second = ga.init("hip0")
    table, ids = gpuarray.zeros((9, 8), context=ctx), gpuarray.zeros((4,), "int64", context=second)
    for call in (lambda: ga.embedding(table, ids, out=gpuarray.zeros((4, 8), context=ctx)),
                 lambda: ga.embedding_grad(gpuarray.zeros((4, 8), context=second), ids, table),
                 lambda: ga.token_logprobs(table[:4], ids, out=ga.TokenLogprobs(gpuarray.zeros((4,), context=ctx), None, None, None, None)),
                 lambda: ga.clip_by_global_norm([table, gpuarray.zeros((3,), context=second)], 1.0)):
        with pytest.raises(_lib.GpuArrayException) as e:
            call()
        assert e.value.code == _lib.GA_INVALID_ERROR
    fixed = gpuarray.from_strided(table, 0, (9, 8), (32, 4), writeable=False)
    with pytest.raises(_lib.GpuArrayException):
        ga.GlobalNorm([fixed]).clip(1.0)
    for call in (lambda: ga.GlobalNorm([table]).clip(-1.0), lambda: ga.GlobalNorm([table]).clip(float("nan")),
                 lambda: ga.GlobalNorm([table]).norm(table[0, :1]), lambda: ga.GlobalNorm([table, table]),
                 lambda: ga.GlobalNorm([ids], context=second), lambda: ga.GlobalNorm([table[:, :3]])):
        with pytest.raises(_lib.GpuArrayException):
            call()
    with pytest.raises(ValueError):
        ga.GlobalNorm([table], out=[])
    with pytest.raises(TypeError):
        ga.GlobalNorm([np.zeros(3)])
