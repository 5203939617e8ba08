"""The gradient of embedding rows where its tokens are sorted: every way the sort is launched, and layouts, ids out of
range and rows between the rows for more tokens than one launch takes."""
import numpy as np
import pytest

import libgpuarray_amd as ga
from libgpuarray_amd import gpuarray
from test_gpu_language import U, check_embedding_grad, on_gpu, vec

pytestmark = pytest.mark.gpu


def check_touched(got, x, ids, base):
    """Like check_embedding_grad, over the rows that have tokens alone; the others are `base`, or zeros."""
    rows, at = np.unique(ids, return_inverse=True)
    want, mag, count = np.zeros((rows.size, x.shape[1])), np.zeros((rows.size, x.shape[1])), np.bincount(at)[:, None]
    order = np.argsort(at, kind="stable")
    first = np.concatenate([[0], np.cumsum(count)[:-1]])
    want[:] = np.add.reduceat(x[order].astype(np.float64), first, axis=0)
    mag[:] = np.add.reduceat(np.abs(x[order]).astype(np.float64), first, axis=0)
    bound = (count + 1) * U * mag
    if base is not None:
        want += base[rows]
        bound += U * np.abs(want)
    off = np.abs(got[rows] - want)
    limit = bound * (1 + 2.0 ** -7) + np.abs(want) * U + 2.0 ** -150
    assert np.all(off <= limit), np.argwhere(off > limit)[:5]
    untouched = np.ones(got.shape[0], bool)
    untouched[rows] = False
    if base is None:
        assert not got[untouched].any()
    else:
        assert np.array_equal(got[untouched], base[untouched])


@pytest.mark.parametrize("n,v,d", [(5000, 280000, 64), (8193, 500000, 64), (16000, 1000000, 64), (16384, 60000, 1024)])
def test_one_group_sorts_while_many_rows_are_cleared(ctx, n, v, d):
    """8 and 16 tokens a lane, where clearing takes longer than the sort."""
    rng = np.random.default_rng(n)
    x = rng.standard_normal((n, d)).astype(np.float32)
    ids = rng.integers(0, v, n)
    ids[rng.random(n) < 0.2] = v - 1
    ids[: n // 50] = 0
    g = gpuarray.empty((v, d), context=ctx)
    ga.embedding_grad(gpuarray.array(x, context=ctx), gpuarray.array(ids, context=ctx), g)
    check_touched(np.asarray(g), x, ids, None)


@pytest.mark.parametrize("n,v,d", [(262145, 50257, 8), (300000, 100, 17), (524288, 1, 4), (1100000, 70001, 4), (1048577, 3000000, 3),
                                   (1100000, 127, 5)])
@pytest.mark.parametrize("accumulate", [False, True])
def test_more_tokens_than_one_a_lane(ctx, n, v, d, accumulate):
    """2 and 4 tokens a lane, of few groups with counts of their own and of many with a launch that adds them up."""
    rng = np.random.default_rng(n)
    x = rng.standard_normal((n, d)).astype(np.float32)
    ids = rng.integers(0, v, n).astype(np.int32)
    ids[rng.random(n) < 0.05] = v // 2
    keep = np.ones(n, bool)
    keep[::101] = False
    sent = np.where(keep, ids, -7777777)
    sent[50::977] -= np.where(keep, v, 0)[50::977].astype(np.int32)     # counted from the end
    base = rng.standard_normal((v, d)).astype(np.float32) if accumulate else None
    g = gpuarray.array(base if accumulate else np.full((v, d), 7, np.float32), context=ctx)
    ga.embedding_grad(gpuarray.array(x, context=ctx), gpuarray.array(sent, context=ctx), g, ignore=-7777777, accumulate=accumulate)
    check_touched(np.asarray(g), x[keep], ids[keep], base)


@pytest.mark.parametrize("pitch,flip,step", [(3, False, 2), (0, True, -1), (13, True, 1), (1, False, 0)])
@pytest.mark.parametrize("accumulate", [False, True])
@pytest.mark.parametrize("n,d", [(257, 45), (700, 45), (4097, 300), (20000, 7)])
def test_layouts_of_sorted_tokens(ctx, pitch, flip, step, accumulate, n, d):
    rng = np.random.default_rng(n)
    v = 900
    x = rng.standard_normal((n, d)).astype(np.float32)
    ids = rng.integers(0, v, n)
    if step == 0:
        ids[:] = ids[0]
    base = rng.standard_normal((v, d)).astype(np.float32)
    g, root_dev, root = on_gpu(ctx, base, pitch, flip, fill=-3)
    dout, _, _ = on_gpu(ctx, x, pitch, flip, fill=1e30)
    ga.embedding_grad(dout, vec(ctx, ids, step), g, accumulate=accumulate)
    check_embedding_grad(g, x, ids, v, 1.0, -100, "float32", base if accumulate else None)
    flat = np.asarray(root_dev)[:root.nbytes].view(np.float32).reshape(root.shape)
    assert np.all(flat[:, d:] == -3)


@pytest.mark.parametrize("accumulate", [False, True])
@pytest.mark.parametrize("n", [257, 700, 20000])
@pytest.mark.parametrize("v", [1, 1023, 1024, 5000])
def test_sorted_tokens_out_of_range(ctx, accumulate, n, v):
    """They are reported, and add to no row; what stands for no token is not reported."""
    rng = np.random.default_rng(v)
    x = rng.standard_normal((n, 12)).astype(np.float32)
    ids = rng.integers(0, v, n)
    sent = ids.copy()
    out = np.zeros(n, bool)
    out[3::5] = True
    sent[out] = np.resize([v, -v - 1, 1 << 40, -(1 << 62), v + 1023], int(out.sum()))
    sent[1::7] = -100
    keep = ~out
    keep[1::7] = False
    base = rng.standard_normal((v, 12)).astype(np.float32)
    g = gpuarray.array(base, context=ctx)
    with pytest.raises(IndexError):
        ga.embedding_grad(gpuarray.array(x, context=ctx), gpuarray.array(sent, context=ctx), g, ignore=-100, accumulate=accumulate)
    check_touched(np.asarray(g), x[keep], ids[keep], base if accumulate else None)
    sent[out] = -100                                       # the error word has been reset
    ga.embedding_grad(gpuarray.array(x, context=ctx), gpuarray.array(sent, context=ctx), g, ignore=-100)
    check_touched(np.asarray(g), x[keep], ids[keep], None)
