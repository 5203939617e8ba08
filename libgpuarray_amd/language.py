"""Operators of language models over the C ABI (include/gpuarray/language.h).

The reference has no counterpart; they stand beside its row gather
(GpuArray_take1, src/gpuarray/array.h:348-366) and its row reductions
(GpuArray_maxandargmax, :607-644) and keep their conventions: negative ids
count from the end, an id out of range raises IndexError with `check` and
sets the context's error word without, results are new arrays unless given.

    h = embedding(table, ids, scale=32.0)
    lp = token_logprobs(logits, targets, top=5, entropy=True)
    dlogits = token_logprobs_grad(logits, targets, lp.stats, dlogp)
    embedding_grad(dh, ids, dtable, scale=32.0)
    norm = clip_by_global_norm(gradients, 1.0)
"""
import collections
import ctypes as C

from . import _lib
from ._lib import lib, check as _check
from . import gpuarray
from .gpuarray import GpuArray

NO_IGNORE = -1 << 63          # GA_NO_IGNORE: no id stands for "no token"


def _finish(err, ctx):
    """The exceptions of GpuArray.take1: IndexError for the bounds flag."""
    if err == _lib.GA_VALUE_ERROR:
        msg = lib.gpucontext_error(ctx.ctx, err)
        if msg == b"Index out of bounds":
            raise IndexError(msg.decode())
    _check(err, ctx.ctx)


def _ignore(ignore):
    """The argument of the C calls, which would take a larger number modulo 2^64."""
    if ignore is None:
        return NO_IGNORE
    if not -1 << 63 <= ignore < 1 << 63:
        raise ValueError("ignore does not fit 64 bits")
    return int(ignore)


def _dims(a, nd, what):
    if a.ndim != nd:
        raise ValueError("%s must have %d dim%s" % (what, nd, "s" if nd > 1 else ""))


def _ref(a):
    return None if a is None else a._ref


def embedding(table, ids, scale=1.0, ignore=None, out=None, dtype=None, check=True):
    """Rows of `table` (v, d) for the 1-D integer array `ids`, times `scale`:
    (n, d), of the table's type unless `dtype` or `out` says another.  The
    rows of the id `ignore` are zeros.  check=False does not wait for the
    bounds flag, as in GpuArray.take1."""
    if out is None:
        _dims(table, 2, "table")
        _dims(ids, 1, "ids")
        out = gpuarray.empty((ids.shape[0], table.shape[1]), table.dtype if dtype is None else dtype,
                             context=table.context, cls=type(table))
    err = lib.GpuArray_embedding(out._ref, table._ref, ids._ref, scale, _ignore(ignore), 1 if check else 0)
    if err:
        _finish(err, out.context)
    return out


def embedding_grad(dout, ids, grad, scale=1.0, ignore=None, accumulate=False, check=True):
    """Gradient of embedding() with respect to its table, into `grad` (v, d):
    every row is scale times the sum of the rows of `dout` that have its id,
    in a fixed order; with `accumulate` that is added to what `grad` holds."""
    err = lib.GpuArray_embedding_grad(grad._ref, dout._ref, ids._ref, scale, _ignore(ignore), 1 if accumulate else 0,
                                      1 if check else 0)
    if err:
        _finish(err, grad.context)
    return grad


#: Results of token_logprobs(); what was not asked for is None.
TokenLogprobs = collections.namedtuple("TokenLogprobs", "logp entropy stats top_logp top_ids")


def token_logprobs(logits, ids=None, scale=1.0, top=0, entropy=False, ignore=None, out=None, check=True):
    """Log probabilities under softmax(scale * logits), row by row of the 2-D
    `logits` (t, v): of the tokens `ids` (t), and the `top` likeliest
    alternatives with their ids, with the entropy if asked for.  `stats` holds what
    token_logprobs_grad() needs.  `out`, a TokenLogprobs, names the arrays to
    write; those it leaves out (None) are not computed.  All values are
    float32."""
    if out is None:
        _dims(logits, 2, "logits")
        if top < 0:
            raise ValueError("top must be 0 or above")
        t, ctx = logits.shape[0], logits.context

        def new(shape, dtype="float32"):
            return gpuarray.empty(shape, dtype, context=ctx, cls=type(logits))

        out = TokenLogprobs(new((t,)) if ids is not None else None, new((t,)) if entropy else None, new((t, 2)),
                            new((t, top)) if top else None, new((t, top), "int64") if top else None)
    logp, h, stats, top_logp, top_ids = out
    err = lib.GpuArray_token_logprobs(_ref(logp), _ref(h), _ref(stats), _ref(top_logp), _ref(top_ids), logits._ref,
                                      _ref(ids), scale, _ignore(ignore), 1 if check else 0)
    if err:
        _finish(err, logits.context)
    return out


def token_logprobs_grad(logits, ids, stats, dlogp, entropy=None, dentropy=None, scale=1.0, ignore=None, out=None,
                        check=True):
    """Gradient with respect to `logits` of sum(dlogp * logp) +
    sum(dentropy * entropy); `stats` and `entropy` come from
    token_logprobs() with the same `scale`.  ids and dlogp may both be None,
    and so may entropy and dentropy.  `out` may be `logits` itself."""
    if out is None:
        out = logits._empty_like_me()
    err = lib.GpuArray_token_logprobs_grad(out._ref, logits._ref, _ref(ids), stats._ref, _ref(dlogp), _ref(entropy),
                                           _ref(dentropy), scale, _ignore(ignore), 1 if check else 0)
    if err:
        _finish(err, out.context)
    return out


def _pointers(arrays):
    for a in arrays:
        if not isinstance(a, GpuArray):
            raise TypeError("expected GpuArrays")
    return (_lib.PA * max(len(arrays), 1))(*[C.pointer(a.ga) for a in arrays])


def _lists(arrays, out, context):
    arrays = list(arrays)
    out = None if out is None else list(out)
    if out is not None and len(out) != len(arrays):
        raise ValueError("%d arrays to clip into for %d" % (len(out), len(arrays)))
    pointers = _pointers(arrays), None if out is None else _pointers(out)
    return arrays, out, arrays[0].context if arrays else gpuarray._ensure_context(context), pointers


class GlobalNorm(object):
    """The 2-norm over all elements of a list of contiguous arrays, and
    clipping by it, for callers that clip the same gradients every step: `out`
    is the list of arrays that clipping writes (None: the arrays themselves,
    no two of which may overlap then; False: none, for norms alone, where an array
    may be listed twice).  Holds the arrays, as they are now, and
    a table of them on the device."""

    def __init__(self, arrays, out=None, context=None):
        alone = out is False
        self.arrays, self.out, self.context, (a, r) = _lists(arrays, None if alone else out, context)
        if r is None and not alone and all(x.flags.writeable for x in self.arrays):
            r = a                  # (read-only arrays have a norm, but are not clipped in place)
        self.g = C.c_void_p()
        _check(lib.GpuGlobalNorm_new(C.byref(self.g), self.context.ctx, a, r, len(self.arrays)), self.context.ctx)

    def __del__(self):
        g = getattr(self, "g", None)
        if g:
            lib.GpuGlobalNorm_free(g)
            self.g = None

    def norm(self, norm=None):
        """The norm, in a 0-d float32 array or in `norm`."""
        if norm is None:
            norm = gpuarray.empty((), "float32", context=self.context)
        err = lib.GpuGlobalNorm_norm(self.g, norm._ref)
        if err:
            _check(err, self.context.ctx)
        return norm

    def clip(self, max_norm, norm=None):
        """Scales the arrays by max_norm / norm where the norm is finite and
        above max_norm; returns the norm before that.  Does not wait."""
        if norm is None:
            norm = gpuarray.empty((), "float32", context=self.context)
        err = lib.GpuGlobalNorm_clip(self.g, max_norm, norm._ref)
        if err:
            _check(err, self.context.ctx)
        return norm


def global_norm(arrays, norm=None, context=None):
    """GlobalNorm(arrays).norm() in one call, for a list that is used once."""
    arrays, _, ctx, (a, _) = _lists(arrays, None, context)
    if norm is None:
        norm = gpuarray.empty((), "float32", context=ctx)
    _check(lib.GpuArray_global_norm(norm._ref, a, len(arrays)), ctx.ctx)
    return norm


def clip_by_global_norm(arrays, max_norm, out=None, norm=None, context=None):
    """GlobalNorm(arrays, out).clip(max_norm) in one call, for a list that is used once."""
    arrays, out, ctx, (a, r) = _lists(arrays, out, context)
    if norm is None:
        norm = gpuarray.empty((), "float32", context=ctx)
    _check(lib.GpuArray_clip_global_norm(r, a, len(arrays), max_norm, norm._ref), ctx.ctx)
    return norm
