"""bfloat16 arrays under expressions and Python's operators: what is computed is the same on floats, rounded once to
nearest even.  The reference has no such type; the rules are those of its half arrays."""
import operator

import numpy as np
import pytest

import libgpuarray_amd as ga
from libgpuarray_amd import GpuElemwise, arg, gpuarray, ndgpuarray

pytestmark = pytest.mark.gpu

X = np.array([-1.5, -0.25, 0.0, 2.75, -7.0, 3.0, 1e30, -1e-30, 0.4375, -2.5], np.float32)
Y = np.array([0.5, 0.75, -1.25, -0.5, 2.0, 3.0, 7.0, 1e-20, 0.125, 1.5], np.float32)


def bf(x):
    """float32 numbers rounded to bfloat16."""
    return ga.from_bfloat16(ga.to_bfloat16(np.asarray(x, np.float32)))


def numbers(a):
    return ga.from_bfloat16(np.asarray(a)) if a.dtype == ga.bfloat16 else np.asarray(a)


def on_gpu(ctx, x, cls=None):
    return gpuarray.array(ga.to_bfloat16(x), context=ctx, cls=cls)


def same(got, want):
    assert got.dtype == ga.bfloat16
    assert np.array_equal(numbers(got), bf(want), equal_nan=True), (numbers(got), bf(want))


EXPRESSIONS = [
    ("r = a > 0 ? a : 0", lambda a, b, s, r: np.where(a > 0, a, 0)),
    ("r = a > 0 ? a : 0.0f", lambda a, b, s, r: np.where(a > 0, a, 0)),
    ("r = a < b ? a : b", lambda a, b, s, r: np.minimum(a, b)),
    ("r += a", lambda a, b, s, r: r + a),
    ("r *= 2", lambda a, b, s, r: r * 2),
    ("r++", lambda a, b, s, r: r + 1),
    ("r -= a * b", lambda a, b, s, r: r - a * b),
    ("r = s > 1 ? s * a : s", lambda a, b, s, r: s * a),
    ("r = fmaf(a, b, s)", lambda a, b, s, r: (a.astype(np.float64) * b + s).astype(np.float32)),
    # several statements and one rounding: 1 + 2^-9 is no bfloat16
    ("r = a; r = r * 0.001953125f; r = r + 1; r = r - 1", lambda a, b, s, r: (a * np.float32(2 ** -9) + np.float32(1)) - np.float32(1)),
    ("ga_float t = a; t += b; r = t > 0 ? t : -t", lambda a, b, s, r: np.abs(a + b)),
]


@pytest.mark.parametrize("convert", [False, True])
@pytest.mark.parametrize("text,of", EXPRESSIONS, ids=[e[0] for e in EXPRESSIONS])
def test_expressions(ctx, text, of, convert):
    """An operand is a float in an expression, with and without GE_CONVERT_F16: the type has no arithmetic of its own."""
    a, b, r = bf(X), bf(Y), bf(Y[::-1])
    k = GpuElemwise(ctx, text, [arg("r", ga.bfloat16, read=True, write=True), arg("a", ga.bfloat16, read=True),
                                arg("b", ga.bfloat16, read=True), arg("s", ga.bfloat16, scalar=True)], convert_f16=convert)
    out, da, db = on_gpu(ctx, r), on_gpu(ctx, a), on_gpu(ctx, b)
    k(out, da, db, 1.25)
    with np.errstate(over="ignore"):
        want = of(a, b, np.float32(1.25), r)
    same(out, want)
    # strided, transposed and broadcast operands go through kernels of their own
    grid = np.resize(np.concatenate([a, b]), (6, 40)).astype(np.float32)
    for view in (lambda x: x[::2, 1::3], lambda x: x.T, lambda x: x):
        da, root = on_gpu(ctx, grid), on_gpu(ctx, grid[:, ::-1])
        db = on_gpu(ctx, grid[:1])
        rows = np.broadcast_to(grid[:1], grid.shape)
        k(view(root), view(da), view(db), 1.25)
        with np.errstate(over="ignore"):
            want = of(view(grid), view(rows), np.float32(1.25), view(grid[:, ::-1]))
        same(view(root), want)


def test_mixed_expressions(ctx):
    """Beside floats, doubles, halves and integers; the scalar takes its value from a Python number."""
    a = bf(X[:5])
    k = GpuElemwise(ctx, "f = a * s; d = a / 3.0; h = a > 0 ? a : h; q = a", [
        arg("f", "float32", write=True), arg("d", "float64", write=True), arg("h", "float16", read=True, write=True),
        arg("q", "int32", write=True), arg("a", ga.bfloat16, read=True), arg("s", ga.bfloat16, scalar=True)], convert_f16=True)
    f, d, i = (gpuarray.empty((5,), t, context=ctx) for t in ("float32", "float64", "int32"))
    h = gpuarray.array(np.full(5, 9, np.float16), context=ctx)
    k(f, d, h, i, on_gpu(ctx, a), 0.1)
    assert np.array_equal(np.asarray(f), a * bf(0.1))
    assert np.array_equal(np.asarray(d), a.astype(np.float64) / 3)
    assert np.array_equal(np.asarray(h), np.where(a > 0, a, 9).astype(np.float16))
    assert np.array_equal(np.asarray(i), a.astype(np.int32))


def test_copies_keep_every_bit(ctx):
    """Signalling NaNs and subnormals too, between any two layouts."""
    host = np.arange(1 << 16, dtype=np.uint16).reshape(256, 256).view(ga.bfloat16)
    a = gpuarray.array(host, context=ctx)
    bits = lambda x: np.ascontiguousarray(np.asarray(x)).view(np.uint16)  # noqa: E731
    want = host.view(np.uint16)
    assert np.array_equal(bits(a.T.copy()), want.T) and np.array_equal(bits(a[::-1, 3:].copy()), want[::-1, 3:])
    assert np.array_equal(bits(a[::2, ::3].copy("F")), want[::2, ::3])
    b = gpuarray.zeros((256, 256), ga.bfloat16, context=ctx)
    b[:, ::-1] = a
    assert np.array_equal(bits(b), want[:, ::-1])
    assert np.array_equal(np.asarray(a.T.astype("float32")), ga.from_bfloat16(host.T), equal_nan=True)


# ---- ndgpuarray -------------------------------------------------------------------------------------

def test_abs(ctx):
    x = np.concatenate([X, [-0.0, np.inf, -np.inf, np.nan]]).astype(np.float32)
    got = abs(on_gpu(ctx, x, ndgpuarray))
    assert type(got) is ndgpuarray
    same(got, np.abs(x))
    same(-on_gpu(ctx, x, ndgpuarray), -x)


FORMS = {"floordiv": lambda a, b: np.floor((a / b).astype(np.float32)), "mod": np.fmod}


@pytest.mark.parametrize("name", ["floordiv", "mod"])
def test_floor_division_and_remainder(ctx, name):
    """floor(a / b) and fmod(a, b) on floats, as for halves: of two arrays, in place and together."""
    a, b = bf(X), bf(Y)
    with np.errstate(all="ignore"):
        want = FORMS[name](a, b)
    x, y = on_gpu(ctx, a, ndgpuarray), on_gpu(ctx, b, ndgpuarray)
    same(getattr(operator, name)(x, y), want)
    same(divmod(x, y)[name == "mod"], want)
    again = getattr(operator, "i" + name)(x, y)
    assert again is x
    same(x, want)


@pytest.mark.parametrize("name", ["floordiv", "mod"])
@pytest.mark.parametrize("other", [2.5, -3, np.float32(0.75)])
def test_floor_division_and_remainder_by_a_number_in_place(ctx, name, other):
    a = bf(X[:6])
    x = on_gpu(ctx, a, ndgpuarray)
    getattr(operator, "i" + name)(x, other)
    same(x, FORMS[name](a, np.float32(other)))


def test_floor_division_of_floats_by_bfloat16_in_place(ctx):
    x = gpuarray.array(X[:6], context=ctx, cls=ndgpuarray)
    y = on_gpu(ctx, bf(Y[:6]), ndgpuarray)
    x //= y
    assert np.array_equal(np.asarray(x), np.floor(X[:6] / bf(Y[:6])))
    x = gpuarray.array(X[:6], context=ctx, cls=ndgpuarray)
    x %= y
    assert np.array_equal(np.asarray(x), np.fmod(X[:6], bf(Y[:6])))


def test_helpers_compute_on_floats(ctx):
    """elemwise2 with the result's type given: operands of more bits keep them."""
    from libgpuarray_amd.elemwise import elemwise2
    a = (X * np.float32(1 + 2.0 ** -9))
    x, y = gpuarray.array(a, context=ctx), on_gpu(ctx, Y)
    same(elemwise2(x, "-", y, x, odtype=ga.bfloat16), a - bf(Y))


def test_division(ctx):
    """bfloat16 is the type of what two of them give, as for + - *."""
    a, b = bf(X), bf(Y)
    x, y = on_gpu(ctx, a, ndgpuarray), on_gpu(ctx, b, ndgpuarray)
    same(x / y, a / b)
    x /= y
    same(x, a / b)
    x *= 0.5                                              # in place a number needs no common type
    same(x, bf(a / b) * np.float32(0.5))
    for what in (lambda: x / 2.0, lambda: 2.0 / x, lambda: x / gpuarray.zeros((10,), context=ctx, cls=ndgpuarray)):
        with pytest.raises(TypeError):
            what()


def test_concatenation(ctx):
    from libgpuarray_amd import operations
    a, b = on_gpu(ctx, X), on_gpu(ctx, Y)
    same(operations.concatenate([a, b, a[:3]]), np.concatenate([X, Y, X[:3]]))
    same(operations.vstack([a, b]), np.stack([X, Y]))


def test_records_of_two_bytes_have_kernels_of_their_own(ctx):
    """NumPy names every record of two bytes alike; what is kept for one type must not serve another."""
    from libgpuarray_amd.elemwise import elemwise1
    pair = np.dtype([("low", "u1"), ("high", "u1")])
    gpuarray.register_dtype(pair, "pair_of_bytes")
    host = np.array([(1, 2), (250, 255), (7, 0)], pair)
    mark = "res = a; "                                  # of this test alone: no kernel is kept for it yet
    same(elemwise1(on_gpu(ctx, X), None, oper=mark), X)
    a = gpuarray.array(host, context=ctx)
    with pytest.raises(ga.GpuArrayException):           # the kernel texts know no type of that name
        elemwise1(a, None, oper=mark)
    text = ("typedef struct { ga_ubyte low, high; } pair_of_bytes;\n")
    out = gpuarray.empty((3,), pair, context=ctx)
    GpuElemwise(ctx, "r.low = a.high; r.high = a.low", [arg("r", pair, write=True), arg("a", pair, read=True)],
                preamble=text)(out, a)
    assert np.array_equal(np.asarray(out)["low"], host["high"]) and np.array_equal(np.asarray(out)["high"], host["low"])
