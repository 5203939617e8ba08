"""The refusals of the language operators where there is no device, against the
stand-in runtime and the three builds of the library; and their kernel texts,
which must compile for gfx950 for every combination of types."""
import ctypes as C
import subprocess
import sys

import pytest

from test_host_logic_without_device import ROOT, build, mock_runtime  # noqa: F401  (fixtures)

HOST_ONLY = ["tests/test_gpu_language.py::test_refusals",
             "tests/test_gpu_language.py::test_refusals_of_more_lanes_than_a_launch_has",
             "tests/test_gpu_language.py::test_refusal_of_arrays_of_two_contexts"]


def test_refusals_without_a_device(build):  # noqa: F811
    variant, env = build
    r = subprocess.run([sys.executable, "-m", "pytest", "-q", "-m", "gpu", "-p", "no:cacheprovider", "--timeout", "300"]
                       + HOST_ONLY, cwd=ROOT, env=env, capture_output=True, text=True, timeout=900)
    assert r.returncode == 0, r.stdout[-4000:] + r.stderr[-2000:]


@pytest.mark.parametrize("x", [11, 23, 320])
@pytest.mark.parametrize("o", [11, 23, 320])
def test_kernel_texts_compile(x, o):
    from libgpuarray_amd import _lib
    source = _lib.extension("hip_language_source", C.c_void_p, [C.c_ulonglong])
    compile_only = _lib.extension("hip_compile_only", C.c_int, [C.c_uint, C.POINTER(C.c_char_p), C.POINTER(C.c_size_t),
                                                                C.POINTER(C.c_char_p)])
    for kind in range(7):
        if kind > 1 and o != 11:
            continue
        for ids, extra in ((5, 0), (8, 0)) if kind != 2 else ((5, 1), (8, 1 | 32 | 64), (7, 4 | 32 | 64 | 128), (7, 16 | 64)):
            text = C.string_at(source(kind | x << 8 | o << 20 | ids << 32 | extra << 44))
            log = C.c_char_p()
            assert compile_only(1, (C.c_char_p * 1)(text), None, C.byref(log)) == 0, (log.value or b"").decode()[-2000:]


def test_refusals_of_scales_without_a_device(build):  # noqa: F811
    variant, env = build
    r = subprocess.run([sys.executable, "-m", "pytest", "-q", "-m", "gpu", "-p", "no:cacheprovider", "--timeout", "300",
                        "tests/test_gpu_language_far.py::test_scales_that_are_too_large_in_powers_of_two_are_refused"],
                       cwd=ROOT, env=env, capture_output=True, text=True, timeout=900)
    assert r.returncode == 0 and "1 passed" in r.stdout, r.stdout[-4000:] + r.stderr[-2000:]


@pytest.mark.parametrize("extra", [0, 1, 2, 3])
def test_texts_of_the_norm_compile(extra):
    """Arrays with the arguments or in a table, without doubles and with."""
    from libgpuarray_amd import _lib
    source = _lib.extension("hip_language_source", C.c_void_p, [C.c_ulonglong])
    compile_only = _lib.extension("hip_compile_only", C.c_int, [C.c_uint, C.POINTER(C.c_char_p), C.POINTER(C.c_size_t),
                                                                C.POINTER(C.c_char_p)])
    text = C.string_at(source(4 | 11 << 8 | 11 << 20 | 5 << 32 | extra << 44))
    assert (b"#define LM_ENDS 1" in text) == (extra > 1)
    log = C.c_char_p()
    assert compile_only(1, (C.c_char_p * 1)(text), None, C.byref(log)) == 0, (log.value or b"").decode()[-2000:]
