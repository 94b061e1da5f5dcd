"""Sizes that the row operators' workspace queries refuse as their calls do (host
only), and those of a token's gradient."""
import ctypes
import os

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LIB = ctypes.CDLL(os.path.join(ROOT, "spira_amd", "libspira_hip.so"))
LIB.spira_hip_last_error.restype = ctypes.c_char_p
I64, NULL, SOME = ctypes.c_int64, ctypes.c_void_p(), ctypes.c_void_p(256)
FP16, FP32 = 0, 1


def refused(code, text):
    assert code != 0 and text in LIB.spira_hip_last_error().decode(), LIB.spira_hip_last_error()


@pytest.mark.timeout(20)
@pytest.mark.parametrize("rows,groups,ci,co,text", [
    (100_000, 70_000, 8, 8, "groups"),  # (more than a launch has blocks in z: no part is long enough)
    (10, 0, 8, 8, "groups"), (-1, 2, 8, 8, "rows"), (1 << 31, 2, 8, 8, "rows"), (10, 2, 8, 0, "widths"),
    (10, 2, 8, 1 << 21, "widths")])
def test_grouped_linear_queries(rows, groups, ci, co, text):
    size = ctypes.c_size_t()
    refused(LIB.spira_hip_grouped_linear_weights_gradient_workspace(I64(rows), groups, ci, co, ctypes.byref(size)), text)
    refused(LIB.spira_hip_grouped_linear_activation_gradient_workspace(I64(rows), groups, co, FP16, ctypes.byref(size)),
            text)


def test_norm_query():
    size, query = ctypes.c_size_t(), LIB.spira_hip_gated_residual_norm_backward_workspace
    for n, c in ((-1, 8), (4, 0), (4, -8)):
        refused(query(I64(n), c, FP16, ctypes.byref(size)), "sizes")
    refused(query(I64(4), 16385, FP16, ctypes.byref(size)), "channels")
    assert query(I64(0), 8, FP16, ctypes.byref(size)) == 0 and size.value == 0


def test_tokens_gradient():
    size, query = ctypes.c_size_t(), LIB.spira_hip_grouped_linear_tokens_gradient_workspace
    for rows, k, ci, text in ((-1, 2, 8, "rows"), (10, 0, 8, "sizes"), (10, 2, 0, "widths")):
        refused(query(I64(rows), k, ci, ctypes.byref(size)), text)
    assert query(I64(1000), 2, 24, ctypes.byref(size)) == 0 and size.value == 4 * 1000 * 24

    def call(offsets=SOME, slots=SOME, tokens=5, k=2, dz=SOME, w=SOME, dx=SOME, workspace=SOME, bytes_=4 * 10 * 8, dtype=FP16):
        return LIB.spira_hip_grouped_linear_tokens_gradient(I64(10), 2, offsets, slots, I64(tokens), k, dz, 8, w, 8, dtype,
                                                            dx, workspace, ctypes.c_size_t(bytes_), NULL)
    refused(call(offsets=NULL), "offsets")
    refused(call(tokens=-1), "sizes")
    refused(call(k=0), "sizes")
    for null in ({"slots": NULL}, {"dz": NULL}, {"w": NULL}, {"dx": NULL}):
        refused(call(**null), "null")
    refused(call(workspace=NULL), "workspace")
    refused(call(bytes_=4 * 10 * 8 - 1), "workspace")
    refused(call(dtype=7), "dtype")


def test_launches_of_too_many_threads():
    """Past 2^32 threads some would not run: refused on the host."""
    def linear(rows, groups, ci, co, dtype):
        return LIB.spira_hip_grouped_linear(I64(rows), groups, SOME, NULL, I64(rows), SOME, ci, SOME, NULL, co, dtype, 0,
                                            SOME, NULL)
    refused(linear(40_000, 32767, 8, 65536, FP16), "too many tiles")   # tiles of 128 rows
    refused(linear(16_384, 32767, 8, 65536, FP32), "too many tiles")   # few rows
    refused(linear((1 << 31) - 1000, 1, 513, 1, FP16), "number of rows")
    refused(LIB.spira_hip_grouped_linear_weights_gradient(I64(40_000), 32767, SOME, NULL, I64(40_000), SOME, 8, SOME, 65_664,
                                                          FP16, SOME, NULL, ctypes.c_size_t(0), NULL), "too many tiles")
