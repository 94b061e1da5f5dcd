"""Refusals and workspace sizes of the row operators' C entry points (host only:
every call returns before a launch), and of CPU tensors."""
import ctypes
import math
import os

import pytest
import torch

from spira_amd.nn import functional as F

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LIB = ctypes.CDLL(os.path.join(ROOT, "spira_amd", "libspira_hip.so"))
LIB.spira_hip_last_error.restype = ctypes.c_char_p
I64, U64, F64, F32, NULL = ctypes.c_int64, ctypes.c_uint64, ctypes.c_double, ctypes.c_float, ctypes.c_void_p()
SOME = ctypes.c_void_p(256)  # (an address that no refused call reads)
FP16, FP32, BF16 = 0, 1, 2


def refused(code, text):
    assert code != 0 and text in LIB.spira_hip_last_error().decode(), LIB.spira_hip_last_error()


def linear(rows=10, groups=2, offsets=SOME, sources=NULL, num_sources=10, ci=8, co=8, dtype=FP16, x=SOME, w=SOME):
    return LIB.spira_hip_grouped_linear(I64(rows), groups, offsets, sources, I64(num_sources), x, ci, w, NULL, co,
                                        dtype, 0, SOME, NULL)


def test_grouped_linear():
    refused(linear(rows=-1), "number of rows")
    refused(linear(rows=1 << 31), "number of rows")
    refused(linear(groups=0), "groups")
    refused(linear(groups=40_000), "groups")
    refused(linear(ci=0), "widths")
    refused(linear(co=1 << 21), "widths")
    refused(linear(offsets=NULL), "offsets")
    refused(linear(w=NULL), "null")
    refused(linear(num_sources=9), "too few sources")
    refused(linear(dtype=7), "dtype")
    assert linear(rows=0, num_sources=0, x=NULL) == 0


def test_workspaces():
    size = ctypes.c_size_t()
    query = LIB.spira_hip_grouped_linear_weights_gradient_workspace
    # enough tiles of the weights for every CU: none; else a share per part and group
    assert query(I64(32768), 64, 1024, 1024, ctypes.byref(size)) == 0 and size.value == 0
    for rows, groups, ci, co in ((1, 1, 1, 1), (100_000, 8, 96, 96), (8_000_000, 3, 16, 16), (70_000, 32767, 8, 8)):
        assert query(I64(rows), groups, ci, co, ctypes.byref(size)) == 0
        assert size.value % (4 * ci * co) == 0 and size.value // (4 * ci * co) < 65536
    sums = LIB.spira_hip_grouped_linear_activation_gradient_workspace
    for rows, groups in ((0, 1), (1, 5), (100_000, 32767), (20_000_000, 32767)):
        assert sums(I64(rows), groups, 24, BF16, ctypes.byref(size)) == 0
        assert size.value % (4 * 24) == 0 and size.value // (4 * 24) < 65536
    refused(LIB.spira_hip_grouped_linear_weights_gradient(I64(1000), 2, SOME, NULL, I64(1000), SOME, 8, SOME, 8, FP16,
                                                          SOME, NULL, ctypes.c_size_t(0), NULL), "workspace")


def test_route_and_combine():
    size = ctypes.c_size_t()
    for experts, k, text in ((0, 1, "experts"), (513, 1, "experts"), (4, 5, "choices"), (64, 17, "choices"), (4, 0, "choices")):
        refused(LIB.spira_hip_route_workspace(I64(10), experts, k, ctypes.byref(size)), text)
    refused(LIB.spira_hip_route_workspace(I64(1 << 31), 4, 1, ctypes.byref(size)), "tokens")
    for tokens in (0, 1, 5000, 1 << 20):
        assert LIB.spira_hip_route_workspace(I64(tokens), 64, 8, ctypes.byref(size)) == 0 and size.value >= 65 * 4
    refused(LIB.spira_hip_route(SOME, I64(9000), 8, 2, FP16, 1, SOME, SOME, SOME, SOME, SOME, SOME, ctypes.c_size_t(8),
                                NULL), "workspace")
    refused(LIB.spira_hip_combine(SOME, I64(10), SOME, NULL, I64(5), 2, 0, FP16, SOME, NULL), "sizes")
    refused(LIB.spira_hip_combine_backward(SOME, I64(10), NULL, SOME, SOME, SOME, I64(5), 2, 8, FP16, SOME, NULL, NULL),
            "null")


def test_norm_and_dropout():
    def norm(c=8, h=SOME, w=SOME, gate=NULL, form=0, r=SOME, next_weight=NULL, following=NULL):
        return LIB.spira_hip_gated_residual_norm(SOME, h, I64(4), c, FP16, w, gate, form, 0, F32(1), next_weight, F32(0),
                                                 r, following, NULL, NULL, NULL)
    refused(norm(c=0), "channels")
    refused(norm(c=16385), "channels")
    refused(norm(form=2), "gate")
    refused(norm(gate=SOME), "gate")
    refused(norm(h=NULL), "no update")
    refused(norm(r=NULL), "fit")
    refused(norm(next_weight=SOME), "fit")
    for p in (-0.1, 1.1, math.nan):
        refused(LIB.spira_hip_dropout(SOME, NULL, I64(8), FP16, F64(p), U64(0), U64(0), SOME, NULL), "p must be")
    refused(LIB.spira_hip_dropout(NULL, NULL, I64(8), FP16, F64(0.5), U64(0), U64(0), SOME, NULL), "null")


def test_cpu_tensors():
    x, w = torch.zeros(4, 8), torch.zeros(2, 8, 8)
    off = torch.zeros(3, dtype=torch.int32)
    routes = F.ExpertRoutes(torch.zeros(4, 1), off, off, off, off)
    for f in (lambda: F.grouped_linear(x, w, off), lambda: F.route_experts(x, 2), lambda: F.combine_experts(x, routes),
              lambda: F.gated_residual_norm(x, x), lambda: F.rms_norm(x, x[0]), lambda: F.dropout(x, 0.5, 0)):
        with pytest.raises(NotImplementedError):
            f()
