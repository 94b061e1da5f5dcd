"""Refusals and workspace sizes of the C entry points of attention, its heads' norms
and the balance loss (host only: every call returns before a launch), and of CPU
tensors."""
import ctypes
import math
import os

import pytest
import torch

from spira_amd.nn import functional as F

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LIB = ctypes.CDLL(os.path.join(ROOT, "spira_amd", "libspira_hip.so"))
LIB.spira_hip_last_error.restype = ctypes.c_char_p
I64, P, I, F32, F64, SIZE = (ctypes.c_int64, ctypes.c_void_p, ctypes.c_int, ctypes.c_float, ctypes.c_double,
                             ctypes.c_size_t)
SOME = 256  # (an address that no refused call reads)
FP16, FP32, BF16 = 0, 1, 2


class Attention(ctypes.Structure):
    _fields_ = ([("rows", I64), ("keys", I64)] +
                [(n, I) for n in ("sequences", "heads", "kv_heads", "head_dim", "dtype", "causal")] + [("scale", F32)] +
                [(n, P) for n in ("offsets", "key_offsets", "key_counts", "queries", "key", "value")] +
                [(n, I64) for n in ("query_row", "query_head", "key_row", "key_head", "value_row", "value_head")])


class Heads(ctypes.Structure):
    _fields_ = ([("rows", I64)] + [(n, I) for n in ("heads", "kv_heads", "head_dim", "dtype", "axes", "interleaved")] +
                [("eps", F32), ("base", F64)] + [(n, P) for n in ("queries", "key", "query_weight", "key_weight")] +
                [(n, I64) for n in ("query_row", "query_head", "key_row", "key_head")] + [("positions", P)])


def refused(code, text):
    assert code != 0 and text in LIB.spira_hip_last_error().decode(), LIB.spira_hip_last_error()


def attention(**kw):
    x = dict(rows=100, keys=100, sequences=2, heads=4, kv_heads=2, head_dim=64, dtype=FP16, causal=1, scale=0.1,
             offsets=SOME, key_offsets=SOME, queries=SOME, key=SOME, value=SOME, query_row=256, query_head=64, key_row=128,
             key_head=64, value_row=128, value_head=64)
    x.update(kw)
    return Attention(**x)


BAD = [(dict(rows=-1), "rows"), (dict(rows=1 << 31), "rows"), (dict(keys=(1 << 31) - 255), "rows"), (dict(sequences=0), "sequences"), (dict(sequences=65537), "sequences"),
       (dict(heads=0), "multiple"), (dict(heads=5), "multiple"), (dict(kv_heads=0), "multiple"), (dict(head_dim=0), "128"),
       (dict(head_dim=129), "128"), (dict(rows=(1 << 31) - 1000, heads=4, kv_heads=1), "queries"), (dict(scale=0), "scale"),
       (dict(scale=math.nan), "scale"), (dict(scale=math.inf), "scale"), (dict(offsets=None), "offsets"),
       (dict(key_offsets=None), "offsets"), (dict(queries=None), "null"), (dict(key=None), "null"), (dict(value=None), "null")]


@pytest.mark.parametrize("bad,text", BAD)
def test_attention(bad, text):
    x, size = attention(**bad), SIZE()
    refused(LIB.spira_hip_attention(ctypes.byref(x), P(SOME), None, None, None, SIZE(0), None), text)
    refused(LIB.spira_hip_attention_workspace(ctypes.byref(x), 0, ctypes.byref(size)), text)
    refused(LIB.spira_hip_attention_backward(ctypes.byref(x), P(SOME), P(SOME), None, P(SOME), P(SOME), P(SOME), P(SOME), P(SOME),
                                             SIZE(1 << 40), None), text)


def test_attention_outputs_and_workspaces():
    x, size = attention(), SIZE()
    refused(LIB.spira_hip_attention(None, P(SOME), None, None, None, SIZE(0), None), "null")
    refused(LIB.spira_hip_attention(ctypes.byref(x), None, None, None, None, SIZE(0), None), "null")
    refused(LIB.spira_hip_attention(ctypes.byref(attention(dtype=7)), P(SOME), None, None, None, SIZE(0), None), "dtype")
    refused(LIB.spira_hip_attention_backward(ctypes.byref(x), P(SOME), None, None, P(SOME), P(SOME), P(SOME), P(SOME), P(SOME),
                                             SIZE(1 << 40), None), "null")
    assert LIB.spira_hip_attention_workspace(ctypes.byref(x), 1, ctypes.byref(size)) == 0 and size.value >= 100 * 4 * 4
    refused(LIB.spira_hip_attention_backward(ctypes.byref(x), P(SOME), P(SOME), None, P(SOME), P(SOME), P(SOME), P(SOME), P(SOME),
                                             SIZE(size.value - 1), None), "workspace")
    # few tokens against a long cache: the parts' sums
    x = attention(rows=2, keys=100_000)
    assert LIB.spira_hip_attention_workspace(ctypes.byref(x), 0, ctypes.byref(size)) == 0 and size.value > 0
    assert size.value % (2 * 4 * 66 * 4) == 0
    refused(LIB.spira_hip_attention(ctypes.byref(x), P(SOME), None, None, P(SOME), SIZE(size.value - 1), None), "workspace")
    refused(LIB.spira_hip_attention(ctypes.byref(x), P(SOME), None, None, None, SIZE(1 << 40), None), "workspace")
    # whatever the sizes, they stay within some hundred MB
    for rows, keys, heads, kv in ((1, (1 << 31) - 256, 64, 1), (4000, 1 << 30, 64, 64), (64, 1 << 20, 128, 2), (1, 0, 1, 1)):
        x = attention(rows=rows, keys=keys, heads=heads, kv_heads=kv, sequences=max(1, rows // 2), head_dim=128)
        assert LIB.spira_hip_attention_workspace(ctypes.byref(x), 0, ctypes.byref(size)) == 0 and size.value < 1 << 29
    assert LIB.spira_hip_attention(ctypes.byref(attention(rows=0, queries=None)), None, None, None, None, SIZE(0), None) == 0


def test_norm_rotate_heads():
    def heads(**kw):
        x = dict(rows=10, heads=4, kv_heads=2, head_dim=64, dtype=FP16, axes=1, interleaved=0, eps=1e-6, base=100.0,
                 queries=SOME, key=SOME, query_weight=SOME, key_weight=SOME, query_row=256, query_head=64, key_row=128,
                 key_head=64, positions=SOME)
        x.update(kw)
        return Heads(**x)
    size = SIZE()
    for bad, text in ((dict(rows=-1), "rows"), (dict(heads=0), "heads"), (dict(kv_heads=70_000), "heads"),
                      (dict(head_dim=0), "128"), (dict(head_dim=130), "128"), (dict(head_dim=33), "even"),
                      (dict(axes=33), "axis"), (dict(axes=-1), "axes"), (dict(base=0.0), "base"), (dict(base=math.nan), "base"),
                      (dict(positions=None), "positions"), (dict(queries=None), "null")):
        x = heads(**bad)
        refused(LIB.spira_hip_norm_rotate_heads(ctypes.byref(x), P(SOME), P(SOME), None), text)
        refused(LIB.spira_hip_norm_rotate_heads_backward_workspace(ctypes.byref(x), ctypes.byref(size)), text)
        refused(LIB.spira_hip_norm_rotate_heads_backward(ctypes.byref(x), P(SOME), P(SOME), P(SOME), P(SOME), None, None,
                                                         None, SIZE(0), None), text)
    x = heads()
    refused(LIB.spira_hip_norm_rotate_heads(ctypes.byref(x), P(SOME), None, None), "null")
    refused(LIB.spira_hip_norm_rotate_heads(ctypes.byref(heads(dtype=9)), P(SOME), P(SOME), None), "dtype")
    assert LIB.spira_hip_norm_rotate_heads_backward_workspace(ctypes.byref(x), ctypes.byref(size)) == 0 and size.value > 0
    refused(LIB.spira_hip_norm_rotate_heads_backward(ctypes.byref(x), P(SOME), P(SOME), P(SOME), P(SOME), P(SOME), None,
                                                     P(SOME), SIZE(size.value - 1), None), "workspace")
    refused(LIB.spira_hip_norm_rotate_heads_backward(ctypes.byref(x), None, P(SOME), P(SOME), None, None, None, None, SIZE(0),
                                                     None), "null")
    refused(LIB.spira_hip_norm_rotate_heads_backward(ctypes.byref(heads(key_weight=None)), P(SOME), P(SOME), None, None, None,
                                                     P(SOME), None, SIZE(0), None), "no weight")


def test_balance():
    size = SIZE()
    for tokens, experts, text in ((-1, 4, "tokens"), (1 << 31, 4, "tokens"), (4, 0, "experts"), (4, 513, "experts")):
        refused(LIB.spira_hip_balance_workspace(I64(tokens), experts, ctypes.byref(size)), text)
        refused(LIB.spira_hip_balance(P(SOME), I64(tokens), experts, FP16, P(SOME), P(SOME), P(SOME), P(SOME), P(SOME),
                                      P(SOME), SIZE(1 << 30), None), text)
        refused(LIB.spira_hip_balance_backward(P(SOME), I64(tokens), experts, FP16, P(SOME), P(SOME), P(SOME), None), text)
    assert LIB.spira_hip_balance_workspace(I64(100), 8, ctypes.byref(size)) == 0 and size.value == 0
    assert LIB.spira_hip_balance_workspace(I64(100_000), 16, ctypes.byref(size)) == 0 and size.value > 0
    refused(LIB.spira_hip_balance(P(SOME), I64(100_000), 16, FP16, P(SOME), P(SOME), P(SOME), P(SOME), P(SOME), P(SOME),
                                  SIZE(size.value - 1), None), "workspace")
    refused(LIB.spira_hip_balance(P(SOME), I64(10), 16, FP16, None, P(SOME), P(SOME), P(SOME), P(SOME), P(SOME), SIZE(0),
                                  None), "null")
    refused(LIB.spira_hip_balance(P(SOME), I64(10), 16, 5, P(SOME), P(SOME), P(SOME), P(SOME), P(SOME), P(SOME), SIZE(0),
                                  None), "dtype")


def test_cpu_tensors():
    x, off = torch.zeros(4, 2, 8), torch.zeros(2, dtype=torch.int32)
    for f in (lambda: F.attention(x, x, x, off), lambda: F.norm_rotate_heads(x, x), lambda: F.balance_loss(x[0], off)):
        with pytest.raises(NotImplementedError):
            f()
