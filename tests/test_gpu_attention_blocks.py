"""Attention's kernels whose blocks own 128 columns, in every width of head, type and way
of fetching tiles, against the reference of test_gpu_attention.py: sequences of several
blocks and tiles, with edges inside them."""
import pytest
import torch

from test_gpu_attention import DTYPES, check, randn

pytestmark = pytest.mark.gpu

# some blocks of columns and tiles of keys each, one that fills neither, none at all
LENGTHS = [700, 130, 0, 65, 705]


def blocks(rows, heads, kv, sequences):
    """Of 128 columns; from 192 on (512 in fp32) the kernels take them."""
    return (rows * (heads // kv) // 128 + sequences) * kv


def least(dtype):
    return 512 if dtype == torch.float32 else 192


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("d", [20, 32, 63, 64, 96, 101, 128])
def test_sequences_of_several_blocks(dev, d, causal, dtype):
    dt, n, group = DTYPES[dtype], sum(LENGTHS), 3
    kv = 13 if dt == torch.float32 else 5
    assert blocks(n, group * kv, kv, len(LENGTHS)) >= least(dt)
    check(dev, randn((n, group * kv, d), dt, 1), randn((n, kv, d), dt, 2), randn((n, kv, d), dt, 3), LENGTHS, causal=causal)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [32, 64, 128])
def test_views_that_start_anywhere(dev, d, dtype):
    """One projection's views at an odd start, fetched through registers."""
    dt, n, kv = DTYPES[dtype], sum(LENGTHS), 13 if dtype == "f32" else 5
    assert blocks(n, 3 * kv, kv, len(LENGTHS)) >= least(dt)
    x = randn((n * 5 * kv * d + 3,), dt, 1).to(dev)[3:].view(n, 5 * kv, d)
    check(dev, x[:, :3 * kv], x[:, 3 * kv:4 * kv], x[:, 4 * kv:], LENGTHS, causal=True)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("causal", [False, True])
def test_keys_of_their_own_in_several_blocks(dev, causal, dtype):
    """Caches longer and shorter than the queries, with room behind their keys, and more sequences than a
    wave looks at at once."""
    dt, kv = DTYPES[dtype], 16 if dtype == "f32" else 6
    queries, room = [300, 5, 0, 200, 650], [400, 90, 70, 100, 900]
    counts = [390, 1, 70, 0, 777]
    n, m = sum(queries), sum(room)
    assert blocks(n, 3 * kv, kv, len(queries)) >= least(dt)
    check(dev, randn((n, 3 * kv, 64), dt, 1), randn((m, kv, 64), dt, 2), randn((m, kv, 64), dt, 3), queries,
          k_lengths=room, counts=counts, causal=causal)
    many = [(i * 53) % 150 for i in range(70)]
    n = sum(many)
    assert blocks(n, 2 * 6, 6, 70) >= least(dt)
    check(dev, randn((n, 12, 32), dt, 1), randn((n, 6, 32), dt, 2), randn((n, 6, 32), dt, 3), many, causal=causal)
