"""8-bit append of many rows and many sequences (several rows per CTA, sequences found 32 ways at a time), and prefill
attention of many query heads per kv head."""
import random

import pytest
import torch

from test_gpu_kv8 import DEV, Appender, Cache, check_prefill, fill, tables_for, values

pytestmark = pytest.mark.gpu


def ragged(sequences, low, high, seed):
    """Row counts, empty ones among them, and starts on and off the borders of blocks."""
    r = random.Random(seed)
    counts = [r.choice([0, low, high, r.randint(low, high)]) for _ in range(sequences)]
    return counts, [r.choice([0, 1, 15, 16, 31, 200, r.randint(0, 300)]) for _ in range(sequences)]


# a CTA takes rows / 296 rows, 1 to 8: calls of 2, 3 and 8, with short last CTAs
MANY = [([592], [0]), ([300, 0, 292], [7, 3, 250]), ([900], [5]), ([700, 0, 1, 1670], [0, 9, 15, 33]), ([4003], [0]),
        ragged(33, 1, 60, 1), ragged(100, 1, 40, 2), ragged(1500, 1, 3, 3)]
SHAPES = [(9, 3, 64, 16, "f32", 64, "half", "int8"), (4, 2, 128, 32, "bf16", 64, "interleaved", "e4m3"),
          (4, 1, 64, 256, "bf16", 24, "half", "int8"), (2, 2, 128, 48, "f32", 40, "interleaved", "e4m3"),
          (5, 1, 64, 64, "f32", 0, "half", "int8"), (3, 1, 128, 16, "bf16", 128, "half", "e4m3")]


@pytest.mark.parametrize("case", range(len(MANY)))
@pytest.mark.parametrize("heads,kv_heads,dim,bt,dtype,rotary,layout,fmt", SHAPES)
def test_append_many_rows(built, case, heads, kv_heads, dim, bt, dtype, rotary, layout, fmt):
    """The whole cache, its scales and the rotated queries as the plain form's; odd cases rotate q in place."""
    counts, starts = MANY[case]
    ends = [s + c for s, c in zip(starts, counts)]
    cache = Cache(sum(-(-n // bt) for n in ends) + 3, kv_heads, dim, bt, fmt)
    tables = tables_for(ends, bt, cache.c.max_blocks, 110)
    fill(cache, tables, starts, 111)
    run = Appender(cache, heads, dtype, rotary, layout, max(ends), in_place=case % 2 == 1)
    run(tables, counts, starts, values(sum(counts), (heads + 2 * kv_heads) * dim, 112), with_q=case != 2, behind=1 + case)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,dim", [(64, 1, 64), (64, 1, 128), (24, 1, 64), (50, 2, 128), (80, 2, 64), (33, 1, 128)])
def test_prefill_many_heads_per_kv_head(built, heads, kv_heads, dim, dtype):
    """Tiles of 2 to 5 rows."""
    counts, starts = [1, 40, 0, 77, 5], [300, 0, 4, 129, 15]
    lengths = [s + c if c else 0 for s, c in zip(starts, counts)]
    cache = Cache(sum(-(-n // 16) for n in lengths), kv_heads, dim, 16, "int8")
    check_prefill(cache, heads, tables_for(lengths, 16, cache.c.max_blocks, 113), counts, starts, dtype)
