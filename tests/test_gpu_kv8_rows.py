"""8-bit append of many rows and many sequences (several rows per CTA, sequences found 32 ways at a time), and prefill
attention of many query heads per kv head."""
import random

import pytest
import torch

import kv8_reference as ref
from test_gpu_kv8 import DEV, Appender, Cache, check_prefill, check_rows, decode, fill, stream, tables_for, values
from tinyinfer_b200 import device as mp

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


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,dim", [(256, 256, 64), (1024, 256, 128), (1024, 16, 64)])
def test_largest_head_counts(built, heads, kv_heads, dim, dtype):
    counts, starts = [3, 0, 21], [30, 0, 2]
    lengths = [s + c if c else 0 for s, c in zip(starts, counts)]
    cache = Cache(sum(-(-n // 16) for n in lengths), kv_heads, dim, 16, "e4m3")
    tables = tables_for(lengths, 16, cache.c.max_blocks, 114)
    check_prefill(cache, heads, tables, counts, starts, dtype)
    q, out = decode(cache, heads, tables, lengths, dtype)
    for i, n in enumerate(lengths):
        if n:
            check_rows(cache, heads, q[i: i + 1], out[i: i + 1], tables[i].tolist(), n, dim ** -0.5, dtype == "bf16")
    run = Appender(cache, heads, dtype, dim, "half", 64)
    run(tables, [1, 0, 2], [32, 0, 14], values(3, (heads + 2 * kv_heads) * dim, 115))


def test_largest_count(built):
    """65536 sequences of 0 to 17 tokens or rows; every operator, checked at some of them."""
    n, heads, kv_heads, dim = 65536, 2, 1, 64
    r = random.Random(116)
    lengths = [r.choice([0, 1, 1, 2, 17]) for _ in range(n)]
    cache = Cache(sum(-(-x // 16) for x in lengths), kv_heads, dim, 16, "int8")
    tables = tables_for(lengths, 16, cache.c.max_blocks, 117, spare=0)
    total = sum(lengths)
    run = Appender(cache, heads, "f32", dim, "half", 32)
    qkv = values(total, (heads + 2 * kv_heads) * dim, 118)
    q_out = torch.full((total, heads * dim), 7.0, device=DEV)
    offsets = [0]
    for x in lengths:
        offsets.append(offsets[-1] + x)
    off, first = torch.tensor(offsets, dtype=torch.int32, device=DEV), torch.zeros(n, dtype=torch.int32, device=DEV)
    mp.kv8_append(cache.c, run.args(qkv, q_out, tables, off, first), run.error.data_ptr(), stream())
    out = torch.full((total, heads * dim), 7.0, device=DEV)
    workspace = torch.zeros(mp.kv8_prefill_workspace(cache.c, heads), dtype=torch.uint8, device=DEV)
    common = dict(tables=tables.data_ptr(), workspace=workspace.data_ptr(), workspace_bytes=workspace.numel(), type=0,
                  heads=heads, table_stride=tables.stride(0), count=n, scale=0.125, q_stride=heads * dim,
                  out_stride=heads * dim)
    mp.kv8_attention_prefill(cache.c, mp.Kv8PrefillArgs(q=q_out.data_ptr(), out=out.data_ptr(), row_offsets=off.data_ptr(),
                             starts=first.data_ptr(), rows=total, **common), run.error.data_ptr(), stream())
    q, last = values(n, heads * dim, 119), torch.full((n, heads * dim), 7.0, device=DEV)
    lens = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    mp.kv8_attention_decode(cache.c, mp.Kv8DecodeArgs(q=q.data_ptr(), out=last.data_ptr(), lengths=lens.data_ptr(), **common),
                            run.error.data_ptr(), stream())
    assert mp.kv8_status(run.error.data_ptr(), stream()) == mp.MP_OK
    assert bool((last[lens == 0] == 0).all())
    for i in [0, 1, 511, 512, n - 1] + [r.randrange(n) for _ in range(60)]:
        x, at = lengths[i], offsets[i]
        if not x:
            continue
        pages, scales = cache.store[:, 0].clone(), cache.scale_store[:, 0].clone()
        y, pos = qkv[at: at + x].double(), torch.arange(x, device=DEV)
        c, s = run.cos[pos].double(), run.sin[pos].double()
        k = ref.rotate(y[:, heads * dim: (heads + 1) * dim].reshape(x, 1, dim), c, s, dim, "half")
        ref.append(pages, scales, "int8", k, y[:, (heads + 1) * dim:].reshape(x, 1, dim), [tables[i].tolist()], [0, x], [0])
        assert torch.equal(pages, cache.store[:, 0]) and torch.equal(scales.view(torch.int32), cache.scale_store[:, 0].view(torch.int32))
        check_rows(cache, heads, q_out[at: at + x], out[at: at + x], tables[i].tolist(), x, 0.125, False)
        check_rows(cache, heads, q[i: i + 1], last[i: i + 1], tables[i].tolist(), x, 0.125, False)
