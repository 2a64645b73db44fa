"""8-bit paged K/V cache operators where they can go wrong: scales at the ends of FP32's range, metadata that leaves
its bounds, very long contexts, calls of many rows."""
import math

import pytest
import torch

import kv8_reference as ref
from test_gpu_kv8 import DEV, DTYPES, Appender, Cache, check_rows, decode, fill, prefill, stream, tables_for, values
from tinyinfer_b200 import device as mp

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rotary", [0, 64])
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_append_under_the_largest_scale(built, fmt, rotary):
    """A held scale of 2^126 or 2^127 stays, and codes are the nearest to value / scale (2^-127 is subnormal)."""
    for held in (2.0 ** 126, 2.0 ** 127):
        cache = Cache(4, 3, 64, 16, fmt)
        tables = tables_for([16], 16, 4, 80)
        fill(cache, tables, [3], 81)
        cache.scales[tables[0, 0].long()] = held
        run = Appender(cache, 9, "f32", rotary, "half", 16)
        x = values(5, 960, 82, 0.0)
        x[:, 576:] *= 2e38 / x[:, 576:].abs().amax()  # rotated magnitudes stay below 2.9e38
        run(tables, [5], [3], x)


@pytest.mark.parametrize("first,late,gap", [(0.0, 2.0 ** 10, 140), (2.0 ** -100, 2.0 ** 20, 140),
                                            (0.0, 2.0 ** 100, 120), (2.0 ** -100, 2.0 ** 100, 100), (1.0, 2.0 ** 60, 90)])
def test_faint_tokens_with_large_value_scales(built, first, late, gap):
    """Tokens whose weights are 2^-gap of the others', with V scales far above theirs, turn about with them; decode and
    prefill row by row. Weights below 2^-126 of a row's largest count as zero (FP32's smallest normal number), so that
    many times the largest V value comes on top of the bound."""
    n = 4096
    cache = Cache(n // 16, 3, 64, 16, "int8")
    tables = tables_for([n], 16, n // 16, 83, spare=0)
    fill(cache, tables, [n], 84, (0, 0))
    faint = tables[0, torch.arange(n // 16, device=DEV) % 4 >= 2].long()  # every other 32 tokens
    loud = tables[0, torch.arange(n // 16, device=DEV) % 4 < 2].long()
    cache.pages[:, :, 0] = 0
    cache.pages[faint, :, 0, :, 0] = -64
    cache.scales[loud, :, 1], cache.scales[faint, :, 1] = first, late
    q = torch.zeros(1, 576, device=DEV)
    q.view(9, 64)[:, 0] = gap * math.log(2) / 8  # the faint tokens' score is -gap ln 2
    want, weight, size, top = ref.attend(q.view(1, 9, 64), cache.pages, cache.scales, "int8", tables[0].tolist(), n, 0.125)
    limit = ref.bound(want, weight, size, top, n, 64, False) + n * 2.0 ** -126 * late * 127
    for _, out in (decode(cache, 9, tables, [n], "f32", q=q), prefill(cache, 9, tables, [1], [n - 1], "f32", q=q)):
        assert bool(torch.isfinite(out).all())
        assert bool(((out.view(1, 9, 64).double() - want).abs() <= limit).all())


@pytest.mark.parametrize("rows", [5, 100])
@pytest.mark.parametrize("scale", [2.0 ** 127, 3.4028234663852886e38])
def test_value_scales_at_the_top_of_the_range(built, scale, rows):
    """V scales up to FP32's largest number, under codes of 0 and of E4M3's smallest step: outputs are the values."""
    cache = Cache(8, 3, 64, 16, "e4m3")
    tables = tables_for([100], 16, 8, 85)
    fill(cache, tables, [100], 86, (-6, -6))
    cache.pages[:, :, 1] = torch.arange(64, device=DEV).to(torch.int8) % 2  # codes 0 and 2^-9 by turns
    cache.scales[:, :, 1] = scale
    want = (torch.arange(64, device=DEV) % 2).double() * 2.0 ** -9 * scale
    # scores, weights and the joined sums have FP32's roundings in common with the normaliser but for their order: 100
    # terms on each side, 2^-24 each, and a few roundings of the result
    for _, out in (prefill(cache, 9, tables, [rows], [100 - rows], "f32"), decode(cache, 9, tables, [100], "f32")):
        off = (out.view(-1, 9, 64).double() - want).abs()
        assert bool(torch.isfinite(out).all()) and bool((off <= want * 210 * 2.0 ** -24).all())


def test_long_bf16_prefill_does_not_fade(built):
    """2^20 tokens of one V value under random scores: the value comes back. (The tensor core cuts its sums by up to
    2^-23 a product; an output added up in one chain over 65536 of them came out 0.5 % small.)"""
    n, rows, count = 1 << 20, 256, 152
    cache = Cache(n // 256, 1, 64, 256, "int8")
    tables = tables_for([n], 256, n // 256, 87, spare=0).repeat(count, 1).contiguous()  # enough items that none is cut
    g = torch.Generator(DEV).manual_seed(88)
    cache.pages[:, :, 0] = torch.randint(-100, 101, cache.pages[:, :, 0].shape, generator=g, device=DEV, dtype=torch.int8)
    cache.pages[:, :, 1] = 100
    cache.scales.fill_(2.0 ** -6)
    _, out = prefill(cache, 1, tables, [rows] * count, [n - rows] * count, "bf16")
    assert bool((out == 100 * 2.0 ** -6).all()), out.unique()


@pytest.mark.parametrize("dim", [64, 128])
def test_bf16_prefill_chains_with_rising_scores_and_scales(built, dim):
    """Contexts of three chains of sums and a rest; scores that rise, stay or fall along them (by head), V scales that
    rise 2^12 times, so that the reference and the unit move within and between chains."""
    n, rows, count, heads = 100000, 100, 150, 4
    cache = Cache(n // 32, 1, dim, 32, "int8")
    table = tables_for([n], 32, n // 32, 95, spare=0)
    fill(cache, table, [n], 96, (0, 0))
    blocks, at = table[0].long(), torch.arange(n // 32, device=DEV)
    keys = torch.zeros(n, dim, dtype=torch.int8, device=DEV)
    marked = torch.arange(0, n, 997, device=DEV)  # every 997th token has a score, from 0 up to 16
    keys[marked, 0] = (marked * 127 // n).to(torch.int8)
    cache.pages[blocks, 0, 0] = keys.view(-1, 32, dim)
    cache.scales[blocks, 0, 1] = torch.exp2((at * 12 // len(at) - 6).float())
    starts = [n - rows - 61 * i for i in range(count)]
    q = torch.zeros(rows * count, heads, dim, device=DEV)
    q[..., 0] = torch.tensor([1.0, 0.5, 0.0, -1.0], device=DEV) * (dim ** 0.5 / 8)
    q, out = prefill(cache, heads, table.repeat(count, 1).contiguous(), [rows] * count, starts, "bf16", q=q.flatten(1))
    for i in (0, 75, 149):
        part = slice(i * rows, (i + 1) * rows)
        want, weight, _, top = ref.attend(q[part].view(rows, heads, dim), cache.pages, cache.scales, "int8",
                                          table[0].tolist(), starts[i] + rows, dim ** -0.5)
        # a weight is one FP16 half (2^-11), its score has two roundings (|score| < 2^5 in powers of two: 2^-18), the
        # chains cut 2^-12, the normaliser adds 2^-12 at most; a rounding of the result; FP16's smallest steps
        limit = weight * (2 ** -11 + 2 ** -17 + 2 ** -11) + want.abs() * 2 ** -8 + top * n * 2 ** -33
        off = (out[part].view(rows, heads, dim).double() - want).abs()
        assert bool((off <= limit).all()), float((off / limit).max())


def test_long_bf16_decode_does_not_fade(built):
    """2^20 tokens per row and a row per warp: values of 64 and 65 whose mean lies just above the border of two BF16
    numbers (64 and 64.5), under random scores. Sums that lost 2^-10 on the way fall on the other side of it."""
    n, rows = 1 << 20, 2 * 148 * 16
    cache = Cache(n // 256, 1, 64, 256, "int8")
    tables = tables_for([n], 256, n // 256, 97, spare=0).repeat(rows, 1).contiguous()
    g = torch.Generator(DEV).manual_seed(98)
    cache.pages[:, :, 0] = torch.randint(-100, 101, cache.pages[:, :, 0].shape, generator=g, device=DEV, dtype=torch.int8)
    cache.pages[:, :, 1] = (64 + (torch.rand(cache.pages[:, :, 1].shape, generator=g, device=DEV) < 0.27)).to(torch.int8)
    cache.scales[..., 0], cache.scales[..., 1] = 2.0 ** -8, 1.0
    q, out = decode(cache, 1, tables, [n] * rows, "bf16")
    for i in range(0, rows, 599):
        want, weight, _, _ = ref.attend(q[i: i + 1].view(1, 1, 64), cache.pages, cache.scales, "int8", tables[i].tolist(), n, 0.125)
        # half a step of the result (0.25), and 2^-13 for the sums
        assert bool(((out[i].double() - want.view(-1)).abs() <= 0.25 + weight.view(-1) * 2 ** -13).all())


@pytest.mark.parametrize("dim,heads,kv_heads", [(64, 9, 3), (128, 8, 2)])
def test_short_contexts_in_long_tables(built, dim, heads, kv_heads):
    """Tables that could hold more than a chain of sums (32768 tokens) beside ones that could not: the same outputs."""
    counts, starts = [70, 0, 130, 9], [500, 3, 0, 1200]
    lengths = [s + c if c else 0 for s, c in zip(starts, counts)]
    cache = Cache(sum(-(-n // 16) for n in lengths), kv_heads, dim, 16, "int8")
    outs = []
    for spare in (0, 2049):
        tables = tables_for(lengths, 16, cache.c.max_blocks, 102, spare=spare)
        fill(cache, tables, lengths, 103)
        q, out = prefill(cache, heads, tables, counts, starts, "bf16")
        outs.append(out)
        at = 0
        for i, (c, n) in enumerate(zip(counts, lengths)):
            if c:
                check_rows(cache, heads, q[at: at + c], out[at: at + c], tables[i].tolist(), n, dim ** -0.5, True)
            at += c
    assert torch.equal(*outs)


@pytest.mark.parametrize("log2n", [17, 20])
@pytest.mark.parametrize("dim", [64, 128])
def test_long_sums_of_like_weights(built, dim, log2n):
    """FP32 rows over 2^17 and 2^20 tokens of one value, all but the first of one weight: a sum that is rounded n times
    on its way up is off by at most n / 2 times 2^-24 of it, all errors alike, and the outputs' chains and the
    normaliser have n = tokens / 128 such sums each (2^-18: those within a chain, and the halves)."""
    n = 1 << log2n
    cache = Cache(n // 256, 1, dim, 256, "int8")
    table = tables_for([n], 256, n // 256, 107, spare=0)
    cache.pages.zero_()
    cache.pages[:, :, 0, :, 0] = -1
    cache.pages[int(table[0, 0]), 0, 0, 0, 0] = 0
    cache.pages[:, :, 1], cache.scales[...] = 100, 2.0 ** -6
    limit = 100 * 2.0 ** -6 * (n / 128 * 2.0 ** -24 + 2.0 ** -18)
    for weight in (0.7, 0.61, 0.9, 0.53):
        rows = 148 * (16 if dim == 64 else 8)  # a row per warp
        q = torch.zeros(rows, dim, device=DEV)
        q[:, 0] = -math.log(weight) * 2.0 ** 6 * dim ** 0.5
        _, out = decode(cache, 1, table.repeat(rows, 1).contiguous(), [n] * rows, "f32", q=q)
        assert float((out.double() - 100 * 2.0 ** -6).abs().max()) <= limit
        count = 152  # items enough that none is cut
        q = q[:1].repeat(256 * count, 1)
        _, out = prefill(cache, 1, table.repeat(count, 1).contiguous(), [256] * count, [n - 256] * count, "f32", q=q)
        assert float((out.double() - 100 * 2.0 ** -6).abs().max()) <= limit


@pytest.mark.parametrize("rows", [10, 900])
@pytest.mark.parametrize("fault", ["table", "rotation", "rows", "order"])
def test_append_leaves_a_bad_sequence_out(built, fault, rows):
    """A sequence that begins in range and ends behind its table, the rotation tables or the call's rows, or whose
    offsets fall: reported, and none of its rows is written; the others are."""
    bt, heads, kh, d = 16, 4, 2, 64
    table = 2 * rows // bt + 3
    cache = Cache(3 * table + 3, kh, d, bt, "int8")
    tables = tables_for([table * bt] * 3, bt, cache.c.max_blocks, 89, spare=0)
    positions = table * bt - (20 if fault == "rotation" else 0)
    run = Appender(cache, heads, "f32", d, "half", positions)
    starts, offsets = [5, 0, 3], [0, rows, 2 * rows, 3 * rows]
    fill(cache, tables, starts, 90)
    good = [0, 2]
    if fault == "rows":
        good, offsets[3] = [0, 1], 3 * rows + 1
    elif fault == "order":
        good, offsets[2:] = [0], [rows - 2, rows]  # the third sequence names rows of the first
    else:
        starts[1] = positions - rows + 3
    x = values(3 * rows, (heads + 2 * kh) * d, 91)
    q_out = torch.full((3 * rows, heads * d), 7.0, device=DEV)
    pages, scales = cache.store.clone(), cache.scale_store.clone()
    off, first = (torch.tensor(a, dtype=torch.int32, device=DEV) for a in (offsets, starts))
    mp.kv8_append(cache.c, run.args(x, q_out, tables, off, first), run.error.data_ptr(), stream())
    assert mp.kv8_status(run.error.data_ptr(), stream()) == mp.MP_ERR_BOUNDS
    for i in good:
        part = slice(i * rows, (i + 1) * rows)
        assert bool((q_out[part] != 7).any(1).all())
        k, v = (x[part, a: a + kh * d].double().view(rows, kh, d) for a in (heads * d, (heads + kh) * d))
        at = torch.arange(rows, device=DEV) + starts[i]
        k = ref.rotate(k, run.cos[at].double(), run.sin[at].double(), d, "half")
        ref.append(pages[:, 0], scales[:, 0], "int8", k, v, [tables[i].tolist()], [0, rows], [starts[i]])
        q_out[part] = 7
    assert bool((q_out == 7).all()), "rows of a sequence that was to be left out"
    assert torch.equal(pages, cache.store) and torch.equal(scales.view(torch.int32), cache.scale_store.view(torch.int32))


def test_prefill_refuses_offsets_that_fall(built):
    """Offsets that fall name rows more than once, more of them than the plan's indexes count: the call is left out."""
    cache = Cache(30, 3, 64, 16, "int8")
    tables = tables_for([100] * 4, 16, 30, 92, spare=0)
    fill(cache, tables, [100] * 4, 93)
    q, out = values(100, 576, 94), torch.full((100, 576), 7.0, device=DEV)
    workspace = torch.zeros(mp.kv8_prefill_workspace(cache.c, 9), dtype=torch.uint8, device=DEV)
    off, first = (torch.tensor(a, dtype=torch.int32, device=DEV) for a in ([0, 100, 0, 100, 0], [0] * 4))
    word = torch.zeros(1, dtype=torch.int32, device=DEV)
    args = mp.Kv8PrefillArgs(q=q.data_ptr(), out=out.data_ptr(), q_stride=576, out_stride=576, tables=tables.data_ptr(),
                             row_offsets=off.data_ptr(), starts=first.data_ptr(), workspace=workspace.data_ptr(),
                             workspace_bytes=workspace.numel(), type=0, heads=9, table_stride=tables.stride(0), count=4,
                             rows=100, scale=0.125)
    mp.kv8_attention_prefill(cache.c, args, word.data_ptr(), stream())
    assert mp.kv8_status(word.data_ptr(), stream()) == mp.MP_ERR_BOUNDS
    assert bool((out == 7).all())
    off.copy_(torch.tensor([0, 40, 40, 95, 100], dtype=torch.int32))  # the workspace serves the next call
    mp.kv8_attention_prefill(cache.c, args, word.data_ptr(), stream())
    assert mp.kv8_status(word.data_ptr(), stream()) == mp.MP_OK
    for i, (lo, hi) in enumerate(((0, 40), (40, 40), (40, 95), (95, 100))):
        if hi > lo:
            check_rows(cache, 9, q[lo:hi], out[lo:hi], tables[i].tolist(), hi - lo, 0.125, False)


@pytest.mark.parametrize("heads,kv_heads,dim,dtype", [(9, 3, 64, "f32"), (32, 8, 128, "bf16")])
def test_prefill_waits_that_run_out(built, heads, kv_heads, dim, dtype):
    """Waits that expire end the kernel with the timeout bit within their bound; the next call, over a workspace that
    was zeroed again, is as ever."""
    cache = Cache(60, kv_heads, dim, 16, "int8")
    tables = tables_for([400, 300], 16, 60, 99)
    fill(cache, tables, [400, 300], 100)
    q = values(170, heads * dim, 101).to(DTYPES[dtype])
    out = torch.zeros_like(q)
    workspace = torch.zeros(mp.kv8_prefill_workspace(cache.c, heads), dtype=torch.uint8, device=DEV)
    off, first = (torch.tensor(a, dtype=torch.int32, device=DEV) for a in ([0, 100, 170], [300, 230]))
    word = torch.zeros(1, dtype=torch.int32, device=DEV)
    args = mp.Kv8PrefillArgs(q=q.data_ptr(), out=out.data_ptr(), q_stride=q.stride(0), out_stride=out.stride(0),
                             tables=tables.data_ptr(), row_offsets=off.data_ptr(), starts=first.data_ptr(),
                             workspace=workspace.data_ptr(), workspace_bytes=workspace.numel(),
                             type=list(DTYPES).index(dtype), heads=heads, table_stride=tables.stride(0), count=2, rows=170,
                             scale=dim ** -0.5)
    for _ in range(3):
        begin, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        mp.kv8_inject_wait_timeout(1000)
        begin.record()
        mp.kv8_attention_prefill(cache.c, args, word.data_ptr(), stream())
        end.record()
        assert mp.kv8_status(word.data_ptr(), stream()) == mp.MP_ERR_TIMEOUT
        assert begin.elapsed_time(end) < 500  # ms: not the 2 s of other calls
        workspace.zero_()
        mp.kv8_attention_prefill(cache.c, args, word.data_ptr(), stream())
        assert mp.kv8_status(word.data_ptr(), stream()) == mp.MP_OK
        for part, i, n in ((slice(0, 100), 0, 400), (slice(100, 170), 1, 300)):
            check_rows(cache, heads, q[part], out[part], tables[i].tolist(), n, dim ** -0.5, dtype == "bf16")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("dim,heads,kv_heads", [(64, 9, 3), (128, 8, 2)])
def test_queries_that_are_not_finite_stay_alone(built, dim, heads, kv_heads, dtype):
    """A NaN or an infinity in one row's head makes that output NaN and no other; decode, row by row and as tiles."""
    n = 400
    cache = Cache(n // 16, kv_heads, dim, 16, "int8")
    tables = tables_for([n], 16, n // 16, 104)
    fill(cache, tables, [n], 105)
    for rows in (5, 100):
        q = values(rows, heads * dim, 106).to(DTYPES[dtype]).view(rows, heads, dim)
        q[1, 2, 7], q[3, 0, 0], q[rows - 1, heads - 1, dim - 1] = float("nan"), float("inf"), -float("inf")
        bad = ~torch.isfinite(q).all(-1)
        good = torch.where(bad[..., None], torch.zeros_like(q), q)
        want, weight, size, top = ref.attend(good, cache.pages, cache.scales, "int8", tables[0].tolist(), n, dim ** -0.5)
        limit = ref.bound(want, weight, size, top, n, dim, dtype == "bf16")
        _, out = prefill(cache, heads, tables, [rows], [n - rows], dtype, q=q.flatten(1))
        outs = [out]
        if rows == 5:
            lengths = [n - rows + 1 + i for i in range(rows)]
            outs.append(decode(cache, heads, tables.repeat(rows, 1).contiguous(), lengths, dtype, q=q.flatten(1))[1])
        for out in outs:
            out = out.view(rows, heads, dim)
            assert bool(torch.isnan(out[bad]).all())
            assert bool(((out[~bad].double() - want[~bad]).abs() <= limit[~bad]).all())
