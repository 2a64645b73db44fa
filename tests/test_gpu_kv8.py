"""8-bit paged K/V cache operators against plain 64-bit forms (kv8_reference.py).

Codes and scales have to be equal; rotated queries and attention outputs lie within
kv8_reference.rotation_bound and kv8_reference.bound, which count the roundings. Blocks that no table names and slots
behind a sequence's last token hold NaN codes (E4M3) and NaN scales, buffers have
strides above their rows and sentinels behind them.
"""
import math

import pytest
import torch

import kv8_reference as ref
from tinyinfer_b200 import device as mp

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
FORMATS = {"int8": mp.MP_KV8_INT8, "e4m3": mp.MP_KV8_E4M3}


def stream():
    return torch.cuda.current_stream().cuda_stream


class Cache:
    """Pages and scales inside larger buffers (strides above a block's), everything stale at first."""

    def __init__(self, blocks, kv_heads, dim, bt, fmt, *, layers=1, layer=0):
        self.fmt, self.bt, self.dim, self.kv_heads = fmt, bt, dim, kv_heads
        self.store = torch.full((blocks, layers, kv_heads, 2, bt, dim), 0x7F, dtype=torch.int8, device=DEV)
        self.pages = self.store[:, layer]
        self.scale_store = torch.full((blocks, layers, kv_heads, 2), float("nan"), device=DEV)
        self.scales = self.scale_store[:, layer]
        self.c = mp.Kv8Cache(pages=self.pages.data_ptr(), scales=self.scales.data_ptr(),
                             page_stride=self.store.stride(0), scale_stride=self.scale_store.stride(0),
                             format=FORMATS[fmt], kv_heads=kv_heads, head_dim=dim, block_tokens=bt, max_blocks=blocks)


def tables_for(lengths, bt, blocks, seed, spare=1):
    """Block tables that permute the pool; unused entries are out of range."""
    g = torch.Generator().manual_seed(seed)
    perm = torch.randperm(blocks, generator=g)
    pages = [-(-n // bt) for n in lengths]
    assert sum(pages) <= blocks
    t = torch.full((len(lengths), max(1, max(pages)) + spare), 1 << 30, dtype=torch.int32)
    at = 0
    for i, n in enumerate(pages):
        t[i, :n] = perm[at: at + n]
        at += n
    return t.to(DEV)


def fill(cache, tables, lengths, seed, exponents=(-9, -4)):
    """Random codes for every sequence's tokens, random power-of-two scales for its blocks."""
    g = torch.Generator(DEV).manual_seed(seed)
    pages = [-(-n // cache.bt) for n in lengths]
    for i, n in enumerate(lengths):
        if not n:
            continue
        blocks = tables[i, : pages[i]].long()
        x = torch.randn(len(blocks), cache.kv_heads, 2, cache.bt, cache.dim, generator=g, device=DEV).double()
        codes = ref.encode(ref.nearest(x * (40 if cache.fmt == "int8" else 60), cache.fmt), cache.fmt)
        past = len(blocks) * cache.bt - n
        if past:
            codes[-1, :, :, cache.bt - past:] = 0x7F
        cache.pages[blocks] = codes
        low, high = exponents
        e = torch.randint(low, high + 1, (len(blocks), cache.kv_heads, 2), generator=g, device=DEV)
        cache.scales[blocks] = torch.exp2(e.double()).float()


def padded(rows, width, dtype, seed, extra=16):
    """A row buffer with a stride above its width and two rows behind it; random values, NaN in the gaps."""
    g = torch.Generator(DEV).manual_seed(seed)
    store = torch.full((rows + 2, width + extra), float("nan"), dtype=dtype, device=DEV)
    store[:rows, :width] = torch.randn(rows, width, generator=g, device=DEV).to(dtype)
    return store, store[:rows, :width]


def decode(cache, heads, tables, lengths, dtype, seed=1, scale=None, q=None, error=None, workspace=None):
    n, d = len(lengths), cache.dim
    qs, qv = padded(n, heads * d, DTYPES[dtype], seed)
    if q is not None:
        qv.copy_(q)
    out = torch.full((n + 1, heads * d + 8), 7.0, dtype=DTYPES[dtype], device=DEV)
    if workspace is None:
        workspace = torch.zeros(mp.kv8_decode_workspace(cache.c, heads), dtype=torch.uint8, device=DEV)
    lens = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    word = torch.zeros(1, dtype=torch.int32, device=DEV) if error is None else error
    args = mp.Kv8DecodeArgs(q=qs.data_ptr(), out=out.data_ptr(), q_stride=qs.stride(0), out_stride=out.stride(0),
                            tables=tables.data_ptr(), lengths=lens.data_ptr(), workspace=workspace.data_ptr(),
                            workspace_bytes=workspace.numel(), type=list(DTYPES).index(dtype), heads=heads,
                            table_stride=tables.stride(0), count=n, scale=d ** -0.5 if scale is None else scale)
    mp.kv8_attention_decode(cache.c, args, word.data_ptr(), stream())
    first = out.clone()
    mp.kv8_attention_decode(cache.c, args, word.data_ptr(), stream())  # the workspace is left as the next call needs it
    if error is None:
        assert mp.kv8_status(word.data_ptr(), stream()) == mp.MP_OK
    assert torch.equal(first.view(torch.int16), out.view(torch.int16)), "two calls differ"
    assert bool((out[n:] == 7).all()) and bool((out[:, heads * d:] == 7).all()), "wrote outside the rows"
    return qv, out[:n, : heads * d]


def check_rows(cache, heads, q, out, table, length, scale, bf16):
    rows, d = q.shape[0], cache.dim
    want, weight, size, top = ref.attend(q.reshape(rows, heads, d), cache.pages, cache.scales, cache.fmt, table, length, scale)
    off = (out.double().reshape(rows, heads, d) - want).abs()
    limit = ref.bound(want, weight, size, top, length, d, bf16)
    assert bool(torch.isfinite(out).all())
    assert bool((off <= limit).all()), (length, float((off / limit).max()), float(off.max()))
    return float((off / limit).max())


GEOMETRIES = [(9, 3, 64, 16), (8, 8, 64, 32), (14, 2, 64, 16), (32, 8, 128, 16), (16, 1, 128, 64), (4, 1, 128, 16),
              (23, 1, 64, 48)]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("heads,kv_heads,dim,bt", GEOMETRIES)
def test_decode(built, heads, kv_heads, dim, bt, fmt, dtype):
    lengths = [0, 1, 2, 15, 16, 17, 31, 33, 0, 64, 100, 257, 1000, 5, 48]
    cache = Cache(sum(-(-n // bt) for n in lengths) + 5, kv_heads, dim, bt, fmt, layers=2, layer=1)
    tables = tables_for(lengths, bt, cache.c.max_blocks, 3)
    fill(cache, tables, lengths, 4)
    q, out = decode(cache, heads, tables, lengths, dtype)
    for i, n in enumerate(lengths):
        if n == 0:
            assert bool((out[i] == 0).all())
        else:
            check_rows(cache, heads, q[i: i + 1], out[i: i + 1], tables[i].tolist(), n, dim ** -0.5, dtype == "bf16")


@pytest.mark.parametrize("heads,kv_heads,dim,lengths", [
    (9, 3, 64, [70001]), (8, 1, 128, [40000, 3]), (9, 3, 64, [16] * 700), (9, 3, 64, [1, 30000] + [7] * 40),
    (9, 3, 64, [2048 + i for i in range(64)]), (64, 1, 64, [5000, 0, 0, 1]), (9, 3, 64, [0] * 50),
    (3, 3, 64, [1] * 1300 + [999])])
def test_decode_runs_over_the_device(built, heads, kv_heads, dim, lengths):
    """One long row over every SM, many short rows per warp, rows that begin and end inside runs."""
    cache = Cache(max(1, sum(-(-n // 16) for n in lengths)), kv_heads, dim, 16, "int8")
    tables = tables_for(lengths, 16, cache.c.max_blocks, 5)
    fill(cache, tables, lengths, 6)
    q, out = decode(cache, heads, tables, lengths, "f32")
    for i in sorted(set(range(0, len(lengths), max(1, len(lengths) // 20))) | {len(lengths) - 1}):
        if lengths[i]:
            check_rows(cache, heads, q[i: i + 1], out[i: i + 1], tables[i].tolist(), lengths[i], dim ** -0.5, False)
    zero = torch.tensor([n == 0 for n in lengths], device=DEV)
    assert bool((out[zero] == 0).all())


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("exponents,magnitude,scale", [((-60, 60), 1.0, 2.0 ** -60), ((-100, -90), 1e28, 0.125),
                                                       ((-6, -6), 1e-30, 0.125), ((-6, -6), 1e30, 1e-31),
                                                       ((-8, -4), 40.0, 0.125), ((-8, -4), 1.0, -0.125)])
def test_decode_ranges(built, fmt, exponents, magnitude, scale):
    """Block scales far apart, queries far from 1, sharp softmaxes, a negative scale."""
    lengths = [300, 40, 1, 777]
    cache = Cache(90, 3, 64, 16, fmt)
    tables = tables_for(lengths, 16, 90, 7)
    fill(cache, tables, lengths, 8, exponents)
    g = torch.Generator(DEV).manual_seed(9)
    q = torch.randn(4, 576, generator=g, device=DEV) * magnitude
    q, out = decode(cache, 9, tables, lengths, "f32", scale=scale, q=q)
    for i, n in enumerate(lengths):
        check_rows(cache, 9, q[i: i + 1], out[i: i + 1], tables[i].tolist(), n, scale, False)


def test_decode_scales_of_any_value(built):
    """Scales that are no powers of two, zero scales, and a zero query."""
    lengths = [333, 20]
    cache = Cache(40, 3, 64, 16, "int8")
    tables = tables_for(lengths, 16, 40, 10)
    fill(cache, tables, lengths, 11)
    cache.scales.mul_(1.37)
    cache.scales[tables[0, 3].long()] = 0.0
    cache.scales[tables[1, 1].long(), :, 1] = 0.0
    q = torch.randn(2, 576, device=DEV)
    q[1] = 0
    q, out = decode(cache, 9, tables, lengths, "f32", q=q)
    for i, n in enumerate(lengths):
        check_rows(cache, 9, q[i: i + 1], out[i: i + 1], tables[i].tolist(), n, 0.125, False)


def prefill(cache, heads, tables, counts, starts, dtype, seed=1, behind=3, error=None, q=None):
    rows, d = sum(counts), cache.dim
    qs, qv = padded(rows + behind, heads * d, DTYPES[dtype], seed)
    if q is not None:
        qv[:rows] = q
    out = torch.full((rows + behind, heads * d + 8), 7.0, dtype=DTYPES[dtype], device=DEV)
    workspace = torch.zeros(mp.kv8_prefill_workspace(cache.c, heads), dtype=torch.uint8, device=DEV)
    offsets = torch.tensor([sum(counts[:i]) for i in range(len(counts) + 1)], dtype=torch.int32, device=DEV)
    first = torch.tensor(starts, dtype=torch.int32, device=DEV)
    word = torch.zeros(1, dtype=torch.int32, device=DEV) if error is None else error
    args = mp.Kv8PrefillArgs(q=qs.data_ptr(), out=out.data_ptr(), q_stride=qs.stride(0), out_stride=out.stride(0),
                             tables=tables.data_ptr(), row_offsets=offsets.data_ptr(), starts=first.data_ptr(),
                             workspace=workspace.data_ptr(), workspace_bytes=workspace.numel(),
                             type=list(DTYPES).index(dtype), heads=heads, table_stride=tables.stride(0),
                             count=len(counts), rows=rows + behind, scale=d ** -0.5)
    mp.kv8_attention_prefill(cache.c, args, word.data_ptr(), stream())
    once = out.clone()
    mp.kv8_attention_prefill(cache.c, args, word.data_ptr(), stream())
    if error is None:
        assert mp.kv8_status(word.data_ptr(), stream()) == mp.MP_OK
    assert torch.equal(once.view(torch.int16), out.view(torch.int16)), "two calls differ"
    assert bool((out[rows:] == 7).all()) and bool((out[:, heads * d:] == 7).all()), "wrote outside the rows"
    return qv[:rows], out[:rows, : heads * d]


def check_prefill(cache, heads, tables, counts, starts, dtype):
    lengths = [s + c if c else 0 for s, c in zip(starts, counts)]
    fill(cache, tables, lengths, 14)
    q, out = prefill(cache, heads, tables, counts, starts, dtype)
    at = 0
    for i, (c, s) in enumerate(zip(counts, starts)):
        for lo in range(0, c, 512):
            n = min(512, c - lo)
            check_rows(cache, heads, q[at + lo: at + lo + n], out[at + lo: at + lo + n], tables[i].tolist(), s + lo + n,
                       cache.dim ** -0.5, dtype == "bf16")
        at += c


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("heads,kv_heads,dim,bt", GEOMETRIES)
def test_prefill(built, heads, kv_heads, dim, bt, fmt, dtype):
    counts = [0, 1, 2, 41, 42, 43, 0, 130, 5, 1, 64, 257]
    starts = [9, 0, 15, 0, 3, 100, 0, 127, 300, 999, 64, 0]
    lengths = [s + c if c else 0 for s, c in zip(starts, counts)]
    cache = Cache(sum(-(-n // bt) for n in lengths) + 5, kv_heads, dim, bt, fmt, layers=2, layer=0)
    check_prefill(cache, heads, tables_for(lengths, bt, cache.c.max_blocks, 12), counts, starts, dtype)


@pytest.mark.parametrize("counts,starts", [([1900], [0]), ([300], [9001]), ([1] * 100, list(range(0, 1000, 10))),
                                           ([7, 1, 500], [4000, 0, 1]), ([0, 0, 1, 0], [5, 0, 0, 3]), ([33], [31])])
def test_prefill_shapes(built, counts, starts):
    lengths = [s + c if c else 0 for s, c in zip(starts, counts)]
    cache = Cache(sum(-(-n // 16) for n in lengths) + 1, 3, 64, 16, "int8")
    check_prefill(cache, 9, tables_for(lengths, 16, cache.c.max_blocks, 13), counts, starts, "f32")


@pytest.mark.parametrize("heads,kv_heads,dim,dtype", [(9, 3, 64, "f32"), (32, 8, 128, "bf16"), (16, 2, 128, "f32"),
                                                      (8, 8, 64, "bf16")])
def test_prefill_many_items_per_sm(built, heads, kv_heads, dim, dtype):
    """Several items of unlike shapes one after the other on every SM: blocks whose rows fill one tile of vectors or
    two, tiles of which one sees fewer tokens, items that end on the next SM."""
    rows = 2 * (128 * kv_heads // heads)
    counts = [1, rows, rows // 2 + 1, 3, 2 * rows + 5, rows // 2] * 24
    starts = [(37 * i) % 700 for i in range(len(counts))]
    lengths = [s + c for s, c in zip(starts, counts)]
    cache = Cache(sum(-(-n // 16) for n in lengths), kv_heads, dim, 16, "int8")
    check_prefill(cache, heads, tables_for(lengths, 16, cache.c.max_blocks, 44), counts, starts, dtype)


@pytest.mark.parametrize("low", [-40, -100])
def test_prefill_tiny_value_scales(built, low):
    """Blocks whose V scale is far below the others' count in the sum of weights alone."""
    counts, starts = [60, 9], [300, 0]
    cache = Cache(40, 3, 64, 16, "int8")
    tables = tables_for([360, 9], 16, 40, 45)
    fill(cache, tables, [360, 9], 46, (-6, -6))
    cache.scales[tables[0, 2:20:3].long(), :, 1] = 2.0 ** low
    cache.scales[tables[1, 0].long(), 1, 1] = 0.0
    q, out = prefill(cache, 9, tables, counts, starts, "f32", q=torch.randn(69, 576, device=DEV) * 6)
    check_rows(cache, 9, q[:60], out[:60], tables[0].tolist(), 360, 0.125, False)
    check_rows(cache, 9, q[60:], out[60:], tables[1].tolist(), 9, 0.125, False)


def test_prefill_ranges(built):
    """Block scales far apart, queries of any size next to each other."""
    counts, starts = [70, 5], [50, 200]
    cache = Cache(30, 3, 64, 16, "e4m3")
    tables = tables_for([120, 205], 16, 30, 15)
    fill(cache, tables, [120, 205], 16, (-30, 20))
    cache.scales[:, :, 0] = 2.0 ** -6
    q = torch.randn(75, 576, device=DEV) * torch.exp2(torch.randint(-90, 1, (75, 1), device=DEV).double()).float()
    q, out = prefill(cache, 9, tables, counts, starts, "f32", q=q)
    check_rows(cache, 9, q[:70], out[:70], tables[0].tolist(), 120, 0.125, False)
    check_rows(cache, 9, q[70:], out[70:], tables[1].tolist(), 205, 0.125, False)


class Appender:
    """Fused q | k | v rows with gaps, rotation tables, and the call."""

    def __init__(self, cache, heads, dtype, rotary, layout, positions, in_place=False):
        self.cache, self.heads, self.dtype, self.rotary, self.layout = cache, heads, dtype, rotary, layout
        self.in_place = in_place
        half = rotary // 2
        angle = torch.arange(positions, device=DEV).double()[:, None] * 10000.0 ** -(
            torch.arange(half, device=DEV).double() / max(1, half))
        self.cos, self.sin = angle.cos().float().contiguous(), angle.sin().float().contiguous()
        self.error = torch.zeros(1, dtype=torch.int32, device=DEV)

    def args(self, qkv, q_out, tables, offsets, starts, with_q=True):
        d, kh, size = self.cache.dim, self.cache.kv_heads, qkv.element_size()
        base, stride = qkv.data_ptr(), qkv.stride(0)
        return mp.Kv8AppendArgs(q=base if with_q else None, k=base + self.heads * d * size,
                                v=base + (self.heads + kh) * d * size, q_out=q_out.data_ptr() if with_q else None,
                                q_stride=stride, k_stride=stride, v_stride=stride, q_out_stride=q_out.stride(0),
                                cos=self.cos.data_ptr(), sin=self.sin.data_ptr(), tables=tables.data_ptr(),
                                row_offsets=offsets.data_ptr(), starts=starts.data_ptr(),
                                type=list(DTYPES).index(self.dtype), heads=self.heads, rotary_dim=self.rotary,
                                rope_layout=mp.MP_ROPE_HALF if self.layout == "half" else mp.MP_ROPE_INTERLEAVED,
                                max_positions=self.cos.shape[0], table_stride=tables.stride(0), count=len(starts),
                                rows=qkv.shape[0])

    def __call__(self, tables, counts, starts, qkv, with_q=True, behind=2):
        """Appends sum(counts) rows; returns rotated q. Checks the whole cache against the plain form."""
        cache, rows, d, kh = self.cache, sum(counts), self.cache.dim, self.cache.kv_heads
        width = (self.heads + 2 * kh) * d
        store = torch.full((rows + behind, width + 8), float("nan"), dtype=DTYPES[self.dtype], device=DEV)
        store[:rows, :width] = qkv.to(store.dtype)
        x = store[:rows, :width].double()
        q_out = store if self.in_place else torch.full((rows + behind, self.heads * d + 8), 7.0, dtype=store.dtype, device=DEV)
        before = q_out.clone()
        offsets = [sum(counts[:i]) for i in range(len(counts) + 1)]
        pages, scales = cache.store.clone(), cache.scale_store.clone()
        layer = cache.pages.storage_offset() // (kh * 2 * cache.bt * d)
        off, first = (torch.tensor(a, dtype=torch.int32, device=DEV) for a in (offsets, starts))
        mp.kv8_append(cache.c, self.args(store, q_out, tables, off, first, with_q), self.error.data_ptr(), stream())
        assert mp.kv8_status(self.error.data_ptr(), stream()) == mp.MP_OK
        pos = torch.cat([torch.arange(s, s + c) for s, c in zip(starts, counts)]).to(DEV)
        c, s = self.cos[pos].double(), self.sin[pos].double()
        q, k, v = (y.reshape(rows, -1, d) for y in x.split([self.heads * d, kh * d, kh * d], 1))
        ref.append(pages[:, layer], scales[:, layer], cache.fmt, ref.rotate(k, c, s, self.rotary, self.layout), v,
                   tables.tolist(), offsets, starts)
        differ = pages != cache.store
        assert torch.equal(pages, cache.store), (int(differ.sum()), differ.nonzero()[:4].tolist(),
                                                 pages[differ][:4].tolist(), cache.store[differ][:4].tolist())
        assert torch.equal(scales.view(torch.int32), cache.scale_store.view(torch.int32))
        if with_q:
            want = ref.rotate(q, c, s, self.rotary, self.layout)
            got = q_out[:rows, : self.heads * d].double().reshape(rows, -1, d)
            assert bool(((got - want).abs() <= ref.rotation_bound(q, want, c, s, self.rotary, self.layout,
                                                                  self.dtype == "bf16")).all())
            before[:rows, : self.heads * d] = q_out[:rows, : self.heads * d]
        assert torch.equal(before.view(torch.int16), q_out.view(torch.int16)), "wrote outside the rows"
        return q_out[:rows, : self.heads * d]


def values(rows, width, seed, spread=1.0):
    g = torch.Generator(DEV).manual_seed(seed)
    return torch.randn(rows, width, generator=g, device=DEV) * torch.exp(
        spread * torch.randn(rows, 1, generator=g, device=DEV))


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("heads,kv_heads,dim,bt,dtype,rotary,layout", [
    (9, 3, 64, 16, "f32", 64, "half"), (9, 3, 64, 16, "f32", 64, "interleaved"), (32, 8, 128, 32, "bf16", 64, "interleaved"),
    (8, 8, 64, 16, "bf16", 24, "half"), (4, 1, 128, 64, "f32", 128, "half"), (6, 2, 128, 48, "f32", 40, "interleaved"),
    (3, 3, 64, 256, "f32", 0, "half"), (2, 1, 64, 16, "f32", 8, "half")])
def test_append(built, heads, kv_heads, dim, bt, dtype, rotary, layout, fmt):
    """Ragged rows from fresh and partly filled blocks, then on top of them twice more; codes, scales and q equal."""
    counts = [[1, 0, 17, 16, 40, 1, 3], [1, 1, 1, 0, 9, 15, 1], [16, 31, 1, 1, 1, 1, 70]]
    starts = [0, 5, 0, 16, 32, 0, 0]
    ends = [s + sum(c[i] for c in counts) for i, s in enumerate(starts)]
    cache = Cache(sum(-(-n // bt) for n in ends) + 3, kv_heads, dim, bt, fmt, layers=2, layer=1)
    tables = tables_for(ends, bt, cache.c.max_blocks, 17)
    # sequences that do not start a block continue what earlier appends left there
    fill(cache, tables, starts, 18)
    run = Appender(cache, heads, dtype, rotary, layout, max(ends), in_place=bt == 48)
    at = list(starts)
    for k, c in enumerate(counts):
        run(tables, c, at, values(sum(c), (heads + 2 * kv_heads) * dim, 19 + k), with_q=k != 1)
        at = [a + n for a, n in zip(at, c)]


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_append_token_by_token(built, fmt):
    """40 single tokens, magnitudes growing and shrinking over 2^30: an INT8 value stays within one scale of what was
    appended, an E4M3 value within a sixteenth (or a subnormal step)."""
    cache = Cache(8, 3, 64, 16, fmt)
    tables = tables_for([48, 48], 16, 8, 20)
    run = Appender(cache, 9, "f32", 0, "half", 64)
    kept = []
    for t in range(40):
        x = values(2, 960, 100 + t) * 2.0 ** (15 * math.sin(t))
        run(tables, [1, 1], [t, t], x)
        kept.append(x)
    for i in range(2):
        for t in range(40):
            block = int(tables[i, t // 16])
            scale = cache.scales[block].double()[..., None]
            got = ref.decode_codes(cache.pages[block, :, :, t % 16], fmt) * scale
            want = kept[t][i, 576:].double().reshape(2, 3, 64).transpose(0, 1)
            room = scale if fmt == "int8" else torch.maximum(want.abs() * 2 ** -4, scale * 2 ** -9)
            assert bool(((got - want).abs() <= room).all())


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_append_extremes(built, fmt):
    """Zero blocks, tiny and huge values, values on the borders between codes."""
    cache = Cache(12, 3, 64, 16, fmt)
    tables = tables_for([16] * 10, 16, 12, 21)
    run = Appender(cache, 9, "f32", 0, "half", 16)
    x = values(160, 960, 22)
    for i, f in enumerate([0.0, 1e-38, 1e-30, 1e-20, 1e37, 3e38]):
        part = x[16 * i: 16 * i + 16]
        x[16 * i: 16 * i + 16] = part / part.abs().amax() * f
    half = torch.arange(960, device=DEV).float() / 2 - 240  # INT8 borders at scale 1 or 2, both ties
    x[96:112] = (half % 127.0) * torch.where(half < 0, -1.0, 1.0)
    grid = ref.e4m3_grid()
    border = ((grid[1:] + grid[:-1]) / 2).float().to(DEV)
    x[112:128] = border[torch.arange(960, device=DEV) % 126]
    x[128:144] = torch.nextafter(border, torch.zeros_like(border))[torch.arange(960, device=DEV) % 126]
    run(tables, [16] * 10, [0] * 10, x)


def test_append_reports_values_it_cannot_hold(built):
    cache = Cache(4, 3, 64, 16, "int8")
    tables = tables_for([16, 16], 16, 4, 23)
    run = Appender(cache, 9, "f32", 0, "half", 16)
    x = values(4, 960, 24)
    x[0, 600], x[1, 900], x[1, 580], x[2, 700] = float("nan"), float("inf"), -float("inf"), 3.0
    q_out = torch.zeros(4, 576, device=DEV)
    off, first = (torch.tensor(a, dtype=torch.int32, device=DEV) for a in ([0, 2, 4], [0, 0]))
    args = run.args(x, q_out, tables, off, first)
    mp.kv8_append(cache.c, args, run.error.data_ptr(), stream())
    assert mp.kv8_status(run.error.data_ptr(), stream()) == mp.MP_ERR_NONFINITE
    assert mp.kv8_status(run.error.data_ptr(), stream()) == mp.MP_OK
    block = int(tables[0, 0])
    assert int(cache.pages[block, 0, 0, 0, 24]) == 0  # k head 0, dim 24: NaN
    assert int(cache.pages[block, 0, 0, 1, 4]) == -127  # -inf
    assert int(cache.pages[block, 2, 1, 1, 900 - 768 - 128]) == 127  # v head 2: inf
    assert bool(torch.isfinite(cache.scales[block]).all())
    cache.scales[block, 1, 0] = 0.3  # no append made this scale
    first += 2
    mp.kv8_append(cache.c, args, run.error.data_ptr(), stream())
    assert mp.kv8_status(run.error.data_ptr(), stream()) == mp.MP_ERR_NONFINITE


def test_bad_metadata_is_reported(built):
    """Block ids, lengths, starts and positions out of range set the bounds bit; nothing outside is touched."""
    lengths = [40, 40]
    cache = Cache(6, 3, 64, 16, "int8")
    good = tables_for(lengths, 16, 6, 25, spare=0)
    fill(cache, good, lengths, 26)
    word = torch.zeros(1, dtype=torch.int32, device=DEV)
    for bad_block in (6, -1, 1 << 30):
        tables = good.clone()
        tables[1, 1] = bad_block
        decode(cache, 9, tables, lengths, "f32", error=word)
        assert mp.kv8_status(word.data_ptr(), stream()) == mp.MP_ERR_BOUNDS
        prefill(cache, 9, tables, [3, 3], [37, 37], "f32", error=word)
        assert mp.kv8_status(word.data_ptr(), stream()) == mp.MP_ERR_BOUNDS
    for n in (49, -1, 1 << 30):
        decode(cache, 9, good, [40, n], "f32", error=word)
        assert mp.kv8_status(word.data_ptr(), stream()) == mp.MP_ERR_BOUNDS
    for s in (46, -1, 2 ** 31 - 2):
        prefill(cache, 9, good, [3, 3], [37, s], "f32", error=word)
        assert mp.kv8_status(word.data_ptr(), stream()) == mp.MP_ERR_BOUNDS
    run = Appender(cache, 9, "f32", 64, "half", 44)
    x, q_out = values(2, 960, 27), torch.zeros(2, 576, device=DEV)
    off = torch.tensor([0, 1, 2], dtype=torch.int32, device=DEV)
    for second, block in ((48, None), (-1, None), (44, None), (2 ** 31 - 1, None), (40, 6), (40, -5)):
        tables = good.clone()
        if block is not None:
            tables[1, 2] = block
        before = cache.store.clone()
        first = torch.tensor([40, second], dtype=torch.int32, device=DEV)
        mp.kv8_append(cache.c, run.args(x, q_out, tables, off, first), run.error.data_ptr(), stream())
        assert mp.kv8_status(run.error.data_ptr(), stream()) == mp.MP_ERR_BOUNDS
        mine = int(good[0, 2])
        before[mine] = cache.store[mine]
        assert torch.equal(before, cache.store)


def test_host_memory_is_refused(built):
    cache = Cache(4, 3, 64, 16, "int8")
    args = mp.Kv8DecodeArgs(q=cache.store.data_ptr(), out=cache.store.data_ptr(), q_stride=576, out_stride=576,
                            tables=cache.store.data_ptr(), lengths=torch.zeros(4, dtype=torch.int32).data_ptr(),
                            workspace=cache.store.data_ptr(), workspace_bytes=1 << 40, type=0, heads=9, table_stride=1,
                            count=1, scale=1.0)
    with pytest.raises(mp.DeviceError) as e:
        mp.kv8_attention_decode(cache.c, args, None, stream())
    assert e.value.code == mp.MP_ERR_INVALID and "current device" in e.value.message


def test_offsets_past_32_bits(built):
    """A cache of over 2^32 bytes whose last blocks are used."""
    blocks, bt = 28000, 16
    cache = Cache(blocks, 3, 64, bt, "e4m3", layers=30, layer=29)
    assert cache.store.numel() > 1 << 32
    tables = torch.tensor([[blocks - 1 - i for i in range(6)]], dtype=torch.int32, device=DEV)
    run = Appender(cache, 9, "f32", 64, "half", 128)
    qkv = values(90, 960, 28)
    store, off, first = qkv.contiguous(), *(torch.tensor(a, dtype=torch.int32, device=DEV) for a in ([0, 90], [0]))
    q_out = torch.zeros(90, 576, device=DEV)
    mp.kv8_append(cache.c, run.args(store, q_out, tables, off, first), run.error.data_ptr(), stream())
    assert mp.kv8_status(run.error.data_ptr(), stream()) == mp.MP_OK
    pos = torch.arange(90, device=DEV)
    k = ref.rotate(qkv[:, 576:768].double().view(90, 3, 64), run.cos[pos].double(), run.sin[pos].double(), 64, "half")
    small = torch.full((6, 3, 2, bt, 64), 0x7F, dtype=torch.int8, device=DEV)
    small_scales = torch.zeros(6, 3, 2, device=DEV)
    ref.append(small, small_scales, "e4m3", k, qkv[:, 768:].double().view(90, 3, 64), [[5, 4, 3, 2, 1, 0]], [0, 90], [0])
    assert torch.equal(cache.pages[blocks - 6:], small) and torch.equal(cache.scales[blocks - 6:], small_scales)
    q, out = decode(cache, 9, tables, [90], "f32")
    check_rows(cache, 9, q, out, tables[0].tolist(), 90, 0.125, False)
    q, out = prefill(cache, 9, tables, [50], [40], "f32")
    check_rows(cache, 9, q, out, tables[0].tolist(), 90, 0.125, False)


@pytest.mark.parametrize("fmt,dtype", [("int8", "f32"), ("e4m3", "bf16")])
def test_a_prompt_and_decode_steps_together(built, fmt, dtype):
    """As a serving loop runs them: two prompts appended and attended to in chunks, then decode steps captured into
    one graph and replayed with advancing positions; every output against the plain attention over the cache, and the
    cache against the plain append."""
    heads, kh, d, bt = 9, 3, 64, 16
    cache = Cache(20, kh, d, bt, fmt)
    tables = tables_for([150, 90], bt, 20, 30)
    run = Appender(cache, heads, dtype, d, "half", 256)
    at = [0, 0]
    for k, counts in enumerate([[100, 33], [21, 40]]):
        x = values(sum(counts), (heads + 2 * kh) * d, 31 + k, 0.3)
        q = run(tables, counts, at, x)
        _, out = prefill(cache, heads, tables, counts, at, dtype, q=q)
        row = 0
        for i in range(2):
            check_rows(cache, heads, q[row: row + counts[i]], out[row: row + counts[i]], tables[i].tolist(),
                       at[i] + counts[i], d ** -0.5, dtype == "bf16")
            row += counts[i]
        at = [a + c for a, c in zip(at, counts)]
    qkv = torch.zeros(2, (heads + 2 * kh) * d, dtype=DTYPES[dtype], device=DEV)
    q_out, out = (torch.zeros(2, heads * d, dtype=DTYPES[dtype], device=DEV) for _ in range(2))
    off = torch.tensor([0, 1, 2], dtype=torch.int32, device=DEV)
    starts = torch.tensor(at, dtype=torch.int32, device=DEV)
    lengths = starts + 1
    workspace = torch.zeros(mp.kv8_decode_workspace(cache.c, heads), dtype=torch.uint8, device=DEV)
    word = torch.zeros(1, dtype=torch.int32, device=DEV)
    append = run.args(qkv, q_out, tables, off, starts)
    attend = mp.Kv8DecodeArgs(q=q_out.data_ptr(), out=out.data_ptr(), q_stride=heads * d, out_stride=heads * d,
                              tables=tables.data_ptr(), lengths=lengths.data_ptr(), workspace=workspace.data_ptr(),
                              workspace_bytes=workspace.numel(), type=list(DTYPES).index(dtype), heads=heads,
                              table_stride=tables.stride(0), count=2, scale=d ** -0.5)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        mp.kv8_append(cache.c, append, word.data_ptr(), stream())
        mp.kv8_attention_decode(cache.c, attend, word.data_ptr(), stream())
    for t in range(20):
        x = values(2, (heads + 2 * kh) * d, 40 + t, 0.3)
        qkv.copy_(x)
        starts.copy_(torch.tensor([a + t for a in at], dtype=torch.int32))
        lengths.copy_(starts + 1)
        pages, scales = cache.store.clone(), cache.scale_store.clone()
        graph.replay()
        assert mp.kv8_status(word.data_ptr(), stream()) == mp.MP_OK
        y = qkv.double()
        c, s = run.cos[starts.long()].double(), run.sin[starts.long()].double()
        k = ref.rotate(y[:, heads * d: (heads + kh) * d].reshape(2, kh, d), c, s, d, "half")
        ref.append(pages[:, 0], scales[:, 0], fmt, k, y[:, (heads + kh) * d:].reshape(2, kh, d), tables.tolist(),
                   [0, 1, 2], [a + t for a in at])
        assert torch.equal(pages, cache.store)
        for i in range(2):
            check_rows(cache, heads, q_out[i: i + 1], out[i: i + 1], tables[i].tolist(), at[i] + t + 1, d ** -0.5,
                       dtype == "bf16")


def test_streams_and_shared_workspaces(built):
    """Two graphs over one workspace, replayed in turn on another stream."""
    lengths = [700, 3, 64]
    cache = Cache(60, 3, 64, 16, "int8")
    tables = tables_for(lengths, 16, 60, 50)
    fill(cache, tables, lengths, 51)
    workspace = torch.zeros(mp.kv8_decode_workspace(cache.c, 9), dtype=torch.uint8, device=DEV)
    runs = []
    for seed in (1, 2):
        q = values(3, 576, 52 + seed)
        out = torch.zeros(3, 576, device=DEV)
        lens = torch.tensor(lengths if seed == 1 else [64, 0, 64], dtype=torch.int32, device=DEV)
        args = mp.Kv8DecodeArgs(q=q.data_ptr(), out=out.data_ptr(), q_stride=576, out_stride=576,
                                tables=tables.data_ptr(), lengths=lens.data_ptr(), workspace=workspace.data_ptr(),
                                workspace_bytes=workspace.numel(), type=0, heads=9, table_stride=tables.stride(0),
                                count=3, scale=0.125)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            mp.kv8_attention_decode(cache.c, args, None, stream())
        runs.append((q, out, lens, graph))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            for _, _, _, graph in runs:
                graph.replay()
    side.synchronize()
    for q, out, lens, _ in runs:
        for i, n in enumerate(lens.tolist()):
            if n:
                check_rows(cache, 9, q[i: i + 1], out[i: i + 1], tables[i].tolist(), n, 0.125, False)
            else:
                assert bool((out[i] == 0).all())


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,dim,counts", [
    (4, 4, 64, [30, 0, 3, 1]), (4, 4, 64, [30, 0, 5]), (5, 1, 128, [100, 45]), (5, 1, 128, [100, 46]),
    (40, 2, 64, [20, 1]), (40, 2, 64, [23])])
def test_prefill_small_calls(built, heads, kv_heads, dim, counts, dtype):
    """Up to 148 items of a row, a kv head and 8 query heads (three of the rows belong to nobody), and one more."""
    starts = [17 * i + (200 if i else 0) for i in range(len(counts))]
    cache = Cache(40, kv_heads, dim, 32, "int8")
    lengths = [s + c for s, c in zip(starts, counts)]
    check_prefill(cache, heads, tables_for(lengths, 32, 40, 61), counts, starts, dtype)


def test_prefill_bad_metadata_in_a_long_call(built):
    """As for a few rows: the bad sequence is reported and left, the others are computed."""
    cache = Cache(30, 3, 64, 16, "int8")
    tables = tables_for([160, 160], 16, 30, 62, spare=0)
    fill(cache, tables, [160, 160], 63)
    word = torch.zeros(1, dtype=torch.int32, device=DEV)
    for rows in (20, 100):
        for start in (161 - rows, -1, 2 ** 31 - 2):
            q, out = prefill(cache, 9, tables, [rows, rows], [160 - rows, start], "f32", error=word)
            assert mp.kv8_status(word.data_ptr(), stream()) == mp.MP_ERR_BOUNDS
            check_rows(cache, 9, q[:rows], out[:rows], tables[0].tolist(), 160, 0.125, False)
            assert bool((out[rows:] == 7).all())


def test_decode_and_prefill_share_a_workspace(built):
    """Calls of both kinds, one after the other, leave a workspace as the next one needs it."""
    cache = Cache(200, 3, 64, 16, "int8")
    tables = tables_for([1500, 900], 16, 200, 64)
    fill(cache, tables, [1500, 900], 65)
    workspace = torch.zeros(max(mp.kv8_decode_workspace(cache.c, 9), mp.kv8_prefill_workspace(cache.c, 9)),
                            dtype=torch.uint8, device=DEV)
    both = dict(tables=tables.data_ptr(), workspace=workspace.data_ptr(), workspace_bytes=workspace.numel(), type=0,
                heads=9, table_stride=tables.stride(0), count=2, scale=0.125, q_stride=576, out_stride=576)
    lens = torch.tensor([1500, 900], dtype=torch.int32, device=DEV)
    word = torch.zeros(1, dtype=torch.int32, device=DEV)
    for rows in (10, 300, 20, 700):
        q, out = values(2 * rows, 576, 66), torch.zeros(2 * rows, 576, device=DEV)
        offsets = torch.tensor([0, rows, 2 * rows], dtype=torch.int32, device=DEV)
        starts = lens - rows
        mp.kv8_attention_prefill(cache.c, mp.Kv8PrefillArgs(q=q.data_ptr(), out=out.data_ptr(), rows=2 * rows,
                                 row_offsets=offsets.data_ptr(), starts=starts.data_ptr(), **both), word.data_ptr(), stream())
        one = torch.zeros(2, 576, device=DEV)
        last = torch.stack([q[rows - 1], q[-1]])
        mp.kv8_attention_decode(cache.c, mp.Kv8DecodeArgs(q=last.data_ptr(), out=one.data_ptr(),
                                lengths=lens.data_ptr(), **both), word.data_ptr(), stream())
        assert mp.kv8_status(word.data_ptr(), stream()) == mp.MP_OK
        for i, n in enumerate((1500, 900)):
            check_rows(cache, 9, q[i * rows: (i + 1) * rows], out[i * rows: (i + 1) * rows], tables[i].tolist(), n, 0.125, False)
            check_rows(cache, 9, last[i: i + 1], one[i: i + 1], tables[i].tolist(), n, 0.125, False)


@pytest.mark.parametrize("scale", [0.0, -0.125])
@pytest.mark.parametrize("rows,dtype", [(4, "f32"), (90, "f32"), (90, "bf16")])
def test_any_factor_of_the_scores(built, rows, dtype, scale):
    """A factor of 0 weighs all tokens alike, a negative one turns the order round; in every kernel."""
    lengths = [333, rows]
    cache = Cache(40, 3, 64, 16, "int8")
    tables = tables_for(lengths, 16, 40, 67)
    fill(cache, tables, lengths, 68)
    q, out = decode(cache, 9, tables, lengths, dtype, scale=scale)
    for i, n in enumerate(lengths):
        check_rows(cache, 9, q[i: i + 1], out[i: i + 1], tables[i].tolist(), n, scale, dtype == "bf16")
    q, out = values(2 * rows, 576, 69).to(DTYPES[dtype]), torch.zeros(2 * rows, 576, dtype=DTYPES[dtype], device=DEV)
    workspace = torch.zeros(mp.kv8_prefill_workspace(cache.c, 9), dtype=torch.uint8, device=DEV)
    offsets = torch.tensor([0, rows, 2 * rows], dtype=torch.int32, device=DEV)
    starts = torch.tensor([333 - rows, 0], dtype=torch.int32, device=DEV)
    mp.kv8_attention_prefill(cache.c, mp.Kv8PrefillArgs(
        q=q.data_ptr(), out=out.data_ptr(), q_stride=576, out_stride=576, tables=tables.data_ptr(),
        row_offsets=offsets.data_ptr(), starts=starts.data_ptr(), workspace=workspace.data_ptr(),
        workspace_bytes=workspace.numel(), type=list(DTYPES).index(dtype), heads=9, table_stride=tables.stride(0),
        count=2, rows=2 * rows, scale=scale), None, stream())
    for i, n in enumerate(lengths):
        part = slice(i * rows, (i + 1) * rows)
        check_rows(cache, 9, q[part], out[part], tables[i].tolist(), n, scale, dtype == "bf16")


def test_prefill_graph_replays_with_other_chunks(built):
    """A captured call follows its metadata buffers: other chunks, other positions, sequences without rows."""
    cache = Cache(300, 3, 64, 16, "e4m3")
    tables = tables_for([1200, 1200, 1200], 16, 300, 70)
    fill(cache, tables, [1200] * 3, 71)
    rows = 600
    q, out = values(rows, 576, 72), torch.zeros(rows, 576, device=DEV)
    workspace = torch.zeros(mp.kv8_prefill_workspace(cache.c, 9), dtype=torch.uint8, device=DEV)
    offsets, starts = torch.zeros(4, dtype=torch.int32, device=DEV), torch.zeros(3, dtype=torch.int32, device=DEV)
    word = torch.zeros(1, dtype=torch.int32, device=DEV)
    args = mp.Kv8PrefillArgs(q=q.data_ptr(), out=out.data_ptr(), q_stride=576, out_stride=576, tables=tables.data_ptr(),
                             row_offsets=offsets.data_ptr(), starts=starts.data_ptr(), workspace=workspace.data_ptr(),
                             workspace_bytes=workspace.numel(), type=0, heads=9, table_stride=tables.stride(0), count=3,
                             rows=rows, scale=0.125)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        mp.kv8_attention_prefill(cache.c, args, word.data_ptr(), stream())
    for counts, first in (([100, 0, 500], [1100, 7, 0]), ([0, 0, 0], [0, 0, 0]), ([1, 1, 1], [0, 1199, 600]),
                          ([0, 600, 0], [0, 600, 0])):
        offsets.copy_(torch.tensor([sum(counts[:i]) for i in range(4)], dtype=torch.int32))
        starts.copy_(torch.tensor(first, dtype=torch.int32))
        out.fill_(7.0)
        graph.replay()
        assert mp.kv8_status(word.data_ptr(), stream()) == mp.MP_OK
        at = 0
        for i, (c, s) in enumerate(zip(counts, first)):
            if c:
                check_rows(cache, 9, q[at: at + c], out[at: at + c], tables[i].tolist(), s + c, 0.125, False)
            at += c
        assert bool((out[at:] == 7).all())
