"""8-bit attention where a single lost, doubled or leaked token, or a half of a product left out, shows at any length.

The general bound of kv8_reference counts every rounding in the worst direction, which at ten thousand tokens is wider
than a token's share. Here the inputs are such that few roundings are left."""
import math

import pytest
import torch

import kv8_reference as ref
from test_gpu_kv8 import DEV, DTYPES, Cache, decode, fill, prefill, tables_for
from tinyinfer_b200 import device as mp

pytestmark = pytest.mark.gpu

DECODES = [[70001], [40000, 3], [9301, 1, 0, 77], [2048 + i for i in range(64)], [1, 30000] + [7] * 40, [333]]
# as tiles; the last one row by row
PREFILLS = [([300], [9001]), ([1900], [0]), ([7, 1, 500], [4000, 0, 1]), ([129, 60], [16000, 127]), ([33], [16000])]
SHAPES = [(9, 3, 64, 16, "int8"), (9, 3, 64, 64, "e4m3"), (8, 1, 128, 16, "e4m3"), (4, 4, 128, 32, "int8")]


def build(heads, kv_heads, dim, bt, fmt, lengths, seed):
    cache = Cache(max(1, sum(-(-n // bt) for n in lengths)), kv_heads, dim, bt, fmt)
    tables = tables_for(lengths, bt, cache.c.max_blocks, seed)
    fill(cache, tables, lengths, seed + 1, (-6, -6))
    return cache, tables


def put(cache, table, part, values):
    """values [tokens, kv heads, dim] (codes' values) as part 0 (K) or 1 (V) of a sequence; the last block's later slots
    stay as they are."""
    n, bt = values.shape[0], cache.bt
    codes = ref.encode(values.double(), cache.fmt)
    token = torch.arange(n, device=DEV)
    blocks = table.long()[token // bt]
    head = torch.arange(cache.kv_heads, device=DEV)
    cache.pages[blocks[:, None], head[None], part, (token % bt)[:, None]] = codes


def whole(n, kv_heads, dim, fmt, g):
    """Positive whole numbers that the format holds."""
    top = 127 if fmt == "int8" else 15
    return torch.randint(1, top + 1, (n, kv_heads, dim), generator=g, device=DEV).double()


def by_head(x, heads, kv_heads):
    return x.repeat_interleave(heads // kv_heads, -2)


@pytest.mark.parametrize("lengths", DECODES, ids=str)
@pytest.mark.parametrize("heads,kv_heads,dim,bt,fmt", SHAPES)
def test_decode_means(built, heads, kv_heads, dim, bt, fmt, lengths):
    """A zero query weighs all tokens alike: the mean of whole numbers. Weights are powers of two (exp2(0) is 1), sums
    stay below 2^24 units and are exact, so what is left is the reciprocal's rounding and the product's (2^-24 each);
    2^-22 allows two more. One token of 70001 changes some dim by more than 2^-18."""
    cache, tables = build(heads, kv_heads, dim, bt, fmt, lengths, 120)
    g = torch.Generator(DEV).manual_seed(121)
    want = torch.zeros(len(lengths), kv_heads, dim, dtype=torch.float64, device=DEV)
    for i, n in enumerate(lengths):
        if n:
            v = whole(n, kv_heads, dim, fmt, g)
            put(cache, tables[i], 1, v)
            want[i] = v.mean(0) * 2.0 ** -6
    _, out = decode(cache, heads, tables, lengths, "f32", q=torch.zeros(len(lengths), heads * dim, device=DEV))
    want = by_head(want, heads, kv_heads)
    assert bool(((out.view(-1, heads, dim).double() - want).abs() <= want * 2.0 ** -22).all())


@pytest.mark.parametrize("counts,starts", PREFILLS, ids=str)
@pytest.mark.parametrize("heads,kv_heads,dim,bt,fmt", SHAPES)
def test_prefill_means(built, heads, kv_heads, dim, bt, fmt, counts, starts):
    """Every row the mean of the tokens up to its own. Weights are 2^(log2 of a block's scale) by the hardware
    approximations, alike for all tokens but not exactly a power of two: halves within 2^-22 on either side, 16 cut
    products a chain of 128 tokens (2^-23 each), and a rounding (2^-24) of sum and normaliser per chain or joined part.
    One token of 16129 changes some dim by more than 2^-15."""
    lengths = [s + c for s, c in zip(starts, counts)]
    cache, tables = build(heads, kv_heads, dim, bt, fmt, lengths, 122)
    g = torch.Generator(DEV).manual_seed(123)
    want = []
    for i, n in enumerate(lengths):
        v = whole(n, kv_heads, dim, fmt, g)
        put(cache, tables[i], 1, v)
        mean = v.cumsum(0) / torch.arange(1, n + 1, device=DEV).double()[:, None, None]
        want.append(mean[starts[i]:] * 2.0 ** -6)
    _, out = prefill(cache, heads, tables, counts, starts, "f32", q=torch.zeros(sum(counts), heads * dim, device=DEV))
    want = by_head(torch.cat(want), heads, kv_heads)
    rel = 2.0 ** -21 + 2.0 ** -19 + (max(lengths) / 128 + 64) * 2.0 ** -23
    assert rel < 2.0 ** -15
    assert bool(((out.view(-1, heads, dim).double() - want).abs() <= want * rel).all())


@pytest.mark.parametrize("n", [100, 1000, 9301, 70001])
@pytest.mark.parametrize("heads,kv_heads,dim,bt,fmt", SHAPES)
def test_low_halves_count(built, heads, kv_heads, dim, bt, fmt, n):
    """Tokens of three weights, 1, just under 2^-1 (1 + 2^-11) and near 2^-9.25, with values in dims of their own: the
    second weight as one FP16 half would be 2^-11 off, the third under an FP16 query 9.25 ln 2 times 2^-12 or so, and
    no average hides it. One product makes a score, so its exponent is off by 2^-22 (the query's halves) and four
    roundings, of 9.25; exp2 2^-22, the weight's halves 2^-22; sums as in the means above."""
    cache, tables = build(heads, kv_heads, dim, bt, fmt, [n], 124)
    g = torch.Generator(DEV).manual_seed(125)
    kind = torch.randint(0, 3, (n,), generator=g, device=DEV)
    kind[: 3] = torch.tensor([0, 1, 2], device=DEV)
    kind[::16] = 0  # the reference score is the largest from the first unit on
    k, v = torch.zeros(n, kv_heads, dim, device=DEV), whole(n, kv_heads, dim, fmt, g)
    k[..., 0] = torch.tensor([0.0, -12.0, -112.0], device=DEV)[kind][:, None]  # held by both formats
    v *= (torch.arange(dim, device=DEV) * 3 // dim == kind[:, None])[:, None]
    put(cache, tables[0], 0, k)
    put(cache, tables[0], 1, v)
    step = -math.log(0.5 * (1 + 2.0 ** -11) * (1 - 2.0 ** -20)) / 12  # of the score, per unit of K
    q = torch.zeros(1, heads, dim, device=DEV)
    q[..., 0] = step * 2.0 ** 6 * dim ** 0.5
    want, weight, _, _ = ref.attend(q, cache.pages, cache.scales, fmt, tables[0].tolist(), n, dim ** -0.5)
    rel = 10 * (2.0 ** -22 + 4 * 2.0 ** -24) + 2 * 2.0 ** -22 + 2.0 ** -19 + (n / 128 + 64) * 2.0 ** -23
    assert rel < 2.0 ** -13
    rows = 1 if n < 300 else 150  # row by row, and as tiles
    outs = [decode(cache, heads, tables, [n], "f32", q=q.flatten(1))[1]]
    if n < 20000:
        outs.append(prefill(cache, heads, tables.repeat(rows, 1).contiguous(), [1] * rows, [n - 1] * rows, "f32",
                            q=q.flatten(1).repeat(rows, 1))[1])
    for out in outs:
        assert bool(((out.view(-1, heads, dim).double() - want).abs() <= weight * rel).all())


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,dim,bt,fmt", SHAPES)
def test_marked_tokens(built, heads, kv_heads, dim, bt, fmt, dtype):
    """All weight on marked tokens: 256 at random, and each of the last rows'. An output is the mean of the marked ones
    it may see; one more or less moves some dim by several times what the roundings allow. Slots behind the last
    token are marked, too."""
    n, rows = 9301, 300
    cache, tables = build(heads, kv_heads, dim, bt, fmt, [n], 126)
    g = torch.Generator(DEV).manual_seed(127)
    room = -(-n // bt) * bt
    marked = torch.zeros(room, dtype=torch.bool, device=DEV)
    marked[torch.randperm(n, generator=g, device=DEV)[:256]] = True
    marked[0] = marked[n - rows - 3:] = True
    k = torch.zeros(room, kv_heads, dim, device=DEV)
    k[..., 0] = marked.double()[:, None].float() * 120
    v = whole(room, kv_heads, dim, fmt, g) * torch.where(torch.rand(room, kv_heads, dim, generator=g, device=DEV) < 0.5, -1, 1)
    put(cache, tables[0], 0, k)
    put(cache, tables[0], 1, v)
    q = torch.zeros(rows, heads, dim, device=DEV)
    q[..., 0] = 24 / (120 * 2.0 ** -6 * dim ** -0.5)  # 24 for marked tokens, else 0: e^24 to 1
    want, weight, _, _ = ref.attend(q.to(DTYPES[dtype]), cache.pages, cache.scales, fmt, tables[0].tolist(), n, dim ** -0.5)
    # all marked weights are alike, as are the others: an FP16 half's step (2^-11, BF16 calls; 2^-22), cut products
    # and added chains as above, and the result's rounding
    bf16 = dtype == "bf16"
    limit = weight * ((2.0 ** -11 if bf16 else 2.0 ** -22) + 2.0 ** -19 + 2 * 24 * 2.0 ** -21 + (n / 128 + 64) * 2.0 ** -23)
    if bf16:
        limit = limit + want.abs() * 2.0 ** -8
    _, out = prefill(cache, heads, tables, [rows], [n - rows], dtype, q=q.flatten(1))
    assert bool(((out.view(rows, heads, dim).double() - want).abs() <= limit).all())
    lengths = [n - i for i in (0, 1, 7, 31, 32, 33, 127, 200)]
    _, out = decode(cache, heads, tables.repeat(len(lengths), 1).contiguous(), lengths, dtype,
                    q=q[: len(lengths)].flatten(1))
    at = [rows - 1 - (n - m) for m in lengths]
    assert bool(((out.view(-1, heads, dim).double() - want[at]).abs() <= limit[at]).all())
