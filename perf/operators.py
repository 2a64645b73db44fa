"""Cases of the 8-bit paged K/V cache operators: rotate-and-append, single-token
(decode) attention and prompt (prefill) attention over the cache.

A cache block holds `block_tokens` tokens of every K/V head as 8-bit codes,
[block][kv head][0 = K, 1 = V][slot][dim], with one power-of-two scale per
(block, kv head, K or V): value = code * scale. `run` returns codes and scales side
by side (E4M3 codes as the float8 values they are): the scales are exact powers of
two, so equal codes and equal scales are equal values, and untouched pages are
compared too. `run` computes an operator with elementary torch operations, or,
with `own`, calls this package's kernels on the same buffers.
"""
import math

import torch

own = False

DEV = "cuda:0"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
# the largest code of each format, and the exponent bias of the smallest scale that holds a
# magnitude m * 2^e (m in [0.5, 1)): 127 = 0.9921875 * 2^7, 448 = 0.875 * 2^9
LIMITS = {"int8": (127.0, 0.9921875, 7), "e4m3": (448.0, 0.875, 9)}
MIN_EXPONENT = -100


def _case(name, op, seqs, low, high, *, ctx_low=0, ctx_high=0, heads=9, kv_heads=3, dim=64, block=16, type="f32",
          format="int8", rope="half", rotary=None, shared=0, pad=0):
    """`seqs` sequences. append / prefill: low..high new rows each, at a start position in ctx_low..ctx_high;
    decode: contexts of low..high tokens, the first `shared` of them on the same pages. `pad`: rows of the
    batch behind the last sequence."""
    return {"name": name, "op": op, "seqs": seqs, "low": low, "high": high, "ctx_low": ctx_low, "ctx_high": ctx_high,
            "heads": heads, "kv_heads": kv_heads, "dim": dim, "block": block, "type": type, "format": format,
            "rope": rope, "rotary": dim if rotary is None else rotary, "shared": shared, "pad": pad}


def listed():
    return [
        # one decode step of a handful of requests: latency
        _case("append 5 x 1", "append", 5, 1, 1, ctx_low=3, ctx_high=900),
        # the decode step of a full batch at the 135M model's widths, 2K contexts
        _case("append 256 x 1", "append", 256, 1, 1, ctx_low=2048, ctx_high=2112),
        # one step of chunked prefill: 16 requests x 512 tokens
        _case("append 16 x 512", "append", 16, 512, 512, ctx_low=0, ctx_high=3584),
        # a batch of whole prompts of very different lengths on a wider model, in bf16; batch padded
        _case("append ragged bf16", "append", 23, 1, 1777, ctx_low=0, ctx_high=50, heads=32, kv_heads=8, dim=128,
              block=32, type="bf16", format="e4m3", rope="interleaved", rotary=64, pad=13),
        # one request alone: latency
        _case("decode 1 x 333", "decode", 1, 333, 333),
        # 64 requests at any point of a 4K context, empty rows among them
        _case("decode 64 x 0..4096", "decode", 64, 0, 4096),
        # 256 requests of 2K tokens sharing a 1K system prompt
        _case("decode 256 x 2048 shared", "decode", 256, 2048, 2112, shared=1024),
        # a wider model in bf16 on an E4M3 cache, up to 8K tokens
        _case("decode 96 x 1..8192 bf16", "decode", 96, 1, 8192, heads=32, kv_heads=8, dim=128, type="bf16",
              format="e4m3"),
        # one short prompt: latency
        _case("prefill 1 x 37", "prefill", 1, 37, 37),
        # the last chunk of 16 requests of 4K tokens
        _case("prefill 16 x 512 at 3584", "prefill", 16, 512, 512, ctx_low=3584, ctx_high=3584),
        # whole prompts of different lengths packed in one call, in bf16 on an E4M3 cache
        _case("prefill ragged bf16", "prefill", 11, 0, 1501, heads=32, kv_heads=8, dim=128, type="bf16",
              format="e4m3", pad=5),
        # one long document, chunk by chunk: few rows over a long context
        _case("prefill 1 x 500 at 16001", "prefill", 1, 500, 500, ctx_low=16001, ctx_high=16001),
    ]


GEOMETRIES = [(9, 3, 64), (9, 3, 64), (32, 8, 128), (8, 8, 64), (16, 2, 128), (14, 2, 64), (4, 1, 128)]


def draw(rng):
    def log_int(low, high):
        return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))

    op = rng.choice(["append", "decode", "prefill"])
    heads, kv_heads, dim = rng.choice(GEOMETRIES)
    width = heads * dim / 576.0
    kw = {"heads": heads, "kv_heads": kv_heads, "dim": dim, "block": rng.choice([16, 16, 16, 32, 64]),
          "type": rng.choice(["f32", "bf16"]), "format": rng.choice(["int8", "e4m3"]),
          "rope": rng.choice(["half", "interleaved"]), "rotary": rng.choice([dim, dim, dim // 2, 24, 0])}
    if op == "append":
        rows = log_int(1, 20000 / width)
        seqs = max(1, min(rows, log_int(1, 512)))
        mean = max(1, rows // seqs)
        low, high = rng.choice([(mean, mean), (max(1, mean // 4), 2 * mean - mean // 4)])
        c = _case("", op, seqs, low, high, ctx_low=0, ctx_high=log_int(1, 8192), pad=rng.choice([0, 0, 7]), **kw)
    elif op == "decode":
        tokens = log_int(64, 256 * 2048 * 192 / (kv_heads * dim))
        seqs = max(1, min(log_int(1, 512), tokens // 8))
        mean = min(tokens // seqs, 40000)
        low, high = rng.choice([(mean, mean), (mean // 2, mean + mean // 2), (0, 2 * mean)])
        shared = rng.choice([0, 0, low // 2])
        c = _case("", op, seqs, low, high, shared=shared, **kw)
    else:
        rows = log_int(1, 4000 / width)
        seqs = max(1, min(rows // 16, log_int(1, 24)))
        mean = max(1, rows // seqs)
        low, high = rng.choice([(mean, mean), (0, 2 * mean)])
        context = max(0, min(log_int(1, 16000), int(1.7e10 / (heads * dim * seqs * max(1, high))) - high))
        c = _case("", op, seqs, low, high, ctx_low=context // 2, ctx_high=context, pad=rng.choice([0, 0, 3]), **kw)
    del c["name"]
    return c


def _layout(case):
    """Starts and row (or token) counts of the case's sequences: part of the case, the same for every seed."""
    g = torch.Generator().manual_seed(1000003 * case["seqs"] + 31 * case["low"] + case["high"])
    n = case["seqs"]
    counts = torch.randint(case["low"], case["high"] + 1, (n,), generator=g)
    starts = torch.randint(case["ctx_low"], case["ctx_high"] + 1, (n,), generator=g)
    if n > 1 and case["high"] > case["low"]:
        counts[0], counts[-1] = case["high"], case["low"]  # both ends of the range occur
    if case["op"] == "decode":
        starts = torch.zeros_like(starts)
    if int(counts.sum()) == 0:
        counts[0] = 1
    return starts, counts


def work(case):
    starts, counts = _layout(case)
    h, kh, d = case["heads"], case["kv_heads"], case["dim"]
    size = 4 if case["type"] == "f32" else 2
    rows, scale_bytes = int(counts.sum()), 8 * kh / case["block"]
    if case["op"] == "append":
        # q, k, v in; q out; codes out; cosines and sines of every position once; a scale pair per block and head
        positions = int((starts + counts).max()) - int(starts.min())
        positions = min(rows, positions)
        return {"bytes": rows * d * (2 * h * size + 2 * kh * size + 2 * kh) + rows * scale_bytes
                + 4 * positions * case["rotary"], "flops": 3.0 * rows * (h + kh) * case["rotary"] + 2.0 * rows * kh * d}
    tokens = int((starts + counts)[counts > 0].sum())
    if case["op"] == "decode":
        tokens -= int((counts >= case["shared"]).sum() - 1) * (case["shared"] // case["block"] * case["block"])
        return {"bytes": tokens * (2 * kh * d + scale_bytes) + 2 * len(counts) * h * d * size,
                "flops": 4.0 * d * h * int(counts.sum())}
    pairs = int((counts * starts + counts * (counts + 1) // 2).sum())
    return {"bytes": tokens * (2 * kh * d + scale_bytes) + 2 * rows * h * d * size, "flops": 4.0 * d * h * pairs}


def _power(exponent):
    """2^exponent in 32 bits, exactly (exponents of normal numbers)."""
    return ((exponent.to(torch.int32) + 127) << 23).view(torch.float32)


def _exponent(amax, format):
    """The exponent x of the smallest power of two with amax <= limit * 2^x."""
    _, mantissa, bias = LIMITS[format]
    m, e = torch.frexp(amax)
    x = e - bias + (m > mantissa).to(e.dtype)
    return torch.where(amax > 0, x, torch.full_like(x, MIN_EXPONENT)).clamp(min=MIN_EXPONENT)


def _round(x, format):
    """x (in units of the scale) as the nearest code's value, ties to even."""
    limit = LIMITS[format][0]
    if format == "int8":
        return torch.round(x).clamp(-limit, limit)
    e = torch.frexp(x.abs())[1] - 1  # 2^e <= |x|
    step = _power(e.clamp(-6, 100) - 3).to(x.dtype)
    return (torch.round(x / step) * step).clamp(-limit, limit)


def _codes(values, format):
    """Code values as bytes."""
    if format == "int8":
        return values.to(torch.int8)
    return values.to(torch.float32).to(torch.float8_e4m3fn).view(torch.int8)


def _values(codes, format):
    return codes.float() if format == "int8" else codes.view(torch.float8_e4m3fn).float()


def prepare(case, seed):
    g = torch.Generator(DEV).manual_seed(int(seed))

    def randn(*shape):
        return torch.randn(*shape, generator=g, device=DEV)

    h, kh, d, bt, format, type = (case[k] for k in ("heads", "kv_heads", "dim", "block", "format", "type"))
    starts, counts = _layout(case)
    lengths = starts + counts
    n, rows = len(counts), int(counts.sum())
    # block tables: a random permutation of a pool with a few blocks to spare; a shared
    # prefix is the same physical blocks in every table that reaches past it
    pages = (lengths + bt - 1) // bt
    width = max(1, int(pages.max()))
    shared = case["shared"] // bt
    need = pages - torch.where(lengths >= case["shared"], shared, 0)
    if case["op"] == "append":  # earlier pages are not touched: any blocks will do
        need = pages - starts // bt
    blocks = int(need.sum()) + shared + 3
    perm = torch.randperm(blocks, generator=g, device=DEV, dtype=torch.int32)
    column = torch.arange(width)
    first = torch.cumsum(need, 0) - need + shared
    own_index = first[:, None] + column[None] - (pages - need)[:, None]
    common = column[None] if shared else blocks - 3 + column[None] % 3
    index = torch.where(column[None] < (pages - need)[:, None], common, own_index)
    used = column[None] < pages[:, None]
    tables = torch.where(used.to(DEV), perm[index.clamp(0, blocks - 1).to(DEV)], torch.tensor(-1, dtype=torch.int32, device=DEV)).contiguous()
    # the cache as earlier appends left it: per-channel gains, a few loud channels
    gain = 0.5 + torch.rand(kh, 2, 1, d, generator=g, device=DEV)
    gain[:, 0, :, :: 17] *= 6.0
    content = randn(blocks, kh, 2, bt, d).mul_(gain)
    scales = _power(_exponent(content.abs().amax((-1, -2)), format))
    cache = _codes(_round(content / scales[..., None, None], format), format)
    del content
    # slots that hold no token keep whatever bytes were there, NaN codes among them; blocks no table names, too
    filled = torch.zeros(blocks, dtype=torch.int64, device=DEV)
    held = starts if case["op"] == "append" else lengths  # append: the new rows' slots are not filled yet
    fill = (held[:, None] - column[None] * bt).clamp(0, bt).to(DEV)
    filled.scatter_reduce_(0, tables.clamp(min=0).long().flatten(), torch.where(tables >= 0, fill, 0).flatten(), "amax")
    stale = torch.arange(bt, device=DEV)[None] >= filled[:, None]
    cache = torch.where(stale[:, None, None, :, None], torch.tensor(0x7F, dtype=torch.int8, device=DEV), cache)
    scales = torch.where((filled > 0)[:, None, None], scales, torch.tensor(float("nan"), device=DEV))
    scales = torch.nan_to_num(scales, nan=3.0) if case["op"] == "append" else scales
    state = {"case": case, "cache": cache.contiguous(), "scales": scales.contiguous(), "tables": tables,
             "scale": d ** -0.5}
    total = n if case["op"] == "decode" else rows + case["pad"]
    state["q"] = randn(total, h * d).mul_(1.5).to(TYPES[type])
    state["out"] = torch.full((total, h * d), 7.0, dtype=TYPES[type], device=DEV)
    if case["op"] == "decode":
        state["lengths"] = lengths.to(torch.int32).to(DEV)
        return state
    state["offsets"] = torch.cat([torch.zeros(1, dtype=torch.int64), torch.cumsum(counts, 0)]).to(torch.int32).to(DEV)
    state["starts"] = starts.to(torch.int32).to(DEV)
    state["rows"], state["longest"] = rows, int(counts.max())
    if case["op"] == "append":
        # one fused projection output: q | k | v columns of each row
        kv = randn(total, 2, kh, d).mul_(gain.squeeze(2).transpose(0, 1)) * torch.exp(0.5 * randn(total, 1, 1, 1))
        state["qkv"] = torch.cat([state.pop("q"), kv.reshape(total, -1).to(TYPES[type])], 1).contiguous()
        half, top = case["rotary"] // 2, int(lengths.max())
        angle = torch.arange(top, device=DEV, dtype=torch.float64)[:, None] * 10000.0 ** (
            -torch.arange(half, device=DEV, dtype=torch.float64) / max(1, half))
        state["cos"], state["sin"] = angle.cos().float().contiguous(), angle.sin().float().contiguous()
    return state


# ---------------------------------------------------------------- the plain forms

def _rotate(x, cos, sin, rotary, layout):
    """x [rows, heads, dim] in 64 bits, cos / sin [rows, rotary / 2]: the first `rotary` dims rotated in pairs."""
    half = rotary // 2
    turn, rest = x[..., :rotary], x[..., rotary:]
    c, s = cos[:, None], sin[:, None]
    if layout == "half":
        a, b = turn[..., :half], turn[..., half:]
        return torch.cat([a * c - b * s, b * c + a * s, rest], -1)
    a, b = turn[..., 0::2], turn[..., 1::2]
    return torch.cat([torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2), rest], -1)


def _plain_append(s):
    case, cache, scales = s["case"], s["cache"], s["scales"]
    h, kh, d, bt, format = (case[k] for k in ("heads", "kv_heads", "dim", "block", "format"))
    rows = s["rows"]
    row = torch.arange(rows, device=DEV)
    seq = torch.searchsorted(s["offsets"][1:].contiguous(), row.to(torch.int32), right=True)
    position = (s["starts"][seq] + row - s["offsets"][seq]).long()
    touched, block = torch.unique(s["tables"][seq, position // bt].long(), return_inverse=True)
    slot, blocks = position % bt, touched.numel()
    q, k, v = s["qkv"][:rows].double().split([h * d, kh * d, kh * d], 1)  # 64 bits: values next to a rounding border
    cos, sin = s["cos"][position].double(), s["sin"][position].double()
    s["out"][:rows] = _rotate(q.view(rows, h, d), cos, sin, case["rotary"], case["rope"]).reshape(rows, -1).to(s["out"].dtype)
    new = torch.stack([_rotate(k.view(rows, kh, d), cos, sin, case["rotary"], case["rope"]), v.view(rows, kh, d)], 2)
    # of each touched block: its largest new magnitude, first new slot, and the scale before (none where it is begun here)
    amax = torch.zeros(blocks, kh, 2, device=DEV)
    amax.scatter_reduce_(0, block[:, None, None].expand(rows, kh, 2), new.float().abs().amax(-1), "amax")
    begin = torch.full((blocks,), bt, device=DEV).scatter_reduce_(0, block, slot, "amin")
    need, held = _power(_exponent(amax, format)), scales[touched]
    fresh = torch.where((begin > 0)[:, None, None], torch.maximum(held, need), need)
    before = (torch.arange(bt, device=DEV)[None] < begin[:, None])[:, None, None, :, None]
    bytes_ = cache[touched]
    old = torch.where(before, _values(bytes_, format) * (held / fresh)[..., None, None], 0.0)
    bytes_ = torch.where(before, _codes(_round(old, format), format), bytes_)
    head, part = torch.arange(kh, device=DEV)[None, :, None], torch.arange(2, device=DEV)[None, None, :]
    bytes_[block[:, None, None], head, part, slot[:, None, None]] = _codes(
        _round(new / fresh[block].double()[..., None], format), format)
    cache[touched] = bytes_
    scales[touched] = fresh
    return s


def _gathered(s, width_type):
    """Keys and values of every sequence, [seqs, kv heads, tokens, dim]."""
    case, tables = s["case"], s["tables"].clamp(min=0).long()
    kv = _values(s["cache"][tables], case["format"]).to(width_type) * s["scales"][tables].to(width_type)[..., None, None]
    kv = kv.permute(3, 0, 2, 1, 4, 5).flatten(3, 4)
    return kv[0], kv[1]


def _attend(q, keys, values, visible, scale):
    """q [seqs, kv heads, queries, dim]; visible [seqs, 1, queries or 1, tokens]."""
    reach = visible.any(2, keepdim=True).transpose(2, 3)  # tokens that no query sees may hold anything
    scores = q @ torch.where(reach, keys, 0.0).transpose(2, 3)
    scores = torch.where(visible, scores * scale, -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    return (p @ torch.where(reach, values, 0.0)) / torch.where(total == 0, 1.0, total)


def _plain_attention(s, width_type):
    case = s["case"]
    h, kh, d = case["heads"], case["kv_heads"], case["dim"]
    keys, values = _gathered(s, width_type)
    token = torch.arange(keys.shape[2], device=DEV)
    if case["op"] == "decode":
        n = s["q"].shape[0]
        visible = (token[None] < s["lengths"][:, None])[:, None, None]
        return _attend(s["q"].to(width_type).view(n, kh, h // kh, d), keys, values, visible, s["scale"]).reshape(n, h * d)
    n, longest, rows = len(s["starts"]), s["longest"], s["rows"]
    step = torch.arange(longest, device=DEV)
    row = s["offsets"][:-1, None] + step[None]
    live = row < s["offsets"][1:, None]
    q = s["q"][torch.where(live, row, 0).long()].to(width_type).view(n, longest, kh, h // kh, d)
    q = q.permute(0, 2, 3, 1, 4).reshape(n, kh, -1, d)
    visible = (token <= s["starts"][:, None, None] + step[None, :, None]) & live[..., None]
    out = _attend(q, keys, values, visible.repeat(1, h // kh, 1)[:, None], s["scale"])
    out = out.view(n, kh, h // kh, longest, d).permute(0, 3, 1, 2, 4).reshape(n, longest, h * d)
    return out[live]


# ---------------------------------------------------------------- this package's kernels

def _call(s):
    """The argument block a serving loop keeps for its fixed buffers."""
    from tinyinfer_b200 import device as mp

    case = s["case"]
    blocks, kh, _, bt, d = s["cache"].shape
    cache = mp.Kv8Cache(pages=s["cache"].data_ptr(), scales=s["scales"].data_ptr(),
                        page_stride=s["cache"].stride(0), scale_stride=s["scales"].stride(0),
                        format=mp.MP_KV8_INT8 if case["format"] == "int8" else mp.MP_KV8_E4M3, kv_heads=kh,
                        head_dim=d, block_tokens=bt, max_blocks=blocks)
    s["error"] = torch.zeros(1, dtype=torch.int32, device=DEV)
    common = {"tables": s["tables"].data_ptr(), "table_stride": s["tables"].shape[1],
              "type": mp.MP_TYPE_F32 if case["type"] == "f32" else mp.MP_TYPE_BF16, "heads": case["heads"],
              "count": s["tables"].shape[0]}
    if case["op"] == "append":
        qkv, size, stride = s["qkv"].data_ptr(), s["qkv"].element_size(), s["qkv"].shape[1]
        args = mp.Kv8AppendArgs(q=qkv, k=qkv + case["heads"] * d * size, v=qkv + (case["heads"] + kh) * d * size,
                                q_out=s["out"].data_ptr(), q_stride=stride, k_stride=stride, v_stride=stride,
                                q_out_stride=s["out"].shape[1], cos=s["cos"].data_ptr(), sin=s["sin"].data_ptr(),
                                rotary_dim=case["rotary"], max_positions=s["cos"].shape[0],
                                rope_layout=mp.MP_ROPE_HALF if case["rope"] == "half" else mp.MP_ROPE_INTERLEAVED,
                                row_offsets=s["offsets"].data_ptr(), starts=s["starts"].data_ptr(),
                                rows=s["qkv"].shape[0], **common)
        call = mp.kv8_append
    else:
        common.update(q=s["q"].data_ptr(), out=s["out"].data_ptr(), q_stride=s["q"].shape[1],
                      out_stride=s["out"].shape[1], scale=s["scale"])
        if case["op"] == "decode":
            size = mp.kv8_decode_workspace(cache, case["heads"])
        else:
            size = mp.kv8_prefill_workspace(cache, case["heads"])
        s["workspace"] = torch.zeros(size, dtype=torch.uint8, device=DEV)
        common.update(workspace=s["workspace"].data_ptr(), workspace_bytes=size)
        if case["op"] == "decode":
            args, call = mp.Kv8DecodeArgs(lengths=s["lengths"].data_ptr(), **common), mp.kv8_attention_decode
        else:
            args = mp.Kv8PrefillArgs(row_offsets=s["offsets"].data_ptr(), starts=s["starts"].data_ptr(),
                                     rows=s["q"].shape[0], **common)
            call = mp.kv8_attention_prefill
    return call, cache, args, s["error"].data_ptr()


def run(state):
    case = state["case"]
    if own:
        if "call" not in state:
            state["call"] = _call(state)
        call, cache, args, error = state["call"]
        call(cache, args, error, torch.cuda.current_stream().cuda_stream)
    elif case["op"] == "append":
        _plain_append(state)
    else:
        out = _plain_attention(state, torch.float32)
        state["out"][: out.shape[0]] = out.to(state["out"].dtype)
    if case["op"] != "append":
        return {"out": state["out"]}
    codes = state["cache"] if case["format"] == "int8" else state["cache"].view(torch.float8_e4m3fn)
    return {"q": state["out"], "codes": codes, "scales": state["scales"]}


# ---------------------------------------------------------------- the definition in 64 bits

def _exact_append(case, s):
    """Sequence by sequence and block by block."""
    h, kh, d, bt = (case[k] for k in ("heads", "kv_heads", "dim", "block"))
    limit = LIMITS[case["format"]][0]
    cache, scales = _values(s["cache"], case["format"]).double(), s["scales"].double()
    out = s["out"].double()
    starts, offsets, tables = s["starts"].tolist(), s["offsets"].tolist(), s["tables"].tolist()
    half, grid = case["rotary"] // 2, None
    if case["format"] == "e4m3":  # every magnitude the format has, and the borders between neighbours
        grid = torch.arange(0, 127, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn).double()
        border = (grid[1:] + grid[:-1]) / 2

    def nearest(x):
        if grid is None:
            return x.round().clamp(-127, 127)
        up = torch.searchsorted(border, x.abs().contiguous(), right=False)
        tie = (up < border.numel()) & (x.abs() == border[up.clamp(max=border.numel() - 1)]) & (up % 2 == 1)
        return torch.where(x < 0, -1.0, 1.0) * grid[up + tie.long()]

    def turned(x, pos):
        a = torch.arange(half, device=DEV)
        i, j = (a, a + half) if case["rope"] == "half" else (2 * a, 2 * a + 1)
        y, z = x.clone(), torch.complex(s["cos"][pos].double(), s["sin"][pos].double())[:, None]
        w = torch.complex(x[..., i], x[..., j]) * z
        y[..., i], y[..., j] = w.real, w.imag
        return y

    for n, start in enumerate(starts):
        lo, hi = offsets[n], offsets[n + 1]
        pos = torch.arange(start, start + hi - lo, device=DEV)
        x = s["qkv"][lo:hi].double()
        out[lo:hi] = turned(x[:, : h * d].view(-1, h, d), pos).flatten(1)
        k = turned(x[:, h * d: (h + kh) * d].view(-1, kh, d), pos)
        v = x[:, (h + kh) * d:].view(-1, kh, d)
        at = lo
        while at < hi:
            p = start + at - lo
            slot, block = p % bt, tables[n][p // bt]
            take = min(bt - slot, hi - at)
            for part, y in ((0, k), (1, v)):
                y = y[at - lo: at - lo + take].transpose(0, 1)  # [kv heads, tokens, dim]
                top = y.abs().amax((1, 2)).float().double()
                need = torch.exp2(torch.ceil(torch.log2(top / limit)))
                need = torch.where(top > need * limit, need * 2, torch.where(top <= need / 2 * limit, need / 2, need))
                need = need.clamp(min=2.0 ** MIN_EXPONENT)
                held = scales[block, :, part]
                scale = torch.maximum(held, need) if slot else need
                if slot:
                    cache[block, :, part, :slot] = nearest(cache[block, :, part, :slot] * (held / scale)[:, None, None])
                cache[block, :, part, slot: slot + take] = nearest(y / scale[:, None, None])
                scales[block, :, part] = scale
            at += take
    codes = cache.to(torch.int8) if case["format"] == "int8" else cache
    return {"q": out, "codes": codes, "scales": scales}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "append":
        blocks = int(s["rows"]) // case["block"] + 2 * len(s["starts"])
        return _exact_append(case, s) if blocks < 3000 else None
    # sequence by sequence, a slice of queries at a time, one K/V head after the other
    h, kh, d, bt = (case[k] for k in ("heads", "kv_heads", "dim", "block"))
    out = s["out"].double()
    tables, per = s["tables"].long(), h // kh
    if case["op"] == "decode":
        spans = [(i, i, 1, length - 1) for i, length in enumerate(s["lengths"].tolist())]
    else:
        offsets = s["offsets"].tolist()
        spans = [(i, offsets[i], offsets[i + 1] - offsets[i], start) for i, start in enumerate(s["starts"].tolist())]
    for i, row, count, start in spans:
        length = start + count
        if case["op"] == "decode" and length == 0:
            out[row] = 0.0
        if count == 0 or length == 0:
            continue
        blocks = tables[i, : (length + bt - 1) // bt]
        kv = _values(s["cache"][blocks], case["format"]).double() * s["scales"][blocks].double()[..., None, None]
        kv = kv.permute(1, 2, 0, 3, 4).reshape(kh, 2, -1, d)[:, :, :length]
        token = torch.arange(length, device=DEV)
        for at in range(0, count, 512):
            take = min(512, count - at)
            q = s["q"][row + at: row + at + take].double().view(take, kh, per, d)
            hidden = token[None] > (start + at + torch.arange(take, device=DEV))[:, None]
            for head in range(kh):
                scores = torch.einsum("tgd,ld->gtl", q[:, head], kv[head, 0]) * s["scale"]
                weights = torch.softmax(scores.masked_fill(hidden, -math.inf), -1)
                y = torch.einsum("gtl,ld->tgd", weights, kv[head, 1])
                out[row + at: row + at + take].view(take, kh, per, d)[:, head] = y
    return {"out": out}
