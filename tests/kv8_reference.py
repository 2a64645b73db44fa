"""Plain 64-bit forms of the 8-bit cache operators, for the tests (torch, any device)."""
import torch

LIMIT = {"int8": 127.0, "e4m3": 448.0}


def e4m3_grid():
    """The non-negative values of E4M3, in code order (0x00 .. 0x7E)."""
    return torch.arange(0, 127, dtype=torch.uint8).view(torch.float8_e4m3fn).double()


def decode_codes(codes, fmt):
    """int8 storage -> values of the codes, 64 bits."""
    return codes.double() if fmt == "int8" else codes.view(torch.float8_e4m3fn).double()


def nearest(x, fmt):
    """x (64 bits, in units of the scale) -> the nearest code's value, ties to even, saturating."""
    if fmt == "int8":
        return x.round().clamp(-127, 127)
    grid = e4m3_grid().to(x.device)
    border = (grid[1:] + grid[:-1]) / 2
    a = x.abs().contiguous()
    up = torch.searchsorted(border, a)
    tie = (up < border.numel()) & (a == border[up.clamp(max=border.numel() - 1)]) & (up % 2 == 1)
    return torch.copysign(grid[up + tie.long()], x)  # a zero keeps its sign


def encode(values, fmt):
    """Code values -> int8 storage."""
    if fmt == "int8":
        return values.to(torch.int8)
    return values.float().to(torch.float8_e4m3fn).view(torch.int8)


def scale_for(amax, fmt):
    """Smallest power of two (at least 2^-100) with amax <= limit * scale; amax rounded to 32 bits."""
    import math

    amax = float(torch.tensor(amax, dtype=torch.float64).float())
    if amax == 0:
        return 2.0 ** -100
    x = math.frexp(amax / LIMIT[fmt])[1] - 2
    while amax > LIMIT[fmt] * 2.0 ** x:
        x += 1
    return 2.0 ** max(x, -100)


def rotate(x, cos, sin, rotary, layout):
    """x [rows, heads, dim] and cos / sin [rows, rotary / 2], 64 bits."""
    y, half = x.clone(), rotary // 2
    i = torch.arange(half, device=x.device)
    a, b = (i, i + half) if layout == "half" else (2 * i, 2 * i + 1)
    c, s = cos[:, None], sin[:, None]
    y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., b] * c + x[..., a] * s
    return y


def rotation_bound(x, rotated, cos, sin, rotary, layout, bf16):
    """How far an FP32 rotation a c - (b s) may be from the 64-bit one: half a step (2^-24) of the rounded product b s,
    and half a step of the sum, which is as large as the result plus the first error; BF16 outputs are rounded once
    more (half a step: 2^-8 of the value)."""
    products = rotate(x.abs(), torch.zeros_like(cos), sin.abs(), rotary, layout).abs()  # |b s| in a's place, |a s| in b's
    products[..., rotary:] = 0
    exact = products * 2 ** -24 + rotated.abs() * 2 ** -24 * (1 + 2 ** -20)
    exact[..., rotary:] = 0
    return exact + products * 2 ** -46 + (rotated.abs() + exact) * 2 ** -8 * (1 if bf16 else 0) + 1e-44


def append(pages, scales, fmt, k, v, tables, offsets, starts):
    """pages [blocks, kv heads, 2, slots, dim] int8 and scales, in place; k (rotated) and v [rows, kv heads, dim]
    in 64 bits, finite."""
    bt = pages.shape[3]
    for n, start in enumerate(starts):
        at, hi = offsets[n], offsets[n + 1]
        while at < hi:
            p = start + at - offsets[n]
            slot, block = p % bt, tables[n][p // bt]
            take = min(bt - slot, hi - at)
            for head in range(pages.shape[1]):
                for part, x in ((0, k), (1, v)):
                    new = x[at: at + take, head]
                    scale, tile = scale_for(float(new.abs().max()), fmt), pages[block, head, part]
                    if slot:
                        held = float(scales[block, head, part])
                        scale = max(scale, held)
                        tile[:slot] = encode(nearest(decode_codes(tile[:slot], fmt) * (held / scale), fmt), fmt)
                    tile[slot: slot + take] = encode(nearest(new / scale, fmt), fmt)
                    scales[block, head, part] = scale
            at += take


def attend(q, pages, scales, fmt, table, length, scale):
    """q [rows, heads, dim] at the last `rows` positions of a sequence of `length` tokens: outputs, and for the
    error bounds sum p |v|, the largest scale * sum |q k|, and the largest p * block scale * largest code."""
    rows, heads, dim = q.shape
    kh, bt = pages.shape[1], pages.shape[3]
    blocks = torch.as_tensor(table[: -(-length // bt)], device=pages.device, dtype=torch.long)
    kv = decode_codes(pages[blocks], fmt) * scales[blocks].double()[..., None, None]
    kv = kv.permute(2, 1, 0, 3, 4).flatten(2, 3)[:, :, :length]  # [2, kv heads, tokens, dim]
    g = q.double().view(rows, kh, heads // kh, dim)
    s = torch.einsum("rhgd,hld->rhgl", g, kv[0]) * scale
    size = torch.einsum("rhgd,hld->rhgl", g.abs(), kv[0].abs()) * abs(scale)
    hidden = torch.arange(length, device=q.device)[None] > (length - rows + torch.arange(rows, device=q.device))[:, None]
    p = torch.softmax(s.masked_fill(hidden[:, None, None], -float("inf")), -1)
    out = torch.einsum("rhgl,hld->rhgd", p, kv[1])
    weight = torch.einsum("rhgl,hld->rhgd", p, kv[1].abs())
    size = size.masked_fill(hidden[:, None, None], 0).amax(-1, keepdim=True).expand_as(out)
    vs = scales[blocks].double()[:, :, 1].t().repeat_interleave(bt, 1)[:, :length]
    top = (p * vs.abs()[None, :, None]).amax(-1, keepdim=True).expand_as(out) * LIMIT[fmt]
    return [x.reshape(rows, heads, dim) for x in (out, weight, size, top)]


def bound(out, weight, size, top, length, dim, bf16):
    """How far an output may be from the 64-bit one.

    A score's error: each FP32 query is two FP16 halves (2^-22 of the value), dim products are added in FP32
    (2^-23 each, adders that cut included), and scaled (2 roundings): e_s = size * (2^-22 + dim 2^-23 + 2^-23). A
    weight's relative error: e_s, 2^-22 from exp2, 2^-22 |score| from the rounded exponent (|score| <= size), and
    2^-22 from its halves (FP16's half step 2^-11 instead for BF16 outputs). It counts twice: in the sum and in the
    normaliser, which also add `length` terms in FP32 (2^-23 each). BF16 outputs are rounded once more (2^-8).

    The halves also have a smallest step: weights times block scales are held in units of which the largest counts 2^8
    or more, and FP16 rounds to multiples of 2^-24 at best, so each is off by up to 2^-25 / 2^8 = 2^-33 of the largest,
    times a code. `length` of those add up, also where the largest itself meets a code of 0 (top = largest * top
    code)."""
    e = size * (2 ** -22 + dim * 2 ** -23 + 2 ** -21) + 2 ** -21 + (2 ** -11 if bf16 else 2 ** -22)
    return weight * (2 * e + length * 2 ** -22) + top * length * 2 ** -33 + (out.abs() * 2 ** -8 if bf16 else 0) + 1e-37
