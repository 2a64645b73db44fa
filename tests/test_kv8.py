"""8-bit paged K/V cache operators: refusals (no GPU: every one comes before a device call) and the plain forms."""
import ctypes
import math

import pytest
import torch

import kv8_reference as ref
from tinyinfer_b200 import device as mp

A = 1 << 20  # a 16-byte aligned address that nothing reads


def cache(**kw):
    fields = dict(pages=A, scales=A, page_stride=3 * 2 * 16 * 64, scale_stride=6, format=mp.MP_KV8_INT8, kv_heads=3,
                  head_dim=64, block_tokens=16, max_blocks=8)
    return mp.Kv8Cache(**{**fields, **kw})


def append_args(**kw):
    fields = dict(q=A, k=A, v=A, q_out=A, q_stride=576, k_stride=192, v_stride=192, q_out_stride=576, cos=A, sin=A,
                  tables=A, row_offsets=A, starts=A, type=mp.MP_TYPE_F32, heads=9, rotary_dim=64,
                  rope_layout=mp.MP_ROPE_HALF, max_positions=64, table_stride=4, count=1, rows=1)
    return mp.Kv8AppendArgs(**{**fields, **kw})


def decode_args(**kw):
    fields = dict(q=A, out=A, q_stride=576, out_stride=576, tables=A, lengths=A, workspace=A, workspace_bytes=1 << 40,
                  type=mp.MP_TYPE_F32, heads=9, table_stride=4, count=1, scale=0.125)
    return mp.Kv8DecodeArgs(**{**fields, **kw})


def prefill_args(**kw):
    fields = dict(q=A, out=A, q_stride=576, out_stride=576, tables=A, row_offsets=A, starts=A, workspace=A,
                  workspace_bytes=1 << 40, type=mp.MP_TYPE_F32, heads=9, table_stride=4, count=1, rows=1, scale=0.125)
    return mp.Kv8PrefillArgs(**{**fields, **kw})


CALLS = {"append": (mp.kv8_append, append_args), "decode": (mp.kv8_attention_decode, decode_args),
         "prefill": (mp.kv8_attention_prefill, prefill_args)}


def refused(op, code, cache_kw=None, error=None, **kw):
    call, make = CALLS[op]
    with pytest.raises(mp.DeviceError) as e:
        call(cache(**(cache_kw or {})), make(**kw), error)
    assert e.value.code == code, e.value
    assert "kv8" in e.value.message


@pytest.mark.parametrize("op", list(CALLS))
@pytest.mark.parametrize("code,kw", [
    (mp.MP_ERR_INVALID, {"pages": None}), (mp.MP_ERR_INVALID, {"scales": None}), (mp.MP_ERR_INVALID, {"pages": A + 8}),
    (mp.MP_ERR_INVALID, {"scales": A + 4}), (mp.MP_ERR_INVALID, {"page_stride": 6143}),
    (mp.MP_ERR_INVALID, {"page_stride": 6144 + 8}), (mp.MP_ERR_INVALID, {"page_stride": 6128}),
    (mp.MP_ERR_INVALID, {"scale_stride": 4}), (mp.MP_ERR_INVALID, {"scale_stride": 7}),
    (mp.MP_ERR_INVALID, {"format": 2}), (mp.MP_ERR_INVALID, {"kv_heads": 0}), (mp.MP_ERR_INVALID, {"kv_heads": 2}),
    (mp.MP_ERR_INVALID, {"max_blocks": 0}), (mp.MP_ERR_UNSUPPORTED, {"head_dim": 96}),
    (mp.MP_ERR_UNSUPPORTED, {"head_dim": 0}), (mp.MP_ERR_UNSUPPORTED, {"block_tokens": 8}),
    (mp.MP_ERR_UNSUPPORTED, {"block_tokens": 24}), (mp.MP_ERR_UNSUPPORTED, {"block_tokens": 272})])
def test_caches_are_checked(built, op, code, kw):
    refused(op, code, kw)


@pytest.mark.parametrize("op,kw", [
    *[(op, {"type": 2}) for op in CALLS], *[(op, {"heads": 10}) for op in CALLS], *[(op, {"heads": 0}) for op in CALLS],
    *[(op, {"heads": 3 * 65}) for op in CALLS], *[(op, {"count": 0}) for op in CALLS],
    *[(op, {"count": 65537}) for op in CALLS], *[(op, {"table_stride": 0}) for op in CALLS],
    *[(op, {"tables": None}) for op in CALLS], *[(op, {"tables": A + 2}) for op in CALLS],
    *[(op, {"q": A + 4}) for op in CALLS], *[(op, {"q_stride": 575}) for op in CALLS],
    *[(op, {"q_stride": 578}) for op in CALLS], *[(op, {"q_stride": 580, "type": mp.MP_TYPE_BF16}) for op in CALLS],
    *[("append", {n: None}) for n in ("k", "v", "q", "q_out", "cos", "sin", "row_offsets", "starts")],
    *[("append", {n: A + 8}) for n in ("k", "v", "q_out", "cos", "sin")],
    *[("append", {n: 191}) for n in ("k_stride", "v_stride", "q_out_stride")],
    *[("append", {"rotary_dim": n}) for n in (-8, 4, 12, 72)], ("append", {"rope_layout": 2}),
    ("append", {"max_positions": 0}), ("append", {"rows": -1}), ("prefill", {"rows": -1}),
    ("prefill", {"row_offsets": None}), ("prefill", {"starts": None}), ("decode", {"lengths": None}),
    *[(op, {n: v}) for op in ("decode", "prefill") for n, v in (
        ("q", None), ("out", None), ("out", A + 4), ("out_stride", 572), ("workspace", None), ("workspace", A + 8),
        ("workspace_bytes", 0))]])
def test_arguments_are_checked(built, op, kw):
    refused(op, mp.MP_ERR_INVALID, **kw)


def test_nulls_and_misaligned_error_words_are_refused(built):
    lib = mp.library()
    for name, (_, make) in CALLS.items():
        entry = getattr(lib, {"append": "mp_kv8_append", "decode": "mp_kv8_attention_decode",
                              "prefill": "mp_kv8_attention_prefill"}[name])
        assert entry(None, make(), None, None) == mp.MP_ERR_INVALID
        assert entry(cache(), None, None, None) == mp.MP_ERR_INVALID
        refused(name, mp.MP_ERR_INVALID, error=A + 2)
    assert lib.mp_kv8_status(None, None) == mp.MP_ERR_INVALID
    assert lib.mp_kv8_status(A + 1, None) == mp.MP_ERR_INVALID


def test_without_a_device_the_calls_fail_loudly(built):
    if torch.cuda.is_available():
        pytest.skip("needs a machine without a GPU")
    for name in CALLS:
        refused(name, mp.MP_ERR_CUDA)


def test_workspace_sizes(built):
    for heads, kv in ((9, 3), (1, 1), (64, 1), (32, 8)):
        for dim in (64, 128):
            c = cache(kv_heads=kv, head_dim=dim)
            assert 0 < mp.kv8_decode_workspace(c, heads) < 1 << 28
            assert 0 < mp.kv8_prefill_workspace(c, heads) < 1 << 29
    assert mp.kv8_decode_workspace(cache(), 10) == 0
    assert mp.kv8_prefill_workspace(cache(head_dim=65), 9) == 0


def test_argument_blocks_mirror_the_header():
    """Field order and count of the ctypes blocks against the header's structs."""
    import os
    import re

    text = open(os.path.join(os.path.dirname(os.path.dirname(__file__)), "include", "miniprefix_b200.h")).read()
    text = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
    for name, block in (("mp_kv8_cache", mp.Kv8Cache), ("mp_kv8_append_args", mp.Kv8AppendArgs),
                        ("mp_kv8_decode_args", mp.Kv8DecodeArgs), ("mp_kv8_prefill_args", mp.Kv8PrefillArgs)):
        body = re.search(r"typedef struct \{([^}]*)\} %s;" % name, text).group(1)
        sizes = {"int32_t": 4, "int64_t": 8, "size_t": 8, "float": 4}
        fields = []
        for line in body.split(";"):
            line = line.replace("const ", "").strip()
            if not line:
                continue
            kind, names = line.split(None, 1) if not line.startswith("void*") else ("void*", line[5:])
            for n in names.split(","):
                pointer = "*" in kind or "*" in n
                fields.append((n.replace("*", "").strip(), 8 if pointer else sizes[kind]))
        assert fields == [(n, ctypes.sizeof(t)) for n, t in block._fields_]


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_reference_rounding_and_scales(fmt):
    """The plain forms that the GPU tests compare with: every code is its own nearest, borders go to even, scales
    are the smallest that hold."""
    codes = torch.arange(-127, 128).to(torch.int8) if fmt == "int8" else torch.tensor(
        [c for c in range(256) if c & 127 != 127], dtype=torch.uint8).view(torch.int8)
    values = ref.decode_codes(codes, fmt)
    assert torch.equal(ref.nearest(values, fmt), values)
    assert torch.equal(ref.decode_codes(ref.encode(values, fmt), fmt), values)
    limit = ref.LIMIT[fmt]
    assert ref.nearest(torch.tensor([1e9, -1e9], dtype=torch.float64), fmt).tolist() == [limit, -limit]
    up = sorted(set(values[values >= 0].tolist()))
    for i in range(len(up) - 1):
        middle = torch.tensor([(up[i] + up[i + 1]) / 2], dtype=torch.float64)
        even = up[i] if i % 2 == 0 else up[i + 1]
        assert ref.nearest(middle, fmt).item() == even
        assert ref.nearest(middle * (1 + 1e-12) + 1e-300, fmt).item() == up[i + 1]
    for amax in (1.0, limit, math.nextafter(limit, 1e9) * (1 + 1e-6), 3.4e38, 1e-30, 0.0):
        s = ref.scale_for(amax, fmt)
        assert limit * s >= float(torch.tensor(amax, dtype=torch.float64).float())
        assert s == 2.0 ** -100 or limit * s / 2 < amax


@pytest.mark.parametrize("op", list(CALLS))
def test_tables_beyond_the_index_range_are_refused(built, op):
    refused(op, mp.MP_ERR_INVALID, table_stride=(1 << 26) // 16 + 1)


@pytest.mark.parametrize("wait_us", [0, -1, 1000001])
def test_wait_limits_out_of_range_are_refused(built, wait_us):
    with pytest.raises(mp.DeviceError) as e:
        mp.kv8_inject_wait_timeout(wait_us)
    assert e.value.code == mp.MP_ERR_INVALID


def test_rotation_in_place_with_another_stride_is_refused(built):
    """Rows would be overwritten before they are read."""
    refused("append", mp.MP_ERR_INVALID, q_out_stride=640)
