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
