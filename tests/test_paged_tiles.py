"""Which tile of rows the attention over pages takes, and the workspace that it asks for, without a GPU: a call that is short of
workspace is refused before any launch, and says how much it needs."""
import random
import re

import pytest

from fstattention_amd import _lib
from paged_shapes import SHAPES, TREES

P = 1 << 20                       # a pointer that nothing follows


def needed(batch, width, tokens, most, page, heads, kv_heads, d, cache_dtype):
    lib = _lib.load()
    exps = P if cache_dtype == _lib.FP8 else None
    rc = lib.fsta_paged_attention(P, heads * d, d, P, P, exps, exps, P, P, P, None, 0, P, None, batch, width, tokens, most, 9, page, heads, kv_heads,
                                  d, _lib.BF16, cache_dtype, _lib.PAGED_CAUSAL, 0.1, None, 0, None)
    assert rc == _lib.EINVAL
    return int(re.search(r"needs (\d+) bytes of workspace", lib.fsta_last_error().decode()).group(1))


def workspace(rows, batch, tokens, heads, kv_heads, d):
    """What tiles of so many rows need: parts of rows x (d + 1) floats, for every unit that the largest cut has beyond whole tiles and
    for every tile that it cuts"""
    tiles = (tokens * (heads // kv_heads) + min(batch, tokens) * (rows - 1)) // rows
    units = 512 if rows == 256 else 768
    runs = (units + units // 256 + kv_heads) // kv_heads
    return 4 * ((runs + min(runs, tiles)) * kv_heads * rows * (d + 1) + 4)


@pytest.mark.parametrize("d,cache_dtype", [(128, _lib.BF16), (64, _lib.BF16), (128, _lib.FP8), (64, _lib.FP8)])
@pytest.mark.parametrize("shape", list(SHAPES.values()) + list(TREES.values()), ids=list(SHAPES) + ["tree_" + name for name in TREES])
def test_the_shapes_take_the_tiles_they_are_listed_for(shape, d, cache_dtype):
    sizes = {rows: workspace(rows, len(shape.new), sum(shape.new), shape.heads, shape.kv_heads, d) for rows in (32, 64, 128, 256)}
    assert len(set(sizes.values())) == 4
    need = needed(len(shape.new), shape.width, sum(shape.new), max(shape.new), shape.page, shape.heads, shape.kv_heads, d, cache_dtype)
    assert need == sizes[shape.rows(d, cache_dtype == _lib.FP8)]


def test_the_workspace_is_enough_for_any_call_of_its_sizes():
    """No page table's width makes a call ask for more than fsta_paged_attention_workspace_bytes says for its other sizes."""
    lib, rng = _lib.load(), random.Random(5)
    log = lambda low, high: int(round(low * (high / low) ** rng.random()))
    for _ in range(20000):
        batch, tokens, kv_heads = log(1, 65536), log(1, 1 << 16), rng.choice([1, 2, 3, 4, 8, 16, 32, 64, 128, 1000, 16384])
        heads = kv_heads * rng.choice([1, 1, 2, 4, 5, 7, 8, 16])
        if tokens * heads > 0x3fffffff:
            continue
        most, d, page = rng.choice([0, 1, log(1, tokens), tokens, 2 * tokens]), rng.choice([64, 128]), 1 << rng.randint(4, 12)
        cache_dtype, width = rng.choice([_lib.BF16, _lib.FP8]), log(1, 0x7fffffc0 // page)
        enough = lib.fsta_paged_attention_workspace_bytes(batch, tokens, most, heads, kv_heads, d, cache_dtype)
        asked = needed(batch, width, tokens, most, page, heads, kv_heads, d, cache_dtype)
        assert 0 < asked <= enough, (batch, width, tokens, most, page, heads, kv_heads, d, cache_dtype)
