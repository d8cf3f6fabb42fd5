"""Calls of the attention over pages that reach each size of a workgroup's tile of rows, with whole keys and with keys dealt to
several workgroups.  ``test_paged_tiles.py`` asks the library which tile each takes, so that a change of its rules that moves one
of them elsewhere is seen; ``test_gpu_paged_tiles.py`` runs them."""
from typing import List, NamedTuple


class Shape(NamedTuple):
    tile: int                  # rows, for keys of 128 in 16 bits
    new: List[int]
    keys: List[int]
    heads: int
    kv_heads: int
    columns: int = 0           # of the page table, that no sequence uses
    page: int = 16

    def rows(self, d, fp8):    # 256 rows are for keys of 128 in 16 bits only
        return 128 if self.tile == 256 and (d == 64 or fp8) else self.tile

    @property
    def width(self):
        return -(-max(self.keys) // self.page) + self.columns


SHAPES = {
    "32": Shape(32, [5, 1, 9], [40, 7, 260], 8, 2),
    "32_many_rows": Shape(32, [70, 33], [200, 33], 8, 4),
    "64": Shape(64, [14, 1, 3], [1900, 50, 33], 8, 2),
    "64_many_rows": Shape(64, [200], [900], 4, 1, page=64),
    "128": Shape(128, [300, 77], [1500, 200], 16, 8),
    "128_whole": Shape(128, [250, 120], [250, 130], 32, 16),
    "128_wide_table": Shape(128, [331, 77], [431, 200], 16, 8, columns=100),
    "128_cut": Shape(128, [300, 1, 40], [4000, 33, 41], 16, 8, page=32),
    "128_below_256": Shape(128, [1100, 940], [1300, 960], 64, 64),
    "256": Shape(256, [1100, 960], [1300, 1031], 64, 64),
    "256_shared_heads": Shape(256, [1200, 941], [1300, 1000], 64, 32, page=128),
    "256_cut": Shape(256, [1900, 200], [2000, 9000], 64, 64, page=64),
}

# Trees of more nodes than a wave keeps mask words for (256), and masks that are none's ancestors
TREES = {
    "32": Shape(32, [300, 5], [351, 77], 4, 4),
    "64": Shape(64, [1000], [1105], 1, 1),
    "32_words_end": Shape(32, [257], [257], 2, 2, page=32),
    "128": Shape(128, [1000, 257, 300], [1105, 301, 2300], 8, 8),
    "256": Shape(256, [1000, 1090], [1105, 1090], 64, 64),
}
