"""The attention over pages at every size of a workgroup's tile (``paged_shapes.SHAPES``) with every type, head size, cache and
mask, against 64 bits, a few of the heads where there are many.  Tolerances: ``test_gpu_paged``'s."""
import math

import pytest
import torch

import fstattention_amd as fsta
from fstattention_amd import trees
from paged_shapes import SHAPES, TREES
from test_gpu_paged import ancestors, check, cuda, make_batch, make_cache, reference, rows_of

pytestmark = pytest.mark.gpu

TYPES = {"bf16": (torch.bfloat16, False), "fp16": (torch.float16, False), "bf16_8bit": (torch.bfloat16, True), "fp16_8bit": (torch.float16, True)}


def of_shapes(shapes, sizes=(64, 128), extra=(None,)):
    """(shape, head size, type, 8-bit, one of `extra`) of each; where there are many rows of many heads only for keys of 128 in 16 bits,
    whose rule of 256 rows they are for"""
    return [pytest.param(shape, d, dtype, fp8, *(() if more is None else (more,)), id="-".join(filter(None, (name, str(d), kind, more))))
            for name, shape in shapes.items() for d in sizes for kind, (dtype, fp8) in TYPES.items() for more in extra
            if shape.heads < 64 or (d == 128 and not fp8)]


def pack(sees, starts, tokens):
    """Rows of bits: word w's bit b says whether column 32 w + b is seen"""
    words = -(-max(s.shape[1] for s in sees) // 32)
    flat = torch.zeros((tokens, words * 32), dtype=torch.int64)
    for b, s in enumerate(sees):
        flat[int(starts[b]):int(starts[b + 1]), :s.shape[1]] = s.long()
    packed = (flat.view(tokens, words, 32) << torch.arange(32)).sum(-1)
    return torch.where(packed >= 1 << 31, packed - (1 << 32), packed).to(torch.int32)


def call(shape, d, dtype, fp8, mode, seed, sees=None, edit=None, table=None):
    """(cache, page table, lengths, starts, q, o, lse) of a call of this shape"""
    tab, lens, starts, pages = make_batch(shape.new, shape.keys, shape.page, seed, width=shape.width)
    if table is not None:
        table(tab)
    cache = make_cache(pages, shape.kv_heads, shape.page, d, dtype, seed + 1, fp8)
    if edit is not None:
        edit(cache, tab)
    tokens = sum(shape.new)
    q = torch.randn((tokens, shape.heads, d), generator=torch.Generator().manual_seed(seed + 2)).to(dtype)
    bits = pack(sees, starts, tokens).cuda() if sees else None
    o, lse = fsta.paged_attention(q.cuda(), cuda(cache), tab.cuda(), lens.cuda(), starts.cuda(), d ** -0.5, causal=mode == "causal",
                                  tree_bits=bits, max_q_len=max(shape.new), return_lse=True)
    return cache, tab, lens, starts, q, o.cpu(), lse.cpu()


def largest_product(q, cache, tab, starts, keys):
    """Largest sum of |q_i k_i| of a query and a key"""
    group, top = q.shape[1] // cache.k.shape[1], 0.0
    for b in range(len(keys)):
        k, _ = rows_of(cache.k, cache.k_exponent, tab, b, keys[b], cache.k.shape[2])
        for h in range(q.shape[1]):
            top = max(top, float((q[int(starts[b]):int(starts[b + 1]), h].abs().float() @ k[h // group].abs().float().t()).max()))
    return top


def compare(shape, d, dtype, fp8, mode, seed, sees=None, edit=None, table=None, large_scores=False):
    """large_scores: where scores are far from 1, what d additions in float32 do to them (d * 2^-24 of the sum of magnitudes) is no
    longer small: a weight is off by that at most, and so are a row's weights together."""
    cache, tab, lens, starts, q, o, lse = call(shape, d, dtype, fp8, mode, seed, sees, edit, table)
    assert o.isfinite().all()
    few = sorted({0, shape.kv_heads // 2, shape.kv_heads - 1})
    of_few = lambda t: t.view(t.shape[0], shape.kv_heads, -1, *t.shape[2:])[:, few].reshape(t.shape[0], -1, *t.shape[2:])
    part = fsta.PagedKV(*(None if t is None else t.view(torch.uint8)[:, few].view(t.dtype) if fp8 else t[:, few] for t in cache))
    want, want_lse, size = reference(of_few(q), part, tab, lens, starts, d ** -0.5, mode, sees)
    if large_scores:
        off = 2 * d * 2.0 ** -24 * largest_product(of_few(q), part, tab, starts, shape.keys) * d ** -0.5
        size = size * (1 + off * 2.0 ** 16)
    check(of_few(o), of_few(lse), want, want_lse, size, shape.keys, dtype, shape.rows(d, fp8), 0.0 if fp8 else 5.0)


@pytest.mark.parametrize("shape,d,dtype,fp8,mode", of_shapes(SHAPES, extra=("causal", "all")))
def test_every_tile(shape, d, dtype, fp8, mode):
    compare(shape, d, dtype, fp8, mode, 101)


@pytest.mark.parametrize("shape,d,dtype,fp8,kind", of_shapes(TREES, extra=("trees", "any_bits")))
def test_masks_of_more_than_256_nodes(shape, d, dtype, fp8, kind):
    """Words beyond those that a wave keeps; lengths in front of the new tokens that no word ends at.  Masks that are no tree's may
    leave rows of the new tokens nothing, and their rows are shorter than the tree."""
    if kind == "trees":
        sees = [ancestors(trees.random_recursive_parents(n, 3 + n, window=16).tolist()) for n in shape.new]
    else:
        g = torch.Generator().manual_seed(7)
        sees = [torch.rand((n, n - n // 7), generator=g) < 0.3 for n in shape.new]
        sees[0][5:9] = False
    compare(shape, d, dtype, fp8, "tree", 111, sees)


ONE_OF_EACH = {name: SHAPES[name] for name in ("32", "64", "128", "128_cut", "256")}


@pytest.mark.parametrize("shape,d,dtype,fp8", of_shapes(ONE_OF_EACH, sizes=(128,)))
def test_pages_outside_the_cache(shape, d, dtype, fp8):
    """Holes in the page table, in steps whose other tiles every row sees whole."""

    def holes(table):
        for b, keys in enumerate(shape.keys):
            for at, entry in ((2, -1), (7, 1 << 30), (8, -7), (31, -1), (90, -(1 << 31))):
                if at < -(-keys // shape.page) - 1:
                    table[b, at] = entry
    compare(shape, d, dtype, fp8, "causal", 121, table=holes)


@pytest.mark.parametrize("shape,d,dtype,fp8", of_shapes(ONE_OF_EACH))
def test_rising_maxima(shape, d, dtype, fp8):
    """Scores that grow along the keys, so that tile after tile raises the running maximum, from ordinary ones up to differences that
    underflow."""
    def edit(cache, table):
        for b, keys in enumerate(shape.keys):
            count = -(-keys // shape.page)
            for j in range(count):
                page = int(table[b, j])
                if fp8:
                    cache.k_exponent[page] += 6 * j // count
                else:
                    cache.k[page] = (cache.k[page].float() * (0.2 + 20.0 * j / count)).to(dtype)
    compare(shape, d, dtype, fp8, "causal", 131, edit=edit, large_scores=True)


@pytest.mark.parametrize("shape,d,dtype,fp8", of_shapes({name: ONE_OF_EACH[name] for name in ("64", "128", "128_cut", "256")}))
def test_values_that_are_not_finite(shape, d, dtype, fp8):
    """NaNs and infinities among the new tokens' values, in the last sequence's and the first one's: rows that see the key get them,
    the others are as without them, bit by bit; what lies in unused rows reaches nobody."""
    tab = make_batch(shape.new, shape.keys, shape.page, 141, width=shape.width)[0]
    bad = {}                                      # (sequence, new token) -> (head dim, value)
    for b in (0, len(shape.new) - 1):
        n = shape.new[b]
        bad[b, 0], bad[b, n // 2], bad[b, n - 1] = (7, math.nan), (d - 1, math.nan if fp8 else math.inf), (33, math.nan if fp8 else -math.inf)

    def dirty(cache, table):
        for (b, i), (col, x) in bad.items():
            at = shape.keys[b] - shape.new[b] + i
            where = (int(tab[b, at // shape.page]), slice(None), at % shape.page, col)
            if fp8:
                cache.v.view(torch.uint8)[where] = 0x7f
            else:
                cache.v[where] = x
        used = torch.zeros((cache.k.shape[0], shape.page), dtype=torch.bool)
        for b, keys in enumerate(shape.keys):
            places = torch.arange(keys)
            used[tab[b][places // shape.page].long(), places % shape.page] = True
        for pool in (cache.k, cache.v):
            raw = pool.view(torch.uint8 if fp8 else torch.int16).permute(0, 2, 1, 3)
            raw[~used] = 0x7f if fp8 else 0x7fff
    got, want = (call(shape, d, dtype, fp8, "causal", 141, edit=edit)[5] for edit in (dirty, None))
    starts = torch.tensor([0] + shape.new).cumsum(0)
    for b in range(len(shape.new)):
        for (c, i), (col, x) in bad.items():
            if c == b:
                want[int(starts[b]) + i:int(starts[b + 1]), :, col] = x
    torch.testing.assert_close(got, want, rtol=0, atol=0, equal_nan=True)


@pytest.mark.parametrize("most", [None, 1, 40, 300])
def test_hints_reach_other_tiles(most):
    """The longest chunk as the caller knows it, or not: tiles of 64 rows (a hint that is too small) and of 128."""
    shape = SHAPES["128"]
    tab, lens, starts, pages = make_batch(shape.new, shape.keys, shape.page, 151)
    cache = make_cache(pages, shape.kv_heads, shape.page, 128, torch.float16, 152)
    q = torch.randn((sum(shape.new), shape.heads, 128), generator=torch.Generator().manual_seed(153)).half()
    out, lse = fsta.paged_attention(q.cuda(), cuda(cache), tab.cuda(), lens.cuda(), starts.cuda(), 128 ** -0.5, max_q_len=most, return_lse=True)
    want, want_lse, size = reference(q, cache, tab, lens, starts, 128 ** -0.5, "causal")
    check(out, lse, want, want_lse, size, shape.keys, torch.float16, 600, 5.0)
