"""The paged KV cache (``fstattention_amd/paged.py``) against plain implementations in 64 bits.

Tolerances of the attention, per element: the output's own rounding ``u |o|`` (u = 2^-8 bfloat16, 2^-11 float16: half a unit in
the last of 8 or 11 bits); the weights' rounding on their way to the matrix cores, at most ``u_p`` each (u, or 2^-16 as a pair), so
``u_p`` times the attention over ``|v|``; float32 sums and scores, 2^-16 of the same; and for float16, whose weights below 2^-14
are denormal, 2^-24 of the largest ``|v|`` per key.
Log-sum-exp: float32 sums, 2^-16 absolute per unit of magnitude.
"""
import math

import pytest
import torch

import fstattention_amd as fsta
from fstattention_amd import trees

pytestmark = pytest.mark.gpu

HALF = [torch.bfloat16, torch.float16]


def make_batch(new, keys, page, seed, spare=2, width=None):
    """(page_table, kv_lens, q_starts, pages): pages in random order, some of nobody's, table entries past the end -1"""
    g = torch.Generator().manual_seed(seed)
    counts = [-(-k // page) for k in keys]
    order = torch.randperm(sum(counts) + spare, generator=g).to(torch.int32)
    width = width or max(max(counts), 1)
    table = torch.full((len(new), width), -1, dtype=torch.int32)
    first = 0
    for b, c in enumerate(counts):
        table[b, :c] = order[first:first + c]
        first += c
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    return table, torch.tensor(keys, dtype=torch.int32), torch.tensor(starts, dtype=torch.int32), sum(counts) + spare


def make_cache(pages, heads, page, d, dtype, seed, fp8=False, fill=None):
    g = torch.Generator().manual_seed(seed)
    k, v = (torch.randn((pages, heads, page, d), generator=g).to(dtype) for _ in range(2))
    if fill is not None:
        k, v = torch.full_like(k, fill), torch.full_like(v, fill)
    if not fp8:
        return fsta.PagedKV(k, v)
    (k8, ke), (v8, ve) = quantise(k), quantise(v)
    return fsta.PagedKV(k8, v8, ke, ve)


def quantise(x):
    """The definition, in 64 bits on the host: smallest e with max |finite x| <= 448 2^e, bytes to nearest even."""
    y = x.double()
    finite = torch.where(y.isfinite(), y.abs(), torch.zeros_like(y))
    amax = finite.amax(-1)
    e = torch.ceil(torch.log2(torch.where(amax > 0, amax, torch.full_like(amax, 448.0)) / 448.0))
    e = torch.where(amax > 0, e.clamp(-110, 120), torch.zeros_like(e)).to(torch.int32)
    scaled = torch.where(y.isfinite(), y / torch.pow(torch.tensor(2.0, dtype=torch.float64), e.double())[..., None], torch.full_like(y, math.nan))
    return scaled.float().to(torch.float8_e4m3fn), (e + 127).to(torch.uint8)


def values(pool, exponent):
    x = pool.double()
    return x if exponent is None else x * torch.pow(torch.tensor(2.0, dtype=torch.float64), exponent.double() - 127)[..., None]


def rows_of(pool, exponent, table, b, keys, page):
    """[Hkv, keys, D] in 64 bits and which keys are on a page"""
    x = values(pool, exponent)
    out = torch.zeros((pool.shape[1], keys, pool.shape[3]), dtype=torch.float64)
    here = torch.zeros(keys, dtype=torch.bool)
    for p in range(0, keys, page):
        id_ = int(table[b, p // page])
        if 0 <= id_ < pool.shape[0]:
            n = min(page, keys - p)
            out[:, p:p + n] = x[id_, :, :n]
            here[p:p + n] = True
    return out, here


def ancestors(parent):
    n = len(parent)
    sees = torch.zeros((n, n), dtype=torch.bool)
    for i, p in enumerate(parent):
        if 0 <= p < i:
            sees[i] = sees[p]
        sees[i, i] = True
    return sees


def reference(q, cache, table, keys, starts, scale, mode, sees=None):
    """(o, lse, attention over |v|, longest) in 64 bits"""
    page, d = cache.k.shape[2], q.shape[2]
    group = q.shape[1] // cache.k.shape[1]
    o, size = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    lse = torch.full(q.shape[:2], -math.inf, dtype=torch.float64)
    for b in range(len(keys)):
        n, kv = int(starts[b + 1] - starts[b]), int(keys[b])
        if n == 0 or kv == 0:
            continue
        k, here = rows_of(cache.k, cache.k_exponent, table, b, kv, page)
        v, _ = rows_of(cache.v, cache.v_exponent, table, b, kv, page)
        number = torch.arange(kv) - (kv - n)
        mask = torch.ones((n, kv), dtype=torch.bool)
        if mode == "causal":
            mask = number[None, :] <= torch.arange(n)[:, None]
        elif mode == "tree":
            mask = (number < 0)[None, :].repeat(n, 1)
            inside = (number >= 0) & (number < sees[b].shape[1])
            mask[:, inside] = sees[b][:, number[inside]]
        mask &= here[None]
        rows = q[int(starts[b]):int(starts[b + 1])].double()
        for h in range(q.shape[1]):
            s = rows[:, h] @ k[h // group].t() * scale
            s = torch.where(mask, s, torch.full_like(s, -math.inf))
            top = s.amax(1, keepdim=True)
            top = torch.where(top == -math.inf, torch.zeros_like(top), top)
            w = torch.exp(s - top)
            w = torch.where(mask, w, torch.zeros_like(w))
            total = w.sum(1, keepdim=True)
            vh = torch.where(mask.any(0)[:, None], v[h // group], torch.zeros_like(v[h // group]))
            dense = w / total.clamp(min=1e-300)
            at = slice(int(starts[b]), int(starts[b + 1]))
            o[at, h], size[at, h] = dense @ vh, dense @ vh.abs()
            lse[at, h] = (top[:, 0] + torch.log(total[:, 0])) / math.log(2.0)
    return o, lse, size


def check(got, got_lse, want, want_lse, size, keys, dtype, rows, largest_v):
    u = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -11
    u_p = u if dtype == torch.float16 or rows > 64 else 2.0 ** -16
    tol = u * want.abs() + (u_p + 2.0 ** -16) * size + 2.0 ** -24
    if dtype == torch.float16:
        tol = tol + 2.0 ** -24 * max(keys) * largest_v
    err = (got.double().cpu() - want).abs()
    worst = (err - tol).amax()
    assert bool((err <= tol).all()), f"{float(worst)} beyond the tolerance, error {float(err.max())}"
    if got_lse is not None:
        got_lse = got_lse.double().cpu()
        empty = want_lse == -math.inf
        assert bool((got_lse[empty] == -math.inf).all())
        err = (got_lse[~empty] - want_lse[~empty]).abs()
        assert err.numel() == 0 or bool((err <= 2.0 ** -16 * want_lse[~empty].abs().clamp(min=1)).all()), float(err.max())


def cuda(cache):
    return fsta.PagedKV(*(None if t is None else t.cuda() for t in cache))


def run(new, keys, heads, kv_heads, d, dtype, page, seed, mode="causal", fp8=False, sees=None, lse=True, table=None, max_q_len="most",
        edit=None, q_view=True):
    tab, lens, starts, pages = make_batch(new, keys, page, seed)
    if table is not None:
        tab = table(tab)
    cache = make_cache(pages, kv_heads, page, d, dtype, seed + 1, fp8)
    if edit is not None:
        edit(cache, tab)
    tokens = int(starts[-1])
    g = torch.Generator().manual_seed(seed + 2)
    fused = torch.randn((tokens, (heads + 2) * d), generator=g).to(dtype)
    q = fused[:, d:d + heads * d].view(tokens, heads, d) if q_view else fused[:, :heads * d].reshape(tokens, heads, d).contiguous()
    scale = 1.0 / math.sqrt(d)
    bits = None
    if mode == "tree":
        words = -(-max(s.shape[1] for s in sees) // 32)
        packed = torch.zeros((tokens, words * 32), dtype=torch.int64)
        for b, s in enumerate(sees):
            packed[int(starts[b]):int(starts[b + 1]), :s.shape[1]] = s.long()
        packed = (packed.view(tokens, words, 32) << torch.arange(32)).sum(-1)
        bits = torch.where(packed >= 1 << 31, packed - (1 << 32), packed).to(torch.int32).cuda()
    dev = fused.cuda()
    q_dev = dev[:, d:d + heads * d].view(tokens, heads, d) if q_view else q.cuda()
    most = max(new) if max_q_len == "most" else max_q_len
    out = fsta.paged_attention(q_dev, cuda(cache), tab.cuda(), lens.cuda(), starts.cuda(), scale, causal=mode == "causal", tree_bits=bits,
                               max_q_len=most, return_lse=lse)
    o, got_lse = out if lse else (out, None)
    want, want_lse, size = reference(q, cache, tab, lens, starts, scale, mode, sees)
    rows = (max(new) if max_q_len == "most" else (max_q_len or tokens)) * (heads // kv_heads)
    check(o, got_lse, want, want_lse, size, keys, dtype, rows, 5.0)
    return o


# ---- attention ----------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("page", [16, 64])
def test_single_tokens(d, dtype, page, fp8):
    run([1] * 7, [1, 2, 31, 32, 33, 257, 700], 8, 2, d, dtype, page, 11, fp8=fp8)


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (4, 4), (14, 2), (32, 1), (40, 8), (64, 1)])
def test_head_layouts(heads, kv_heads):
    run([1, 3, 1], [45, 203, 1], heads, kv_heads, 128, torch.bfloat16, 32, 12)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("new,keys", [([17], [17]), ([33, 1, 64], [90, 5, 64]), ([127, 200], [130, 1201]), ([300, 2, 0, 75], [1300, 700, 50, 75])])
def test_chunks(new, keys, d, dtype, fp8):
    run(new, keys, 6, 2, d, dtype, 16, 13, fp8=fp8)


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256, 4096])
def test_page_sizes(page):
    run([5, 40], [page + 3, 2 * page if page < 4096 else 900], 4, 2, 64, torch.bfloat16, page, 14)


@pytest.mark.parametrize("most", [None, 1, 8, 1000])
def test_the_hint_of_the_longest_chunk_changes_the_kernel_only(most):
    run([20, 1, 30], [400, 300, 31], 4, 2, 128, torch.float16, 16, 15, max_q_len=most)


@pytest.mark.parametrize("kv_heads,keys", [(1, 40000), (8, 9001), (2, 700)])
def test_keys_cut_into_runs(kv_heads, keys):
    """Few sequences with many keys: the keys are dealt to several workgroups and their parts joined."""
    run([1], [keys], 4 * kv_heads, kv_heads, 128, torch.bfloat16, 64, 16)
    run([9, 1], [keys, 50], 4 * kv_heads, kv_heads, 64, torch.float16, 64, 17, fp8=True)


def test_cut_chunks_and_long_chunks_together():
    run([130, 1, 3], [6000, 9000, 40], 8, 2, 128, torch.bfloat16, 128, 18)


def test_many_sequences():
    """More sequences than lanes: 150, some without new tokens, some without keys (their tokens see nothing)."""
    g = torch.Generator().manual_seed(5)
    new = torch.randint(0, 4, (150,), generator=g).tolist()
    keys = [0 if i % 37 == 5 else n + int(torch.randint(0, 200, (1,), generator=g)) for i, n in enumerate(new)]
    run(new, keys, 4, 2, 64, torch.bfloat16, 16, 19)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("dtype,d", [(torch.bfloat16, 128), (torch.float16, 64)])
@pytest.mark.parametrize("batch,kv_heads,low,high", [(3, 1, 500, 9000), (5, 8, 1, 3000), (70, 2, 1, 1500), (200, 4, 300, 700), (130, 1, 1, 40)])
def test_keys_dealt_evenly(batch, kv_heads, low, high, dtype, d, fp8):
    """Lengths of all kinds in one batch, cut into runs of keys or not, sequences without keys among them."""
    g = torch.Generator().manual_seed(batch + high)
    new = torch.randint(0, 3, (batch,), generator=g).tolist()
    keys = [n + int(torch.randint(low, high, (1,), generator=g)) for n in new]
    keys[batch // 2] = new[batch // 2]
    run(new, keys, 2 * kv_heads, kv_heads, d, dtype, 64, 60, fp8=fp8)


def test_every_position_is_seen_without_a_mask():
    run([5, 70], [64, 333], 4, 2, 128, torch.bfloat16, 16, 20, mode="all")


def test_tokens_in_front_of_the_first_position_see_nothing():
    """Fewer positions than new tokens: the first ones have no place and no key."""
    run([40, 3], [25, 2], 2, 1, 64, torch.float16, 16, 21)
    run([40, 3], [25, 0], 2, 1, 128, torch.bfloat16, 16, 22)


@pytest.mark.parametrize("new,keys", [([1], [1]), ([13, 64], [13, 500]), ([64, 61, 5], [700, 61, 40]), ([256, 100], [1031, 100])])
@pytest.mark.parametrize("dtype,d,fp8", [(torch.bfloat16, 128, False), (torch.float16, 64, False), (torch.bfloat16, 64, True)])
def test_trees(new, keys, dtype, d, fp8):
    sees = [ancestors(trees.random_recursive_parents(n, 3 + n, window=16).tolist()) for n in new]
    run(new, keys, 4, 4, d, dtype, 16, 23, mode="tree", sees=sees, fp8=fp8)


def test_masks_with_empty_rows():
    """Rows of bits that leave a token nothing, with and without positions in front of the new tokens."""
    g = torch.Generator().manual_seed(3)
    sees = [torch.rand((n, n), generator=g) < 0.05 for n in (40, 70)]
    sees[0][3:9] = False
    sees[1][:] = False
    run([40, 70], [40, 70], 4, 2, 128, torch.bfloat16, 16, 24, mode="tree", sees=sees)
    run([40, 70], [47, 200], 4, 2, 64, torch.float16, 16, 25, mode="tree", sees=sees)


def test_rows_of_bits_shorter_than_the_chunk():
    sees = [torch.ones((50, 32), dtype=torch.bool)]
    run([50], [90], 2, 2, 64, torch.bfloat16, 16, 26, mode="tree", sees=sees)


def test_unused_rows_and_pages_may_hold_anything():
    """NaN and infinities in every row that belongs to no position, largest exponents in 8-bit ones."""
    for fp8 in (False, True):
        def edit(cache, table):
            used = torch.zeros(cache.k.shape[0], cache.k.shape[2], dtype=torch.bool)
            for b, kv in enumerate(keys):
                for p in range(kv):
                    used[int(table[b, p // 16]), p % 16] = True
            for pool in (cache.k, cache.v):
                flat = pool.view(torch.uint8 if fp8 else torch.int16)
                flat.copy_(torch.where(used[:, None, :, None], flat, torch.full_like(flat, 0x7f if fp8 else 0x7fff)))
            for e in (cache.k_exponent, cache.v_exponent) if fp8 else ():
                e.copy_(torch.where(used[:, None, :], e, torch.full_like(e, 255)))
        new, keys = [1, 20, 3], [37, 52, 3]
        run(new, keys, 4, 2, 128, torch.bfloat16, 16, 27, fp8=fp8, edit=edit)


def test_keys_on_no_page_are_not_seen():
    def holes(table):
        table = table.clone()
        table[0, 1], table[0, 4], table[1, 0] = -1, 1 << 30, -7
        return table
    for new in ([1, 1], [16, 9], [33, 40]):
        run(new, [150, 90], 4, 2, 64, torch.bfloat16, 16, 28, table=holes)


def test_large_scores_and_rising_maxima():
    """Scores that grow along the keys, so that every tile raises the running maximum, up to differences that underflow."""
    def edit(cache, table):
        for b in range(table.shape[0]):
            for j, page in enumerate(table[b].tolist()):
                if page >= 0:
                    cache.k[page] = (cache.k[page].float() * (0.2 + 0.7 * j)).to(cache.k.dtype)
    for dtype in HALF:
        run([1, 50], [400, 500], 4, 2, 64, dtype, 16, 29, edit=edit)


def test_contiguous_queries():
    run([3, 1], [70, 4], 4, 2, 64, torch.float16, 16, 30, q_view=False)


def test_offsets_past_32_bits():
    """A cache of more than 4 GiB per tensor, the sequence's keys on its last pages."""
    page, d, heads = 4096, 128, 1
    pages = (4 << 30) // (page * heads * d * 2) + 5
    k = torch.zeros((pages, heads, page, d), dtype=torch.bfloat16, device="cuda")
    v = torch.zeros_like(k)
    g = torch.Generator().manual_seed(1)
    tail = [torch.randn((3, heads, page, d), generator=g).to(torch.bfloat16) for _ in range(2)]
    k[-3:], v[-3:] = tail[0].cuda(), tail[1].cuda()
    table = torch.tensor([[pages - 2, pages - 1]], dtype=torch.int32)
    lens, starts = torch.tensor([5000], dtype=torch.int32), torch.tensor([0, 2], dtype=torch.int32)
    q = torch.randn((2, 2, d), generator=g).to(torch.bfloat16)
    cache = fsta.PagedKV(k, v)
    o, lse = fsta.paged_attention(q.cuda(), cache, table.cuda(), lens.cuda(), starts.cuda(), 0.1, return_lse=True)
    small = fsta.PagedKV(tail[0], tail[1])
    want, want_lse, size = reference(q, small, table - (pages - 3), lens, starts, 0.1, "causal")
    check(o, lse, want, want_lse, size, [5000], torch.bfloat16, 4, 5.0)
    dense_k, dense_v = fsta.read_paged_kv(cache, table.cuda(), lens.cuda(), 5000)
    assert torch.equal(dense_k[0, 0].cpu(), tail[0][1:, 0].reshape(-1, d)[:5000])
    rows = torch.randn((2, heads, d), generator=g).to(torch.bfloat16)
    fsta.write_paged_kv(cache, rows.cuda(), rows.cuda(), table.cuda(), lens.cuda(), starts.cuda())
    assert torch.equal(k[-1, 0, 4998 - 4096:5000 - 4096].cpu(), rows[:, 0]) and torch.equal(v[-1, 0, 902:904].cpu(), rows[:, 0])


def test_results_do_not_change_from_call_to_call():
    """The same call gives the same bits, also where keys are cut into runs."""
    tab, lens, starts, pages = make_batch([1, 70], [9000, 3000], 16, 1)
    cache = cuda(make_cache(pages, 2, 16, 128, torch.bfloat16, 2))
    q = torch.randn((71, 8, 128), generator=torch.Generator().manual_seed(3)).bfloat16().cuda()
    args = (q, cache, tab.cuda(), lens.cuda(), starts.cuda(), 0.09)
    first = fsta.paged_attention(*args, max_q_len=70, return_lse=True)
    for _ in range(3):
        again = fsta.paged_attention(*args, max_q_len=70, return_lse=True)
        assert all(torch.equal(a, b) for a, b in zip(first, again))


def test_parts_of_the_keys_join_to_the_whole():
    """Attention over the pages without the new tokens, joined with the tree part of ``fst_attention``."""
    n, prefix, heads, d = 64, 500, 4, 128
    parent = trees.random_recursive_parents(n, 4, window=16)
    g = torch.Generator().manual_seed(9)
    q, k, v = (torch.randn((n, heads, d), generator=g).bfloat16().cuda() for _ in range(3))
    tab, lens, starts, pages = make_batch([n], [prefix + n], 16, 3)
    cache = cuda(make_cache(pages, heads, 16, d, torch.bfloat16, 4))
    tab, lens, starts = tab.cuda(), lens.cuda(), starts.cuda()
    fsta.write_paged_kv(cache, k, v, tab, lens, starts)
    bits = fsta.tree_mask_bits(torch.from_numpy(parent).cuda())
    scale = 1.0 / math.sqrt(d)
    whole = fsta.paged_attention(q, cache, tab, lens, starts, scale, tree_bits=bits)
    front = fsta.paged_attention(q, cache, tab, lens - n, starts, scale, causal=False, return_lse=True)
    dense = [t.transpose(0, 1).contiguous()[None] for t in (q, k, v)]
    lineage, level = trees.lineage_from_parents(parent)
    max_anc = trees.required_max_ancestors(parent, 64)
    inputs = fsta.create_fst_attention_kernel_inputs(lineage.cuda(), level.cuda(), 64, max_anc)
    tree = fsta.fst_attention(*dense, *inputs, scale, BLOCK_M=64, MAX_ANCESTORS=max_anc, return_lse=True)
    front_o, front_lse = front[0].transpose(0, 1).contiguous()[None], front[1].t().contiguous()
    joined, _ = fsta.merge_attention_states(front_o, front_lse, tree[0], tree[1])
    want = whole.transpose(0, 1)[None].double()
    # three roundings to bfloat16 (both parts and the join) and the whole's own
    assert bool(((joined.double() - want).abs() <= 4 * 2.0 ** -8 * (want.abs() + 1.0)).all())


def test_other_streams_and_graphs():
    tab, lens, starts, pages = make_batch([1, 4, 2], [900, 77, 2], 16, 6)
    cache = cuda(make_cache(pages, 2, 16, 64, torch.bfloat16, 7))
    g = torch.Generator().manual_seed(8)
    q, k, v = (torch.randn((7, h, 64), generator=g).bfloat16().cuda() for h in (8, 2, 2))
    parent = torch.tensor([-1, -1, 0, 0, 1, -1, 0]).cuda()
    tab, lens, starts = tab.cuda(), lens.cuda(), starts.cuda()

    def step():
        bits = fsta.tree_mask_bits(parent, starts, 4)
        fsta.write_paged_kv(cache, k, v, tab, lens, starts)
        return fsta.paged_attention(q, cache, tab, lens, starts, 0.125, tree_bits=bits, max_q_len=4), fsta.read_paged_kv(cache, tab, lens, 900)[1]
    want = step()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(want[0], got[0]) and torch.equal(want[1], got[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for i in range(4):
        q.copy_(torch.randn(q.shape, generator=g).bfloat16())
        k.copy_(torch.randn(k.shape, generator=g).bfloat16())
        graph.replay()
        torch.cuda.synchronize()
        replayed = [t.clone() for t in got]
        eager = step()
        assert torch.equal(eager[0], replayed[0]) and torch.equal(eager[1], replayed[1]), i


# ---- writing and reading ------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("new,keys,heads,page", [([1], [1], 1, 16), ([1, 1, 1], [16, 17, 40], 8, 16), ([70, 3, 0, 9], [100, 3, 50, 64], 3, 64),
                                                 ([2] * 100, list(range(2, 102)), 2, 32)])
def test_write_and_read(new, keys, heads, page, fp8, dtype, d):
    tab, lens, starts, pages = make_batch(new, keys, page, 31)
    cache = make_cache(pages, heads, page, d, dtype, 32, fp8)
    tokens = sum(new)
    g = torch.Generator().manual_seed(33)
    fused = (torch.randn((tokens, 3, heads, d), generator=g) * torch.logspace(-3, 3, tokens)[:, None, None, None]).to(dtype)
    k, v = fused[:, 1], fused[:, 2]
    want = [t.clone() if t is not None else None for t in cache]
    (k8, ke), (v8, ve) = quantise(k), quantise(v)
    for b in range(len(new)):
        for i in range(new[b]):
            t, pos = int(starts[b]) + i, keys[b] - new[b] + i
            page_id, row = int(tab[b, pos // page]), pos % page
            if fp8:
                want[0].view(torch.uint8)[page_id, :, row], want[1].view(torch.uint8)[page_id, :, row] = k8[t].view(torch.uint8), v8[t].view(torch.uint8)
                want[2][page_id, :, row], want[3][page_id, :, row] = ke[t], ve[t]
            else:
                want[0][page_id, :, row], want[1][page_id, :, row] = k[t], v[t]
    dev, got = fused.cuda(), cuda(cache)
    fsta.write_paged_kv(got, dev[:, 1], dev[:, 2], tab.cuda(), lens.cuda(), starts.cuda())
    for a, b in zip(got, want):
        if a is not None:
            assert torch.equal(a.cpu().view(torch.uint8 if fp8 else torch.int16), b.view(torch.uint8 if fp8 else torch.int16))
    for max_len in (max(keys), max(keys) + 5, max(1, max(keys) // 2)):
        dense = fsta.read_paged_kv(got, tab.cuda(), lens.cuda(), max_len, dtype=dtype)
        for out, pool, e in zip(dense, want[:2], want[2:]):
            full = torch.zeros((len(new), heads, max_len, d), dtype=torch.float64)
            for b in range(len(new)):
                rows, _ = rows_of(pool, e, tab, b, keys[b], page)
                full[b, :, :min(keys[b], max_len)] = rows[:, :max_len]
            assert torch.equal(out.cpu(), full.to(dtype))


def test_write_leaves_out_tokens_without_a_place():
    page, heads, d = 16, 2, 64
    tab, lens, starts, pages = make_batch([20, 5], [12, 40], page, 41)
    tab[1, 2] = -1                       # positions 32 .. 39 of sequence 1: all its new ones
    cache = cuda(make_cache(pages, heads, page, d, torch.bfloat16, 42))
    before = [cache.k.clone(), cache.v.clone()]
    rows = torch.ones((25, heads, d), dtype=torch.bfloat16, device="cuda")
    fsta.write_paged_kv(cache, rows, rows, tab.cuda(), lens.cuda(), starts.cuda())
    for pool, old in zip((cache.k, cache.v), before):
        changed = (pool != old).any(-1).any(1)
        assert int(changed.sum()) == 12 and bool(changed[int(tab[0, 0]), :12].all())
    # arrays that say more than the tensors hold
    bad_starts = torch.tensor([0, 9, 1 << 30], dtype=torch.int32).cuda()
    bad_lens = torch.tensor([1 << 30, -5], dtype=torch.int32).cuda()
    fsta.write_paged_kv(cache, rows, rows, tab.cuda(), bad_lens, bad_starts)
    o = fsta.paged_attention(torch.ones((25, 2, d), dtype=torch.bfloat16, device="cuda"), cache, tab.cuda(), bad_lens, bad_starts, 0.1)
    dense = fsta.read_paged_kv(cache, tab.cuda(), bad_lens, 100)
    torch.cuda.synchronize()
    assert bool(torch.isfinite(o[:9].float()).all()) and float(dense[0][1].abs().max()) == 0.0


@pytest.mark.parametrize("dtype", HALF)
def test_quantised_rows_at_the_ends_of_the_range(dtype):
    """Zeros, one value, exact powers of two and 448, infinities and NaN, the largest and smallest magnitudes."""
    info = torch.finfo(dtype)
    rows = torch.zeros((12, 1, 64))
    rows[1, 0, 5] = -3.0
    rows[2, 0] = 448.0
    rows[3, 0, :] = 449.0 if dtype == torch.float16 else 450.0
    rows[4, 0, ::2] = info.max
    rows[5, 0, 1::2] = info.tiny
    rows[6, 0] = torch.linspace(-1, 1, 64)
    rows[6, 0, 3] = math.inf
    rows[7, 0] = torch.linspace(-1, 1, 64)
    rows[7, 0, 9], rows[7, 0, 11] = math.nan, -math.inf
    rows[8, 0] = math.nan
    rows[9, 0] = torch.arange(64) * 2.0 ** -6
    rows[10, 0] = info.tiny * 2.0 ** -6 if dtype == torch.bfloat16 else 2.0 ** -24
    rows[11, 0] = torch.logspace(-20, 0, 64, base=2.0)
    rows = rows.to(dtype)
    tab, lens, starts, pages = make_batch([12], [12], 16, 1)
    cache = fsta.paged_kv_cache(pages, 1, 16, 64, torch.float8_e4m3fn)
    fsta.write_paged_kv(cache, rows.cuda(), rows.cuda(), tab.cuda(), lens.cuda(), starts.cuda())
    want, e = quantise(rows)
    page = int(tab[0, 0])
    assert torch.equal(cache.k_exponent[page, 0, :12].cpu(), e[:, 0])
    got = cache.k[page, 0, :12].cpu().float()
    torch.testing.assert_close(got, want[:, 0].float(), rtol=0, atol=0, equal_nan=True)
    dense, _ = fsta.read_paged_kv(cache, tab.cuda(), lens.cuda(), 12, dtype=dtype)
    torch.testing.assert_close(dense[0, 0].cpu().double(), values(want, e)[:, 0].to(dtype).double(), rtol=0, atol=0, equal_nan=True)


# ---- masks of trees -----------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("dtype,d,new,keys", [(torch.bfloat16, 128, 5, 40), (torch.float16, 64, 20, 100), (torch.bfloat16, 64, 33, 33),
                                              (torch.float16, 128, 90, 300)])
def test_values_that_are_not_finite_reach_the_rows_that_see_them(dtype, d, new, keys, fp8):
    """A NaN and an infinity of either sign among the new tokens' values, at several head dims: rows that see the key get them,
    the others what they would have got without."""
    tab, lens, starts, pages = make_batch([new], [keys], 16, 50)
    cache = make_cache(pages, 1, 16, d, dtype, 51, fp8)
    clean = fsta.PagedKV(*(None if t is None else t.clone() for t in cache))
    place = lambda i: (int(tab[0, (keys - new + i) // 16]), 0, (keys - new + i) % 16)
    bad = {2: (7, math.nan), 3: (d - 1, math.nan if fp8 else math.inf), new - 1: (33, math.nan if fp8 else -math.inf)}
    for i, (col, x) in bad.items():
        if fp8:
            cache.v.view(torch.uint8)[(*place(i), col)] = 0x7f
        else:
            cache.v[(*place(i), col)] = x
    g = torch.Generator().manual_seed(52)
    q = torch.randn((new, 2, d), generator=g).to(dtype).cuda()
    sees = torch.ones((new, new), dtype=torch.bool).tril()
    sees[4] = False
    sees[4, 3:5] = True
    words = -(-new // 32)
    packed = torch.zeros((new, words * 32), dtype=torch.int64)
    packed[:, :new] = sees
    packed = (packed.view(new, words, 32) << torch.arange(32)).sum(-1)
    bits = torch.where(packed >= 1 << 31, packed - (1 << 32), packed).to(torch.int32).cuda()
    args = (tab.cuda(), lens.cuda(), starts.cuda(), 0.125)
    for kwargs, mask in (({}, torch.ones((new, new), dtype=torch.bool).tril()), ({"tree_bits": bits}, sees)):
        got = fsta.paged_attention(q, cuda(cache), *args, max_q_len=new, **kwargs).cpu()
        want = fsta.paged_attention(q, cuda(clean), *args, max_q_len=new, **kwargs).cpu()
        for i, (col, x) in bad.items():
            want[mask[:, i], :, col] = x
        torch.testing.assert_close(got, want, rtol=0, atol=0, equal_nan=True)


@pytest.mark.parametrize("nodes,window", [([1], 8), ([32, 33, 31], 4), ([64, 1, 200, 0, 7], 16), ([300], None), ([2048, 1000], 3)])
def test_tree_mask_bits(nodes, window):
    parents = [trees.random_recursive_parents(n, 5 + n, window=window) if n else torch.zeros(0).numpy() for n in nodes]
    starts = [0]
    for n in nodes:
        starts.append(starts[-1] + n)
    flat = torch.cat([torch.from_numpy(p).to(torch.int64) for p in parents]).cuda()
    bits = fsta.tree_mask_bits(flat, torch.tensor(starts, dtype=torch.int32).cuda(), max(nodes)).cpu()
    assert bits.shape == (sum(nodes), -(-max(nodes) // 32))
    unpacked = ((bits.long()[:, :, None] >> torch.arange(32)) & 1).bool().view(sum(nodes), -1)
    for b, p in enumerate(parents):
        want = torch.zeros((nodes[b], unpacked.shape[1]), dtype=torch.bool)
        want[:, :nodes[b]] = ancestors(p.tolist())
        assert torch.equal(unpacked[starts[b]:starts[b + 1]], want)


def test_tree_mask_bits_of_odd_inputs():
    """A chain of the largest depth, parents that are none, fewer words than nodes, tokens of no tree."""
    chain = torch.arange(-1, 999, dtype=torch.int64)
    bits = fsta.tree_mask_bits(chain.cuda()).cpu()
    unpacked = ((bits.long()[:, :, None] >> torch.arange(32)) & 1).view(1000, -1)[:, :1000]
    assert torch.equal(unpacked, torch.ones((1000, 1000), dtype=torch.int64).tril())
    odd = torch.tensor([-9, 0, 2, 77, 1 << 40, 4], dtype=torch.int64)
    assert fsta.tree_mask_bits(odd.cuda()).cpu()[:, 0].tolist() == [1, 3, 4, 8, 16, 48]
    few = fsta.tree_mask_bits(chain[:100].cuda(), max_nodes=40).cpu()
    assert few.shape == (100, 2) and few[99].tolist() == [-1, -1] and few[3].tolist() == [15, 0]
    part = fsta.tree_mask_bits(chain[:10].cuda(), torch.tensor([2, 5], dtype=torch.int32).cuda(), 32).cpu()[:, 0].tolist()
    assert part[:2] == [0, 0] and part[5:] == [0] * 5
    assert fsta.tree_mask_bits(torch.zeros(0, dtype=torch.int64).cuda()).shape == (0, 0)


# ---- refusals -----------------------------------------------------------------------------------------------------------

def test_refusals():
    tab, lens, starts, pages = (t.cuda() if torch.is_tensor(t) else t for t in make_batch([2, 1], [20, 3], 16, 1))
    cache = cuda(make_cache(pages, 2, 16, 64, torch.bfloat16, 2))
    q = torch.zeros((3, 4, 64), dtype=torch.bfloat16, device="cuda")
    k = torch.zeros((3, 2, 64), dtype=torch.bfloat16, device="cuda")
    attend = lambda **c: fsta.paged_attention(*{**dict(q=q, cache=cache, page_table=tab, kv_lens=lens, q_starts=starts, sm_scale=0.1), **c}.values())
    assert attend().shape == q.shape
    for change, word in ((dict(q=q.half()), "dtype"), (dict(q=q[:, :3]), "evenly"), (dict(q=q.float()), "float16"), (dict(q=q.cpu()), "device"),
                         (dict(q=torch.zeros((3, 4, 128), dtype=torch.bfloat16, device="cuda")), "head_dim"),
                         (dict(q=torch.zeros((3, 4, 68), dtype=torch.bfloat16, device="cuda")[..., 4:]), "aligned"),
                         (dict(q=torch.zeros((3, 64, 4), dtype=torch.bfloat16, device="cuda").transpose(1, 2)), "contiguous"),
                         (dict(page_table=tab.long()), "int32"), (dict(kv_lens=lens[:1]), "batch"), (dict(q_starts=starts[:2]), "batch"),
                         (dict(kv_lens=lens.cpu()), "device"), (dict(sm_scale=0.0), "positive"), (dict(sm_scale=float("nan")), "positive"),
                         (dict(sm_scale=-1.0), "positive"), (dict(cache=fsta.PagedKV(cache.k, cache.v[:1])), "one shape"),
                         (dict(cache=fsta.PagedKV(cache.k.float(), cache.v.float())), "float8"),
                         (dict(cache=fsta.PagedKV(cache.k.cpu(), cache.v.cpu())), "GPU"),
                         (dict(cache=fsta.PagedKV(cache.k.transpose(1, 2), cache.v.transpose(1, 2))), "contiguous"),
                         (dict(cache=fsta.PagedKV(cache.k, cache.v, tab, tab)), "8-bit"),
                         (dict(cache=fsta.PagedKV(cache.k.to(torch.float8_e4m3fn), cache.v.to(torch.float8_e4m3fn))), "exponent"),
                         (dict(q=q.clone().requires_grad_()), "backward")):
        with pytest.raises(ValueError, match=word):
            attend(**change)
    for bits in (torch.zeros((3, 1), device="cuda"), torch.zeros((2, 1), dtype=torch.int32, device="cuda"), torch.zeros((3, 1), dtype=torch.int32)):
        with pytest.raises(ValueError, match="tree_bits"):
            fsta.paged_attention(q, cache, tab, lens, starts, 0.1, tree_bits=bits)
    with pytest.raises(ValueError, match="pages"):
        fsta.paged_attention(q, cuda(fsta.PagedKV(cache.k[:0], cache.v[:0])), tab, lens, starts, 0.1)
    with pytest.raises(ValueError, match="one dtype"):
        fsta.write_paged_kv(cache, k, k[:2], tab, lens, starts)
    with pytest.raises(ValueError, match="dtype"):
        fsta.write_paged_kv(cache, k.half(), k.half(), tab, lens, starts)
    with pytest.raises(ValueError, match="dtype"):
        fsta.read_paged_kv(cache, tab, lens, 10, dtype=torch.float16)
    with pytest.raises(ValueError, match="max_len"):
        fsta.read_paged_kv(cache, tab, lens, -1)
    for size in (8, 24, 8192):
        odd = fsta.paged_kv_cache(2, 1, size, 64)
        with pytest.raises(fsta._lib.FstaError, match="page_size"):
            fsta.read_paged_kv(odd, tab[:, :1].contiguous(), lens, 4)
    with pytest.raises(fsta._lib.FstaError, match="head_dim"):
        fsta.read_paged_kv(fsta.paged_kv_cache(2, 1, 16, 96), tab, lens, 4)
    for parent in (torch.zeros(3, device="cuda"), torch.zeros((3, 1), dtype=torch.int64, device="cuda")):
        with pytest.raises(ValueError, match="int64"):
            fsta.tree_mask_bits(parent)
    with pytest.raises(ValueError, match="GPU"):
        fsta.tree_mask_bits(torch.zeros(3, dtype=torch.int64))
    # nothing to do
    empty = torch.zeros((0, 4, 64), dtype=torch.bfloat16, device="cuda")
    assert fsta.paged_attention(empty, cache, tab, lens, torch.zeros_like(starts), 0.1).shape == empty.shape
    fsta.write_paged_kv(cache, k[:0], k[:0], tab, lens, torch.zeros_like(starts))
    assert fsta.read_paged_kv(cache, tab, lens, 0)[0].shape == (2, 2, 0, 64)
