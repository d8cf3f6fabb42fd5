"""The page table's operators (fit_pages, fork_pages), rows of accepted paths moved together (compact_paged_kv) and pages copied
(copy_pages), against the host's account of them: everything is equal to the bit, what no call names included."""
import random

import numpy as np
import pytest
import torch

import fstattention_amd as fsta
from decoding_oracle import Server

pytestmark = pytest.mark.gpu

BF16, F16, FP8 = torch.bfloat16, torch.float16, torch.float8_e4m3fn


def make_pools(pages, page, layers, seed=0):
    """`layers`: (heads, head_dim, dtype) each; every byte is random."""
    g = torch.Generator().manual_seed(seed)
    out = []
    for heads, d, dtype in layers:
        size = 1 if dtype == FP8 else 2
        rows = [torch.randint(256, (pages, heads, page, d * size), generator=g, dtype=torch.uint8).cuda().view(dtype) for _ in range(2)]
        exponents = [torch.randint(256, (pages, heads, page), generator=g, dtype=torch.uint8).cuda() if dtype == FP8 else None for _ in range(2)]
        out.append(fsta.PagedKV(*rows, *exponents))
    return out


def bytes_of(caches):
    return [t.view(torch.uint8).cpu().numpy() for c in caches for t in c if t is not None]


def same(caches, server, table=None, refs=None, lens=None):
    for name, t, want in (("page_table", table, server.table), ("refs", refs, server.refs), ("lens", lens, server.lens)):
        if t is not None:
            np.testing.assert_array_equal(t.cpu().numpy(), want, err_msg=name)
    for i, (a, b) in enumerate(zip(bytes_of(caches), server.pools)):
        assert (a == b).all(), f"pool {i}: pages {np.unique(np.nonzero((a != b).reshape(len(a), -1).any(1))[0])[:10]}"


def int32(x):
    return torch.as_tensor(np.asarray(x), dtype=torch.int32).cuda()


def start(slots, width, pages, page, layers, seed=0):
    caches = make_pools(pages, page, layers, seed)
    table, refs, lens = np.full((slots, width), -1, np.int32), np.zeros(pages, np.int32), np.zeros(slots, np.int32)
    return caches, int32(table), int32(refs), int32(lens), Server(table, refs, lens, bytes_of(caches), page)


SMALL = [(2, 64, BF16)]
MIXED = [(2, 64, BF16), (3, 128, F16), (5, 128, FP8), (1, 64, FP8)]


@pytest.mark.parametrize("slots,width,pages,page,layers", [(1, 1, 1, 16, SMALL), (3, 5, 9, 16, MIXED), (7, 70, 300, 32, SMALL), (40, 9, 120, 64, MIXED),
                                                           (5, 200, 5000, 16, SMALL), (300, 3, 700, 16, SMALL), (2, 0, 4, 16, SMALL)])
def test_lengths_come_and_go(slots, width, pages, page, layers):
    """Rounds of random lengths, until pages run out and come back."""
    caches, table, refs, lens, server = start(slots, width, pages, page, layers)
    rng = random.Random(slots * 100 + pages)
    short = 0
    for round_ in range(8):
        most = width * page
        wanted = [rng.choice([0, most, rng.randint(0, most), rng.randint(0, most), -3, most + 40]) for _ in range(slots)]
        missing = fsta.fit_pages(caches if round_ % 2 else tuple(caches), refs, table, int32(wanted))
        np.testing.assert_array_equal(missing.cpu().numpy(), server.fit(wanted), err_msg=f"round {round_}")
        same(caches, server, table, refs)
        short += int(missing.sum())
    assert (short > 0) == (pages < slots * width) or slots == 1 or width == 0
    missing = fsta.fit_pages(caches, refs, table, int32([0] * slots))
    assert not refs.any() and (table == -1).all() and not missing.any()


@pytest.mark.parametrize("slots,width,pages,page,layers", [(2, 1, 3, 16, MIXED), (6, 5, 20, 16, MIXED), (30, 12, 500, 32, SMALL), (12, 90, 700, 16, SMALL),
                                                           (200, 4, 450, 64, [(1, 128, F16)])])
def test_forks_writes_and_lengths(slots, width, pages, page, layers):
    """Forks in random patterns (slots that are source and target at once, targets named twice, numbers outside the batch), lengths that
    grow and shrink into pages that others hold, until pages run out."""
    caches, table, refs, lens, server = start(slots, width, pages, page, layers, 1)
    rng = random.Random(slots + 7)
    most = width * page
    for round_ in range(10):
        pairs = rng.choice([1, slots, rng.randint(1, 2 * slots)])
        if round_ % 2 == 0:
            wanted = [rng.choice([int(n), rng.randint(0, most) if rng.random() < 0.5 else rng.randint(0, max(1, most // 4)), 0]) for n in server.lens]
            missing = fsta.fit_pages(caches, refs, table, int32(wanted))
            np.testing.assert_array_equal(missing.cpu().numpy(), server.fit(wanted), err_msg=f"round {round_}")
            server.lens[:] = wanted
            lens.copy_(int32(wanted))
        else:
            sources = [rng.randint(-1, slots) if rng.random() < 0.1 else rng.randrange(slots) for _ in range(pairs)]
            targets = [rng.randint(-1, slots) if rng.random() < 0.1 else rng.randrange(slots) for _ in range(pairs)]
            missing = fsta.fork_pages(caches, refs, table, lens, int32(sources), int32(targets))
            np.testing.assert_array_equal(missing.cpu().numpy(), server.fork(sources, targets), err_msg=f"round {round_}")
        same(caches, server, table, refs, lens)
        held = np.bincount(server.table[server.table >= 0], minlength=pages)
        np.testing.assert_array_equal(refs.cpu().numpy(), held, err_msg="a page is held as often as tables name it")


def test_beams_change_places():
    """A beam search's step: every slot goes on from another one, all at once."""
    caches, table, refs, lens, server = start(8, 6, 80, 16, MIXED, 2)
    for wanted in ([33, 96, 1, 0, 16, 47, 80, 95],):
        fsta.fit_pages(caches, refs, table, int32(wanted))
        server.fit(wanted)
        lens.copy_(int32(wanted))
        server.lens[:] = wanted
    for order in ([1, 0, 3, 2, 5, 4, 7, 6], [0, 0, 0, 0, 5, 5, 5, 5], [7, 6, 5, 4, 3, 2, 1, 0], [2, 3, 2, 3, 2, 3, 2, 3]):
        missing = fsta.fork_pages(caches, refs, table, lens, int32(order), int32(range(8)))
        np.testing.assert_array_equal(missing.cpu().numpy(), server.fork(order, range(8)))
        same(caches, server, table, refs, lens)


def test_entries_that_name_no_page():
    """Tables with garbage: entries outside the pool are as good as -1."""
    caches, table, refs, lens, server = start(4, 5, 12, 16, SMALL, 3)
    junk = np.array([[99, 3, -7, 2 ** 31 - 1, 4], [12, 13, 5, -1, -2 ** 31], [6, 7, 8, 50, 51], [-1, -1, -1, -1, -1]], np.int32)
    refs[3:9] = 1
    table.copy_(int32(junk))
    server.table[:], server.refs[3:9] = junk, 1
    for wanted in ([70, 40, 33, 17], [16, 0, 80, 80]):
        missing = fsta.fit_pages(caches, refs, table, int32(wanted))
        np.testing.assert_array_equal(missing.cpu().numpy(), server.fit(wanted))
        same(caches, server, table, refs)
    table.copy_(int32(junk))
    server.table[:] = junk
    lens.copy_(int32([70, 80, -5, 1000]))
    server.lens[:] = [70, 80, -5, 1000]
    missing = fsta.fork_pages(caches, refs, table, lens, int32([0, 1, 2, 3]), int32([1, 2, 3, 0]))
    np.testing.assert_array_equal(missing.cpu().numpy(), server.fork([0, 1, 2, 3], [1, 2, 3, 0]))
    same(caches, server, table, refs, lens)


def make_paths(rng, fresh, most):
    """Ascending node numbers from 0, one path per sequence; lengths from none to all."""
    path, counts = np.full((len(fresh), most), -1, np.int32), np.zeros(len(fresh), np.int32)
    for b, n in enumerate(fresh):
        if n == 0:
            continue
        count = min(rng.choice([1, 2, 5, n, rng.randint(1, n)]), n, most)
        nodes = sorted(rng.sample(range(1, n), count - 1)) if count > 1 else []
        path[b, :count], counts[b] = [0] + nodes, count
    return path, counts


@pytest.mark.parametrize("page", [16, 64, 256])
@pytest.mark.parametrize("layers", [SMALL, MIXED, [(1, 128, FP8)], [(9, 128, BF16)]])
def test_accepted_rows_move_together(page, layers):
    rng = random.Random(page)
    fresh = [0, 1, 2, 5, 16, 17, 40, 64, 65, 130, 200, 300, 7, 3]
    lens = [n + rng.choice([0, 1, 15, 16, 100, 333]) for n in fresh]
    width = max(-(-n // page) for n in lens) + 1
    caches, table, refs, _, server = start(len(fresh), width, sum(-(-n // page) for n in lens) + 3, page, layers, 4)
    fsta.fit_pages(caches, refs, table, int32(lens))
    server.fit(lens)
    order = torch.randperm(len(server.refs), generator=torch.Generator().manual_seed(1))          # not in the order they were given in
    table = torch.where(table >= 0, order.cuda().int()[table.long().clamp(min=0)], table)
    server.table = table.cpu().numpy().copy()
    starts = np.cumsum([0] + fresh)
    for most in (1, 6, 70, 300):
        path, counts = make_paths(rng, fresh, most)
        got = fsta.compact_paged_kv(caches, int32(path), int32(counts), table, int32(lens), int32(starts))
        np.testing.assert_array_equal(got.cpu().numpy(), server.compact(path, counts, lens, starts))
        same(caches, server)


def test_paths_counts_and_lengths_out_of_range():
    """Counts past a path or a tree, nodes that are none, lengths past the table, missing pages: nothing outside the rows concerned moves."""
    caches, table, refs, _, server = start(6, 4, 30, 16, MIXED, 5)
    lens = [40, 64, 30, 50, 10, 64]
    fsta.fit_pages(caches, refs, table, int32(lens))
    server.fit(lens)
    table[3, 2] = -1
    table[5, 3] = 77
    server.table[3, 2], server.table[5, 3] = -1, 77
    lens[1] = 1000
    starts = [0, 12, 30, 30, 55, 75, 90]                     # 12, 18, 0, 25, 20 (of 10), 15 new tokens
    path = np.array([[0, 5, 12, 90, 2 ** 31 - 1], [0, 3, 9, 17, -1], [0, 1, 2, 3, 4], [0, 7, 13, 20, 24], [0, 4, 8, 9, 15], [0, 9, 11, 13, 14]], np.int32)
    counts = [9, 4, 3, 5, 5, -2]
    got = fsta.compact_paged_kv(caches, int32(path), int32(counts), table, int32(lens), int32(starts))
    np.testing.assert_array_equal(got.cpu().numpy(), server.compact(path, counts, lens, starts))
    same(caches, server)
    counts[5] = 5
    got = fsta.compact_paged_kv(caches, int32(path), int32(counts), table, int32(lens), int32(starts))
    np.testing.assert_array_equal(got.cpu().numpy(), server.compact(path, counts, lens, starts))
    same(caches, server)
    got = fsta.compact_paged_kv(caches, int32(path[:, :0]), int32(counts), table, int32(lens), int32(starts))
    np.testing.assert_array_equal(got.cpu().numpy(), server.compact(path[:, :0], counts, lens, starts))


@pytest.mark.parametrize("layers", [SMALL, MIXED, [(7, 128, FP8)], [(3, 64, F16)] * 35])
@pytest.mark.parametrize("page", [16, 128])
def test_pages_are_copied(layers, page):
    pages = 40
    caches = make_pools(pages, page, layers, 6)
    want = bytes_of(caches)
    r = random.Random(page)
    places = r.sample(range(pages), 30)
    sources, targets = [r.choice(places[:12]) for _ in range(18)], places[12:]
    for p in want:
        p[targets] = p[sources]
    sources += [-1, 40, 3, 2 ** 31 - 1, 5]
    targets += [4, 4, -1, 4, 40]
    fsta.copy_pages(caches, int32(sources), int32(targets))
    for a, b in zip(bytes_of(caches), want):
        assert (a == b).all()
    fsta.copy_pages(caches, int32([7, 9]), int32([7, 9]))     # onto themselves
    fsta.copy_pages(caches, int32([]), int32([]))
    for a, b in zip(bytes_of(caches), want):
        assert (a == b).all()


def test_pages_go_to_a_larger_pool():
    caches, into = make_pools(20, 32, MIXED, 7), make_pools(50, 32, MIXED, 8)
    want, before = bytes_of(into), bytes_of(caches)
    sources, targets = list(range(20)), [2 * i + 7 for i in range(20)]
    for a, b in zip(want, before):
        a[targets] = b[sources]
    fsta.copy_pages(caches, int32(sources + [21, 3]), int32(targets + [0, 50]), into)
    fsta.copy_pages(caches, int32([5]), int32([5]), into)     # the same number, another pool
    for a, b in zip(want, before):
        a[5] = b[5]
    for a, b in zip(bytes_of(into) + bytes_of(caches), want + before):
        assert (a == b).all()


def test_many_layers_and_large_pages():
    caches, table, refs, lens, server = start(3, 2, 9, 1024, [(2, 64, F16)] * 70, 9)
    wanted = [1500, 2048, 0]
    fsta.fit_pages(caches, refs, table, int32(wanted))
    server.fit(wanted)
    lens.copy_(int32(wanted))
    server.lens[:] = wanted
    fsta.fork_pages(caches, refs, table, lens, int32([0]), int32([2]))
    server.fork([0], [2])
    same(caches, server, table, refs, lens)
    path, counts, starts = np.array([[0, 30, 77, 399], [0, 1, 2, 3], [0, -1, -1, -1]]), [4, 4, 1], [0, 400, 410, 415]
    got = fsta.compact_paged_kv(caches, int32(path), int32(counts), table, lens, int32(starts))
    np.testing.assert_array_equal(got.cpu().numpy(), server.compact(path, counts, server.lens, starts))
    same(caches, server)


def test_more_pages_than_one_wave_lists():
    """A pool of many groups of pages, almost all of them held: free ones are found far apart, and one sequence wants many."""
    pages, rng = 70001, np.random.default_rng(5)
    caches = make_pools(pages, 16, [(1, 64, FP8)], 10)
    refs = np.ones(pages, np.int32)
    refs[rng.choice(pages, 3000, replace=False)] = 0
    refs[20000:40000] = 1
    refs[2047:2049] = 0
    table, wanted = np.full((50, 2600), -1, np.int32), [16 * int(n) for n in rng.integers(0, 20, 50)]
    wanted[7], wanted[30] = 16 * 2500 - 3, 16 * 1000
    server = Server(table, refs, np.zeros(50, np.int32), bytes_of(caches), 16)
    table, refs = int32(table), int32(refs)
    missing = fsta.fit_pages(caches, refs, table, int32(wanted))
    np.testing.assert_array_equal(missing.cpu().numpy(), server.fit(wanted))
    assert int(missing.sum()) > 0
    same(caches, server, table, refs)


def test_far_pages():
    """Rows behind the 2^32nd element of a pool."""
    pages, shape = 270000, (2, 64, 128)                      # 16384 elements a page
    k, v = (torch.zeros((pages, *shape), dtype=BF16, device="cuda") for _ in range(2))
    assert k.numel() > 2 ** 32
    cache = fsta.PagedKV(k, v)
    k[3], v[3] = 1.5, 2.5
    fsta.copy_pages(cache, int32([3]), int32([pages - 1]))
    assert (k[pages - 1] == 1.5).all() and (v[pages - 1] == 2.5).all() and k[:3].sum() == 0
    v[pages - 1, 1, 40] = 7.0
    got = fsta.compact_paged_kv(cache, int32([[0, 30]]), int32([2]), int32([[pages - 1]]), int32([50]), int32([0, 40]))
    assert got.item() == 12 and (v[pages - 1, 1, 11] == 7.0).all() and (k[pages - 1, 0, 11] == 1.5).all() and (v[pages - 1, 0, 11] == 2.5).all()
    refs = torch.ones(pages, dtype=torch.int32, device="cuda")
    refs[pages - 2] = 0
    table, lens = int32([[pages - 1], [-1]]), int32([41, 0])
    missing = fsta.fork_pages(cache, refs, table, lens, int32([0]), int32([1]))
    assert missing.item() == 0 and table[1].item() == pages - 2 and refs[pages - 2].item() == 1 and lens.tolist() == [41, 41]
    assert (v[pages - 2, 1, 40] == 7.0).all() and (v[pages - 2, :, 41:] == 0).all()


def test_captured_and_replayed():
    """A step's room, its rows moved together and the room given back, as one graph over new lengths and paths each time."""
    caches, table, refs, lens, server = start(5, 8, 60, 16, MIXED, 11)
    first = [20, 3, 77, 16, 50]
    fsta.fit_pages(caches, refs, table, int32(first))
    server.fit(first)
    lens.copy_(int32(first))
    fresh, starts = 12, [12 * i for i in range(6)]
    path, counts, gpu_starts = int32(np.zeros((5, 4))), int32([1] * 5), int32(starts)

    def step():
        grown = lens + fresh
        a = fsta.fit_pages(caches, refs, table, grown)
        kept = fsta.compact_paged_kv(caches, path, counts, table, grown, gpu_starts)
        lens.copy_(kept)
        return a, fsta.fit_pages(caches, refs, table, lens)

    step()
    torch.cuda.synchronize()
    server.fit(np.array(first) + fresh)
    server.compact(np.zeros((5, 4)), [1] * 5, np.array(first) + fresh, starts)
    now = np.array(first) + 1
    server.fit(now)
    same(caches, server, table, refs)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    rng = random.Random(2)
    for turn in range(5):
        p, c = make_paths(rng, [fresh] * 5, 4)
        path.copy_(int32(p))
        counts.copy_(int32(c))
        if turn == 3:
            step()
        else:
            graph.replay()
        torch.cuda.synchronize()
        missing = server.fit(now + fresh)
        if turn != 3:
            np.testing.assert_array_equal(out[0].cpu().numpy(), missing)
        now = server.compact(p, c, now + fresh, starts).astype(np.int64)
        server.fit(now)
        np.testing.assert_array_equal(lens.cpu().numpy(), now)
        same(caches, server, table, refs)


def test_another_stream():
    caches, table, refs, lens, server = start(6, 10, 80, 16, MIXED, 12)
    wanted = [100, 20, 0, 0, 0, 60]
    stream = torch.cuda.Stream()
    args = [int32(x) for x in (wanted, [0, 1, 5], [2, 3, 4])]
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        fsta.fit_pages(caches, refs, table, args[0])
        lens.copy_(args[0])
        fsta.fork_pages(caches, refs, table, lens, args[1], args[2])
        fsta.copy_pages(caches, args[1], args[2] + 70)
    stream.synchronize()
    server.fit(wanted)
    server.lens[:] = wanted
    server.fork([0, 1, 5], [2, 3, 4])
    for p in server.pools:
        p[[72, 73, 74]] = p[[0, 1, 5]]
    same(caches, server, table, refs, lens)


def test_version_counters_move():
    caches, table, refs, lens, _ = start(2, 3, 9, 16, [(2, 64, BF16), (2, 64, FP8)], 13)
    tensors = [t for c in caches for t in c if t is not None]
    some = int32([0])

    def moved(call, *written):
        before = [t._version for t in tensors + [table, refs, lens]]
        call()
        for t, v in zip(tensors + [table, refs, lens], before):
            assert (t._version > v) == any(t is w for w in written)

    moved(lambda: fsta.fit_pages(caches, refs, table, lens), *tensors, table, refs)
    moved(lambda: fsta.fork_pages(caches, refs, table, lens, some, some), *tensors, table, refs, lens)
    moved(lambda: fsta.copy_pages(caches, some, some), *tensors)
    moved(lambda: fsta.copy_pages([caches[0]], some, some, into=[caches[0]]), *tensors[:2])
    moved(lambda: fsta.compact_paged_kv(caches, int32([[0], [0]]), int32([1, 1]), table, lens, int32([0, 1, 2])), *tensors)
    with torch.inference_mode():
        fsta.fit_pages(caches, refs, table, lens)


def test_refusals():
    caches, table, refs, lens, _ = start(2, 3, 9, 16, [(2, 64, BF16), (2, 64, FP8)], 14)
    pairs, starts, path = int32([0, 1]), int32([0, 1, 2]), int32([[0], [0]])
    fit = lambda **c: fsta.fit_pages(*{**dict(caches=caches, refs=refs, table=table, lens=lens), **c}.values())
    fork = lambda **c: fsta.fork_pages(*{**dict(caches=caches, refs=refs, table=table, lens=lens, sources=pairs, targets=pairs), **c}.values())
    copy = lambda **c: fsta.copy_pages(*{**dict(caches=caches, sources=pairs, targets=pairs, into=None), **c}.values())
    compact = lambda **c: fsta.compact_paged_kv(*{**dict(caches=caches, path=path, counts=pairs, table=table, lens=lens, starts=starts), **c}.values())
    other, larger = make_pools(9, 32, SMALL), make_pools(10, 16, SMALL)
    for call in (fit, fork, copy, compact):
        for bad, word in (([], "at least one"), (caches + other, "share"), (caches + larger, "share"), ([caches[0]._replace(k=caches[0].k.transpose(1, 2))], "must be"),
                          ([caches[1]._replace(k_exponent=None)], "exponent"), ([caches[0]._replace(k=caches[0].k.float(), v=caches[0].v.float())], "float16"),
                          ([fsta.PagedKV(caches[0].k.clone().requires_grad_(), caches[0].v)], "gradient")):
            with pytest.raises(ValueError, match=word):
                call(caches=bad)
    for call in (fit, fork):
        for change, word in ((dict(refs=refs[:8]), "refs"), (dict(refs=refs.long()), "refs"), (dict(table=table.long()), "page_table"), (dict(table=table[0]), "page_table"),
                             (dict(table=table.t().contiguous().t()), "page_table"), (dict(lens=lens[:1]), "lens"), (dict(lens=lens.cpu()), "lens")):
            with pytest.raises(ValueError, match=word):
                call(**change)
    for call in (fork, copy):
        for change, word in ((dict(sources=pairs[:1]), "targets"), (dict(sources=pairs.long()), "sources"), (dict(targets=pairs.cpu()), "targets"),
                             (dict(sources=path), "sources")):
            with pytest.raises(ValueError, match=word):
                call(**change)
    for change, word in ((dict(path=path[:1]), "path"), (dict(path=pairs), "path"), (dict(counts=pairs[:1]), "counts"), (dict(starts=pairs), "q_starts"),
                         (dict(lens=lens.float()), "kv_lens")):
        with pytest.raises(ValueError, match=word):
            compact(**change)
    for bad in ([caches[0], caches[1], caches[0]], [caches[0]._replace(v=caches[0].k)], [caches[0], caches[0]._replace(k=caches[0].v, v=caches[0].k)]):
        with pytest.raises(Exception, match="twice"):
            compact(caches=bad)
    for into, word in (([caches[0]], "layers"), (make_pools(9, 32, [(2, 64, BF16), (2, 64, FP8)]), "layers"), (make_pools(9, 16, [(2, 64, BF16), (3, 64, FP8)]), "layers"),
                       (make_pools(9, 16, [(2, 64, F16), (2, 64, FP8)]), "layers"), (make_pools(9, 16, [(2, 128, BF16), (2, 64, FP8)]), "layers")):
        with pytest.raises(ValueError, match=word):
            copy(into=into)


def test_no_sequences_and_no_pairs():
    caches, table, refs, lens, server = start(2, 3, 9, 16, MIXED, 15)
    none = int32([])
    assert fsta.fit_pages(caches, refs, table[:0], lens[:0]).shape == (0,)
    assert fsta.fork_pages(caches, refs, table, lens, none, none).shape == (0,)
    assert fsta.fork_pages(caches, refs, table[:0], lens[:0], int32([0]), int32([0])).tolist() == [0]
    assert fsta.compact_paged_kv(caches, int32(np.zeros((0, 3))), none, table[:0], lens[:0], int32([0])).shape == (0,)
    same(caches, server, table, refs, lens)
