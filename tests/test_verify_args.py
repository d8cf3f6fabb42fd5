"""What the operators between two passes of a model refuse, without a GPU: every refusal comes before a launch."""
import ctypes

import pytest
import torch

import fstattention_amd as fsta
from fstattention_amd import _lib

P = 1 << 20                       # a pointer that nothing follows: every call below ends in its checks

VERIFY = dict(logits=P, stride=100, dtype=_lib.BF16, draft=None, draft_stride=0, draft_dtype=_lib.F32, tokens=P, parent=P, starts=P, u_accept=P,
              u_next=P, temperatures=None, temperature=1.0, path=P, counts=P, next=P, batch=2, nodes=5, vocabulary=100, max_path=4,
              work=P, work_bytes=1 << 40, stream=None)
COMPACT = dict(pools=None, layers=2, pages=9, page_size=16, path=P, max_path=4, counts=P, table=P, lens=P, starts=P, batch=2, width=3, out=P, stream=None)
COPY = dict(pools=None, into=None, layers=2, pages=9, into_pages=9, page_size=16, sources=P, targets=P, pairs=3, stream=None)
FIT = dict(pools=None, layers=2, pages=9, page_size=16, refs=P, table=P, lens=P, batch=2, width=3, missing=P, work=P, work_bytes=1 << 40, stream=None)
FORK = dict(pools=None, layers=2, pages=9, page_size=16, refs=P, table=P, lens=P, batch=2, width=3, sources=P, targets=P, pairs=3, missing=P,
            work=P, work_bytes=1 << 40, stream=None)


def _pools(**change):
    pools = (_lib.PagedPool * 2)()
    for p in pools:
        p.k, p.v, p.kv_heads, p.head_dim, p.cache_dtype = P, P, 2, 64, _lib.BF16
    for name, value in change.items():
        setattr(pools[1], name, value)
    return pools


def _refused(entry, base, change, word, pool=None):
    lib = _lib.load()
    args = {**base, **{k: v for k, v in change.items() if k in base}}
    for name in ("pools", "into"):
        if name in base and name not in change:
            args[name] = _pools(**(pool or {}))
    rc = getattr(lib, entry)(*args.values())
    assert rc in (_lib.EINVAL, _lib.EUNSUPPORTED)
    assert entry in lib.fsta_last_error().decode() and word in lib.fsta_last_error().decode(), lib.fsta_last_error()


@pytest.mark.parametrize("change,word", [
    (dict(logits=None), "null"), (dict(tokens=None), "null"), (dict(parent=None), "null"), (dict(starts=None), "null"), (dict(u_accept=None), "null"),
    (dict(u_next=None), "null"), (dict(path=None), "null"), (dict(counts=None), "null"), (dict(next=None), "null"), (dict(batch=-1), "batch"),
    (dict(nodes=-1), "nodes"), (dict(vocabulary=0), "vocabulary"), (dict(vocabulary=2 ** 31 - 1), "vocabulary"), (dict(batch=2 ** 31 - 1), "batch"), (dict(max_path=0), "max_path"),
    (dict(dtype=_lib.FP8), "logits_dtype"), (dict(dtype=_lib.F64), "logits_dtype"), (dict(draft=P, draft_dtype=_lib.FP8), "draft_dtype"),
    (dict(temperature=-0.5), "temperature"), (dict(temperature=float("nan")), "temperature"), (dict(temperature=float("inf")), "temperature"),
    (dict(stride=-1), "stride"), (dict(draft=P, draft_stride=-4), "stride"), (dict(logits=P + 1), "aligned"), (dict(draft=P + 2), "aligned"),
    (dict(tokens=P + 4), "aligned"), (dict(next=P + 4), "aligned"), (dict(starts=P + 2), "aligned"), (dict(u_next=P + 1), "aligned"),
    (dict(temperatures=P + 2), "aligned")])
def test_verify(change, word):
    _refused("fsta_verify_drafts", VERIFY, change, word)


POOLS = [(dict(head_dim=96), "head_dim"), (dict(cache_dtype=_lib.F32), "cache_dtype"), (dict(kv_heads=0), "kv_heads"), (dict(kv_heads=20000), "kv_heads"),
         (dict(k=None), "null"), (dict(v=None), "null"), (dict(k=P + 8), "aligned"), (dict(cache_dtype=_lib.FP8), "null")]
SHARED = [(dict(layers=0), "layers"), (dict(pages=-1), "num_pages"), (dict(page_size=8), "page_size"), (dict(page_size=48), "page_size"),
          (dict(page_size=8192), "page_size"), (dict(pools=None), "null")]
TABLE = SHARED + [(dict(batch=-1), "batch"), (dict(width=-1), "width"), (dict(width=1 << 28), "keys in a sequence"), (dict(table=None), "null"),
                  (dict(lens=None), "null"), (dict(table=P + 2), "aligned"), (dict(lens=P + 1), "aligned")]


@pytest.mark.parametrize("entry,base", [("fsta_compact_paged_kv", COMPACT), ("fsta_copy_pages", COPY), ("fsta_fit_pages", FIT), ("fsta_fork_pages", FORK)])
@pytest.mark.parametrize("pool,word", POOLS)
def test_pools(entry, base, pool, word):
    _refused(entry, base, {}, word, pool)


@pytest.mark.parametrize("change,word", TABLE + [(dict(max_path=-1), "max_path"), (dict(path=None), "null"), (dict(counts=None), "null"),
                                                 (dict(starts=None), "null"), (dict(out=None), "null"), (dict(out=P + 2), "aligned"), (dict(path=P + 1), "aligned")])
def test_compact(change, word):
    _refused("fsta_compact_paged_kv", COMPACT, change, word)


@pytest.mark.parametrize("change,word", SHARED + [(dict(into=None), "null"), (dict(into_pages=-1), "into_pages"), (dict(pairs=-1), "pairs"),
                                                  (dict(sources=None), "null"), (dict(targets=None), "null"), (dict(sources=P + 2), "aligned")])
def test_copy(change, word):
    _refused("fsta_copy_pages", COPY, change, word)


def test_copy_between_unlike_layers():
    for change in (dict(kv_heads=4), dict(head_dim=128), dict(cache_dtype=_lib.F16)):
        _refused("fsta_copy_pages", COPY, dict(into=_pools(**change)), "another")


@pytest.mark.parametrize("entry,base", [("fsta_fit_pages", FIT), ("fsta_fork_pages", FORK)])
@pytest.mark.parametrize("change,word", TABLE + [(dict(refs=None), "null"), (dict(missing=None), "null"), (dict(refs=P + 2), "aligned"),
                                                 (dict(work=None), "workspace"), (dict(work=P + 4), "workspace"), (dict(work_bytes=64), "workspace")])
def test_tables(entry, base, change, word):
    _refused(entry, base, change, word)


def test_compact_with_a_pool_twice():
    for at in ((1, 2, 1, 3), (1, 2, 3, 2), (1, 2, 2, 3), (1, 2, 3, 1), (1, 1, 2, 3), (1, 2, 3, 3)):
        pools = _pools()
        for pool, k, v in zip(pools, at[::2], at[1::2]):
            pool.k, pool.v = k * P, v * P
        _refused("fsta_compact_paged_kv", COMPACT, dict(pools=pools), "twice")


def test_more_rows_than_31_bits_count():
    for entry, base, change, word in (("fsta_fit_pages", FIT, dict(batch=2 ** 31 - 1), "batch"), ("fsta_fit_pages", FIT, dict(batch=1 << 16, width=1 << 15), "width"),
                                      ("fsta_fork_pages", FORK, dict(batch=1 << 16, width=1 << 15), "width"), ("fsta_fork_pages", FORK, dict(pairs=(1 << 16) + 1), "pairs"),
                                      ("fsta_copy_pages", COPY, dict(pairs=2 ** 31 - 1), "pairs"), ("fsta_compact_paged_kv", COMPACT, dict(batch=(1 << 16) + 1), "batch")):
        _refused(entry, base, change, word)


@pytest.mark.parametrize("change,word", [(dict(sources=None), "null"), (dict(targets=None), "null"), (dict(targets=P + 1), "aligned"), (dict(pairs=-1), "pairs")])
def test_fork(change, word):
    _refused("fsta_fork_pages", FORK, change, word)


def test_nothing_to_do_is_no_error():
    lib = _lib.load()
    for entry, base, change in (("fsta_verify_drafts", VERIFY, dict(batch=0, path=None)), ("fsta_compact_paged_kv", COMPACT, dict(batch=0, path=None)),
                                ("fsta_copy_pages", COPY, dict(pairs=0, sources=None)), ("fsta_copy_pages", COPY, dict(pages=0)),
                                ("fsta_fit_pages", FIT, dict(batch=0, refs=None)), ("fsta_fork_pages", FORK, dict(pairs=0, refs=None))):
        args = {**base, **change}
        for name in ("pools", "into"):
            if name in args:
                args[name] = _pools()
        assert getattr(lib, entry)(*args.values()) == _lib.OK, entry


def test_workspaces():
    lib = _lib.load()
    assert lib.fsta_fit_pages_workspace_bytes(-1, 5) == 0 and lib.fsta_fork_pages_workspace_bytes(3, -1, 5) == 0
    assert 0 < lib.fsta_fit_pages_workspace_bytes(1, 1) < lib.fsta_fit_pages_workspace_bytes(1000, 1 << 20) < 1 << 20
    assert lib.fsta_fork_pages_workspace_bytes(10, 1000, 64) >= 40000
    assert ctypes.sizeof(_lib.PagedPool) == 48


def test_python_refuses_what_is_not_on_the_gpu():
    cache = fsta.PagedKV(*(torch.zeros((4, 2, 16, 64), dtype=torch.bfloat16) for _ in range(2)))
    table, lens, starts = torch.zeros((1, 2), dtype=torch.int32), torch.ones(1, dtype=torch.int32), torch.tensor([0, 1], dtype=torch.int32)
    refs, some = torch.zeros(4, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    for call in (lambda: fsta.compact_paged_kv(cache, table, some, table, lens, starts), lambda: fsta.copy_pages([cache], some, some),
                 lambda: fsta.fit_pages((cache,), refs, table, lens), lambda: fsta.fork_pages([tuple(cache)], refs, table, lens, some, some),
                 lambda: fsta.verify_drafts(torch.zeros((1, 5)), torch.zeros(1, dtype=torch.int64), torch.zeros(1, dtype=torch.int64), starts,
                                            torch.zeros(1), torch.zeros(1), 2)):
        with pytest.raises(ValueError, match="GPU"):
            call()
    with pytest.raises(ValueError, match="at least one"):
        fsta.fit_pages([], refs, table, lens)
