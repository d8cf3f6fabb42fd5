"""What the paged operators refuse, through the C ABI and through Python, without a GPU: every refusal comes before a launch."""
import ctypes

import pytest
import torch

import fstattention_amd as fsta
from fstattention_amd import _lib

P = 1 << 20                       # a pointer that nothing follows: every call below ends in its checks

WRITE = dict(k=P, v=P, kts=256, khs=128, vts=256, vhs=128, k_cache=P, v_cache=P, k_exp=None, v_exp=None, table=P, lens=P, starts=P,
             batch=2, width=3, tokens=5, pages=9, page_size=16, kv_heads=2, d=128, dtype=_lib.BF16, cache_dtype=_lib.BF16, stream=None)
READ = dict(k_cache=P, v_cache=P, k_exp=None, v_exp=None, table=P, lens=P, k=P, v=P, batch=2, width=3, max_len=40, pages=9, page_size=16,
            kv_heads=2, d=128, dtype=_lib.BF16, cache_dtype=_lib.BF16, stream=None)
ATTEND = dict(q=P, qts=1024, qhs=128, k_cache=P, v_cache=P, k_exp=None, v_exp=None, table=P, lens=P, starts=P, bits=None, words=0, o=P,
              lse=None, batch=2, width=3, tokens=5, most=4, pages=9, page_size=16, heads=8, kv_heads=2, d=128, dtype=_lib.BF16,
              cache_dtype=_lib.BF16, mask=_lib.PAGED_CAUSAL, scale=0.1, work=P, work_bytes=1 << 40, stream=None)
BITS = dict(parent=P, starts=P, batch=2, tokens=5, words=1, bits=P, stream=None)

BOTH = [(dict(page_size=8), "page_size"), (dict(page_size=24), "page_size"), (dict(page_size=8192), "page_size"), (dict(d=96), "head_dim"),
        (dict(d=256), "head_dim"), (dict(dtype=_lib.FP8), "dtype"), (dict(dtype=_lib.F32), "dtype"), (dict(cache_dtype=_lib.F32), "cache_dtype"),
        (dict(cache_dtype=_lib.F16), "cache_dtype"), (dict(batch=-1), "batch"), (dict(width=-1), "width"), (dict(pages=-1), "num_pages"),
        (dict(kv_heads=0), "kv_heads"), (dict(kv_heads=20000, heads=20000), "kv_heads"), (dict(table=None), "null"), (dict(lens=None), "null"),
        (dict(table=P + 2), "aligned"), (dict(lens=P + 1), "aligned"), (dict(k_cache=None), "null"), (dict(v_cache=None), "null"),
        (dict(k_cache=P + 8), "aligned"), (dict(cache_dtype=_lib.FP8), "null"), (dict(width=1 << 20, page_size=4096), "keys in a sequence")]


def _refused(entry, base, change, word):
    lib = _lib.load()
    args = {**base, **{k: v for k, v in change.items() if k in base}}
    rc = getattr(lib, entry)(*args.values())
    assert rc in (_lib.EINVAL, _lib.EUNSUPPORTED)
    assert entry in lib.fsta_last_error().decode() and word in lib.fsta_last_error().decode()


@pytest.mark.parametrize("change,word", BOTH + [
    (dict(k=None), "null"), (dict(v=None), "null"), (dict(k=P + 8), "aligned"), (dict(kts=260), "aligned"), (dict(vhs=4), "aligned"),
    (dict(tokens=-1), "tokens"), (dict(starts=None), "null"), (dict(starts=P + 2), "aligned")])
def test_write(change, word):
    _refused("fsta_paged_write", WRITE, change, word)


@pytest.mark.parametrize("change,word", BOTH + [(dict(k=None), "null"), (dict(v=P + 4), "aligned"), (dict(max_len=-1), "max_len")])
def test_read(change, word):
    _refused("fsta_paged_read", READ, change, word)


@pytest.mark.parametrize("change,word", BOTH + [
    (dict(q=None), "null"), (dict(o=None), "null"), (dict(q=P + 8), "aligned"), (dict(qts=4), "aligned"), (dict(qhs=12), "aligned"),
    (dict(o=P + 2), "aligned"), (dict(lse=P + 2), "aligned"), (dict(heads=7), "heads"), (dict(heads=0), "heads"), (dict(mask=7), "mask"),
    (dict(scale=0.0), "sm_scale"), (dict(scale=-1.0), "sm_scale"), (dict(scale=float("nan")), "sm_scale"), (dict(scale=float("inf")), "sm_scale"),
    (dict(mask=_lib.PAGED_TREE, words=1), "tree_words"), (dict(words=-1), "tree_words"), (dict(bits=P + 1, words=1, mask=_lib.PAGED_TREE), "aligned"),
    (dict(batch=0), "no sequence"), (dict(pages=0), "pages"), (dict(width=0), "pages"), (dict(work=None), "workspace"),
    (dict(work_bytes=64), "workspace"), (dict(work=P + 4), "aligned"), (dict(tokens=1 << 28), "tokens"), (dict(starts=None), "null"),
    (dict(batch=70000), "batch")])
def test_attention(change, word):
    _refused("fsta_paged_attention", ATTEND, change, word)


@pytest.mark.parametrize("change,word", [(dict(parent=None), "null"), (dict(bits=None), "null"), (dict(starts=None), "null"), (dict(batch=-1), "batch"),
                                         (dict(tokens=-1), "tokens"), (dict(words=-1), "words"), (dict(batch=0), "no sequence"),
                                         (dict(parent=P + 4), "aligned"), (dict(bits=P + 2), "aligned"), (dict(words=1 << 27), "words")])
def test_tree_bits(change, word):
    _refused("fsta_tree_bits", BITS, change, word)


def test_nothing_to_do_is_no_error():
    lib = _lib.load()
    for entry, base, change in (("fsta_paged_write", WRITE, dict(tokens=0, k=None)), ("fsta_paged_write", WRITE, dict(pages=0, k_cache=None)),
                                ("fsta_paged_read", READ, dict(max_len=0, k=None)), ("fsta_paged_attention", ATTEND, dict(tokens=0, q=None)),
                                ("fsta_tree_bits", BITS, dict(tokens=0)), ("fsta_tree_bits", BITS, dict(words=0, bits=None))):
        assert getattr(lib, entry)(*{**base, **change}.values()) == _lib.OK, entry


def test_workspace():
    """Big enough for any width of the page table, 0 for nothing; more tokens never need less."""
    lib = _lib.load()
    size = lambda batch, tokens, most, heads, kv_heads, d, dtype: lib.fsta_paged_attention_workspace_bytes(batch, tokens, most, heads, kv_heads, d, dtype)
    assert size(0, 0, 0, 8, 2, 128, _lib.BF16) == 0 and size(1, 1, 1, 7, 2, 128, _lib.BF16) == 0
    for d in (64, 128):
        for heads, kv_heads in ((8, 8), (8, 2), (64, 8), (28, 4)):
            sizes = [size(1, n, n, heads, kv_heads, d, _lib.BF16) for n in (1, 8, 64, 512, 4096)]
            assert all(a > 0 for a in sizes) and sizes[0] < sizes[-1] < 1 << 30


def test_python_refuses_what_is_not_on_the_gpu():
    cache = fsta.PagedKV(*(torch.zeros((4, 2, 16, 64), dtype=torch.bfloat16) for _ in range(2)))
    table, lens, starts = torch.zeros((1, 2), dtype=torch.int32), torch.ones(1, dtype=torch.int32), torch.tensor([0, 1], dtype=torch.int32)
    rows = torch.zeros((1, 2, 64), dtype=torch.bfloat16)
    for call in (lambda: fsta.write_paged_kv(cache, rows, rows, table, lens, starts), lambda: fsta.read_paged_kv(cache, table, lens, 4),
                 lambda: fsta.paged_attention(rows, cache, table, lens, starts, 0.1), lambda: fsta.tree_mask_bits(torch.zeros(3, dtype=torch.int64))):
        with pytest.raises(ValueError, match="GPU"):
            call()
    with pytest.raises(ValueError, match="float8"):
        fsta.paged_kv_cache(4, 2, 16, 64, torch.float32, device="cpu")
    eight = fsta.paged_kv_cache(4, 2, 16, 64, torch.float8_e4m3fn, device="cpu")
    assert eight.k_exponent.shape == (4, 2, 16) and int(eight.k_exponent[0, 0, 0]) == 127
