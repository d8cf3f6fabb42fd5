"""The operators of the paged KV cache at the ends of what they accept."""
import types

import pytest
import torch

import fstattention_amd as fsta
from test_gpu_paged import check, cuda, make_batch, make_cache, reference, values

pytestmark = pytest.mark.gpu


def test_masks_wider_than_32_bits_count():
    """64 nodes of 2^25 words: the words of a workgroup's rows are 2^31 in number.  Memory that held something else before."""
    nodes, most = 64, 1 << 30
    dirty = torch.full((nodes, most // 32), -1, dtype=torch.int32, device="cuda")
    del dirty
    bits = fsta.tree_mask_bits(torch.arange(-1, nodes - 1).cuda(), torch.tensor([0, nodes], dtype=torch.int32).cuda(), most)
    assert bits.shape == (nodes, most // 32)
    chain = [(2 << i) - 1 for i in range(nodes)]
    signed = lambda x: x - (1 << 32) if x >> 31 else x
    assert bits[:, :2].tolist() == [[signed(x & 0xffffffff), signed(x >> 32)] for x in chain]
    for row in bits:
        assert int(row[2:].count_nonzero()) == 0


@pytest.mark.parametrize("most", [-1, 1 << 31, 1 << 37])
def test_more_nodes_than_a_tree_can_have_are_refused(most):
    """2^37 nodes are 2^32 words, which the library's 32-bit count would take for none."""
    with pytest.raises(ValueError, match="max_nodes"):
        fsta.tree_mask_bits(torch.zeros(1, dtype=torch.int64).cuda(), max_nodes=most)


# ---- float16 queries over 8-bit rows of any range ------------------------------------------------------------------------
# Rows written from bfloat16 may be larger than float16 holds; the queries and the result are float16.  Tolerances: those of
# test_gpu_paged.check, per unit of the attention over |v| (the largest value here is 4.5 * 2^17).

def _wide_batch(new, keys, columns, seed):
    """A batch whose page table is as wide as a server's: `columns` more that no sequence uses"""
    tab, lens, starts, pages = make_batch(new, keys, 16, seed)
    return torch.cat([tab, torch.full((len(new), columns), -1, dtype=torch.int32)], 1), lens, starts, pages


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("new,columns", [([1, 1], 0), ([15, 9], 0), ([500, 70], 1000)])
def test_float16_queries_over_large_8_bit_values(d, new, columns):
    """Every 50th key's values beyond float16's range: the weighted means are within it, at every size of tile."""
    keys = [700, 333]
    tab, lens, starts, pages = _wide_batch(new, keys, columns, 61)
    cache = make_cache(pages, 2, 16, d, torch.bfloat16, 62, fp8=True)
    cache.v_exponent[:, :, 5] += torch.where(torch.arange(pages) % 3 == 0, 17, 0).to(torch.uint8)[:, None]
    q = (torch.randn((sum(new), 8, d), generator=torch.Generator().manual_seed(63)) * 0.5).half()
    out, lse = fsta.paged_attention(q.cuda(), cuda(cache), tab.cuda(), lens.cuda(), starts.cuda(), d ** -0.5, causal=False, max_q_len=max(new),
                                    return_lse=True)
    want, want_lse, size = reference(q, cache, tab, lens, starts, d ** -0.5, "all")
    assert want.abs().max() > 500 and out.isfinite().all()
    check(out, lse, want, want_lse, size, keys, torch.float16, max(new) * 4, 0.0)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("new,columns", [([1, 1], 0), ([15, 9], 0), ([500, 70], 1000)])
@pytest.mark.parametrize("power", [17, -30])
def test_float16_queries_over_8_bit_keys_of_any_range(power, d, new, columns):
    """Keys beyond float16's range, or below its smallest numbers, whose scores are ordinary: sm_scale makes up for it."""
    keys = [700, 333]
    tab, lens, starts, pages = _wide_batch(new, keys, columns, 64)
    cache = make_cache(pages, 2, 16, d, torch.bfloat16, 65, fp8=True)
    cache.k_exponent.copy_((cache.k_exponent.int() + power).to(torch.uint8))
    q = torch.randn((sum(new), 8, d), generator=torch.Generator().manual_seed(66)).half()
    scale = d ** -0.5 * 2.0 ** -power
    out, lse = fsta.paged_attention(q.cuda(), cuda(cache), tab.cuda(), lens.cuda(), starts.cuda(), scale, max_q_len=max(new), return_lse=True)
    want, want_lse, size = reference(q, cache, tab, lens, starts, scale, "causal")
    check(out, lse, want, want_lse, size, keys, torch.float16, max(new) * 4, 0.0)


# ---- gradients and what autograd keeps --------------------------------------------------------------------------------------

def _small_call():
    tab, lens, starts, pages = (t.cuda() if torch.is_tensor(t) else t for t in make_batch([2, 1], [20, 3], 16, 71))
    cache = cuda(make_cache(pages, 2, 16, 64, torch.bfloat16, 72))
    q, k = (torch.randn((3, h, 64), device="cuda").bfloat16() for h in (4, 2))
    return cache, tab, lens, starts, q, k


def _without_plain_calls(monkeypatch):
    """Every call through the checks in Python"""
    calls = types.SimpleNamespace(**{name: lambda *args: NotImplemented for name in ("paged_attention", "paged_read", "paged_write", "tree_bits")})
    monkeypatch.setattr("fstattention_amd.paged._calls", lambda: calls)


@pytest.mark.parametrize("which", ["k", "v"])
def test_a_cache_that_requires_a_gradient_is_refused(which):
    """A learned prefix among the pages: no operator has a backward pass, so none takes it for one that has."""
    cache, tab, lens, starts, q, k = _small_call()
    learned = cache._replace(**{which: getattr(cache, which).clone().requires_grad_()})
    calls = (lambda: fsta.write_paged_kv(learned, k, k, tab, lens, starts), lambda: fsta.read_paged_kv(learned, tab, lens, 20),
             lambda: fsta.paged_attention(q, learned, tab, lens, starts, 0.1))
    for call in calls:
        with pytest.raises(ValueError, match="backward"):
            call()
        with torch.no_grad():
            call()


def test_tangents_are_refused():
    """Forward-mode derivatives of new rows or of the cache: dropped without a word otherwise."""
    from torch.autograd import forward_ad
    cache, tab, lens, starts, q, k = _small_call()
    with forward_ad.dual_level():
        dual = lambda t: forward_ad.make_dual(t.clone(), torch.ones_like(t))
        learned = cache._replace(v=dual(cache.v))
        calls = (lambda: fsta.paged_attention(dual(q), cache, tab, lens, starts, 0.1), lambda: fsta.write_paged_kv(cache, dual(k), k, tab, lens, starts),
                 lambda: fsta.write_paged_kv(cache, k, dual(k), tab, lens, starts), lambda: fsta.paged_attention(q, learned, tab, lens, starts, 0.1),
                 lambda: fsta.write_paged_kv(learned, k, k, tab, lens, starts), lambda: fsta.read_paged_kv(learned, tab, lens, 20))
        for call in calls:
            with pytest.raises(ValueError, match="tangent"):
                call()
        fsta.write_paged_kv(cache, k, k, tab, lens, starts)
        assert fsta.paged_attention(q, cache, tab, lens, starts, 0.1).shape == q.shape


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("plain_call", [True, False])
def test_writing_moves_the_version_counters(plain_call, fp8, monkeypatch):
    """Autograd notices that a tensor it has kept for a backward pass was written to; inference tensors have no counter."""
    cache, tab, lens, starts, q, k = _small_call()
    if not plain_call:
        _without_plain_calls(monkeypatch)
    if fp8:
        cache = fsta.paged_kv_cache(*cache.k.shape, torch.float8_e4m3fn)
    before = [t._version for t in cache if t is not None]
    fsta.write_paged_kv(cache, k, k, tab, lens, starts)
    assert [t._version for t in cache if t is not None] == [n + 1 for n in before]
    if not fp8:
        w = torch.ones_like(cache.k).requires_grad_()
        kept = (w * cache.k).sum()
        fsta.write_paged_kv(cache, k, k, tab, lens, starts)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            kept.backward()
    with torch.inference_mode():
        fresh = fsta.paged_kv_cache(*cache.k.shape, cache.k.dtype)
        fsta.write_paged_kv(fresh, k, k, tab, lens, starts)
    got, want = (fsta.read_paged_kv(c, tab, lens, 20)[0][0, :, 18:] for c in (fresh, cache))
    assert torch.equal(got, want) and got.abs().amax() > 0


def test_masks_of_one_tree_in_a_captured_call():
    """Without ``q_starts`` the operator makes them itself, on the GPU: nothing comes from the host, so a capture takes it."""
    parent = torch.tensor([-1, 0, 0, 1, 2, 2, 4, -1]).cuda()
    want = fsta.tree_mask_bits(parent)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = fsta.tree_mask_bits(parent)
    for shift in range(4):
        parent.copy_(torch.tensor([-1, 0, 0, 1, 2, 2, 4, -1]).roll(shift))
        got.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, fsta.tree_mask_bits(parent)), shift
        assert shift > 0 or torch.equal(got, want)


@pytest.mark.parametrize("tokens,most", [(200, None), (200, 0), (300, None), (300, 300), (1, None), (40, 3)])
def test_slots_without_new_tokens(tokens, most):
    """A server's fixed slots, one of which brings a chunk, without a word about its length (or with a wrong one)."""
    new, keys = [0] * 256, [16] * 256
    new[7], keys[7] = tokens, 500 + tokens
    tab, lens, starts, pages = make_batch(new, keys, 16, 81)
    cache = make_cache(pages, 2, 16, 64, torch.bfloat16, 82)
    q = torch.randn((tokens, 8, 64), generator=torch.Generator().manual_seed(83)).bfloat16()
    out, lse = fsta.paged_attention(q.cuda(), cuda(cache), tab.cuda(), lens.cuda(), starts.cuda(), 0.125, max_q_len=most, return_lse=True)
    want, want_lse, size = reference(q, cache, tab, lens, starts, 0.125, "causal")
    check(out, lse, want, want_lse, size, keys, torch.bfloat16, tokens * 4, 5.0)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("new,columns", [([1, 1], 0), ([15, 9], 0), ([500, 70], 1000)])
def test_values_as_large_as_documented(new, columns, fp8):
    """Values up to 1e24, whose weights grow along the keys: the float32 sums in front of the division by the weights' sum hold them."""
    keys = [700, 333]
    tab, lens, starts, pages = _wide_batch(new, keys, columns, 91)
    cache = make_cache(pages, 2, 16, 128, torch.bfloat16, 92, fp8)
    if fp8:
        cache.v_exponent.copy_((cache.v_exponent.int() + 77).to(torch.uint8))
    else:
        cache.v.mul_(2.0 ** 77)
    # (scores of the later keys are greater by up to 7: the running maximum is raised from 8 powers of two on)
    q = (torch.randn((sum(new), 8, 128), generator=torch.Generator().manual_seed(93)) * 0.5).bfloat16()
    for b in range(2):
        for p in range(keys[b]):
            place = (int(tab[b, p // 16]), slice(None), p % 16)
            if not fp8:
                cache.k[place] = cache.k[place] * (0.1 + 2.0 * p / keys[b])
    assert values(cache.v, cache.v_exponent).abs().max() < 1e24
    out, lse = fsta.paged_attention(q.cuda(), cuda(cache), tab.cuda(), lens.cuda(), starts.cuda(), 128 ** -0.5, max_q_len=max(new), return_lse=True)
    want, want_lse, size = reference(q, cache, tab, lens, starts, 128 ** -0.5, "causal")
    assert want.abs().max() > 2.0 ** 70 and out.isfinite().all()
    check(out, lse, want, want_lse, size, keys, torch.bfloat16, max(new) * 4, 0.0)
