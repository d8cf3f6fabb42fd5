"""The operators of the paged KV cache where the first tests do not go: trees larger than shared memory, few rows on few keys,
infinities that every row sees."""
import math
import random

import pytest
import torch

import fstattention_amd as fsta

pytestmark = pytest.mark.gpu


def _pool(pages, heads, page_size, d, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    k, v = (torch.randn((pages, heads, page_size, d), generator=g).to(dtype) for _ in range(2))
    return fsta.PagedKV(k.cuda(), v.cuda(), None, None)


def _batch(new, keys, page_size, seed):
    """Page table, lengths, starts (int32, on the host) and the number of pages; pages in a random order, a few of them unused."""
    need = [-(-k // page_size) for k in keys]
    order = list(range(sum(need) + 3))
    random.Random(seed).shuffle(order)
    table = torch.full((len(keys), max(need)), -1, dtype=torch.int32)
    for b, n in enumerate(need):
        table[b, :n] = torch.tensor(order[:n], dtype=torch.int32)
        order = order[n:]
    starts = torch.tensor([0] + list(torch.tensor(new).cumsum(0)), dtype=torch.int32)
    return table, torch.tensor(keys, dtype=torch.int32), starts, sum(need) + 3


def _rows_of_bits(parent, words):
    """Rows of a tree's masks, from Python's integers"""
    rows = []
    for i, p in enumerate(parent):
        rows.append((1 << i) | (rows[p] if 0 <= p < i else 0))
    signed = lambda x: x - (1 << 32) if x >> 31 else x
    return torch.tensor([[signed((r >> (32 * w)) & 0xffffffff) for w in range(words)] for r in rows], dtype=torch.int32).reshape(len(parent), words)


@pytest.mark.parametrize("nodes,window,most", [([9000], None, 9000), ([8300, 40], 9, 8300), ([700, 3], 1, 40), ([1, 2, 33, 64, 65, 31], 4, 65),
                                               ([700, 10, 90], 30, 700), ([127, 129, 0, 0, 5], 2, 256), ([3000], 2, 96)])
def test_tree_mask_bits_of_large_trees(nodes, window, most):
    """Trees that shared memory does not hold, rows with fewer bits than their trees have nodes, and chains."""
    words, parent, want = -(-most // 32), [], []
    for at, n in enumerate(nodes):
        rng = random.Random(100 * at + n)
        tree = [-1] + [rng.randint(0 if window is None else max(0, i - window), i - 1) for i in range(1, n)] if n else []
        parent += tree
        want.append(_rows_of_bits(tree, words))
    starts = torch.tensor([0] + list(torch.tensor(nodes).cumsum(0)), dtype=torch.int32).cuda()
    got = fsta.tree_mask_bits(torch.tensor(parent).cuda(), starts, most).cpu()
    assert torch.equal(got, torch.cat(want))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("new,keys,group", [(1, 64, 1), (1, 1000, 4), (3, 200, 8), (40, 200, 8), (200, 900, 4)])
def test_infinities_that_every_row_sees(dtype, new, keys, group):
    """An infinity among the values of the oldest keys: every row's sum holds it with a positive weight."""
    table, lens, starts, pages = _batch([new], [keys], 16, 7)
    cache = _pool(pages, 1, 16, 64, dtype, 8)
    cache.v[int(table[0, 0]), 0, 5, 9] = math.inf
    cache.v[int(table[0, 0]), 0, 11, 60] = -math.inf
    q = torch.randn((new, group, 64), generator=torch.Generator().manual_seed(9)).to(dtype).cuda()
    out = fsta.paged_attention(q, cache, table.cuda(), lens.cuda(), starts.cuda(), 0.125).cpu()
    assert (out[:, :, 9] == math.inf).all() and (out[:, :, 60] == -math.inf).all()
    rest = [c for c in range(64) if c not in (9, 60)]
    assert out[:, :, rest].isfinite().all()


# Scores are off by float32 sums of d terms (d * 2^-24 relative of sums of about sqrt(d)), far below the rest; a weight is rounded
# to half a unit in the last place (2^-8 bfloat16, 2^-11 float16) at most, and so is the result.  A row's result is a weighted mean
# of values of size max |v|, so the weights' rounding moves it by 2^-8 * max |v| at most, its own rounding by 2^-8 of itself.
_UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


@pytest.mark.parametrize("dtype,d", [(torch.bfloat16, 128), (torch.float16, 64)])
@pytest.mark.parametrize("new,keys,heads,kv_heads,page,width", [
    ([64], [256], 8, 2, 16, 0), ([5, 38, 1, 17], [362, 40, 1, 99], 16, 2, 32, 0), ([256], [300], 4, 4, 64, 0), ([64], [256], 8, 2, 16, 4000),
    ([90, 1, 70], [600, 33, 71], 8, 1, 16, 0), ([33] * 9, [128] * 9, 4, 4, 16, 0), ([48], [5000], 4, 1, 64, 0), ([512], [512], 4, 4, 16, 0)])
def test_few_rows_on_few_keys(dtype, d, new, keys, heads, kv_heads, page, width):
    """Every size of a workgroup's tile that the page table's width and the number of rows choose (`width`: columns that no sequence
    uses), against softmax in 64 bits."""
    table, lens, starts, pages = _batch(new, keys, page, 21)
    if width:
        table = torch.cat([table, torch.full((len(new), width), -1, dtype=torch.int32)], 1)
    cache = _pool(pages, kv_heads, page, d, dtype, 22)
    q = torch.randn((sum(new), heads, d), generator=torch.Generator().manual_seed(23)).to(dtype)
    got = fsta.paged_attention(q.cuda(), cache, table.cuda(), lens.cuda(), starts.cuda(), d ** -0.5, max_q_len=max(new)).cpu().double()
    for b, (n, total) in enumerate(zip(new, keys)):
        places = table[b, : -(-total // page)].long()
        k, v = (t.cpu()[places].permute(1, 0, 2, 3).reshape(kv_heads, -1, d)[:, :total].double().repeat_interleave(heads // kv_heads, 0)
                for t in (cache.k, cache.v))
        rows = q[starts[b] : starts[b + 1]].double().permute(1, 0, 2)
        score = rows @ k.transpose(1, 2) * d ** -0.5
        score = score.masked_fill(torch.arange(total)[None, :] > torch.arange(total - n, total)[:, None], -math.inf)
        want = (score.softmax(-1) @ v).permute(1, 0, 2)
        top = v.abs().amax()
        torch.testing.assert_close(got[starts[b] : starts[b + 1]], want, rtol=_UNIT[dtype], atol=float(1.1 * _UNIT[dtype] * top))


# The model of the example has logits of standard deviation 1, the largest of 512 about 3.  Some ten roundings to bfloat16 (2^-8
# each) on a token's way move a logit by 0.03 or so; 8-bit keys and values (2^-4 of a value, averaged over the keys seen, times the
# 0.3 that a layer's result counts, four layers) by 0.04.  Eight times that is asked for, far below what a wrong key would do.
@pytest.mark.parametrize("fp8,off", [(False, 0.25), (True, 0.5)])
def test_speculative_decoding_over_pages(fp8, off):
    """The example's answers against its model in float32 on the CPU, whole sequences at a time and without a cache: every token is
    the likeliest one but for roundings, and trees say more than a token a step."""
    from fstattention_amd.examples import speculative_decoding as example
    model = example.make_model()
    g = torch.Generator().manual_seed(3)
    prompts = [torch.randint(512, (n,), generator=g).tolist() for n in (7, 130, 64, 33)]
    steps = 24
    answers, talk = example.answer(model, prompts, steps, draft=32, fp8=fp8)
    assert talk.lens.tolist() == [len(p) + len(a) - 1 for p, a in zip(prompts, answers)]
    assert all(steps < len(a) - 1 < 5 * steps for a in answers)
    embed, unembed = model.embed.cpu().float(), model.unembed.cpu().float()
    norm = lambda x: x * (x.square().mean(-1, keepdim=True) + 1e-6).rsqrt()
    h, hk, d = model.heads, model.kv_heads, model.head_dim
    for prompt, said in zip(prompts, answers):
        tokens = torch.tensor(prompt + said[:-1])
        n = len(tokens)
        x = embed[tokens] + 0.1 * example._place(torch.arange(n), embed.shape[1]).float()
        hidden = torch.ones(n, n, dtype=torch.bool).triu(1)
        for w_qkv, w_out in zip(model.qkv, model.out):
            fused = (norm(x) @ w_qkv.cpu().float()).view(n, h + 2 * hk, d).permute(1, 0, 2)
            k, v = (t.repeat_interleave(h // hk, 0) for t in (fused[h:h + hk], fused[h + hk:]))
            weights = (fused[:h] @ k.transpose(1, 2) * d ** -0.5).masked_fill(hidden, -math.inf).softmax(-1)
            x = x + 0.3 * ((weights @ v).permute(1, 0, 2).reshape(n, h * d) @ w_out.cpu().float())
        logits = (norm(x) @ unembed)[len(prompt) - 1:]
        short = logits.amax(-1) - logits.gather(1, torch.tensor(said)[:, None])[:, 0]
        assert short.max() <= off


def test_speculative_decoding_one_token_a_step():
    """The example without trees says one token a step, and leaves as many rows in its pages as there were tokens."""
    from fstattention_amd.examples import speculative_decoding as example
    model = example.make_model()
    prompts = [[5, 6, 7], [9] * 100]
    answers, talk = example.answer(model, prompts, 6, draft=0)
    assert [len(a) for a in answers] == [7, 7] and talk.lens.tolist() == [9, 106]
    dense, _ = fsta.read_paged_kv(talk.pools[0], talk.page_table, talk.lens, 110)
    used = dense.abs().amax((1, 3)).cpu() > 0
    assert torch.equal(used, torch.arange(110)[None, :] < talk.lens.cpu()[:, None])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float8_e4m3fn])
def test_pages_beyond_32_bits(dtype):
    """A pool of more than 2^32 elements: rows written to its last pages are read from there, by both kernels that read."""
    pages, heads, page, d = (1 << 20) + 40, 2, 16, 128
    shape = (pages, heads, page, d)
    exps = (None, None) if dtype == torch.bfloat16 else tuple(torch.full(shape[:3], 127, dtype=torch.uint8, device="cuda") for _ in range(2))
    cache = fsta.PagedKV(torch.empty(shape, dtype=dtype, device="cuda"), torch.empty(shape, dtype=dtype, device="cuda"), *exps)
    keys = 300
    need = -(-keys // page)
    places = [pages - 1 - 2 * i for i in range(need)]
    low = [p - (1 << 20) for p in places]                        # where they would lie by 32-bit offsets
    table = torch.tensor([places, low], dtype=torch.int32).cuda()
    lens = torch.tensor([keys, keys], dtype=torch.int32).cuda()
    starts = torch.tensor([0, keys, 2 * keys], dtype=torch.int32).cuda()
    g = torch.Generator().manual_seed(5)
    k, v = (torch.randn((2 * keys, heads, d), generator=g).bfloat16().cuda() for _ in range(2))
    fsta.write_paged_kv(cache, k, v, table, lens, starts)
    near = fsta.PagedKV(*(None if t is None else t[torch.tensor(places + low, device="cuda")].clone() for t in cache))
    near_table = torch.arange(2 * need, dtype=torch.int32).view(2, need).cuda()
    got, want = (fsta.read_paged_kv(c, t, lens, keys, torch.bfloat16) for c, t in ((cache, table), (near, near_table)))
    if dtype == torch.bfloat16:
        assert torch.equal(got[0].transpose(1, 2).reshape(2 * keys, heads, d), k) and torch.equal(got[1].transpose(1, 2).reshape(2 * keys, heads, d), v)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    for new in (1, 40, 300):
        q = torch.randn((2 * new, 4, d), generator=g).bfloat16().cuda()
        q_starts = torch.tensor([0, new, 2 * new], dtype=torch.int32).cuda()
        outs = [fsta.paged_attention(q, c, t, lens, q_starts, d ** -0.5, max_q_len=new) for c, t in ((cache, table), (near, near_table))]
        assert torch.equal(*outs) and outs[0].isfinite().all()
