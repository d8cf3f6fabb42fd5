"""Performance cases of the paged KV cache: a serving program's cache in pages, written, read back and attended to.

A case is a dict of plain values.  ``listed()`` are the fixed ones, ``draw(rng)`` gives further ones of the same ranges;
``prepare`` makes on the GPU what a program holds before the call, ``run`` is one pass, ``work`` the bytes and operations
that pass cannot do without, ``exact`` its result in 64 bits.  ``own`` chooses between the package's operators and their
plain form in elementary tensor operations.

``op`` says which use a case is of:

* ``attention``  one layer's attention of the new tokens of a batch over each sequence's pages: single tokens, chunks of a
  prompt, or both in one batch; the keys and values of the new tokens are in the cache already.
* ``tree_step``  a decoding step of draft trees: the trees' masks from their parent arrays, then for every layer the new
  tokens' keys and values into the cache and the attention over it.
* ``write``      keys and values of new tokens go to their places in the pages.
* ``read``       the pages of a batch of sequences are brought back to dense tensors.
* ``store_read`` a prompt's keys and values are quantised as they are written and read back as 16-bit values.
* ``tree_bits``  parent arrays of draft trees to the masks that say which tokens of a tree see which.

Lengths come from the case alone, values and the order of the pages from the seed.
"""
import math
import random

import torch

own = False

DTYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16}


def _attention(name, batch, new, keys, heads, kv_heads, head_dim, dtype, page, fp8=False, lse=False):
    """`new` and `keys`: [fewest, most] new tokens and cached keys (new ones included) of a sequence."""
    return _named(name, {"op": "attention", "batch": batch, "new_low": new[0], "new_high": new[1], "keys_low": keys[0],
                         "keys_high": keys[1], "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim, "dtype": dtype,
                         "page": page, "fp8": fp8, "lse": lse})


def _cache(name, op, batch, new, keys, kv_heads, head_dim, dtype, page, fp8=False):
    return _named(name, {"op": op, "batch": batch, "new_low": new[0], "new_high": new[1], "keys_low": keys[0],
                         "keys_high": keys[1], "heads": kv_heads, "kv_heads": kv_heads, "head_dim": head_dim, "dtype": dtype,
                         "page": page, "fp8": fp8})


def _tree_step(name, batch, nodes, keys, heads, kv_heads, head_dim, dtype, page, layers):
    return _named(name, {"op": "tree_step", "batch": batch, "new_low": nodes, "new_high": nodes, "keys_low": keys[0],
                         "keys_high": keys[1], "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim, "dtype": dtype,
                         "page": page, "fp8": False, "layers": layers})


def _tree_bits(name, batch, nodes, window):
    return _named(name, {"op": "tree_bits", "batch": batch, "new_low": nodes[0], "new_high": nodes[1], "window": window})


def _named(name, case):
    return dict(case, name=name) if name else case


def listed():
    return [
        # the smallest call: the next token of one short conversation, where only latency counts
        _attention("decode_1", 1, [1, 1], [333, 333], 32, 8, 128, "bfloat16", 16),
        # the ordinary decoding call of a server: a batch of conversations of very different lengths
        _attention("decode_64_ragged", 64, [1, 1], [16, 8192], 32, 8, 128, "bfloat16", 64),
        # long documents whose cache is kept in 8 bits
        _attention("decode_16_long_fp8", 16, [1, 1], [8192, 32768], 64, 8, 128, "bfloat16", 64, fp8=True),
        # a long prompt taken in chunks: the largest call, bound by the matrix products
        _attention("chunk_4096_after_16384", 1, [4096, 4096], [20480, 20480], 32, 8, 128, "bfloat16", 128),
        # chunks of prompts and single tokens in one batch, odd sizes throughout; the log-sum-exp is wanted because another
        # part of the keys is attended to elsewhere
        _attention("mixed_17_odd", 17, [1, 501], [37, 5003], 28, 4, 64, "float16", 32, lse=True),
        # a step of speculative decoding: draft trees of 256 nodes, four layers
        _tree_step("tree_256_4_layers", 2, 256, [1256, 1500], 32, 32, 128, "bfloat16", 16, 4),
        # the new tokens of a decoding batch go to their pages
        _cache("write_decode_61", "write", 61, [1, 1], [16, 2048], 8, 128, "float16", 16),
        # so do those of a prompt
        _cache("write_8192", "write", 1, [8192, 8192], [8192, 8192], 16, 128, "bfloat16", 64),
        # cached conversations leave the pages: for a dense kernel, another machine or the host's memory
        _cache("read_8_ragged", "read", 8, [1, 1], [100, 8192], 8, 128, "bfloat16", 64),
        # a prompt's cache kept in 8 bits, and what a later reader gets
        _cache("store_read_8192_fp8", "store_read", 2, [4000, 8192], [4000, 8192], 8, 128, "bfloat16", 64, fp8=True),
        # the masks of a batch of ordinary draft trees, and of a few large ones of long chains
        _tree_bits("tree_bits_16x256", 16, [40, 256], 64),
        _tree_bits("tree_bits_4x2048", 4, [1500, 2048], 48),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    """Batches of 1 to 128 sequences of up to 32768 keys (8 bits) or 20480, chunks of up to 4096 tokens, trees of 16 to 2048 nodes."""
    op = rng.choices(["decode", "chunk", "mixed", "tree_step", "write", "read", "store_read", "tree_bits"], weights=[5, 3, 3, 2, 2, 2, 2, 2])[0]
    if op == "tree_bits":
        high = _log_int(rng, 16, 2048)
        return _tree_bits(None, max(1, min(_log_int(rng, 1, 64), 8192 // high)), [max(1, high // rng.randint(1, 6)), high], _log_int(rng, 8, 128))
    dtype, head_dim, page = rng.choice(["bfloat16", "float16"]), rng.choice([64, 128, 128]), rng.choice([16, 32, 64, 128, 256])
    kv_heads = rng.choice([1, 2, 4, 8, 16])
    group = rng.choice([1, 2, 4, 5, 7, 8])
    heads = kv_heads * group
    if op == "decode":
        fp8 = rng.random() < 0.4
        high = _log_int(rng, 33, 32768 if fp8 else 20480)
        batch = max(1, min(_log_int(rng, 1, 128), (1 << 20) // (high * kv_heads)))
        return _attention(None, batch, [1, rng.choice([1, 1, 1, 4])], [max(5, high // rng.randint(1, 50)), high], heads, kv_heads, head_dim,
                          dtype, page, fp8=fp8, lse=rng.random() < 0.2)
    if op in ("chunk", "mixed"):
        high = _log_int(rng, 16, 4096)
        before = _log_int(rng, 1, 16384)
        batch = 1 if op == "chunk" else rng.randint(2, 20)
        while batch > 1 and batch * high * (high + before) * heads > 2 << 30:
            batch -= 1
        while high > 16 and batch * high * (high + before) * heads > 2 << 30:
            high //= 2
        low = high if op == "chunk" else 1
        return _attention(None, batch, [low, high], [low + (before if op == "chunk" else 0), high + before], heads, kv_heads, head_dim, dtype,
                          page, fp8=rng.random() < 0.25, lse=rng.random() < 0.3)
    if op == "tree_step":
        nodes = _log_int(rng, 16, 256)
        high = nodes + _log_int(rng, 64, 2048)
        batch = max(1, min(rng.randint(1, 8), (1 << 16) // (high * kv_heads)))
        return _tree_step(None, batch, nodes, [nodes + 1 if batch > 1 else high, high], heads, kv_heads, head_dim, dtype, page, rng.randint(1, 4))
    high = _log_int(rng, 16, 8192)
    batch = max(1, min(_log_int(rng, 1, 64), (1 << 17) // (high * kv_heads)))
    low = max(1, high // rng.randint(1, 20))
    if op == "write":
        new = [1, 1] if rng.random() < 0.5 else [max(1, low // 2), low]
        return _cache(None, op, batch, new, [low, high], kv_heads, head_dim, dtype, page)
    if op == "read":
        return _cache(None, op, batch, [1, 1], [low, high], kv_heads, head_dim, dtype, page, fp8=rng.random() < 0.4)
    return _cache(None, op, batch, [low, high], [low, high], kv_heads, head_dim, dtype, page, fp8=True)


# ---- the lengths of a case ----------------------------------------------------------------------------------------------

def _spread(rng, low, high, count):
    """`count` lengths over the logarithm of [low, high], the largest among them."""
    values = [high] + [min(high, max(low, _log_int(rng, low, high))) for _ in range(count - 1)]
    rng.shuffle(values)
    return values


def _lengths(case):
    """(new tokens, keys) of every sequence, new ones included in keys."""
    rng = random.Random(case["batch"] * 1000003 + case["new_high"] * 1009 + case.get("keys_high", 0))
    new = _spread(rng, case["new_low"], case["new_high"], case["batch"])
    if case["op"] == "tree_bits":
        return new, new
    if case["op"] == "store_read":          # whole prompts
        return new, list(new)
    keys = _spread(rng, case["keys_low"], case["keys_high"], case["batch"])
    return [min(n, k) for n, k in zip(new, keys)], keys


def _starts(lengths):
    out = [0]
    for n in lengths:
        out.append(out[-1] + n)
    return out


# ---- what a program holds before the call -------------------------------------------------------------------------------

def _parents(new, window, seed):
    """Random recursive trees: a node's parent is one of the `window` nodes in front of it, node 0 the root."""
    rng = random.Random(seed)
    out = []
    for n in new:
        out += [-1] + [rng.randint(max(0, i - window), i - 1) for i in range(1, n)]
    return torch.tensor(out, dtype=torch.int64).cuda()


def _projection(case, tokens, generator, dtype):
    """q, k, v [tokens, heads, head_dim]: views of one fused projection's output, as a layer has them."""
    h, hk, d = case["heads"], case["kv_heads"], case["head_dim"]
    fused = torch.randn((tokens, (h + 2 * hk) * d), generator=generator, dtype=dtype, device="cuda")
    q, k, v = fused.split([h * d, hk * d, hk * d], dim=1)
    return q.view(tokens, h, d), k.view(tokens, hk, d), v.view(tokens, hk, d)


def _pool(case, pages, generator, dtype):
    """(k, v, k_exponent, v_exponent): pages of a cache that has been in use for a while; every place holds something."""
    shape = (pages, case["kv_heads"], case["page"], case["head_dim"])
    k = torch.randn(shape, generator=generator, dtype=dtype, device="cuda")
    v = torch.randn(shape, generator=generator, dtype=dtype, device="cuda")
    if not case["fp8"]:
        return k, v, None, None
    (k8, ke), (v8, ve) = _quantise(k), _quantise(v)
    return k8, v8, ke, ve


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    new, keys = _lengths(case)
    state = {"case": dict(case), "tokens": sum(new), "most_new": max(new), "most_keys": max(keys),
             "starts": torch.tensor(_starts(new), dtype=torch.int32).cuda()}
    if case["op"] in ("tree_bits", "tree_step"):
        state["parent"] = _parents(new, case.get("window", 32), seed)
    if case["op"] == "tree_bits":
        return state
    dtype, page = DTYPES[case["dtype"]], case["page"]
    width = -(-max(keys) // page)
    used = sum(-(-k // page) for k in keys)
    order = torch.randperm(used + 3, generator=g, device="cuda").to(torch.int32)      # a few pages belong to nobody
    table = torch.full((case["batch"], width), -1, dtype=torch.int32, device="cuda")
    for b, first in enumerate(_starts([-(-k // page) for k in keys])[:-1]):
        count = -(-keys[b] // page)
        table[b, :count] = order[first:first + count]
    state.update(table=table, keys=torch.tensor(keys, dtype=torch.int32).cuda(), scale=1.0 / math.sqrt(case["head_dim"]))
    state["layers"] = [(_projection(case, sum(new), g, dtype), _pool(case, used + 3, g, dtype)) for _ in range(case.get("layers", 1))]
    return state


# ---- one pass -----------------------------------------------------------------------------------------------------------

def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(state):
    import fstattention_amd as fsta
    case, op = state["case"], state["case"]["op"]
    starts = state["starts"]
    if op == "tree_bits":
        return fsta.tree_mask_bits(state["parent"], starts, state["most_new"])
    table, keys = state["table"], state["keys"]
    (q, k, v), pool = state["layers"][0]
    cache = fsta.PagedKV(*pool)
    if op == "attention":
        return fsta.paged_attention(q, cache, table, keys, starts, state["scale"], max_q_len=state["most_new"], return_lse=case["lse"])
    if op == "read":
        return fsta.read_paged_kv(cache, table, keys, state["most_keys"], dtype=q.dtype)
    if op in ("write", "store_read"):
        fsta.write_paged_kv(cache, k, v, table, keys, starts)
        return (cache.k, cache.v) if op == "write" else fsta.read_paged_kv(cache, table, keys, state["most_keys"], dtype=q.dtype)
    bits = fsta.tree_mask_bits(state["parent"], starts, state["most_new"])
    out = []
    for (q, k, v), pool in state["layers"]:
        cache = fsta.PagedKV(*pool)
        fsta.write_paged_kv(cache, k, v, table, keys, starts)
        out.append((fsta.paged_attention(q, cache, table, keys, starts, state["scale"], tree_bits=bits, max_q_len=state["most_new"]),
                    cache.k, cache.v))
    return out


def _run_plain(state):
    case, op = state["case"], state["case"]["op"]
    if op == "tree_bits":
        return _pack(_tree_reach(state))
    (q, k, v), pool = state["layers"][0]
    if op == "attention":
        o, lse = _attend(state, q, pool, _causal(state))
        return (o, lse) if case["lse"] else o
    if op == "read":
        return _read(state, pool, q.dtype)
    if op == "write":
        return _store(state, pool, k, v)[:2]
    if op == "store_read":
        return _read(state, _store(state, pool, k, v), q.dtype)
    sees = _pack(_tree_reach(state))
    out = []
    for (q, k, v), pool in state["layers"]:
        pool = _store(state, pool, k, v)
        out.append((_attend(state, q, pool, _tree(state, sees))[0],) + pool[:2])
    return out


def _grid(state):
    """[batch, most_new] places of the new tokens in the packed tensors, and which of them exist."""
    starts = state["starts"].long()
    i = torch.arange(state["most_new"], device=starts.device)
    at = starts[:-1, None] + i
    return at.clamp(max=state["tokens"] - 1), at < starts[1:, None]


def _sequence(state):
    """Of every new token: its sequence, and its number among the new ones of that sequence."""
    starts = state["starts"].long()
    t = torch.arange(state["tokens"], device=starts.device)
    seq = (starts[1:, None] <= t).sum(0)
    return seq, t - starts[seq]


def _quantise(x):
    """Rows as e4m3 bytes times a power of two: the smallest under which the row's largest magnitude is at most 448."""
    amax = x.float().abs().amax(-1)
    mantissa, exponent = torch.frexp(amax)
    e = torch.where(mantissa > 0.875, exponent - 8, exponent - 9)      # 448 = 0.875 * 2^9
    e = torch.where(amax > 0, e.clamp(-110, 120), torch.zeros_like(e))
    return (x.float() * _power(-e)[..., None]).to(torch.float8_e4m3fn), (e + 127).to(torch.uint8)


def _power(e):
    """2^e in 32 bits, exactly."""
    return ((e.int() + 127) << 23).view(torch.float32)


def _values(rows, exponents):
    return rows.float() * _power(exponents.int() - 127)[..., None]


def _places(state, seq, position):
    """(page, row in it) of positions of sequences."""
    page = state["case"]["page"]
    return state["table"].long()[seq, position // page], position % page


def _store(state, pool, k, v):
    k_pool, v_pool, k_exp, v_exp = pool
    seq, i = _sequence(state)
    count = (state["starts"][1:] - state["starts"][:-1]).long()
    page, row = _places(state, seq, state["keys"].long()[seq] - count[seq] + i)
    if k_exp is None:
        k_pool[page, :, row] = k
        v_pool[page, :, row] = v
    else:
        k8, k_exp[page, :, row] = _quantise(k)
        v8, v_exp[page, :, row] = _quantise(v)
        k_pool.view(torch.uint8)[page, :, row] = k8.view(torch.uint8)
        v_pool.view(torch.uint8)[page, :, row] = v8.view(torch.uint8)
    return pool


def _dense(state, rows, exponents):
    """[batch, kv_heads, most_keys, head_dim] in 32 bits, zero past each sequence's end."""
    position = torch.arange(state["most_keys"], device=rows.device).expand(state["case"]["batch"], -1)
    seq = torch.arange(state["case"]["batch"], device=rows.device)[:, None]
    page, row = _places(state, seq, position)
    here = position < state["keys"][:, None]
    page = page.clamp(min=0)
    if exponents is None:
        x = rows[page, :, row].float()
    else:
        x = _values(rows.view(torch.uint8)[page, :, row].view(rows.dtype), exponents[page, :, row])
    return torch.where(here[:, :, None, None], x, torch.zeros_like(x)).transpose(1, 2).contiguous()


def _read(state, pool, dtype):
    return _dense(state, pool[0], pool[2]).to(dtype), _dense(state, pool[1], pool[3]).to(dtype)


def _tree_reach(state):
    """[batch, most_new, most_new] truth values: row i sees column j where j is i or one of its ancestors."""
    at, here = _grid(state)
    n = state["most_new"]
    parent = state["parent"][at]
    j = torch.arange(n, device=parent.device)
    step = ((parent[:, :, None] == j) & here[:, :, None]).float()
    reach = step + torch.eye(n, device=parent.device)
    hops = 1
    while hops < n:                      # paths of up to twice the length
        reach = (torch.matmul(reach, reach) > 0).float()
        hops *= 2
    return (reach > 0) & here[:, :, None]


def _pack(reach):
    """Bit b of word w: column 32 w + b.  One row for every new token."""
    batch, n, _ = reach.shape
    words = -(-n // 32)
    full = torch.zeros((batch, n, 32 * words), dtype=torch.int64, device=reach.device)
    full[:, :, :n] = reach
    packed = (full.view(batch, n, words, 32) << torch.arange(32, device=reach.device)).sum(-1)
    packed = torch.where(packed >= 1 << 31, packed - (1 << 32), packed).to(torch.int32)
    return packed[reach.diagonal(dim1=1, dim2=2)]


def _limits(state):
    """[batch, most_new, most_keys]: the key's number among the sequence's new tokens (below 0: older), the row's own, and whether the key exists."""
    keys = state["keys"].long()
    count = (state["starts"][1:] - state["starts"][:-1]).long()
    position = torch.arange(state["most_keys"], device=keys.device)
    number = position[None, None, :] - (keys - count)[:, None, None]
    row = torch.arange(state["most_new"], device=keys.device)[None, :, None]
    return number, row, (position[None, None, :] < keys[:, None, None])


def _causal(state):
    number, row, here = _limits(state)
    return (number <= row) & here


def _tree(state, packed):
    number, row, here = _limits(state)
    at, _ = _grid(state)
    words = packed.long()[at]                                    # [batch, most_new, words]
    word = (number // 32).clamp(0, words.shape[2] - 1).expand(-1, words.shape[1], -1)
    bit = (torch.gather(words, 2, word) >> (number % 32)) & 1
    return ((number < 0) | (bit > 0)) & here


def _attend(state, q, pool, sees):
    case = state["case"]
    batch, n, hk, d = case["batch"], state["most_new"], case["kv_heads"], case["head_dim"]
    group = case["heads"] // hk
    k, v = _dense(state, pool[0], pool[2]), _dense(state, pool[1], pool[3])
    at, _ = _grid(state)
    rows = q[at].float().view(batch, n, hk, group, d).permute(0, 2, 3, 1, 4).reshape(batch, hk, group * n, d)
    s = torch.matmul(rows, k.transpose(2, 3)).view(batch, hk, group, n, -1).mul_(state["scale"])
    s.masked_fill_(~sees[:, None, None], -math.inf)
    top = s.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    s.sub_(top).exp_()
    total = s.sum(-1, keepdim=True)
    o = torch.matmul(s.view(batch, hk, group * n, -1), v).view(batch, hk, group, n, d) / total.clamp(min=1e-38)
    seq, i = _sequence(state)
    lse = (top + torch.log(total)) * (1.0 / math.log(2.0))
    o = o.permute(0, 3, 1, 2, 4).reshape(batch, n, case["heads"], d)[seq, i]
    return o.to(q.dtype), lse.permute(0, 3, 1, 2, 4).reshape(batch, n, case["heads"])[seq, i]


# ---- the result in 64 bits ----------------------------------------------------------------------------------------------

def exact(case, seed):
    state = prepare(case, seed)
    new, keys = _lengths(case)
    op, first = case["op"], _starts(new)
    if op == "tree_bits":
        return None
    page, table = case["page"], state["table"].tolist()

    def rows_of(b):
        """pool indices of the keys of sequence b, pool seen as [pages * page] rows"""
        return torch.tensor([table[b][p // page] * page + p % page for p in range(keys[b])], device="cuda")

    def flat(pool):
        return pool.transpose(1, 2).reshape(-1, case["kv_heads"], pool.shape[3])

    def stored(pool, exponents):
        x = flat(pool).double()
        return x if exponents is None else x * 2.0 ** (flat(exponents[..., None]).double() - 127)

    def rounded(x):
        """What e4m3 with a power of two of its own per row keeps of x."""
        x = x.double().cpu()
        amax = x.abs().amax(-1, keepdim=True)
        e = torch.ceil(torch.log2(torch.where(amax > 0, amax, torch.ones_like(amax)) / 448.0))
        unit = torch.floor(torch.log2(torch.where(x == 0, torch.ones_like(x), x).abs() / 2.0 ** e)).clamp(min=-6) - 3
        return (torch.round(x / 2.0 ** (e + unit)) * 2.0 ** (e + unit)).cuda()

    def dense(of_sequence):
        out = torch.zeros((case["batch"], case["kv_heads"], max(keys), case["head_dim"]), dtype=torch.float64, device="cuda")
        for b in range(case["batch"]):
            out[b, :, :keys[b]] = of_sequence(b).transpose(0, 1)
        return out

    def filled(pool, x):
        out = flat(pool).double()
        for b in range(case["batch"]):
            out[rows_of(b)[keys[b] - new[b]:]] = x[first[b]:first[b + 1]].double()
        return out

    def as_pool(rows):
        return rows.view(-1, page, *rows.shape[1:]).transpose(1, 2)

    def ancestors(b):
        parent = state["parent"][first[b]:first[b + 1]].tolist()
        sees = torch.zeros((new[b], new[b]), dtype=torch.bool)
        for i, p in enumerate(parent):
            if p >= 0:
                sees[i] = sees[p]
            sees[i, i] = True
        return sees.cuda()

    def attended(q, k_rows, v_rows):
        group = case["heads"] // case["kv_heads"]
        o = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
        lse = torch.zeros(q.shape[:2], dtype=torch.float64, device="cuda")
        for b in range(case["batch"]):
            at = rows_of(b)
            old = keys[b] - new[b]
            sees = torch.ones((new[b], keys[b]), dtype=torch.bool, device="cuda")
            sees[:, old:] = ancestors(b) if op == "tree_step" else torch.ones((new[b], new[b]), dtype=torch.bool, device="cuda").tril()
            for h in range(case["heads"]):
                s = q[first[b]:first[b + 1], h].double() @ k_rows[at, h // group].t() * state["scale"]
                s = torch.where(sees, s, torch.full_like(s, -math.inf))
                o[first[b]:first[b + 1], h] = torch.softmax(s, -1) @ v_rows[at, h // group]
                lse[first[b]:first[b + 1], h] = torch.logsumexp(s, -1) / math.log(2.0)
        return o, lse

    (q, k, v), pool = state["layers"][0]
    if op == "attention":
        o, lse = attended(q, stored(pool[0], pool[2]), stored(pool[1], pool[3]))
        return (o, lse) if case["lse"] else o
    if op == "read":
        k_rows, v_rows = stored(pool[0], pool[2]), stored(pool[1], pool[3])
        return dense(lambda b: k_rows[rows_of(b)]), dense(lambda b: v_rows[rows_of(b)])
    if op == "write":
        return as_pool(filled(pool[0], k)), as_pool(filled(pool[1], v))
    if op == "store_read":
        k, v = rounded(k), rounded(v)
        return dense(lambda b: k[first[b]:first[b + 1]]), dense(lambda b: v[first[b]:first[b + 1]])
    out = []
    for (q, k, v), pool in state["layers"]:
        k_rows, v_rows = filled(pool[0], k), filled(pool[1], v)
        out.append((attended(q, k_rows, v_rows)[0], as_pool(k_rows), as_pool(v_rows)))
    return out


# ---- what a pass cannot do without --------------------------------------------------------------------------------------

def work(case):
    new, keys = _lengths(case)
    if case["op"] == "tree_bits":
        return {"bytes": 8 * sum(new) + 4 * sum(new) * (-(-max(new) // 32)) + 4 * len(new), "flops": 0}
    hk, d, h = case["kv_heads"], case["head_dim"], case["heads"]
    row = d + 1 if case["fp8"] else 2 * d                      # a key or a value in the cache
    tables = 4 * sum(-(-k // case["page"]) for k in keys) + 8 * len(keys)
    if case["op"] == "write":
        return {"bytes": 2 * hk * sum(new) * (2 * d + row) + tables, "flops": 0}
    if case["op"] == "read":
        return {"bytes": 2 * hk * (sum(keys) * row + len(keys) * max(keys) * 2 * d) + tables, "flops": 0}
    if case["op"] == "store_read":
        return {"bytes": 2 * hk * (sum(new) * (2 * d + row) + sum(keys) * row + len(keys) * max(keys) * 2 * d) + tables, "flops": 6 * hk * d * sum(new)}
    pairs = sum(n * (k - n) + n * (n + 1) // 2 for n, k in zip(new, keys))
    layer = {"bytes": 2 * 2 * h * d * sum(new) + 2 * hk * sum(keys) * row + tables + (4 * h * sum(new) if case.get("lse") else 0),
             "flops": 4 * h * d * pairs}
    if case["op"] == "attention":
        return layer
    pairs = sum(n * (k - n) + n * max(1, math.ceil(math.log2(n))) for n, k in zip(new, keys))      # a tree's paths are short
    bits = 8 * sum(new) + 4 * sum(new) * (-(-max(new) // 32))
    return {"bytes": case["layers"] * (layer["bytes"] + 2 * hk * sum(new) * 4 * d) + bits, "flops": case["layers"] * 4 * h * d * pairs}
