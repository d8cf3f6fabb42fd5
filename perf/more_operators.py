"""Performance cases of what a serving program does between two passes of its model over a paged KV cache: which drafted
tokens stand, the accepted branch's keys and values moved together, pages given to sequences, shared and taken back.

A case is a dict of plain values.  ``listed()`` are the fixed ones, ``draw(rng)`` gives further ones of the same ranges;
``prepare`` makes on the GPU what a program holds before the call, ``run`` is one pass, ``work`` the bytes and operations
that pass cannot do without, ``exact`` its result in 64 bits.  ``own`` chooses between the package's operators and their
plain form in elementary tensor operations.

``op`` says which use a case is of:

* ``verify``   trees or chains of drafted tokens against the model's logits, from given random numbers: the accepted path of every
  tree and the token behind it.  ``sampled``: the drafts were drawn from probabilities that are known; otherwise they are a
  ranked list's.
* ``compact``  the rows of the accepted paths move to the places directly behind each conversation, in every layer.
* ``fit``      a step's room: pages for the trees' rows are taken, and given back when the trees are done with.
* ``fork``     slots of a batch give up what they hold and become copies of other slots: further answers to the same prompt.
* ``copy``     whole pages go to other pages, in every layer.

Shapes and lengths come from the case alone, values and the order of the pages from the seed.
"""
import heapq
import math
import random

import torch

own = False

DTYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
SIGMA = 3.0                     # spread of the logits that no draft names


def _verify(name, batch, nodes, depth, children, vocabulary, dtype, sampled="", pad=0, mixed=False):
    """`nodes`: [fewest, most] of a tree; `sampled`: dtype of the draft's probabilities; `mixed`: a temperature per sequence, some 0."""
    return _named(name, {"op": "verify", "batch": batch, "nodes_low": nodes[0], "nodes_high": nodes[1], "depth": depth, "children": children,
                         "vocabulary": vocabulary, "dtype": dtype, "sampled": sampled, "pad": pad, "mixed": mixed})


def _pages(name, op, batch, keys, nodes, layers, kv_heads, head_dim, dtype, page, fp8=False):
    """`keys`: [fewest, most] positions of a sequence before the step; `nodes`: of its tree (compact, fit), its copies (fork), the pages (copy)."""
    return _named(name, {"op": op, "batch": batch, "keys_low": keys[0], "keys_high": keys[1], "nodes": nodes, "layers": layers,
                         "kv_heads": kv_heads, "head_dim": head_dim, "dtype": dtype, "page": page, "fp8": fp8})


def _named(name, case):
    return dict(case, name=name) if name else case


def listed():
    return [
        # one conversation whose draft model proposes five tokens in a row: latency is all
        _verify("verify_chain_1", 1, [6, 6], 5, 1, 32000, "bfloat16", sampled="float32"),
        # trees of a draft head's best guesses in a batch whose users chose different temperatures, some greedy
        _verify("verify_trees_16x64", 16, [64, 64], 5, 6, 32000, "float32", mixed=True),
        # trees drawn from a draft model, odd sizes throughout, logits with a padded row
        _verify("verify_sampled_32x23", 32, [5, 23], 6, 3, 50021, "float16", sampled="float16", pad=27),
        # a large vocabulary in a large batch: bound by reading the logits
        _verify("verify_trees_128x64", 128, [64, 64], 6, 6, 131072, "bfloat16"),
        # the accepted tokens of one conversation, a model's 32 layers
        _pages("compact_1", "compact", 1, [700, 700], 64, 32, 8, 128, "bfloat16", 16),
        # a batch with its cache in 8 bits
        _pages("compact_96_fp8", "compact", 96, [40, 900], 61, 24, 8, 128, "bfloat16", 32, fp8=True),
        # a step's room in an ordinary batch
        _pages("fit_48", "fit", 48, [16, 2048], 64, 2, 2, 64, "bfloat16", 16),
        # a large server: a thousand long conversations in some 300000 pages
        _pages("fit_1024_long", "fit", 1024, [400, 16000], 61, 1, 1, 64, "bfloat16", 16),
        # three more answers to each of two prompts
        _pages("fork_2x3", "fork", 2, [133, 715], 3, 16, 8, 128, "float16", 32),
        # many answers to many prompts, 8-bit rows
        _pages("fork_48x7_fp8", "fork", 48, [20, 3001], 7, 12, 8, 128, "bfloat16", 64, fp8=True),
        # a few pages to the places of others
        _pages("copy_37", "copy", 1, [0, 0], 37, 4, 4, 64, "bfloat16", 16),
        # a pool's pages are moved together before it is made smaller: bound by the copy
        _pages("copy_1024", "copy", 1, [0, 0], 1024, 8, 8, 128, "bfloat16", 64),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    """Batches of 1 to 256 trees of 2 to 256 nodes over 1000 to 150000 tokens, pools of up to 32 layers, up to 1024 pages copied."""
    op = rng.choices(["trees", "sampled", "compact", "fit", "fork", "copy"], weights=[4, 3, 3, 2, 2, 2])[0]
    if op in ("trees", "sampled"):
        vocabulary, dtype = _log_int(rng, 1000, 150000), rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
        high = _log_int(rng, 2, 256 if op == "trees" else 64)
        room = (1 << 29 if op == "trees" else 1 << 26) // (vocabulary * high)
        batch = max(1, min(_log_int(rng, 1, 256), room))
        low = max(2, high // rng.randint(1, 5))
        children = rng.randint(1, 8)
        return _verify(None, batch, [low, high], rng.randint(1, 12) if children > 1 else high - 1, children, vocabulary, dtype,
                       sampled=rng.choice(["float32", "bfloat16", "float16"]) if op == "sampled" else "", pad=rng.choice([0, 0, 8, 13]),
                       mixed=rng.random() < 0.4)
    kv_heads, head_dim, page = rng.choice([1, 2, 4, 8, 16]), rng.choice([64, 128, 128]), rng.choice([16, 32, 64, 128])
    dtype, fp8, layers = rng.choice(["bfloat16", "float16"]), rng.random() < 0.4, rng.randint(1, 32)
    row = layers * kv_heads * head_dim            # values of one position, K or V, in all layers
    if op == "copy":
        nodes = max(1, min(_log_int(rng, 1, 1024), (1 << 29) // (row * page)))
        return _pages(None, op, 1, [0, 0], nodes, layers, kv_heads, head_dim, dtype, page, fp8)
    if op == "fit":
        high = _log_int(rng, 30, 16000)
        batch = max(1, min(_log_int(rng, 1, 1024), (1 << 24) // (high + 256)))
        return _pages(None, op, batch, [max(1, high // rng.randint(1, 30)), high], _log_int(rng, 1, 256), 1, 1, 64, dtype, page, False)
    high = _log_int(rng, 10, 3000)
    nodes = rng.randint(1, 8) if op == "fork" else _log_int(rng, 2, 256)
    rows = high + page * (nodes + 1) if op == "fork" else high + nodes
    batch = max(1, min(_log_int(rng, 1, 128), (1 << 29) // (row * rows)))
    return _pages(None, op, batch, [max(1, high // rng.randint(1, 30)), high], nodes, layers, kv_heads, head_dim, dtype, page, fp8)


# ---- shapes and lengths of a case ---------------------------------------------------------------------------------------

def _spread(rng, low, high, count):
    """`count` lengths over the logarithm of [low, high], the largest among them."""
    values = [high] + [min(high, max(low, _log_int(rng, low, high))) for _ in range(count - 1)]
    rng.shuffle(values)
    return values


def _starts(lengths):
    out = [0]
    for n in lengths:
        out.append(out[-1] + n)
    return out


def _chance(rank):
    """How likely the model says the draft's guess of a rank."""
    return 0.5 * 0.45 ** rank


def _tree(nodes, depth, children):
    """Parents of the most likely paths of ranked guesses, numbered by depth (fewer nodes where the shape has no more)."""
    heap, taken = [(-1.0, ())], []
    while heap and len(taken) < nodes:
        score, path = heapq.heappop(heap)
        taken.append(path)
        if len(path) < depth:
            for r in range(children):
                heapq.heappush(heap, (score * _chance(r), path + (r,)))
    taken.sort(key=lambda p: (len(p), p))
    at = {p: i for i, p in enumerate(taken)}
    return [at[p[:-1]] if p else -1 for p in taken]


def _trees(case):
    rng = random.Random(case["batch"] * 1000003 + case["nodes_high"])
    known = {}
    out = []
    for n in _spread(rng, case["nodes_low"], case["nodes_high"], case["batch"]):
        if n not in known:
            known[n] = _tree(n, case["depth"], case["children"])
        out.append(known[n])
    return out


def _keys(case):
    rng = random.Random(case["batch"] * 1000003 + case["keys_high"] * 1009 + case["nodes"])
    return _spread(rng, case["keys_low"], case["keys_high"], case["batch"])


def _paths(case):
    """Accepted paths of a batch of trees: node numbers from the root.  No row of a path has its place where another one comes from,
    so that a second pass over the same rows leaves the same."""
    rng = random.Random(case["batch"] * 7919 + case["nodes"])
    parent = _tree(case["nodes"], 5, 6)
    below = [[j for j, p in enumerate(parent) if p == i] for i in range(len(parent))]
    out = []
    for _ in range(case["batch"]):
        path = [0]
        while below[path[-1]] and rng.random() < 0.85:
            path.append(below[path[-1]][min(len(below[path[-1]]) - 1, int(rng.expovariate(0.8)))])
        while any(p != i and p < len(path) for i, p in enumerate(path)):
            path.pop()
        out.append(path)
    return len(parent), out


# ---- what a program holds before the call -------------------------------------------------------------------------------

def _random_rows(shape, generator, dtype):
    return torch.randn(shape, generator=generator, dtype=dtype, device="cuda")


def _prepare_verify(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    trees, vocabulary = _trees(case), case["vocabulary"]
    starts = _starts([len(t) for t in trees])
    total = starts[-1]
    parent = torch.tensor([p for t in trees for p in t], dtype=torch.int64).cuda()
    above = torch.tensor([s + p if p >= 0 else -1 for t, s in zip(trees, starts) for p in t], dtype=torch.int64).cuda()
    ranks = []
    for t in trees:
        seen = {}
        for p in t:
            ranks.append(seen.get(p, 0))
            seen[p] = ranks[-1] + 1
    rank = torch.tensor(ranks, dtype=torch.int64).cuda()
    logits = _random_rows((total, vocabulary + case["pad"]), g, DTYPES[case["dtype"]])[:, :vocabulary]
    logits *= SIGMA
    tokens = torch.randint(vocabulary, (total,), generator=g, device="cuda")
    child = above >= 0
    up = above[child]
    state = {"case": dict(case), "logits": logits, "parent": parent, "starts": torch.tensor(starts, dtype=torch.int32).cuda(), "draft": None,
             "most_path": case["depth"] + 1, "most_children": max(ranks) + 1,
             "u_accept": torch.rand((total,), generator=g, device="cuda"), "u_next": torch.rand((case["batch"],), generator=g, device="cuda"),
             "temperature": 1.0}
    if case["sampled"]:
        # the draft model's probabilities, and children drawn from them one after the other, no token twice
        draft = torch.empty((total, vocabulary), dtype=DTYPES[case["sampled"]], device="cuda")
        most = int(state["most_children"])
        drawn = torch.empty((total, most), dtype=torch.int64, device="cuda")
        for a in range(0, total, 256):
            rows = logits[a:a + 256].float()
            q = torch.softmax(rows + 0.7 * torch.randn(rows.shape, generator=g, device="cuda"), -1)
            draft[a:a + 256] = q
            race = draft[a:a + 256].float() / torch.empty_like(q).exponential_(generator=g)
            drawn[a:a + 256] = race.topk(most, -1).indices
        tokens[child] = drawn[up, rank[child]]
        state["draft"] = draft
    else:
        # a draft head's ranked guesses; at one node in five the model says something else
        base = torch.randint(vocabulary, (total,), generator=g, device="cuda")
        tokens[child] = (base[up] + rank[child] * 101) % vocabulary
        miss = torch.rand((total,), generator=g, device="cuda") < 0.2
        rest = 1.0 - sum(_chance(r) for r in range(case["children"]))
        likely = math.log(vocabulary) + SIGMA ** 2 / 2 + torch.log(_chance(rank[child].double()) / rest)
        logits[up, tokens[child]] = torch.where(miss[up], likely - 9.0, likely).to(logits.dtype)
        logits[torch.arange(total, device="cuda"), (base + 50) % vocabulary] = torch.where(miss, math.log(vocabulary) + 5.5, 0.0).to(logits.dtype)
    if case["mixed"]:
        choice = torch.tensor([0.0, 0.6, 0.8, 1.0, 1.3])
        state["temperature"] = choice[torch.arange(case["batch"]) % 5].cuda()
    state["tokens"] = tokens
    return state


def _pool(case, pages, g):
    """k, v [layers, pages, heads, page, head_dim] (one allocation, a layer is a view) and the exponents of 8-bit rows."""
    shape = (case["layers"], pages, case["kv_heads"], case["page"], case["head_dim"])
    if not case["fp8"]:
        return [_random_rows(shape, g, DTYPES[case["dtype"]]) for _ in range(2)] + [None, None]
    rows = []
    for _ in range(2):
        rows.append(torch.empty(shape, dtype=torch.float8_e4m3fn, device="cuda"))
        for layer in range(case["layers"]):
            rows[-1][layer] = (_random_rows(shape[1:], g, torch.bfloat16) * 100.0).to(torch.float8_e4m3fn)
    return rows + [torch.randint(115, 125, shape[:4], generator=g, dtype=torch.uint8, device="cuda") for _ in range(2)]


def _prepare_pages(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    page, op = case["page"], case["op"]
    state = {"case": dict(case)}
    if op == "copy":
        total = 2 * case["nodes"] + 3
        order = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
        state.update(sources=order[:case["nodes"]].clone(), targets=order[case["nodes"]:2 * case["nodes"]].clone())
    else:
        keys = _keys(case)
        grown, slots = case["nodes"] if op != "fork" else 0, case["batch"] * (1 + case["nodes"]) if op == "fork" else case["batch"]
        width = -(-(max(keys) + grown) // page)
        held = [-(-(k + (case["nodes"] if op == "compact" else 0)) // page) for k in keys]
        spare = sum(-(-(k + grown) // page) for k in keys) - sum(held) if op == "fit" else case["batch"] * case["nodes"]
        total = sum(held) + spare + spare // 8 + 3
        order = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
        first, count = torch.tensor(_starts(held)[:-1]).cuda(), torch.tensor(held).cuda()
        at = torch.arange(width, device="cuda")
        table = torch.full((slots, width), -1, dtype=torch.int32, device="cuda")
        table[:case["batch"]] = torch.where(at < count[:, None], order[(first[:, None] + at).clamp(max=total - 1)], -1)
        refs = torch.zeros((total,), dtype=torch.int32, device="cuda")
        refs[order[:sum(held)].long()] = 1
        state.update(table=table, refs=refs, lens=torch.tensor(keys + [0] * (slots - case["batch"]), dtype=torch.int32).cuda())
        if op == "compact":
            count, paths = _paths(case)
            most = max(map(len, paths))
            state.update(path=torch.tensor([p + [-1] * (most - len(p)) for p in paths], dtype=torch.int32).cuda(),
                         counts=torch.tensor([len(p) for p in paths], dtype=torch.int32).cuda(),
                         starts=torch.arange(case["batch"] + 1, dtype=torch.int32, device="cuda") * count)
            state["lens"] += count
        if op == "fit":
            state["grown"] = state["lens"] + case["nodes"]
        if op == "fork":
            state["sources"] = torch.arange(case["batch"], dtype=torch.int32, device="cuda").repeat_interleave(case["nodes"])
            state["targets"] = torch.arange(case["batch"], slots, dtype=torch.int32, device="cuda")
    pool = _pool(case, total, g)
    state["pool"] = [x for x in pool if x is not None]
    state["layers"] = [tuple(None if x is None else x[i] for x in pool) for i in range(case["layers"])]
    return state


def prepare(case, seed):
    return _prepare_verify(case, seed) if case["op"] == "verify" else _prepare_pages(case, seed)


# ---- one pass -----------------------------------------------------------------------------------------------------------

def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(state):
    import fstattention_amd as fsta
    op = state["case"]["op"]
    if op == "verify":
        return tuple(fsta.verify_drafts(state["logits"], state["tokens"], state["parent"], state["starts"], state["u_accept"], state["u_next"],
                                        state["most_path"], temperature=state["temperature"], draft_probs=state["draft"]))
    layers = state["layers"]
    if op == "copy":
        fsta.copy_pages(layers, state["sources"], state["targets"])
        return state["pool"]
    table, refs, lens = state["table"], state["refs"], state["lens"]
    if op == "compact":
        return state["pool"] + [fsta.compact_paged_kv(layers, state["path"], state["counts"], table, lens, state["starts"])]
    if op == "fit":
        short = fsta.fit_pages(layers, refs, table, state["grown"])
        grown = table.clone()
        return short, grown, fsta.fit_pages(layers, refs, table, lens), table, refs
    fsta.fit_pages(layers, refs, table, lens)
    lens = lens.clone()
    return [fsta.fork_pages(layers, refs, table, lens, state["sources"], state["targets"]), table, refs, lens] + state["pool"]


def _run_plain(state):
    op = state["case"]["op"]
    if op == "verify":
        return _verify_plain(state)
    if op == "copy":
        for x in state["pool"]:
            x = _bytes(x)
            x[:, state["targets"].long()] = x[:, state["sources"].long()]
        return state["pool"]
    table, refs, lens = state["table"], state["refs"], state["lens"]
    if op == "compact":
        return state["pool"] + [_compact_plain(state)]
    if op == "fit":
        short = _fit_plain(state, refs, table, state["grown"])
        grown = table.clone()
        return short, grown, _fit_plain(state, refs, table, lens), table, refs
    _fit_plain(state, refs, table, lens)
    lens = lens.clone()
    return [_fork_plain(state, refs, table, lens), table, refs, lens] + state["pool"]


def _bytes(x):
    return x.view(torch.uint8) if x.dtype == torch.float8_e4m3fn else x


def _children(state):
    """[nodes, most_children] packed numbers of every node's children in order, -1 where there are no more."""
    starts, parent = state["starts"].long(), state["parent"]
    total = parent.shape[0]
    t = torch.arange(total, device=parent.device)
    first = starts[(starts[1:, None] <= t).sum(0)]
    above = torch.where((parent >= 0) & (parent < t - first), first + parent, total)
    order = above.argsort(stable=True)
    rows = above[order]
    rank = t - torch.searchsorted(rows, rows)
    table = torch.full((total + 1, max(state["most_children"], 1)), -1, dtype=torch.int64, device=parent.device)
    table[rows, torch.where(rows < total, rank, 0)] = order
    return table[:total], first


def _verify_plain(state):
    logits, tokens, draft = state["logits"], state["tokens"], state["draft"]
    batch, vocabulary = state["case"]["batch"], logits.shape[1]
    children, _ = _children(state)
    first = state["starts"].long()[:-1]
    tau = torch.as_tensor(state["temperature"], dtype=torch.float32, device=logits.device).double().expand(batch)
    u_accept, u_next = state["u_accept"].double(), state["u_next"].double()
    node = first
    going = torch.ones((batch,), dtype=torch.bool, device=logits.device)
    path = torch.full((batch, state["most_path"]), -1, dtype=torch.int32, device=logits.device)
    weights = torch.zeros((batch, vocabulary), dtype=torch.float64, device=logits.device)
    counts = torch.zeros((batch,), dtype=torch.int32, device=logits.device)
    column = torch.arange(vocabulary, device=logits.device)
    for step in range(state["most_path"]):
        path[:, step] = torch.where(going, node - first, -1).int()
        counts += going
        rows = logits[node].double()
        top = rows.amax(1, keepdim=True)
        best = torch.where(rows == top, column, vocabulary).amin(1, keepdim=True)
        p = torch.where(tau[:, None] > 0, torch.exp((rows - top) / tau.clamp(min=1e-30)[:, None]), (column == best).double())
        q = torch.where(tau[:, None] > 0, draft[node].double(), 0.0) if draft is not None else None
        w = p.clone()
        z = w.sum(1)
        shift, left = torch.zeros_like(z), torch.ones_like(z)
        goes_on = torch.zeros_like(going)
        after = node
        for r in range(state["most_children"] if step + 1 < state["most_path"] else 0):
            child = children[node, r]
            x = tokens[child.clamp(min=0)][:, None]
            asked = going & ~goes_on & (child >= 0)
            wx, u = w.gather(1, x)[:, 0], u_accept[child.clamp(min=0)]
            if q is None:
                good = u * z < wx
            else:
                qx = q.gather(1, x)[:, 0]
                drawn = (qx > 0) & (left > 0)
                good = torch.where(drawn, u * z * qx < wx * left, u * z < wx)
                fell = asked & ~good & drawn
                shift = torch.where(fell, shift + z / left, shift)
                left = torch.where(fell, left - qx, left)
            after = torch.where(asked & good, child, after)
            goes_on |= asked & good
            p.scatter_(1, x, torch.where((asked & ~good)[:, None], 0.0, p.gather(1, x)))
            w = p if q is None else (p - shift[:, None] * q).clamp_(min=0)
            z = w.sum(1)
        weights = torch.where((going & ~goes_on)[:, None], w, weights)
        going, node = goes_on, after
    sums = weights.cumsum(1)
    choice = torch.searchsorted(sums, (u_next * sums[:, -1])[:, None], right=True)[:, 0]
    last = torch.where(weights > 0, column, -1).amax(1)
    return path, counts, torch.where(choice < vocabulary, choice, last)


def _compact_plain(state):
    path, table, page = state["path"].long(), state["table"].long(), state["case"]["page"]
    lens, starts = state["lens"].long(), state["starts"].long()
    base = lens - (starts[1:] - starts[:-1])
    i = torch.arange(path.shape[1], device=path.device).expand_as(path)
    moved = (i < state["counts"][:, None]) & (path != i)
    seq, i = moved.nonzero(as_tuple=True)
    old, new = base[seq] + path[seq, i], base[seq] + i
    source, target = (table[seq, old // page], old % page), (table[seq, new // page], new % page)
    for layer in state["layers"]:
        for x in layer:
            if x is not None:
                x = _bytes(x)
                x[target[0], :, target[1]] = x[source[0], :, source[1]]
    return (base + state["counts"]).int()


def _named_pages(table, refs):
    return (table >= 0) & (table < refs.shape[0])


def _copy_tails(state, old, new, rows):
    """The first `rows` rows of pages `old` to pages `new`, in every layer."""
    here = torch.arange(state["case"]["page"], device=rows.device) < rows[:, None]
    which, row = here.nonzero(as_tuple=True)
    for x in state["pool"]:
        x = _bytes(x)
        x[:, new[which], :, row] = x[:, old[which], :, row]


def _free_pages(refs):
    """Pages that nobody has, the lowest first, and how many there are."""
    free = refs <= 0
    return (~free).to(torch.uint8).argsort(stable=True), free.sum()


def _fit_plain(state, refs, table, lens):
    page = state["case"]["page"]
    n = lens.long().clamp(min=0, max=table.shape[1] * page)[:, None]
    keep, slot = (n + page - 1) // page, torch.arange(table.shape[1], device=table.device)
    named = _named_pages(table, refs)
    at = torch.where(named, table, 0).long()
    inside = slot < keep
    shared = inside & named & (slot == keep - 1) & (n % page != 0) & (refs[at] > 1)
    wanted = (inside & ~named) | shared
    free, count = _free_pages(refs)
    number = wanted.view(-1).cumsum(0).view_as(wanted) - 1
    got = wanted & (number < count)
    new = free[number.clamp(min=0, max=free.shape[0] - 1)]
    copied = (shared & got).nonzero(as_tuple=True)
    _copy_tails(state, at[copied], new[copied], n[copied[0], 0] % page)
    gone = (named & ~inside) | (shared & got)
    refs.index_add_(0, at.view(-1), -gone.view(-1).int())
    refs[new[got]] = 1
    table.copy_(torch.where(got, new.int(), torch.where(inside & named, table, -1)))
    return (wanted & ~got).sum(1).int()


def _fork_plain(state, refs, table, lens):
    page = state["case"]["page"]
    source, target = state["sources"].long(), state["targets"].long()
    n = lens[source].long().clamp(min=0, max=table.shape[1] * page)[:, None]
    keep, slot = (n + page - 1) // page, torch.arange(table.shape[1], device=table.device)
    rows = table[source]
    named = _named_pages(rows, refs) & (slot < keep)
    tail = named & (slot == keep - 1) & (n % page != 0)
    free, count = _free_pages(refs)
    number = (tail.any(1).cumsum(0) - 1)[:, None].expand_as(tail)
    good = ~tail.any(1) | (number[:, 0] < count)
    new = free[number.clamp(min=0, max=free.shape[0] - 1)]
    at = torch.where(named, rows, 0).long()
    copied = (tail & good[:, None]).nonzero(as_tuple=True)
    _copy_tails(state, at[copied], new[copied], n[copied[0], 0] % page)
    old = table[target]
    gone = _named_pages(old, refs)
    refs.index_add_(0, torch.where(gone, old, 0).long().view(-1), -gone.view(-1).int())
    refs.index_add_(0, at.view(-1), (named & ~tail & good[:, None]).view(-1).int())
    refs[new[copied]] = 1
    table[target] = torch.where(good[:, None] & named, torch.where(tail, new.int(), rows), -1)
    lens[target] = torch.where(good, n[:, 0], 0).int()
    return (~good).int()


# ---- the result in 64 bits ----------------------------------------------------------------------------------------------

def exact(case, seed):
    """Rows that move are what they were; where they end is worked out here one by one."""
    if case["op"] in ("verify", "fit"):
        return None                     # whole numbers only
    state, page = prepare(case, seed), case["page"]

    def value(x):
        return x.double() if "float" in str(x.dtype) else None

    pairs = []                          # (page, row) from, (page, row) to
    if case["op"] == "copy":
        for a, b in zip(state["sources"].tolist(), state["targets"].tolist()):
            pairs += [((a, r), (b, r)) for r in range(page)]
    table = state["table"].tolist() if case["op"] != "copy" else None
    if case["op"] == "compact":
        starts, lens = state["starts"].tolist(), state["lens"].tolist()
        for b, path in enumerate(state["path"].tolist()):
            base = lens[b] - (starts[b + 1] - starts[b])
            for i, p in enumerate(path):
                if p >= 0:
                    pairs.append(((table[b][(base + p) // page], (base + p) % page), (table[b][(base + i) // page], (base + i) % page)))
    if case["op"] == "fork":
        free = [i for i, n in enumerate(state["refs"].tolist()) if n == 0]
        lens = state["lens"].tolist()
        for a in state["sources"].tolist():
            if lens[a] % page:
                new = free.pop(0)
                pairs += [((table[a][lens[a] // page], r), (new, r)) for r in range(lens[a] % page)]
    moved = []
    old, new = (torch.tensor([p[k] for p in pairs] or [(0, 0)]).cuda() for k in (0, 1))
    for x in state["pool"]:
        y = value(x)
        if y is not None:
            y[:, new[:, 0], :, new[:, 1]] = y[:, old[:, 0], :, old[:, 1]]
        moved.append(y)
    return moved + [None] if case["op"] == "compact" else [None] * 4 + moved if case["op"] == "fork" else moved


# ---- what a pass cannot do without --------------------------------------------------------------------------------------

def work(case):
    if case["op"] == "verify":
        trees, size = _trees(case), {"float32": 4, "float16": 2, "bfloat16": 2}
        # the rows of the nodes on an accepted path and the draft's row of the one where it ends, as often as the inputs are likely to go on
        on = 0.75 if case["sampled"] else 0.8 * sum(_chance(r) for r in range(case["children"]))
        rows = 0.0
        for t in trees:
            depth = [0] * len(t)
            for i, p in enumerate(t[1:], 1):
                depth[i] = depth[p] + 1
            rows += sum(on ** d for d in range(max(depth) + 1))
        read = case["vocabulary"] * (rows * size[case["dtype"]] + (len(trees) * size[case["sampled"]] if case["sampled"] else 0))
        nodes = sum(map(len, trees))
        return {"bytes": read + 20 * nodes + len(trees) * (4 * (case["depth"] + 1) + 20), "flops": 4 * case["vocabulary"] * rows}
    row = 2 * case["layers"] * case["kv_heads"] * (case["head_dim"] + 1 if case["fp8"] else 2 * case["head_dim"])
    if case["op"] == "copy":
        return {"bytes": 2 * row * case["page"] * case["nodes"] + 8 * case["nodes"], "flops": 0}
    keys, page = _keys(case), case["page"]
    if case["op"] == "compact":
        _, paths = _paths(case)
        moved = sum(p != i for path in paths for i, p in enumerate(path))
        return {"bytes": 2 * row * moved + 8 * moved + 4 * sum(map(len, paths)) + 12 * len(keys), "flops": 0}
    if case["op"] == "fit":
        width = -(-(max(keys) + case["nodes"]) // page)
        taken = sum(-(-(k + case["nodes"]) // page) - -(-k // page) for k in keys)
        # both calls look for what the table lacks or has over; who is free is looked for once
        pages = sum(-(-k // page) for k in keys) + taken
        return {"bytes": 2 * 4 * len(keys) * width + 4 * (pages + taken // 8 + 3) + 4 * 4 * taken + 16 * len(keys) + 2 * 4 * len(keys) * width, "flops": 0}
    copies = case["nodes"]
    held = sum(-(-k // page) for k in keys)
    return {"bytes": copies * sum(2 * row * (k % page) for k in keys) + 4 * held * (1 + 3 * copies) + 12 * len(keys) * copies, "flops": 0}
