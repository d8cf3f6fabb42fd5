"""Speculative decoding of a batch of conversations over a paged KV cache, with draft trees:
``python -m fstattention_amd.examples.speculative_decoding``.

A small transformer of random weights reads prompts of different lengths in chunks, then answers each one or several times.  Every
step drafts a tree of likely continuations per conversation (:func:`medusa_parents_gpu`: its shape), turns it into masks
(:func:`tree_mask_bits`), and runs the model once over all nodes: per layer their keys and values go to the pages behind the
conversation's (:func:`write_paged_kv`) and every node attends to the conversation and to its own branch (:func:`paged_attention`).  The
branch that the model agrees with, and the token behind it, come from :func:`verify_drafts`; its keys and values move to the places
directly behind the conversation's (:func:`compact_paged_kv`).  Pages are given out before a pass and taken back behind it
(:func:`fit_pages`); several answers share the prompt's (:func:`fork_pages`); where they could run out they move to a larger pool
(:func:`copy_pages`).  Nothing in a step waits for the GPU: lengths, starts, the page table and who holds which page live there.

The answers are those of decoding one token at a time (``draft=0``), in fewer steps; where two tokens are equally likely but for
the rounding of bfloat16, either may be taken.  At a temperature they are drawn as the model alone would draw them.
"""
from typing import List, NamedTuple, Optional

import torch

import fstattention_amd as fsta


class Model(NamedTuple):
    embed: torch.Tensor             # [vocabulary, width]
    unembed: torch.Tensor           # [width, vocabulary]
    qkv: List[torch.Tensor]         # [width, (H + 2 Hkv) * D]
    out: List[torch.Tensor]         # [H * D, width]
    heads: int
    kv_heads: int
    head_dim: int


def make_model(vocabulary=512, width=256, layers=4, heads=8, kv_heads=2, head_dim=64, seed=0, device="cuda") -> Model:
    g = torch.Generator().manual_seed(seed)
    draw = lambda *shape: (torch.randn(shape, generator=g) * shape[0] ** -0.5).to(device=device, dtype=torch.bfloat16)
    embed = draw(vocabulary, width) * vocabulary ** 0.5
    return Model(embed, draw(width, vocabulary), [draw(width, (heads + 2 * kv_heads) * head_dim) for _ in range(layers)],
                 [draw(heads * head_dim, width) for _ in range(layers)], heads, kv_heads, head_dim)


class Conversations:
    """The pages of a batch: a pool per layer and one page table for all of them, empty at first; on the GPU the lengths so far, and
    by how many entries of the table each page is held."""

    def __init__(self, model: Model, batch: int, most_tokens: int, page_size: int = 16, fp8: bool = False, pages: Optional[int] = None):
        width = -(-most_tokens // page_size)
        dtype = torch.float8_e4m3fn if fp8 else torch.bfloat16
        self.page_size = page_size
        self._make = lambda pages: [fsta.paged_kv_cache(pages, model.kv_heads, page_size, model.head_dim, dtype, device="cuda") for _ in model.qkv]
        self.pools = self._make(batch * width if pages is None else pages)
        self.refs = torch.zeros(self.pools[0].k.shape[0], dtype=torch.int32, device="cuda")
        self.page_table = torch.full((batch, width), -1, dtype=torch.int32, device="cuda")
        self.lens = torch.zeros(batch, dtype=torch.int32, device="cuda")

    def fit(self, lens):
        """Pages for lengths ``lens``, and no others -> how many there were not, per conversation"""
        return fsta.fit_pages(self.pools, self.refs, self.page_table, lens)

    def grow(self, pages: int):
        """To pools of ``pages`` pages; those there are keep their numbers"""
        held = torch.arange(self.refs.shape[0], dtype=torch.int32, device="cuda")
        larger = self._make(pages)
        fsta.copy_pages(self.pools, held, held, into=larger)
        self.pools, self.refs = larger, torch.nn.functional.pad(self.refs, (0, pages - self.refs.shape[0]))


def _norm(x):
    return x * (x.float().square().mean(-1, keepdim=True) + 1e-6).rsqrt().to(x.dtype)


def _place(positions, width):
    """Sines and cosines of a token's position"""
    rate = 10000.0 ** (-torch.arange(width // 2, device=positions.device) / (width // 2))
    angle = positions[:, None].float() * rate
    return torch.cat([angle.sin(), angle.cos()], 1).bfloat16()


def forward(model: Model, talk: Conversations, tokens, positions, kv_lens, q_starts, tree_bits=None, most_new: Optional[int] = None):
    """Packed new tokens ``[T]`` of a batch -> logits ``[T, vocabulary]``; their keys and values are in the pages then."""
    x = model.embed[tokens] + 0.1 * _place(positions, model.embed.shape[1])
    h, hk, d = model.heads, model.kv_heads, model.head_dim
    for pool, w_qkv, w_out in zip(talk.pools, model.qkv, model.out):
        fused = (_norm(x) @ w_qkv).view(-1, h + 2 * hk, d)
        q, k, v = fused[:, :h], fused[:, h:h + hk], fused[:, h + hk:]
        fsta.write_paged_kv(pool, k, v, talk.page_table, kv_lens, q_starts)
        o = fsta.paged_attention(q, pool, talk.page_table, kv_lens, q_starts, d ** -0.5, tree_bits=tree_bits, max_q_len=most_new)
        x = x + 0.3 * (o.reshape(-1, h * d) @ w_out)
    return _norm(x).float() @ model.unembed.float()


def say(logits, starts, temperature: float):
    """A token per row of logits, as the model alone says it: a tree of one node"""
    batch = logits.shape[0]
    none = torch.full((batch,), -1, dtype=torch.int64, device="cuda")
    u = torch.rand(2, batch, device="cuda")
    return fsta.verify_drafts(logits, none, none, starts, u[0], u[1], 1, temperature=temperature).next_tokens


def read_prompts(model: Model, talk: Conversations, prompts: List[List[int]], chunk: int = 64):
    """Prompts in chunks of up to ``chunk`` tokens a conversation -> the logits behind each ``[B, vocabulary]``"""
    last = torch.zeros((len(prompts), model.unembed.shape[1]), device="cuda")
    for at in range(0, max(map(len, prompts)), chunk):
        parts = [p[at:at + chunk] for p in prompts]
        new = torch.tensor([len(p) for p in parts], dtype=torch.int32, device="cuda")
        starts = torch.nn.functional.pad(new.cumsum(0, dtype=torch.int32), (1, 0))
        tokens = torch.tensor([t for p in parts for t in p], device="cuda")
        positions = torch.tensor([at + i for p in parts for i in range(len(p))], device="cuda")
        talk.lens += new
        talk.fit(talk.lens)
        logits = forward(model, talk, tokens, positions, talk.lens, starts, most_new=max(map(len, parts)))
        ends = (starts[1:].long() - 1).clamp(min=0)
        last = torch.where((new > 0)[:, None], logits[ends], last)
    return last


class Drafts:
    """One tree shape for all conversations (from the draft's chances per depth and rank) and the draft itself: what the model
    would say next if it had no layers, its ``topk`` best guesses per token."""

    def __init__(self, model: Model, batch: int, nodes: int, depths: int = 4, topk: int = 4):
        chances = torch.softmax(-torch.arange(topk, dtype=torch.float64) * 1.5, 0).expand(depths, topk).contiguous()
        self.depths, self.nodes = depths, nodes
        self.parent = fsta.medusa_parents_gpu(chances.to("cuda"), nodes)
        siblings = (self.parent[:, None] == self.parent[None, :]).tril(-1)
        self.rank = siblings.sum(1)                                  # of a node among its parent's children
        self.depth = torch.zeros_like(self.parent)
        for _ in range(depths):
            self.depth = torch.where(self.parent >= 0, self.depth[self.parent.clamp(min=0)] + 1, 0)
        self.guesses = (_norm(model.embed).float() @ model.unembed.float()).topk(topk, -1).indices       # [vocabulary, topk]
        self.starts = torch.arange(batch + 1, dtype=torch.int32, device="cuda") * nodes
        self.parents = self.parent.repeat(batch)
        self.bits = fsta.tree_mask_bits(self.parents, self.starts, nodes)

    def tokens(self, last):
        """Token of every node ``[B, nodes]`` below the roots ``last [B]``"""
        up = self.parent.clamp(min=0)
        t = last[:, None].expand(-1, self.nodes)
        for _ in range(self.depths):
            t = torch.where(self.parent >= 0, self.guesses[t[:, up], self.rank], last[:, None])
        return t


def tree_step(model: Model, talk: Conversations, drafts: Drafts, last, temperature: float = 0.0):
    """One step: ``last [B]`` is every conversation's newest token, not in the cache yet.  Returns the tokens of the step ``[B,
    depths + 1]`` (-1 behind the last one) and the next ``last``."""
    batch, n = last.shape[0], drafts.nodes
    tokens = drafts.tokens(last)
    positions = (talk.lens[:, None] + drafts.depth).reshape(-1)
    grown = talk.lens + n
    talk.fit(grown)
    logits = forward(model, talk, tokens.reshape(-1), positions, grown, drafts.starts, drafts.bits, n)
    path, counts, following = fsta.verify_drafts(logits, tokens.reshape(-1), drafts.parents, drafts.starts, torch.rand(batch * n, device="cuda"),
                                                 torch.rand(batch, device="cuda"), drafts.depths + 1, temperature=temperature)
    talk.lens = fsta.compact_paged_kv(talk.pools, path, counts, talk.page_table, grown, drafts.starts)
    talk.fit(talk.lens)
    # the drafts that stand, below the root that was said before, and the token behind them
    said = tokens.gather(1, torch.nn.functional.pad(path[:, 1:], (0, 1)).clamp(min=0).long())
    at = counts[:, None].long() - 1
    said = torch.where(torch.arange(drafts.depths + 1, device="cuda") < at, said, -1).scatter(1, at, following[:, None])
    return said, following


def answer(model: Model, prompts: List[List[int]], steps: int, draft: int = 32, fp8: bool = False, each: int = 1, temperature: float = 0.0):
    """``steps`` steps for a batch of prompts, each answered ``each`` times; ``draft``: nodes of a tree, 0 for one token a step.
    Returns the answers (lists of tokens, a prompt's behind each other) and the conversations."""
    prompts = [p for q in prompts for p in [q] + [[]] * (each - 1)]
    batch, most = len(prompts), max(map(len, prompts)) + steps * 5 + draft + 1
    starts = torch.arange(batch + 1, dtype=torch.int32, device="cuda")
    # pages that hold the prompts and some tokens behind each; what a step may need is known without a look at the GPU
    lens = [len(prompts[i - i % each]) + draft + 1 for i in range(batch)]
    needed = lambda steps: sum(-(-(n + steps * 5) // 16) for n in lens)
    talk = Conversations(model, batch, most, 16, fp8, pages=needed(4))
    logits = read_prompts(model, talk, prompts)
    if each > 1:
        first = torch.arange(batch, dtype=torch.int32, device="cuda") // each * each
        fsta.fork_pages(talk.pools, talk.refs, talk.page_table, talk.lens, first, starts[:-1])
        logits = logits[first]
    last = say(logits, starts, temperature)
    said = [last[:, None]]
    drafts = Drafts(model, batch, draft) if draft else None
    for i in range(steps):
        if needed(i) > talk.refs.shape[0]:
            talk.grow(needed(min(2 * i, steps)))
        if draft:
            tokens, last = tree_step(model, talk, drafts, last, temperature)
            said.append(tokens)
        else:
            talk.lens += 1
            talk.fit(talk.lens)
            last = say(forward(model, talk, last, talk.lens - 1, talk.lens, starts, most_new=1), starts, temperature)
            said.append(last[:, None])
    return [[t for t in row if t >= 0] for row in torch.cat(said, 1).tolist()], talk


def main():
    model = make_model()
    g = torch.Generator().manual_seed(3)
    prompts = [torch.randint(512, (n,), generator=g).tolist() for n in (7, 130, 64, 33)]
    fast, talk = answer(model, prompts, 24)
    plain, _ = answer(model, prompts, max(map(len, fast)) - 1, draft=0)
    for i, (a, b) in enumerate(zip(fast, plain)):
        same = next((j for j, (x, y) in enumerate(zip(a, b)) if x != y), min(len(a), len(b)))
        print(f"conversation {i}: {len(prompts[i])} tokens of prompt, {len(a)} tokens in 24 steps, the first {same} as one at a time")
    k, v = fsta.read_paged_kv(talk.pools[0], talk.page_table, talk.lens, int(talk.lens.max()))
    print(f"the first layer's cache leaves its pages as {tuple(k.shape)}, {k.dtype}")
    several, talk = answer(model, prompts, 24, each=4, temperature=0.5)
    print(f"four answers each at a temperature of 0.5: {sum(map(len, several))} tokens; {int((talk.refs > 0).sum())} pages hold what "
          f"{int(talk.refs.sum())} would if none were shared")


if __name__ == "__main__":
    main()
