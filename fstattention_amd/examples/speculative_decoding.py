"""Speculative decoding of a batch of conversations over a paged KV cache, with draft trees:
``python -m fstattention_amd.examples.speculative_decoding``.

A small transformer of random weights reads prompts of different lengths in chunks, then answers.  Every step drafts a tree of
likely continuations per conversation (:func:`medusa_parents_gpu`: its shape), turns it into masks (:func:`tree_mask_bits`), and
runs the model once over all nodes: per layer their keys and values go to the pages behind the conversation's
(:func:`write_paged_kv`) and every node attends to the conversation and to its own branch (:func:`paged_attention`).  The branch
that the model agrees with is kept: its keys and values are written again, to the places directly behind the conversation's.
Nothing in a step waits for the GPU: lengths, starts and the page table live there.

The answers are those of decoding one token at a time (``draft=0``), in fewer steps; where two tokens are equally likely but for
the rounding of bfloat16, either may be taken.
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
    """The pages of a batch: a pool per layer, one page table for all of them (drawn in a random order, as a long-running server's
    pages lie), and on the GPU the lengths so far."""

    def __init__(self, model: Model, batch: int, most_tokens: int, page_size: int = 16, fp8: bool = False):
        per = -(-most_tokens // page_size)
        dtype = torch.float8_e4m3fn if fp8 else torch.bfloat16
        self.pools = [fsta.paged_kv_cache(batch * per, model.kv_heads, page_size, model.head_dim, dtype, device="cuda") for _ in model.qkv]
        order = torch.randperm(batch * per, generator=torch.Generator().manual_seed(1))
        self.page_table = order.view(batch, per).to(device="cuda", dtype=torch.int32)
        self.lens = torch.zeros(batch, dtype=torch.int32, device="cuda")


def _norm(x):
    return x * (x.float().square().mean(-1, keepdim=True) + 1e-6).rsqrt().to(x.dtype)


def _place(positions, width):
    """Sines and cosines of a token's position"""
    rate = 10000.0 ** (-torch.arange(width // 2, device=positions.device) / (width // 2))
    angle = positions[:, None].float() * rate
    return torch.cat([angle.sin(), angle.cos()], 1).bfloat16()


def forward(model: Model, talk: Conversations, tokens, positions, kv_lens, q_starts, tree_bits=None, most_new: Optional[int] = None):
    """Packed new tokens ``[T]`` of a batch -> logits ``[T, vocabulary]`` and, per layer, their keys and values (views)."""
    x = model.embed[tokens] + 0.1 * _place(positions, model.embed.shape[1])
    h, hk, d = model.heads, model.kv_heads, model.head_dim
    kept = []
    for pool, w_qkv, w_out in zip(talk.pools, model.qkv, model.out):
        fused = (_norm(x) @ w_qkv).view(-1, h + 2 * hk, d)
        q, k, v = fused[:, :h], fused[:, h:h + hk], fused[:, h + hk:]
        fsta.write_paged_kv(pool, k, v, talk.page_table, kv_lens, q_starts)
        o = fsta.paged_attention(q, pool, talk.page_table, kv_lens, q_starts, d ** -0.5, tree_bits=tree_bits, max_q_len=most_new)
        x = x + 0.3 * (o.reshape(-1, h * d) @ w_out)
        kept.append((k, v))
    return _norm(x).float() @ model.unembed.float(), kept


def read_prompts(model: Model, talk: Conversations, prompts: List[List[int]], chunk: int = 64):
    """Prompts in chunks of up to ``chunk`` tokens a conversation -> each one's next token ``[B]``"""
    last = torch.zeros(len(prompts), dtype=torch.int64, device="cuda")
    for at in range(0, max(map(len, prompts)), chunk):
        parts = [p[at:at + chunk] for p in prompts]
        new = torch.tensor([len(p) for p in parts], dtype=torch.int32, device="cuda")
        starts = torch.nn.functional.pad(new.cumsum(0, dtype=torch.int32), (1, 0))
        tokens = torch.tensor([t for p in parts for t in p], device="cuda")
        positions = torch.tensor([at + i for p in parts for i in range(len(p))], device="cuda")
        talk.lens += new
        logits, _ = forward(model, talk, tokens, positions, talk.lens, starts, most_new=max(map(len, parts)))
        ends = (starts[1:].long() - 1).clamp(min=0)
        last = torch.where(new > 0, logits[ends].argmax(-1), last)
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
        self.bits = fsta.tree_mask_bits(self.parent.repeat(batch), self.starts, nodes)

    def tokens(self, last):
        """Token of every node ``[B, nodes]`` below the roots ``last [B]``"""
        up = self.parent.clamp(min=0)
        t = last[:, None].expand(-1, self.nodes)
        for _ in range(self.depths):
            t = torch.where(self.parent >= 0, self.guesses[t[:, up], self.rank], last[:, None])
        return t


def tree_step(model: Model, talk: Conversations, drafts: Drafts, last):
    """One step: ``last [B]`` is every conversation's newest token, not in the cache yet.  Returns the tokens of the step ``[B,
    depths + 1]`` (-1 behind the accepted ones) and the next ``last``."""
    batch, n, up = last.shape[0], drafts.nodes, drafts.parent.clamp(min=0)
    tokens = drafts.tokens(last)
    positions = (talk.lens[:, None] + drafts.depth).reshape(-1)
    logits, kept = forward(model, talk, tokens.reshape(-1), positions, talk.lens + n, drafts.starts, drafts.bits, n)
    says = logits.argmax(-1).view(batch, n)
    # a node is accepted where the model says its token at its parent, and the parent is accepted
    agrees = (tokens == says[:, up]) | (drafts.parent < 0)
    accepted = agrees
    for _ in range(drafts.depths):
        accepted = agrees & (accepted[:, up] | (drafts.parent < 0))
    # one branch at most: its nodes in order, padded
    order = torch.where(accepted, drafts.depth, drafts.depths + 1).argsort(dim=1, stable=True)[:, :drafts.depths + 1]
    counts = accepted.sum(1)
    valid = torch.arange(drafts.depths + 1, device="cuda") < counts[:, None]
    said = torch.where(valid, says.gather(1, order), -1)
    # the branch's rows, all conversations' behind each other (rows behind the last one are of no conversation)
    first = torch.arange(batch, device="cuda")[:, None] * n
    rows = (first + order).reshape(-1)[(~valid).reshape(-1).byte().argsort(dim=0, stable=True)]
    starts = torch.nn.functional.pad(counts.cumsum(0), (1, 0)).int()
    talk.lens += counts.int()
    for pool, (k, v) in zip(talk.pools, kept):
        fsta.write_paged_kv(pool, k[rows], v[rows], talk.page_table, talk.lens, starts)
    return said, said.gather(1, counts[:, None] - 1)[:, 0]


def answer(model: Model, prompts: List[List[int]], steps: int, draft: int = 32, fp8: bool = False):
    """``steps`` steps for a batch of prompts; ``draft``: nodes of a tree, 0 for one token a step.  Returns the answers (lists of
    tokens) and the conversations."""
    batch, most = len(prompts), max(map(len, prompts)) + steps * 5 + draft + 1
    talk = Conversations(model, batch, most, fp8=fp8)
    last = read_prompts(model, talk, prompts)
    said = [last[:, None]]
    if draft:
        drafts = Drafts(model, batch, draft)
        for _ in range(steps):
            tokens, last = tree_step(model, talk, drafts, last)
            said.append(tokens)
    else:
        starts = torch.arange(batch + 1, dtype=torch.int32, device="cuda")
        for _ in range(steps):
            talk.lens += 1
            logits, _ = forward(model, talk, last, talk.lens - 1, talk.lens, starts, most_new=1)
            last = logits.argmax(-1)
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


if __name__ == "__main__":
    main()
