"""A whole decoder block: attention over a paged cache, then the MoE layer.

    h1  = h + Wo . attention(norm(h))          DecoderBlock.attend
    out = h1 + MoE(norm(h1))                   MoELayer.forward_block / prefill

The projections are trunk matrices (Q4 or Q8, ops.mvq_matvec), their fp32
results go straight to ops.kv_append (norm for each head, rotation, cache), and
ops.paged_attention reads the pages.  A Step holds what the layers of one step
share: which tokens belong to which request, where their keys go, and a prefix
that the requests have in common.

    step = Step.plan(q_lens, kv_lens, pages, page_size)      # once a step
    for block, (k_pages, v_pages) in zip(blocks, caches):
        h = block.forward(h, k_pages, v_pages, step)

A step of drafted tokens (Step.draft) is planned on the device, pages included, and
its attention is that of trees.  Decoder runs such steps from tokens to tokens:
plan, embedding, blocks, head, pick, accept.
"""
from dataclasses import dataclass

import torch

from . import ops

TRUNK_TOKENS = 64               # tokens ops.mvq_matvec takes at once


@dataclass
class Trunk:
    """A Q4 or Q8 matrix [out][in] on the device, as ops.mvq_matvec takes it."""
    w: torch.Tensor
    scales: torch.Tensor
    out: int
    in_: int
    group: int
    bits: int

    def __call__(self, x):
        """x [T][in] -> fp32 [T][out]."""
        y = [ops.mvq_matvec(self.w, self.scales, part, self.out, self.in_, self.group, self.bits)
             for part in x.split(TRUNK_TOKENS)]
        return y[0] if len(y) == 1 else torch.cat(y)


@dataclass
class Step:
    """One step's batch: request b brings q_lens[b] tokens, the last of its
    kv_lens[b] own keys, and keeps its keys in the pages of pages[b].  With a
    prefix, prefix_len keys of prefix_pages come before every request's own.  seen:
    the masks of a step whose requests bring trees of drafted tokens."""
    q_start: torch.Tensor
    kv_len: torch.Tensor
    pages: torch.Tensor
    max_q: int
    max_kv: int
    positions: torch.Tensor
    slots: torch.Tensor
    prefix_pages: torch.Tensor = None
    prefix_len: int = 0
    seen: torch.Tensor = None

    @classmethod
    def plan(cls, q_lens, kv_lens, pages, page_size, prefix_pages=None, prefix_len=0):
        """q_lens and kv_lens are lists; pages int32 [batch][n] on the device.  What
        the page numbers themselves leave out is for ops.attn_status to say."""
        if len(q_lens) != len(kv_lens) or not q_lens:
            raise ValueError("q_lens and kv_lens must name the same requests, one at least")
        if pages.dim() != 2 or pages.shape[0] != len(q_lens):
            raise ValueError("pages must have a row for each request")
        held = pages.shape[1] * page_size
        for b, (n, kv) in enumerate(zip(q_lens, kv_lens)):
            if not 0 <= n <= kv <= held:
                raise ValueError(f"request {b}: {n} tokens, the last of {kv} keys, in pages for "
                                 f"{held}")
        front = 0 if prefix_pages is None else prefix_pages.numel() * page_size
        if not 0 <= prefix_len <= front:
            raise ValueError(f"a prefix of {prefix_len} keys in pages for {front}")
        starts = [0]
        for n in q_lens:
            starts.append(starts[-1] + n)
        q_start = torch.tensor(starts, dtype=torch.int32, device=pages.device)
        kv_len = torch.tensor(kv_lens, dtype=torch.int32, device=pages.device)
        positions, slots = ops.kv_slots(q_start, kv_len, pages, page_size, starts[-1],
                                        base=prefix_len)
        return cls(q_start, kv_len, pages, max(q_lens), max(kv_lens), positions, slots,
                   prefix_pages, prefix_len)

    @classmethod
    def draft(cls, q_start, kv_len, pages, page_size, tokens, max_q, parents=None, held=None,
              pool=None, prefix_pages=None, prefix_len=0):
        """A step whose lengths are on the device (ops.step_plan, which hands out the
        pages with held and pool): request b brings tokens q_start[b] ..
        q_start[b+1]-1, max_q at most, of `tokens` in all.  With parents they are the
        nodes of a tree, else they follow one another."""
        planned = ops.step_plan(q_start, kv_len, pages, page_size, tokens, base=prefix_len,
                                held=held, pool=pool, parents=parents, max_q=max_q)
        return cls(q_start, kv_len, pages, max_q, pages.shape[1] * page_size, *planned[:2],
                   prefix_pages, prefix_len, planned[2] if len(planned) > 2 else None)


class DecoderBlock:
    """One decoder block on the device.

    qkv: Trunk [(q_heads + 2 kv_heads) * head_dim][hidden]; proj: Trunk
    [hidden][q_heads * head_dim]; norm1 / norm2 fp32 [hidden] (before attention
    and before the MoE layer); q_norm / k_norm fp32 [head_dim] or None;
    inv_freq, rot_scale from ops.rope_inv_freq; moe: ops.MoELayer."""

    def __init__(self, moe, qkv, proj, q_heads, kv_heads, head_dim, norm1, norm2, inv_freq,
                 rot_scale=1.0, q_norm=None, k_norm=None, interleaved=False, eps=1e-6,
                 scale=None):
        if qkv.out != (q_heads + 2 * kv_heads) * head_dim or proj.in_ != q_heads * head_dim or \
                proj.out != qkv.in_ or qkv.in_ != moe.hidden:
            raise ValueError("the projections do not fit the heads or the MoE layer")
        self.moe, self.qkv, self.proj = moe, qkv, proj
        self.q_heads, self.kv_heads, self.head_dim = q_heads, kv_heads, head_dim
        self.norm1, self.norm2 = norm1, norm2
        self.inv_freq, self.rot_scale, self.interleaved = inv_freq, rot_scale, interleaved
        self.q_norm, self.k_norm, self.eps, self.scale = q_norm, k_norm, eps, scale

    def attend(self, h, k_pages, v_pages, step):
        """h + the attention half; the step's keys and values are in the pages after it."""
        T = h.shape[0]
        x = self.qkv(ops.rmsnorm(h, self.norm1, self.eps))
        x = x.view(T, self.q_heads + 2 * self.kv_heads, self.head_dim)
        q, k, v = x.split((self.q_heads, self.kv_heads, self.kv_heads), 1)
        q = ops.kv_append(q, k, v, k_pages, v_pages, step.slots, step.positions, self.inv_freq,
                          q_norm=self.q_norm, k_norm=self.k_norm, eps=self.eps,
                          interleaved=self.interleaved, rot_scale=self.rot_scale)
        over = (q, k_pages, v_pages, step.pages, step.kv_len, step.q_start)
        how = dict(max_q=step.max_q, max_kv=step.max_kv, scale=self.scale,
                   prefix_pages=step.prefix_pages, prefix_len=step.prefix_len)
        if step.seen is None:
            o = ops.paged_attention(*over, **how)
        else:
            o = ops.tree_attention(*over, step.seen, **how)
        o = o.view(T, -1)
        # the trunk takes bf16 or fp32
        return h + self.proj(o if o.dtype is torch.bfloat16 else o.float())

    def forward(self, h, k_pages, v_pages, step):
        """h fp32 [T][hidden], the tokens in the step's order -> the same after the block."""
        h = self.attend(h, k_pages, v_pages, step)
        if h.shape[0] <= self.moe.max_tokens:
            return self.moe.forward_block(h, torch.empty_like(h), self.norm2, self.eps)
        return self.moe.prefill(ops.rmsnorm(h, self.norm2, self.eps), residual=h)


class Decoder:
    """Blocks between an embedding and an output head, over the caches of all layers,
    for a fixed number of requests whose pages come from one pool.

    embed fp32 [vocabulary][hidden]; norm fp32 [hidden]; head: Trunk
    [vocabulary][hidden]; k_pages / v_pages
    [layers][pages][page_size][kv_heads][head_dim].  kv_len (int32 [requests], on the
    device) is how many keys each request has: set it to 0 for one that ends, and its
    pages go back with the next step.  A request that a step leaves without pages for all
    its keys (the pool ran empty, or its row of pages is full; ops.attn_status raises) stays
    as it was, with -1 or a count of 0 for its result: bring the same tokens again when
    there are pages.  Nothing here waits for the device.  A number outside the vocabulary is
    read as the nearest in it (and is never accepted)."""

    def __init__(self, blocks, embed, norm, head, k_pages, v_pages, requests,
                 pages_per_request, eps=1e-6):
        if k_pages.dim() != 5 or k_pages.shape != v_pages.shape or len(blocks) != len(k_pages):
            raise ValueError("the caches must be [layers][pages][page_size][kv_heads][head_dim], "
                             "a layer for each block")
        if head.in_ != embed.shape[1] or head.out != embed.shape[0]:
            raise ValueError("the head does not fit the embedding")
        self.blocks, self.embed, self.norm, self.head, self.eps = blocks, embed, norm, head, eps
        self.k_pages, self.v_pages, self.page_size = k_pages, v_pages, k_pages.shape[2]
        dev = k_pages.device
        self.pool = ops.page_pool(k_pages.shape[1], dev)
        self.pages = torch.full((requests, pages_per_request), -1, dtype=torch.int32, device=dev)
        self.held = torch.zeros(requests, dtype=torch.int32, device=dev)
        self.kv_len = torch.zeros(requests, dtype=torch.int32, device=dev)

    def _forward(self, tokens, q_start, max_q, parents=None):
        """(states behind the last block, the step)."""
        if not tokens.numel():
            raise ValueError("a step needs a token")
        kv_len = self.kv_len + (q_start[1:] - q_start[:-1])
        step = Step.draft(q_start, kv_len, self.pages, self.page_size, tokens.numel(), max_q,
                          parents, self.held, self.pool)
        h = self.embed[tokens.clamp(0, len(self.embed) - 1)]
        for block, k, v in zip(self.blocks, self.k_pages, self.v_pages):
            h = block.forward(h, k, v, step)
        return h, step

    def _placed(self, step):
        """Which requests have pages for all keys of the step, bool [requests]."""
        return self.held * self.page_size >= step.kv_len

    def _logits(self, h):
        return self.head(ops.rmsnorm(h, self.norm, self.eps))

    def extend(self, tokens, q_start, max_q, **choice):
        """The requests' next tokens (int32, certain ones: a prompt, a chunk of one or a
        single token), max_q a request at most, through the blocks; returns the
        token picked behind each request's last, int32 [requests] (of no meaning where a
        request brings none, -1 where its keys have no place).  choice: what ops.pick_tokens
        weighs, a row a request."""
        h, step = self._forward(tokens, q_start, max_q)
        last = (q_start[1:] - 1).clamp(0, len(h) - 1)
        picked = ops.pick_tokens(self._logits(h[last]), **choice)
        placed = self._placed(step)
        torch.where(placed, step.kv_len, self.kv_len, out=self.kv_len)
        return torch.where(placed, picked, -1)

    def verify(self, drafted, parents, q_start, max_q, **choice):
        """A step of drafted trees: request b's nodes are tokens q_start[b] ..
        q_start[b+1]-1, node 0 the last certain token, which is not in the cache yet.
        Returns (count, chosen) of ops.tree_accept: chosen[b][:count[b]] are the
        request's new tokens, the last of which is the next tree's node 0; count is 0 for a
        request whose keys have no place."""
        h, step = self._forward(drafted, q_start, max_q, parents)
        picked = ops.pick_tokens(self._logits(h), q_start, max_q, drafted=drafted, seen=step.seen,
                                 **choice)
        count, _, chosen, kv_len = ops.tree_accept(
            drafted, picked, step.seen, q_start, step.kv_len, max_q,
            caches=(self.k_pages, self.v_pages), pages=self.pages)
        placed = self._placed(step)
        torch.where(placed, kv_len, self.kv_len, out=self.kv_len)
        return torch.where(placed, count, 0), torch.where(placed[:, None], chosen, -1)
