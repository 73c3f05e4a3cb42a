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
    prefix, prefix_len keys of prefix_pages come before every request's own."""
    q_start: torch.Tensor
    kv_len: torch.Tensor
    pages: torch.Tensor
    max_q: int
    max_kv: int
    positions: torch.Tensor
    slots: torch.Tensor
    prefix_pages: torch.Tensor = None
    prefix_len: int = 0

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
        o = ops.paged_attention(q, k_pages, v_pages, step.pages, step.kv_len, step.q_start,
                                step.max_q, step.max_kv, scale=self.scale,
                                prefix_pages=step.prefix_pages, prefix_len=step.prefix_len)
        o = o.view(T, -1)
        # the trunk takes bf16 or fp32
        return h + self.proj(o if o.dtype is torch.bfloat16 else o.float())

    def forward(self, h, k_pages, v_pages, step):
        """h fp32 [T][hidden], the tokens in the step's order -> the same after the block."""
        h = self.attend(h, k_pages, v_pages, step)
        if h.shape[0] <= self.moe.max_tokens:
            return self.moe.forward_block(h, torch.empty_like(h), self.norm2, self.eps)
        return self.moe.prefill(ops.rmsnorm(h, self.norm2, self.eps), residual=h)
