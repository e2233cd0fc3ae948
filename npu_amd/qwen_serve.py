"""The decoder for several sequences at once: a paged KV cache, one step over the new
tokens of all of them, and sampling.

The reference's decoder runs one sequence (qwen/forward.py:834-893); ``qwen_core.forward``
keeps that contract.  Here a step takes any number of new tokens of every sequence
(prompts, single tokens, or both): the projections and the MoE blocks run over all tokens
of the step, the attention layers through ``ops.rope_append`` and ``ops.paged_attention``
(every sequence has one new token) or ``ops.prompt_attention``, the Gated DeltaNet layers
per sequence (their state is a recurrence over the sequence).  ``generate`` adds
``ops.sample``.

The cache holds k (rotated) and v in 16 bits, half the traffic of the single-sequence
path's fp32 cache at one rounding of each, 2^-9 (bf16) of the value.
"""
from __future__ import annotations

from dataclasses import dataclass

import torch

from npu_amd import ops
from npu_amd._dropin import device
from npu_amd.gguf_types import GGMLQuantizationType
from npu_amd.profiler import profile
from npu_amd.qwen_core import (AttnLayer, Config, GpuAttn, Model, _bf16_dev, _f32_dev, _moe_residual, _rms_norm_dev,
                               ssm_forward)


def build_rope_axes(rope_dim: int, theta: float, sections=None, dev=None) -> tuple[torch.Tensor, torch.Tensor | None]:
    """``(inv_freq, axis)`` for ``ops.rope_append``: the radians per position of every pair in
    64 bits (the angles of ``qwen_core.build_partial_rope_cache``, without its fp32 rounding at
    far positions), and the axis of positions that turns it: ``sections`` pairs in turn, None
    for one axis."""
    dev = dev or device()
    half = rope_dim // 2
    inv = theta ** (-torch.arange(half, dtype=torch.float64, device=dev) / max(half, 1))
    if sections is None:
        return inv, None
    if sum(sections) != half:
        raise ValueError(f"sections {list(sections)} do not add up to rope_dim / 2 = {half}")
    return inv, torch.tensor([i for i, n in enumerate(sections) for _ in range(n)], dtype=torch.int32, device=dev)


@dataclass
class Step:
    """Where a step's new tokens go, on the device: ``seqs`` have ``counts`` of them each."""

    seqs: list
    counts: list
    positions: torch.Tensor       # int32 [T]
    slots: torch.Tensor           # int32 [T]
    cu_q: torch.Tensor            # int32 [len(seqs) + 1]
    lengths: torch.Tensor         # int32 [len(seqs)], the new tokens counted
    table: torch.Tensor           # int32 [len(seqs), width]

    @property
    def single(self) -> bool:
        return all(n == 1 for n in self.counts)


class PagedCache:
    """What ``n_seq`` sequences have cached: for every attention layer ``n_pages`` pages of
    ``page_size`` positions, shared by the sequences (one table for all layers), and for
    every other layer each sequence's DeltaNet state."""

    def __init__(self, cfg: Config, n_seq: int, n_pages: int, *, page_size: int = 16, dtype=torch.bfloat16, dev=None):
        if n_seq < 1 or n_pages < 1 or page_size < 1:
            raise ValueError(f"PagedCache: n_seq={n_seq}, n_pages={n_pages} and page_size={page_size} must be positive")
        if dtype not in (torch.bfloat16, torch.float16):
            raise TypeError(f"PagedCache: pages are bf16 or fp16, not {dtype}")
        if n_pages * page_size >= 2 ** 31:
            raise ValueError("PagedCache: more than 2^31 positions")
        self.cfg, self.n_seq, self.n_pages, self.page_size = cfg, int(n_seq), int(n_pages), int(page_size)
        self.dev = dev or device()
        shape = (n_pages, page_size, cfg.n_head_kv, cfg.head_dim)
        self.k, self.v = ([torch.zeros(shape, dtype=dtype, device=self.dev) if cfg.is_attention[i] else None
                           for i in range(cfg.n_layer)] for _ in range(2))
        self.ssm = [[None] * cfg.n_layer for _ in range(n_seq)]
        self.pages: list[list[int]] = [[] for _ in range(n_seq)]
        self.length = [0] * n_seq
        self.free = list(range(n_pages - 1, -1, -1))

    def reserve(self, counts) -> Step:
        """Make room for ``counts[b]`` new tokens of every sequence b.  Raises MemoryError, with
        nothing changed, where the pages do not suffice."""
        counts = [int(n) for n in counts]
        if len(counts) != self.n_seq or min(counts) < 0:
            raise ValueError(f"counts must be {self.n_seq} numbers of at least 0, got {counts}")
        P = self.page_size
        seqs = [b for b in range(self.n_seq) if counts[b]]
        more = {b: -(-(self.length[b] + counts[b]) // P) - len(self.pages[b]) for b in seqs}
        if sum(more.values()) > len(self.free):
            raise MemoryError(f"PagedCache: {sum(more.values())} pages needed, {len(self.free)} of {self.n_pages} free")
        pos, slots, cu = [], [], [0]
        for b in seqs:
            self.pages[b] += [self.free.pop() for _ in range(more[b])]
            at = range(self.length[b], self.length[b] + counts[b])
            pos += at
            slots += [self.pages[b][p // P] * P + p % P for p in at]
            cu.append(len(pos))
            self.length[b] += counts[b]
        width = max((len(self.pages[b]) for b in seqs), default=0)
        lengths = [self.length[b] for b in seqs]
        table = [p for b in seqs for p in self.pages[b] + [-1] * (width - len(self.pages[b]))]
        parts = [pos, slots, cu, lengths, table]
        ints = torch.tensor([x for part in parts for x in part], dtype=torch.int32).to(self.dev)     # one copy
        pos, slots, cu, lengths, table = ints.split([len(part) for part in parts])
        return Step(seqs, [counts[b] for b in seqs], pos, slots, cu, lengths, table.view(len(seqs), width))

    def release(self, b: int) -> None:
        """Forget sequence b: its pages are free for others."""
        self.free += reversed(self.pages[b])
        self.pages[b], self.length[b], self.ssm[b] = [], 0, [None] * self.cfg.n_layer


def attn_step(x: torch.Tensor, layer: AttnLayer, cfg: Config, rope, step: Step, k_pages: torch.Tensor,
              v_pages: torch.Tensor) -> torch.Tensor:
    """x [T, D] + gated attention of the step's tokens over the cache, which gets their keys
    and values (the layer of ``qwen_core.attn_forward``)."""
    T, D = x.shape
    hq, hkv, dh = cfg.n_head, cfg.n_head_kv, cfg.head_dim
    if layer.gpu is None:
        layer.gpu = GpuAttn(layer, cfg)
    w = layer.gpu
    inv, axis = rope
    row = ops.matvec(GGMLQuantizationType.BF16, w.wqkv, w.wqkv.shape[0], D,
                     _rms_norm_dev(x, layer.attn_norm, cfg.rms_eps, w_dev=w.attn_norm))
    qg, k, v = row.split([2 * hq * dh, hkv * dh, hkv * dh], 1)
    qg = qg.view(T, hq, 2 * dh)
    gate = qg[..., dh:]
    one = step.single
    q = ops.rope_append(qg[..., :dh], k.view(T, hkv, dh), v.view(T, hkv, dh), step.positions, inv, k_pages, v_pages,
                        step.slots, axis=axis, q_norm=w.q_norm, k_norm=w.k_norm, eps=cfg.rms_eps,
                        out_dtype=torch.float32 if one else k_pages.dtype)
    if one:
        y = ops.paged_attention(q, k_pages, v_pages, step.table, step.lengths, gate=gate)
    else:
        y = ops.prompt_attention(q, k_pages, v_pages, step.cu_q, block_table=step.table, lengths=step.lengths,
                                 gate=gate)
    return x + ops.matvec(GGMLQuantizationType.BF16, w.wo, D, hq * dh, y.view(T, hq * dh))


def forward_step(model: Model, tokens, cache: PagedCache, *, skip_moe: bool = False) -> torch.Tensor:
    """One step: ``tokens[b]`` are sequence b's new tokens, behind what ``cache`` has of it
    (empty: not in this step).  Returns the logits [n, vocab] of the last token of every
    sequence that has any, in their order.  A step that raises leaves ``cache`` to be
    released."""
    cfg, g = model.cfg, model.gpu
    flat = [int(t) for seq in tokens for t in seq]
    if flat and not (0 <= min(flat) and max(flat) < model.token_embd.shape[0]):
        raise ValueError(f"tokens must be 0 .. {model.token_embd.shape[0] - 1}")
    step = cache.reserve([len(seq) for seq in tokens])
    if "embd" not in g:
        g["embd"] = model.token_embd.to(device(), torch.float32).contiguous()
        g["onorm"] = _f32_dev(model.output_norm)
        g["lm_head"] = _bf16_dev(model.lm_head)
    if "rope_axes" not in g:
        g["rope_axes"] = build_rope_axes(cfg.rope_dim, cfg.rope_theta)
    if not flat:
        return torch.empty(0, model.lm_head.shape[0], device=device())
    x = g["embd"][torch.tensor(flat, dtype=torch.long).to(device())]
    T, D = x.shape
    for i in range(cfg.n_layer):
        core, moe = model.layers[i]
        if cfg.is_attention[i]:
            with profile("step.attn"):
                x = attn_step(x, core, cfg, g["rope_axes"], step, cache.k[i], cache.v[i])
        else:
            with profile("step.ssm"):
                ys = []
                for b, part in zip(step.seqs, x.split(step.counts)):
                    y, cache.ssm[b][i] = ssm_forward(part[None], core, cfg, cache.ssm[b][i], residual=True)
                    ys.append(y[0])
                x = torch.cat(ys)
        if not skip_moe:
            with profile("step.moe"):
                x = _moe_residual(g, i, x[None], core, moe, cfg)[0]
    last = _rms_norm_dev(x[step.cu_q[1:].long() - 1], model.output_norm, cfg.rms_eps, w_dev=g["onorm"])
    with profile("step.lm_head"):
        return ops.matvec(GGMLQuantizationType.BF16, g["lm_head"], g["lm_head"].shape[0], D, last)


def generate(model: Model, prompts, max_new: int, cache: PagedCache, *, temperature=1.0, top_k=None, top_p=None,
             min_p=None, stop: int | None = None, generator: torch.Generator | None = None,
             skip_moe: bool = False) -> list[list[int]]:
    """Up to ``max_new`` tokens behind every prompt, by ``ops.sample`` with its parameters (one
    value each, for all); a sequence ends with the token ``stop``, and its pages are free for
    the others' from then on.  ``generator`` (of the cache's device) draws the numbers.  The
    sequences of ``cache`` are new ones; afterwards all are released."""
    if len(prompts) != cache.n_seq or any(cache.length):
        raise ValueError(f"generate: {len(prompts)} prompts for {cache.n_seq} sequences of a cache that must be empty")
    if any(len(p) == 0 for p in prompts):
        raise ValueError("generate: a prompt needs a token")
    out: list[list[int]] = [[] for _ in prompts]
    new = [list(p) for p in prompts]
    try:
        for _ in range(max_new):
            live = [b for b, seq in enumerate(new) if seq]
            if not live:
                break
            logits = forward_step(model, new, cache, skip_moe=skip_moe)
            u = torch.rand(len(live), generator=generator, device=logits.device)
            ids = ops.sample(logits, u, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p).tolist()
            for b, t in zip(live, ids):
                if t < 0:
                    raise FloatingPointError(f"generate: sequence {b} has no finite logit")
                out[b].append(t)
                new[b] = [] if t == stop else [t]
                if t == stop:
                    cache.release(b)
    finally:
        for b in range(cache.n_seq):
            cache.release(b)
    return out


__all__ = ["build_rope_axes", "Step", "PagedCache", "attn_step", "forward_step", "generate"]
