"""Tensor-parallel, sequence-parallel mixture-of-experts SwiGLU block.

``y[t] = sum over the experts e chosen for token t of
weight[t, e] * (silu(x @ W_gate[e]) * (x @ W_up[e])) @ W_down[e]``, every expert's FFN dimension
sharded over the ranks and the activations sharded over tokens:

    x_shard [T/ws, H] --all-gather--> X [T, H]
    weights, ids = route_experts(X @ W_router)            the same on every rank
    slots = expert_slots(ids)
    H1 = silu(X @ W_gate) * (X @ W_up)                    [T * top_k, F/ws], gathered by slot
    part = expert_combine(H1 @ W_down, weights)           [T, H]
    part --reduce-scatter--> y_shard [T/ws, H]

The block beside :class:`tileccl_b200.models.TPMLP` for models whose MLP is split into experts;
the collectives are the tile collectives of ``ops``.  The router runs in fp32 from the product
on.  Nothing synchronises with the host, so ``forward`` can be captured into a CUDA graph.
"""

from __future__ import annotations

from typing import Optional

import torch

from .. import ops
from .tp_mlp import GATE_BLOCK, pack_gate_up


class TPMoE:
    """One rank's shard of the block.  Weights: N(0, 0.02); the router's are the same on every
    rank, the experts' are seeded per (seed, rank)."""

    def __init__(self, ctx, *, tokens: int, hidden: int = 4096, ffn: int = 14336, experts: int = 8,
                 top_k: int = 2, dtype: torch.dtype = torch.bfloat16, score: str = "softmax",
                 renormalize: bool = True, scale: float = 1.0, groups: int = 1,
                 top_groups: Optional[int] = None, balance: bool = False, seed: int = 0,
                 weights: Optional[tuple] = None):
        """``weights``: ``(w_router [H, E], w_gate [E, H, F/ws], w_up [E, H, F/ws], w_down
        [E, F/ws, H])``, this rank's shards.  ``balance``: keep a bias per expert
        (``self.bias``, zeros) that steers the choice."""
        ws, rank = ctx.world_size, ctx.rank
        if ffn % ws or tokens % ws:
            raise ValueError("ffn and tokens must be divisible by world_size")
        if (ffn // ws) % GATE_BLOCK:
            raise ValueError(f"FFN shard width {ffn // ws} must be a multiple of {GATE_BLOCK}")
        if hidden % 8 or experts % 8:
            raise ValueError("hidden and experts must be multiples of 8 (16-byte rows)")
        if not 1 <= top_k <= experts:
            raise ValueError(f"top_k={top_k} must be in 1..{experts}")
        self.ctx = ctx
        self.tokens, self.hidden, self.ffn, self.experts, self.top_k = tokens, hidden, ffn, experts, top_k
        self.dtype, self.f_local, self.t_local = dtype, ffn // ws, tokens // ws
        self.routing = dict(score=score, renormalize=renormalize, scale=scale, groups=groups,
                            top_groups=top_groups)
        dev = ctx.torch_device
        if weights is None:
            gen = torch.Generator(device=dev)
            mk = lambda *shape: (torch.randn(*shape, device=dev, generator=gen) * 0.02).to(dtype)
            gen.manual_seed(seed * 1000)
            w_router = mk(hidden, experts)
            gen.manual_seed(seed * 1000 + 1 + rank)
            f = self.f_local
            w_gate, w_up, w_down = mk(experts, hidden, f), mk(experts, hidden, f), mk(experts, f, hidden)
        else:
            w_router, w_gate, w_up, w_down = (w.to(device=dev, dtype=dtype) for w in weights)
        self.w_router = w_router.contiguous().unsqueeze(0)          # a product of one expert
        self.w_gate, self.w_up, self.w_down = w_gate, w_up, w_down.contiguous()
        self.w_gu = torch.stack([pack_gate_up(g, u) for g, u in zip(w_gate, w_up)])
        self.bias = torch.zeros(experts, device=dev) if balance else None
        # every token is a row of the router's one expert
        rows = torch.arange(tokens, dtype=torch.int32, device=dev)
        self._all_tokens = ops.ExpertSlots(
            torch.tensor([0, tokens], dtype=torch.int32, device=dev), rows, rows.unsqueeze(1))
        # Buffers the collectives touch live on the heap.
        self.x_local = ctx.zeros(self.t_local, hidden, dtype=dtype)
        self.x_full = self.x_local if ws == 1 else ctx.zeros(tokens, hidden, dtype=dtype)
        self.part = ctx.zeros(tokens, hidden, dtype=dtype)
        self.y = self.part if ws == 1 else ctx.zeros(self.t_local, hidden, dtype=dtype)
        self.counts = None               # int32 [experts + 1] slot offsets of the last forward

    # The three parts of `forward`.  One process that emulates several ranks on one GPU runs each
    # part for all of its ranks before the next (the collectives of emulated ranks take place once
    # the last rank has called).
    def gather(self, x_shard: Optional[torch.Tensor] = None) -> None:
        if x_shard is not None and x_shard.data_ptr() != self.x_local.data_ptr():
            self.x_local.copy_(x_shard)
        if self.ctx.world_size > 1:
            ops.allgather(self.x_local, self.x_full, ctx=self.ctx)

    def compute(self) -> None:
        x = self.x_full
        logits = ops.expert_gemm(x, self.w_router, self._all_tokens, rows="slots",
                                 out_dtype=torch.float32)
        weights, ids = ops.route_experts(logits, self.top_k, bias=self.bias, **self.routing)
        slots = ops.expert_slots(ids, self.experts)
        self.counts = slots.offsets
        h = ops.expert_gemm(x, self.w_gu, slots, epilogue="silu_gate")
        y = ops.expert_gemm(h, self.w_down, slots, rows="slots")
        ops.expert_combine(y, slots, weights, self.part)

    def scatter(self) -> torch.Tensor:
        if self.ctx.world_size > 1:
            ops.reduce_scatter(self.part, self.y, ctx=self.ctx)
        return self.y

    def forward(self, x_shard: Optional[torch.Tensor] = None) -> torch.Tensor:
        if self.ctx.emulated:
            raise RuntimeError("ranks that share a GPU run gather(), compute() and scatter() in turn, "
                               "each for all ranks")
        self.gather(x_shard)
        self.compute()
        return self.scatter()

    __call__ = forward

    def flops(self) -> float:
        """FLOPs of this rank's expert products per forward."""
        return 2.0 * self.tokens * self.top_k * self.hidden * self.f_local * 3


def reference_moe_forward(x_full: torch.Tensor, shards: list) -> torch.Tensor:
    """fp32 PyTorch reference of the unsharded block (softmax or sigmoid scores, no groups, no
    bias) from the per-rank shards: every expert applied to every token."""
    x, m0 = x_full.float(), shards[0]
    logits = x @ m0.w_router[0].float().to(x.device)
    p = torch.softmax(logits, 1) if m0.routing["score"] == "softmax" else torch.sigmoid(logits)
    top = p.topk(m0.top_k, 1)
    w = top.values / top.values.sum(1, keepdim=True) if m0.routing["renormalize"] else top.values
    w = torch.zeros_like(p).scatter(1, top.indices, w * m0.routing["scale"])
    y = torch.zeros_like(x)
    for m in shards:
        for e in range(m.experts):
            g, u, d = (t[e].float().to(x.device) for t in (m.w_gate, m.w_up, m.w_down))
            y += w[:, e:e + 1] * ((torch.nn.functional.silu(x @ g) * (x @ u)) @ d)
    return y


def smoke_moe_forward(ctxs, tokens: int = 256, hidden: int = 256, ffn: int = 1024, experts: int = 8,
                      top_k: int = 2) -> None:
    """Tiny forward on the given single-process contexts, checked against fp32 PyTorch."""
    ws = len(ctxs)
    moes = [TPMoE(ctx, tokens=tokens, hidden=hidden, ffn=ffn, experts=experts, top_k=top_k)
            for ctx in ctxs]
    gen = torch.Generator(device=ctxs[0].torch_device)
    gen.manual_seed(7)
    x = torch.randn(tokens, hidden, device=ctxs[0].torch_device, generator=gen).to(torch.bfloat16)
    t = tokens // ws
    for it in range(2):
        for r, m in enumerate(moes):
            with torch.cuda.device(m.x_local.device):
                m.gather(x[r * t:(r + 1) * t].to(m.x_local.device))
        for m in moes:
            with torch.cuda.device(m.x_local.device):
                m.compute()
        for m in moes:
            with torch.cuda.device(m.x_local.device):
                m.scatter()
    for ctx in ctxs:
        ops.check_expert_status(ctx.torch_device)
    ref = reference_moe_forward(x, moes)
    for r, m in enumerate(moes):
        want = ref[r * t:(r + 1) * t].to(m.y.device)
        err = (m.y.float() - want).abs().max().item() / (want.abs().max().item() + 1e-9)
        if not err <= 3e-2:
            raise AssertionError(f"TP-MoE mismatch on rank {r}: rel err {err:.3e}")
