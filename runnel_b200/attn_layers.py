"""The full-attention half of a decoder layer over a paged cache, for serving:
:class:`PagedKVCache` (pages, block table, lengths and free list of a batch of
requests) and :class:`GatedAttention` (mlx-lm's ``self_attn`` of a Qwen3.5 layer: quantized
projections, normed and rotated heads, causal attention, output gate).

:class:`runnel_b200.stack.LayerStack` runs them with the MoE blocks.  A step:

    cache = PagedKVCache(n_layers, num_pages, n_kv_heads, head_dim, max_requests, max_len)
    plan = cache.plan(new_lens, max_tokens)       # pages, slots, positions of the step's tokens
    out = stack.forward(x, cache=cache, plan=plan, max_q=longest)   # x [max_tokens, H], requests in order
    cache.commit(plan)
    cache.release(finished)                       # requests that are done, before the next plan

Everything that varies from step to step (lengths, pages, positions) is on the
device, so a step of fixed ``max_tokens`` can be captured in a CUDA graph.  Neither
the cache nor the layers read :func:`runnel_b200.attention.status`, which waits for the
device: the caller does, every so many steps (a plan that did not fit, a page id out
of range, and ``STATUS_TIMEOUT``: a call's outputs are void, a captured one's until it is
read).
"""
from __future__ import annotations

from dataclasses import dataclass

import torch

from . import attention, probes
from .switch_layers import QuantizedLinear, _cat


class PagedKVCache:
    """Paged keys and values of ``n_layers`` attention layers for up to
    ``max_requests`` requests of up to ``max_len`` tokens.

    ``k[layer]`` / ``v[layer]`` are ``[num_pages, n_kv_heads, page_size, head_dim]``; one
    block table serves all layers."""

    def __init__(self, n_layers: int, num_pages: int, n_kv_heads: int, head_dim: int, max_requests: int, max_len: int,
                 page_size: int = 64, dtype: torch.dtype = torch.bfloat16, device="cuda"):
        self.page_size, self.num_pages = page_size, num_pages
        shape = (num_pages, n_kv_heads, page_size, head_dim)
        self.k = [torch.empty(shape, dtype=dtype, device=device) for _ in range(n_layers)]
        self.v = [torch.empty(shape, dtype=dtype, device=device) for _ in range(n_layers)]
        cols = max(1, -(-max_len // page_size))
        self.table = torch.zeros((max_requests, cols), dtype=torch.int32, device=device)
        self.lens = torch.zeros(max_requests, dtype=torch.int32, device=device)
        # taken from the end: page 0 first
        self.free_pages = torch.arange(num_pages - 1, -1, -1, dtype=torch.int32, device=device)
        self.free_count = torch.full((1,), num_pages, dtype=torch.int32, device=device)
        self._stale = False  # a release came after the last plan
        self._captured = False  # a plan is part of a graph, whose replays are not seen here

    def plan(self, new_lens: torch.Tensor, max_tokens: int) -> attention.KVPlan:
        """Pages, slots and positions for ``new_lens`` ``[max_requests]`` more tokens;
        nothing is taken over before :meth:`commit`."""
        self._stale = False
        self._captured = self._captured or (self.lens.is_cuda and torch.cuda.is_current_stream_capturing())
        return attention.kv_plan(self.table, self.lens, new_lens, self.free_pages, self.free_count,
                                 page_size=self.page_size, num_pages=self.num_pages, max_tokens=max_tokens)

    def commit(self, plan: attention.KVPlan) -> None:
        """The step's tokens are cached now (in place, so captured steps keep their addresses).
        A plan from before a :meth:`release` is refused: its lengths and free count would undo it."""
        if self._stale and not self._captured:
            raise RuntimeError("pages were released after this plan: plan again")
        self.lens.copy_(plan.seq_lens)
        self.free_count.copy_(plan.free_count)

    def release(self, finished: torch.Tensor) -> None:
        """Requests with ``finished[b] != 0`` (int32) give their pages back and become empty;
        between a step's :meth:`commit` and the next :meth:`plan`, or instead of a commit."""
        self._stale = True
        lens, count = attention.kv_release(self.table, self.lens, finished, self.free_pages, self.free_count,
                                           page_size=self.page_size, num_pages=self.num_pages)
        self.lens.copy_(lens)
        self.free_count.copy_(count)


@dataclass
class RotarySpec:
    """How heads are rotated: the first ``rot`` elements, frequencies
    ``theta ** (-2 i / rot)``, dealt over axes by ``sections`` (see
    :func:`runnel_b200.attention.rope_append`)."""

    rot: int
    theta: float = 1e7
    sections: tuple | None = None
    interleaved: bool = True

    def inv_freq(self, device) -> torch.Tensor:
        i = torch.arange(self.rot // 2, dtype=torch.float64)
        return (self.theta ** (-2.0 * i / self.rot)).float().to(device)


class GatedAttention(torch.nn.Module):
    """mlx-lm's ``self_attn`` with affine-quantized projections.

    ``q_proj`` gives each head its queries and, behind them, its output gate
    (``[heads, 2, head_dim]`` a token; with ``gated`` False queries alone).  The q, k and v
    rows are packed into one quantized matrix, so a forward is one quantized
    product, the rotary append, the attention (which applies the gate) and the
    output product."""

    def __init__(self, q_proj: QuantizedLinear, k_proj: QuantizedLinear, v_proj: QuantizedLinear,
                 o_proj: QuantizedLinear, q_norm: torch.Tensor | None, k_norm: torch.Tensor | None, head_dim: int,
                 rotary: RotarySpec, gated: bool = True, eps: float = 1e-6):
        super().__init__()
        if len({(p.bits, p.group_size, p.mode) for p in (q_proj, k_proj, v_proj)}) != 1:
            raise ValueError("q, k and v projections must share one quantization format")
        for p in (q_proj, k_proj, v_proj, o_proj):
            if p.group_size != 64 or p.mode != "affine" or p.get("biases") is None or "bias" in p:
                raise ValueError("projections must be affine-quantized in groups of 64, without module biases")
        # the products read as many scales and biases as the codes' shape says
        for name, p in (("q_proj", q_proj), ("k_proj", k_proj), ("v_proj", v_proj), ("o_proj", o_proj)):
            groups = (p.weight.shape[0], p.weight.shape[1] * 32 // p.bits // 64)
            if p.weight.dtype not in (torch.uint32, torch.int32) or any(
                    t.dtype != torch.bfloat16 or tuple(t.shape) != groups for t in (p.scales, p.biases)):
                raise ValueError(f"{name} must have 32-bit codes, and bf16 scales and biases of shape {groups}")
        self.hidden = q_proj.weight.shape[1] * 32 // q_proj.bits
        if o_proj.weight.shape[0] != self.hidden or any(p.weight.shape[1] != q_proj.weight.shape[1]
                                                        for p in (k_proj, v_proj)):
            raise ValueError(f"projections must all fit the hidden size of q_proj, {self.hidden}")
        self.head_dim, self.rotary, self.gated, self.eps = head_dim, rotary, gated, eps
        self.bits, self.o_bits = q_proj.bits, o_proj.bits
        self.n_heads = o_proj.weight.shape[-1] * 32 // o_proj.bits // head_dim
        self.n_kv_heads = k_proj.weight.shape[0] // head_dim
        q_rows = self.n_heads * head_dim * (2 if gated else 1)
        if q_proj.weight.shape[0] != q_rows or v_proj.weight.shape[0] != k_proj.weight.shape[0]:
            raise ValueError(f"q_proj must have {q_rows} rows, k_proj and v_proj as many as each other")
        if k_proj.weight.shape[0] % head_dim or self.n_kv_heads == 0 or self.n_heads % self.n_kv_heads:
            raise ValueError(f"k_proj must have the rows of heads of {head_dim}, of which the {self.n_heads} query heads "
                             "are a multiple")
        for name, w in (("q_norm", q_norm), ("k_norm", k_norm)):
            if w is not None and (w.dtype != torch.bfloat16 or tuple(w.shape) != (head_dim,)):
                raise ValueError(f"{name} must be bf16 [{head_dim}]")
        for n in ("weight", "scales", "biases"):
            self.register_buffer(n, _cat([getattr(m, n) for m in (q_proj, k_proj, v_proj)], 0))
        self.o_proj = o_proj
        self.register_buffer("q_norm", q_norm)
        self.register_buffer("k_norm", k_norm)
        self.register_buffer("inv_freq", rotary.inv_freq(q_proj.weight.device))

    def forward(self, x: torch.Tensor, cache: PagedKVCache, layer: int, plan: attention.KVPlan,
                max_q: int | None = None, positions: torch.Tensor | None = None, window: int = 0,
                record: dict | None = None) -> torch.Tensor:
        """``[T, H]`` bf16 -> ``[T, H]``; T is the plan's ``max_tokens``, rows behind the
        plan's last token come out undefined but finite.  ``layer`` indexes the
        cache's layers; ``positions`` (``[axes, T]``) replaces the plan's for images.
        ``record`` (a dict) receives the intermediate tensors, for checking."""
        if x.dtype != torch.bfloat16 or x.dim() != 2 or x.shape[1] != self.hidden:
            raise ValueError(f"x must be bf16 [tokens, {self.hidden}], not {x.dtype} {tuple(x.shape)}")
        if x.shape[0] == 0:
            return torch.empty_like(x)
        with torch.cuda.device_of(x):  # (the products launch on the current device)
            return self._forward(x, cache, layer, plan, max_q, positions, window, record)

    def _forward(self, x, cache, layer, plan, max_q, positions, window, record):
        T, D, Hq, Hkv = x.shape[0], self.head_dim, self.n_heads, self.n_kv_heads
        y = probes.qmm(self.bits, self.weight, self.scales, self.biases, x, out_f32=False)
        n = Hq * D * (2 if self.gated else 1)
        qg = y[:, :n].view(T, Hq, -1)
        q, gate = qg[..., :D], qg[..., D:] if self.gated else None
        k, v = y[:, n:n + Hkv * D].view(T, Hkv, D), y[:, n + Hkv * D:].view(T, Hkv, D)
        r = self.rotary
        # rows behind the step's last token keep these zeros, so the output product stays finite
        qr = torch.zeros((T, Hq, D), dtype=x.dtype, device=x.device)
        attention.rope_append(q, k, v, plan.positions if positions is None else positions, self.inv_freq, plan.slots,
                              cache.k[layer], cache.v[layer], sections=r.sections, interleaved=r.interleaved,
                              q_norm=self.q_norm, k_norm=self.k_norm, eps=self.eps, out=qr)
        o = torch.zeros_like(qr)
        attention.paged_attention(qr, cache.k[layer], cache.v[layer], cache.table, plan.seq_lens, cu_q=plan.cu_q,
                                  max_q=max_q, window=window, gate=gate, out=o)
        out = probes.qmm(self.o_bits, self.o_proj.weight, self.o_proj.scales, self.o_proj.biases, o.view(T, Hq * D),
                         out_f32=False)
        if record is not None:
            record.update(qkv=y, q=q, gate=gate, k=k, v=v, q_rot=qr, attn=o, out=out)
        return out
