"""Host side of the operators around the hot path in a gpt-oss decoder layer (RMSNorm, rotary tables, KV write).

The reference leaves these to upstream vLLM; their arithmetic is taken from transformers'
models/gpt_oss/modeling_gpt_oss.py (GptOssRMSNorm :47-62, GptOssRotaryEmbedding.forward :187-200,
_apply_rotary_emb :217-225) and modeling_rope_utils._compute_yarn_parameters.
"""
from __future__ import annotations

import math
from typing import Tuple

import torch

# gpt-oss-20b (transformers GptOssConfig defaults)
GPT_OSS_ROPE = dict(rope_theta=150000.0, factor=32.0, beta_fast=32.0, beta_slow=1.0,
                    original_max_position_embeddings=4096, truncate=False)
RMS_EPS = 1e-5


def yarn_inv_freq(head_dim: int, rope_theta: float, factor: float, beta_fast: float, beta_slow: float,
                  original_max_position_embeddings: int, truncate: bool = True) -> Tuple[torch.Tensor, float]:
    """(inv_freq fp32 [head_dim/2], attention scaling) of YaRN, computed as _compute_yarn_parameters does: the
    same torch fp32 expressions in the same order, so the values are that function's bit for bit."""
    dim = head_dim

    def correction_dim(num_rotations):
        return (dim * math.log(original_max_position_embeddings / (num_rotations * 2 * math.pi))) / (2 * math.log(rope_theta))

    low, high = correction_dim(beta_fast), correction_dim(beta_slow)
    if truncate:
        low, high = math.floor(low), math.ceil(high)
    low, high = max(low, 0), min(high, dim - 1)
    if low == high:
        high += 0.001
    pos_freqs = rope_theta ** (torch.arange(0, dim, 2).to(dtype=torch.float) / dim)
    extrapolation = 1.0 / pos_freqs
    interpolation = 1.0 / (factor * pos_freqs)
    ramp = torch.clamp((torch.arange(dim // 2, dtype=torch.float32) - low) / (high - low), 0, 1)
    extrapolation_factor = 1 - ramp
    inv_freq = interpolation * (1 - extrapolation_factor) + extrapolation * extrapolation_factor
    scaling = 1.0 if factor <= 1 else 0.1 * math.log(factor) + 1.0
    return inv_freq, scaling


def rope_tables(max_pos: int, head_dim: int = 64, dtype: torch.dtype = torch.float16, **rope) -> Tuple[torch.Tensor, torch.Tensor]:
    """cos, sin [max_pos][head_dim/2] in `dtype`, the values GptOssRotaryEmbedding.forward returns for positions
    0..max_pos-1: fp32 outer product, cos/sin, times the attention scaling, then the cast."""
    params = dict(GPT_OSS_ROPE)
    params.update(rope)
    inv_freq, scaling = yarn_inv_freq(head_dim, **params)
    freqs = (inv_freq[:, None].float() @ torch.arange(max_pos)[None, :].float()).transpose(0, 1)
    return (freqs.cos() * scaling).to(dtype).contiguous(), (freqs.sin() * scaling).to(dtype).contiguous()


def validate_paging(block_tables: torch.Tensor, slots: torch.Tensor, ctx_lens: torch.Tensor, kcache: torch.Tensor) -> None:
    """Host-side check (synchronises) that the paging metadata stays inside the cache: the kernels trust it, and an
    out-of-range block id is an out-of-bounds access on the GPU.  Meant to run once per configuration, before the
    step is launched or captured."""
    nblocks, block_size = kcache.shape[0], kcache.shape[1]
    bt = block_tables.detach().cpu()
    used = (ctx_lens.detach().cpu().to(torch.int64) + block_size - 1) // block_size
    if bt.shape[0] != used.numel():
        raise ValueError(f"block_tables has {bt.shape[0]} rows for {used.numel()} sequences")
    if int(used.max()) > bt.shape[1]:
        raise ValueError(f"a context of {int(ctx_lens.max())} tokens needs {int(used.max())} blocks, block_tables holds {bt.shape[1]}")
    for b in range(bt.shape[0]):
        row = bt[b, :int(used[b])]
        if row.numel() and (int(row.min()) < 0 or int(row.max()) >= nblocks):
            raise ValueError(f"sequence {b}: block id outside [0, {nblocks})")
    sl = slots.detach().cpu()
    if int(sl.max()) >= nblocks * block_size:
        raise ValueError(f"slot {int(sl.max())} outside the cache of {nblocks * block_size} rows")


def validate_eviction(block_tables: torch.Tensor, ctx_lens: torch.Tensor, dst_tables: torch.Tensor, kcache: torch.Tensor, *, keep: int,
                      prefix_len: int = 0) -> None:
    """Host-side check (synchronises) of what kv_evict trusts: the pages that will receive kept tokens lie inside the cache,
    are handed out once, and are none of those that the call reads.  Meant to run where the pages are handed out."""
    nblocks, block_size = kcache.shape[0], kcache.shape[1]
    src, dst = block_tables.detach().cpu(), dst_tables.detach().cpu()
    first, seen = prefix_len // block_size, set()
    # the shared pages (row 0's leading entries; the other rows' may hold anything) and every sequence's own ones
    read = set(src[0, :first].tolist()) if src.shape[0] else set()
    for b, ctx in enumerate(ctx_lens.detach().cpu().tolist()):
        if ctx > prefix_len:
            read.update(src[b, first:(ctx + block_size - 1) // block_size].tolist())
    for b, ctx in enumerate(ctx_lens.detach().cpu().tolist()):
        end = prefix_len + min(max(ctx - prefix_len, 0), keep)
        need = (end + block_size - 1) // block_size
        if need > dst.shape[1]:
            raise ValueError(f"sequence {b} keeps {end} tokens in {need} pages, dst_tables holds {dst.shape[1]}")
        for page in dst[b, first:need].tolist():
            if page < 0 or page >= nblocks:
                raise ValueError(f"sequence {b}: destination page {page} outside [0, {nblocks})")
            if page in seen or page in read:
                raise ValueError(f"sequence {b}: destination page {page} is in use")
            seen.add(page)


def evict_tokens(caches, scores, block_tables: torch.Tensor, ctx_lens: torch.Tensor, dst_tables: torch.Tensor, *, keep: int, recent: int,
                 max_ctx: int, prefix_len: int = 0, new_lens=None) -> torch.Tensor:
    """Trim every layer's cache by its own scores: caches [(kcache, vcache)] and scores [blocks][Hkv][block_size] per layer,
    tables and lengths shared by the layers.  Layers and heads keep different tokens but equally many, in order, so the new
    tables and lengths (returned) serve them all; `recent` of at least a sliding window leaves windowed layers unharmed.
    Rotary positions go on counting from the old lengths: keys were rotated when they were written."""
    from . import lib
    caches, scores = list(caches), list(scores)
    if len(caches) != len(scores):
        raise ValueError(f"{len(caches)} layers' caches, {len(scores)} layers' scores: the layers left out would not fit the new lengths")
    for (kc, vc), sc in zip(caches, scores):
        _, new_lens = lib.kv_evict(kc, vc, sc, block_tables, ctx_lens, dst_tables, keep=keep, recent=recent, max_ctx=max_ctx,
                                   prefix_len=prefix_len, new_lens=new_lens)
    return new_lens


# ---------------------------------------------------------------------------------------------
# One gpt-oss decoder layer at decode time, as a fixed sequence of library calls on preallocated buffers
# ---------------------------------------------------------------------------------------------
class PendingCombine:
    """The expert output of a layer whose forward skipped the combine step: the experts' rows and the routing still sit
    in that layer's workspace.  The next layer consumes it in its first kernel; materialize() runs the plain combine."""

    def __init__(self, layer):
        self.layer, self.workspace, self.w = layer, layer.moe_ws, layer.wts
        self.FF, self.E, self.flags = layer.FF, layer.E, 0

    def materialize(self):
        lay, lib, w = self.layer, self.layer.lib, self.layer.w
        skip = lib.FLAG_SKIP_ROUTE | lib.FLAG_SKIP_GATE_UP | lib.FLAG_SKIP_DOWN
        lib.moe_nf4_forward(lay.h2, lay.ids, lay.wts, w["w13_q"], w["w13_absmax"], w["w2_q"], w["w2_absmax"], E_local=lay.E,
                            e_first=0, H=lay.H, FF=lay.FF, workspace=lay.moe_ws, out=lay.moe_out, act_mode=lay.act_mode,
                            flags=self.flags | skip, b13=w.get("b13"), b2=w.get("b2"))
        return lay.moe_out


class GptOssDecodeLayer:
    """GptOssDecoderLayer.forward (transformers models/gpt_oss/modeling_gpt_oss.py:347-379) for one new token per
    sequence: RMSNorm -> fused q/k/v projection -> rotary + KV-cache write -> paged attention (sinks, optional sliding
    window) -> o projection + residual -> RMSNorm -> router top-k -> NF4 experts.  The second residual add is left to
    the next layer's first RMSNorm call (or `finish`), which fuses it.

    weights: dict with ln1, ln2 [H]; wqkv [(Hq + 2 Hkv) D][H], bqkv; wo [H][Hq D], bo; sinks [Hq] or None;
    router_w [E][H], router_b [E] or None; w13_q, w13_absmax, w2_q, w2_absmax (tile order), b13 / b2 or None -- fp16
    unless NF4.  Every intermediate lives in buffers sized for max_tokens, so a step allocates nothing (but for
    the attention's workspace, where it needs a larger one than any step before) and can be captured in a HIP graph.
    """

    def __init__(self, weights, *, hidden: int, heads: int, kv_heads: int, head_dim: int, ffn: int, experts: int,
                 top_k: int, max_tokens: int, eps: float = RMS_EPS, window: int = 0, act_mode: int = 1,
                 device=None):
        from . import lib
        self.lib, self.w = lib, weights
        self.H, self.Hq, self.Hkv, self.D, self.FF, self.E, self.k = hidden, heads, kv_heads, head_dim, ffn, experts, top_k
        self.eps, self.window, self.act_mode, self.T = eps, window, act_mode, max_tokens
        dev = device if device is not None else weights["wqkv"].device
        f16 = dict(dtype=torch.float16, device=dev)
        T = max_tokens
        self.h1 = torch.empty((T, hidden), **f16)
        self.resid = torch.empty((T, hidden), **f16)
        self.qkv = torch.empty((T, (heads + 2 * kv_heads) * head_dim), **f16)
        self.q = torch.empty((T, heads, head_dim), **f16)
        self.attn = torch.empty((T, heads, head_dim), **f16)
        self.resid2 = torch.empty((T, hidden), **f16)
        self.h2 = torch.empty((T, hidden), **f16)
        self.ids = torch.empty((T, top_k), dtype=torch.int32, device=dev)
        self.wts = torch.empty((T, top_k), dtype=torch.float32, device=dev)
        self.moe_out = torch.empty((T, hidden), **f16)
        self.moe_ws = torch.empty(max(256, lib.moe_workspace_bytes(T, top_k, hidden, ffn, experts)), dtype=torch.uint8, device=dev)
        self.attn_ws = None
        self._captured, self._outgrown = False, []

    def _attn_workspace(self, need: int):
        """The attention's workspace of at least `need` bytes.  One that a captured graph writes to on every replay is kept
        when a later call (another form, a longer context) needs a larger one."""
        if need and (self.attn_ws is None or self.attn_ws.numel() < need):
            if self._captured:
                self._outgrown.append(self.attn_ws)
            self.attn_ws, self._captured = torch.empty(need, dtype=torch.uint8, device=self.q.device), False
        if self.attn_ws is not None and torch.cuda.is_current_stream_capturing():
            self._captured = True
        return self.attn_ws

    def write_kv_only(self, x, positions, slots, kcache, vcache, cos, sin):
        """RMSNorm + q/k/v projection + rotary + cache write for tokens whose attention output is not needed
        (filling the cache with a prompt through the decode kernels)."""
        lib, w = self.lib, self.w
        h = lib.add_rmsnorm(x, None, w["ln1"], self.eps)
        qkv = lib.linear_f16(h, w["wqkv"], w.get("bqkv"))
        lib.rope_kv_write(qkv, cos, sin, positions, slots, kcache, vcache, Hq=self.Hq, Hkv=self.Hkv, D=self.D)

    def prefill(self, resid_in, delta, positions, slots, seq_starts, max_seq: int, kcache, vcache, cos, sin, *, block_tables=None,
                ctx_lens=None, max_ctx: int = 0, prefix_len: int = 0):
        """The same layer over whole prompts: resid_in [tokens][H] holds the sequences one after another, seq_starts
        int32 [B + 1] their first rows, positions the rotary positions, slots the cache rows of the tokens (negative:
        not cached).  Attention is causal within each sequence (m355_attn_prefill) over the rotated keys of this
        call, so the sequences must start at position 0 of their context -- unless block_tables [B][max_blocks], ctx_lens
        [B] (these tokens counted) and max_ctx are given: then the tokens continue what the cache already holds, of which
        the first prefix_len tokens are shared by all sequences (m355_shared_prefix_attn), and every token needs a slot.
        Buffers are allocated per call (prompt sizes vary).  Returns (residual stream after attention, expert output), as
        forward does."""
        if block_tables is None and (ctx_lens is not None or max_ctx or prefix_len):
            raise ValueError("ctx_lens, max_ctx and prefix_len belong to prompts that continue a cache: block_tables is missing")
        if block_tables is not None and (ctx_lens is None or max_ctx <= 0):
            raise ValueError("prompts that continue a cache need ctx_lens and max_ctx")
        lib, w = self.lib, self.w
        T, dev = resid_in.shape[0], resid_in.device
        resid = torch.empty_like(resid_in)
        h1 = lib.add_rmsnorm(resid_in, delta, w["ln1"], self.eps, resid_out=resid)
        qkv = lib.linear_f16(h1, w["wqkv"], w.get("bqkv"))
        if block_tables is not None:
            q = lib.rope_kv_write(qkv, cos, sin, positions, slots, kcache, vcache, Hq=self.Hq, Hkv=self.Hkv, D=self.D)
            attn = lib.shared_prefix_attn(q, kcache, vcache, block_tables, ctx_lens, prefix_len=prefix_len, max_ctx=max_ctx,
                                          scale=self.D ** -0.5, seq_starts=seq_starts, max_q=max_seq, sinks=w.get("sinks"),
                                          window=self.window)
        else:
            # rotated keys and the values of the prompt, token-major, for the attention; then the same rows into the cache
            k_rows = torch.empty((T, 1, self.Hkv, self.D), dtype=torch.float16, device=dev)
            v_rows = torch.empty_like(k_rows)
            q = lib.rope_kv_write(qkv, cos, sin, positions, torch.arange(T, dtype=torch.int64, device=dev), k_rows, v_rows,
                                  Hq=self.Hq, Hkv=self.Hkv, D=self.D)
            lib.rope_kv_write(qkv, cos, sin, positions, slots, kcache, vcache, Hq=self.Hq, Hkv=self.Hkv, D=self.D, q_out=q)
            attn = lib.attn_prefill(q, k_rows.view(T, self.Hkv, self.D), v_rows.view(T, self.Hkv, self.D), seq_starts, max_seq,
                                    scale=self.D ** -0.5, sinks=w.get("sinks"), window=self.window)
        resid2 = lib.linear_f16(attn.view(T, self.Hq * self.D), w["wo"], w.get("bo"), resid=resid)
        h2 = lib.add_rmsnorm(resid2, None, w["ln2"], self.eps)
        moe_out, _, _ = lib.moe_nf4_forward_routed(h2, w["router_w"], w.get("router_b"), self.k, w["w13_q"], w["w13_absmax"],
                                                   w["w2_q"], w["w2_absmax"], E_local=self.E, e_first=0, H=self.H, FF=self.FF,
                                                   act_mode=self.act_mode, flags=0, b13=w.get("b13"), b2=w.get("b2"))
        return resid2, moe_out

    def forward(self, resid_in, delta, positions, slots, block_tables, ctx_lens, kcache, vcache, cos, sin, max_ctx: int,
                defer_combine: bool = False, prefix_len: int = 0, scores=None):
        """resid_in [T][H]: the residual stream entering the layer, delta: the previous layer's expert output still to
        be added (None for the first layer; a PendingCombine when that layer ran with defer_combine).  ctx_lens counts
        the new token.  Returns (residual stream after attention, expert output): their sum is the layer's output.
        defer_combine: the expert output is returned as a PendingCombine (the experts' rows still unsummed in this
        layer's workspace); the next layer's first kernel then forms it together with the residual add and its
        RMSNorm, one launch less per layer, same bits.
        prefix_len: the first tokens of every sequence are the same, read through row 0 of block_tables once for all.
        scores [blocks][Hkv][block_size] fp32: every own token's attention weight is added there, for evict_tokens."""
        lib, w = self.lib, self.w
        T = resid_in.shape[0]
        if T != self.T:
            raise ValueError(f"built for {self.T} tokens per step, got {T}")
        # residual add (or the previous layer's combine), input norm, q/k/v projection, rotary embedding and cache write:
        # one launch up to 4 tokens, the norm's launch and the projection's one or two beyond (same bits)
        pending = (delta.workspace, delta.w, delta.FF, delta.E, delta.flags) if isinstance(delta, PendingCombine) else delta
        lib.norm_qkv_rope_kv_write(resid_in, pending, w["ln1"], self.eps, w["wqkv"], w.get("bqkv"), cos, sin, positions, slots,
                                   kcache, vcache, Hq=self.Hq, Hkv=self.Hkv, D=self.D, resid_out=self.resid, q_out=self.q,
                                   h_scratch=self.h1, qkv_scratch=self.qkv)
        if scores is not None:
            need = lib.paged_attn_decode_scored_workspace_bytes(T, self.Hq, self.Hkv, self.D, max_ctx, prefix_len)
        elif prefix_len:
            need = lib.shared_prefix_attn_workspace_bytes(T, T, 1, self.Hq, self.Hkv, self.D, max_ctx, prefix_len)
        else:
            need = lib.paged_attn_workspace_bytes(T, self.Hq, self.D, max_ctx)
        attn_args = dict(max_ctx=max_ctx, scale=self.D ** -0.5, workspace=self._attn_workspace(need), out=self.attn, sinks=w.get("sinks"), window=self.window)
        if scores is not None:
            lib.paged_attn_decode_scored(self.q, kcache, vcache, scores, block_tables, ctx_lens, prefix_len=prefix_len, **attn_args)
        elif prefix_len:
            lib.shared_prefix_attn(self.q, kcache, vcache, block_tables, ctx_lens, prefix_len=prefix_len, **attn_args)
        else:
            lib.paged_attn_decode(self.q, kcache, vcache, block_tables, ctx_lens, **attn_args)
        lib.linear_f16(self.attn.view(T, self.Hq * self.D), w["wo"], w.get("bo"), resid=self.resid, out=self.resid2)
        # the router rides in the launch of the norm in front of the MoE block (one workgroup per token has the normalised
        # row at hand).  Measured against the norm alone followed by m355_moe_nf4_forward_routed (logits as a launch of
        # their own over every CU, top-k inside the gate_up launch): the whole stack runs 1.387 against 1.391 ms per step
        # at bs=1 (one launch more there), and 2.795 against 2.851 at bs=32 where the router is a launch of its own
        lib.add_rmsnorm_router(self.resid2, None, w["ln2"], self.eps, w["router_w"], w.get("router_b"), self.k, out=self.h2,
                               ids=self.ids, w=self.wts)
        lib.moe_nf4_forward(self.h2, self.ids, self.wts, w["w13_q"], w["w13_absmax"], w["w2_q"], w["w2_absmax"],
                            E_local=self.E, e_first=0, H=self.H, FF=self.FF, workspace=self.moe_ws, out=self.moe_out,
                            act_mode=self.act_mode, flags=lib.FLAG_SKIP_COMBINE if defer_combine else 0, b13=w.get("b13"),
                            b2=w.get("b2"))
        if defer_combine:
            return self.resid2, PendingCombine(self)
        return self.resid2, self.moe_out
