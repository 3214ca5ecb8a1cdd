"""Measured cases of the paged-cache operators for long contexts: attention of a batch that shares a prefix, decode
attention that accumulates every cached token's attention weight, and eviction from the cache by that weight.

`listed()` and `draw()` give cases, `prepare()` their inputs on the GPU, `run()` one pass: in elementary torch operations
in 32 bits, or, with `own` set, through the framework's entry points.  `exact()` is the definition in 64 bits.
"""
import random

import torch

own = False

_DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


# ---------------------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------------------
def _case(name, op, B, layout, block, prefix, own, n=(1, 1), window=0, sinks=False, keep=0, recent=0):
    """layout = (query heads, KV heads, head size, type).  prefix: tokens that all sequences share; own: range of the
    sequences' own cached tokens (the new ones among them); n: range of new tokens per sequence."""
    Hq, Hkv, D, dtype = layout
    c = dict(op=op, B=B, Hq=Hq, Hkv=Hkv, D=D, dtype=dtype, block=block, prefix=prefix, own_lo=own[0], own_hi=own[1],
             n_lo=n[0], n_hi=n[1], window=window, sinks=sinks, keep=keep, recent=recent)
    if name:
        c["name"] = name
    return c


_A64 = (64, 8, 64, "fp16")        # this repository's own decoder layer


def listed():
    return [
        # a handful of answers to one short system prompt: only latency counts
        _case("prefix_few", "prefix", 4, _A64, 16, 200, (1, 33), sinks=True),
        # a decode batch over one long document, answers of different lengths, full-attention layer with sinks
        _case("prefix_batch", "prefix", 32, _A64, 16, 8192, (1, 512), sinks=True),
        # wide sampling from one very long prompt whose end lies inside a page; larger heads, bfloat16
        _case("prefix_wide", "prefix", 96, (32, 8, 128, "bf16"), 64, 20011, (64, 1024)),
        # the same batch on a sliding-window layer: a query still sees some or none of the prefix
        _case("prefix_window", "prefix", 32, _A64, 16, 4099, (1, 300), window=128, sinks=True),
        # several drafted tokens per sequence checked at once (a few query tokens each, ragged)
        _case("prefix_drafts", "prefix", 24, (40, 8, 128, "fp16"), 32, 6001, (6, 700), n=(1, 6)),
        # questions of a few hundred tokens, all about the same cached document: prompts that continue a shared prefix
        _case("prefix_prompts", "prefix", 6, _A64, 16, 8192, (150, 420), n=(150, 420), sinks=True),
        # two short conversations, weights accumulated for a later eviction
        _case("scored_few", "scored", 2, _A64, 16, 0, (1, 300), sinks=True),
        # a decode batch with a shared system prompt; only the conversations' own tokens are candidates and are scored
        _case("scored_batch", "scored", 32, _A64, 16, 2048, (1000, 4096), sinks=True),
        # few very long contexts
        _case("scored_long", "scored", 4, (32, 4, 128, "bf16"), 64, 0, (50001, 65536)),
        # two short conversations trimmed
        _case("evict_few", "evict", 2, _A64, 16, 0, (100, 300), keep=128, recent=32),
        # a batch trimmed to a quarter behind a shared system prompt
        _case("evict_batch", "evict", 32, _A64, 16, 512, (700, 4096), keep=1024, recent=128),
        # long contexts cut to a quarter
        _case("evict_long", "evict", 3, (32, 8, 128, "bf16"), 64, 0, (50001, 65536), keep=16385, recent=512),
    ]


def _log(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    import math
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _cost(c):
    w = work(c)
    return w["bytes"] / 4e12 + w["flops"] / 4e14


def draw(rng):
    tops = {}
    for c in listed():
        tops[c["op"]] = max(tops.get(c["op"], 0.0), _cost(c))
    op = rng.choice(["prefix", "prefix", "scored", "evict"])
    while True:
        layout = rng.choice([_A64, _A64, (32, 8, 128, "bf16"), (40, 8, 128, "fp16"), (16, 16, 64, "bf16"), (32, 4, 128, "bf16"),
                             (12, 4, 64, "fp16"), (8, 1, 64, "bf16"), (24, 2, 128, "fp16")])
        block = rng.choice([16, 16, 32, 64, 20, 128])
        B = _log(rng, 1, 96)
        if op == "prefix":
            n_hi = rng.choice([1, 1, 1, _log(rng, 2, 12), _log(rng, 13, 420)])
            n_lo = 1 if n_hi == 1 else rng.randint(1, n_hi)
            own_hi = n_hi + _log(rng, 1, 1024) - 1
            c = _case(None, op, B, layout, block, _log(rng, 1, 20011), (rng.randint(n_hi, own_hi), own_hi), n=(n_lo, n_hi),
                      window=rng.choice([0, 0, 0, _log(rng, 1, 5000)]), sinks=rng.random() < 0.5)
        elif op == "scored":
            own_hi = _log(rng, 1, 65536)
            c = _case(None, op, B, layout, block, rng.choice([0, 0, _log(rng, 1, 4096)]), (rng.randint(max(1, own_hi // 3), own_hi), own_hi),
                      window=rng.choice([0, 0, 0, _log(rng, 1, 5000)]), sinks=rng.random() < 0.5)
        else:
            own_hi = _log(rng, 16, 65536)
            keep = _log(rng, 1, min(own_hi, 16385))
            c = _case(None, op, B, layout, block, block * rng.choice([0, 0, 1, _log(rng, 2, 40)]), (rng.randint(1, own_hi), own_hi),
                      keep=keep, recent=rng.randint(0, keep))
        rows = B * c["own_hi"] + c["prefix"]
        pool = 4 * c["Hkv"] * c["D"] * (rows + B * c["keep"])              # bytes of the cache that prepare() fills
        dense = B * c["n_hi"] * c["Hq"] * (c["prefix"] + c["own_hi"])      # logits of the plain form, windows or not
        if _cost(c) <= tops[op] and pool <= 1 << 30 and dense <= 1.4e9:
            return c


# ---------------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------------
def _lengths(case, seed):
    """Own lengths and numbers of new tokens of the sequences: the range's two ends, then numbers between them, the same
    ones for every seed, dealt out to the sequences by the seed."""
    r = random.Random(case["own_lo"] * 1000003 + case["own_hi"])
    B, lo, hi = case["B"], case["own_lo"], case["own_hi"]
    own_len = [hi, lo][:B] + [r.randint(lo, hi) for _ in range(max(0, B - 2))]
    n = [1] * B
    if case["n_hi"] > 1:
        n = [case["n_hi"], case["n_lo"]][:B] + [r.randint(case["n_lo"], case["n_hi"]) for _ in range(max(0, B - 2))]
        # (where both ranges end alike the prompts are fresh: all own tokens are new)
        own_len = n if hi == case["n_hi"] else [max(o, k) for o, k in zip(own_len, n)]
    pairs = list(zip(own_len, n))
    random.Random(seed).shuffle(pairs)
    return [o for o, _ in pairs], [k for _, k in pairs]


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    host = random.Random(seed + 1)
    B, Hq, Hkv, D, bs, P = (case[k] for k in ("B", "Hq", "Hkv", "D", "block", "prefix"))
    dtype = _DTYPES[case["dtype"]]
    own_len, n = _lengths(case, seed)
    ctx = [P + o for o in own_len]
    max_ctx = P + case["own_hi"]
    max_blocks = (max_ctx + bs - 1) // bs
    first_own = P // bs                                   # page of a sequence's first own token
    used = [(c + bs - 1) // bs - first_own for c in ctx]
    dst_blocks = (P + case["keep"] + bs - 1) // bs if case["op"] == "evict" else 0
    num_blocks = (P + bs - 1) // bs + sum(used) + B * max(0, dst_blocks - first_own) + 3
    ids = list(range(num_blocks))
    host.shuffle(ids)
    shared = [ids.pop() for _ in range((P + bs - 1) // bs)]
    tables = []
    for b in range(B):
        row = shared[:first_own] + [ids.pop() for _ in range(used[b])]
        if b == 0 and len(shared) > first_own:            # the first sequence goes on in the prefix's last page
            ids.append(row[first_own])
            row[first_own] = shared[first_own]
        tables.append(row + [0] * (max_blocks - len(row)))
    randn = lambda *shape: torch.randn(*shape, generator=gen, device=dev, dtype=torch.float32)      # noqa: E731
    s = dict(case=case, block_tables=torch.tensor(tables, dtype=torch.int32, device=dev),
             ctx_lens=torch.tensor(ctx, dtype=torch.int32, device=dev), max_ctx=max_ctx, scale=D ** -0.5, window=case["window"],
             kcache=torch.empty((num_blocks, bs, Hkv, D), dtype=dtype, device=dev).normal_(generator=gen),
             vcache=torch.empty((num_blocks, bs, Hkv, D), dtype=dtype, device=dev).normal_(generator=gen))
    if case["op"] in ("scored", "evict"):
        # weights add up to a few units over many steps, unevenly; some tokens were never attended to
        acc = torch.exp(1.5 * randn(num_blocks, Hkv, bs) - 2.0)
        s["scores"] = acc * (torch.rand(acc.shape, generator=gen, device=dev) > 0.1)
    if case["op"] == "evict":
        dst = [shared[:first_own] + [ids.pop() for _ in range(dst_blocks - first_own)] for _ in range(B)]
        s.update(dst_tables=torch.tensor(dst, dtype=torch.int32, device=dev), keep=case["keep"], recent=case["recent"])
        return s
    starts = [0]
    for k in n:
        starts.append(starts[-1] + k)
    # queries somewhat larger than the keys: attention that picks out tokens instead of averaging over all
    s["q"] = (1.5 * randn(starts[-1], Hq, D)).to(dtype)
    s["sinks"] = (0.5 + randn(Hq)).to(dtype) if case["sinks"] else None
    s["seq_starts"] = torch.tensor(starts, dtype=torch.int32, device=dev) if case["n_hi"] > 1 else None
    s["max_q"] = case["n_hi"]
    if own:
        # what a serving loop keeps over its steps
        from gpt_oss_vllm_amd import lib
        s["out"] = torch.empty_like(s["q"])
        if case["op"] == "prefix":
            need = lib.shared_prefix_attn_workspace_bytes(starts[-1], B, case["n_hi"], Hq, Hkv, D, max_ctx, P)
        else:
            need = lib.paged_attn_decode_scored_workspace_bytes(B, Hq, Hkv, D, max_ctx, P)
        s["workspace"] = torch.empty(max(need, 256), dtype=torch.uint8, device=dev)
    return s


# ---------------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------------
def run(s):
    op = s["case"]["op"]
    if own:
        from gpt_oss_vllm_amd import lib
        if op == "prefix":
            return lib.shared_prefix_attn(s["q"], s["kcache"], s["vcache"], s["block_tables"], s["ctx_lens"], prefix_len=s["case"]["prefix"],
                                          max_ctx=s["max_ctx"], scale=s["scale"], seq_starts=s["seq_starts"], max_q=s["max_q"],
                                          sinks=s["sinks"], window=s["window"], workspace=s["workspace"], out=s["out"])
        if op == "scored":
            out = lib.paged_attn_decode_scored(s["q"], s["kcache"], s["vcache"], s["scores"], s["block_tables"], s["ctx_lens"],
                                               max_ctx=s["max_ctx"], scale=s["scale"], prefix_len=s["case"]["prefix"], sinks=s["sinks"],
                                               window=s["window"], workspace=s["workspace"], out=s["out"])
            return out, s["scores"]
        kept, new_lens = lib.kv_evict(s["kcache"], s["vcache"], s["scores"], s["block_tables"], s["ctx_lens"], s["dst_tables"],
                                      keep=s["keep"], recent=s["recent"], prefix_len=s["case"]["prefix"], max_ctx=s["max_ctx"])
        return kept, new_lens, s["kcache"], s["vcache"], s["scores"]
    if op == "evict":
        return _plain_evict(s)
    out, w = _plain_attention(s)
    if op == "prefix":
        return out
    # the own tokens' weights, summed over the query heads of a KV head, onto what earlier steps left there
    blk, off = _own_slots(s)
    heads = torch.arange(s["case"]["Hkv"], device=blk.device)
    s["scores"].index_put_((blk[:, None, :], heads[None, :, None], off[None, None, :]), w, accumulate=True)
    return out, s["scores"]


def _own_slots(s):
    """Page [B][O] and offset [O] of every sequence's own positions (past its end: page 0 of the table's padding)."""
    P, bs = s["case"]["prefix"], s["case"]["block"]
    pos = torch.arange(P, s["max_ctx"], device=s["ctx_lens"].device)
    return s["block_tables"][:, pos // bs].long(), pos % bs


def _plain_attention(s):
    """softmax(q K^T) V over the shared prefix, read once, and every sequence's own tokens; [T][Hq][D] and the own tokens'
    weights [B][Hkv][O] summed over a KV head's queries."""
    c = s["case"]
    B, Hq, Hkv, D, bs, P, N = (c[k] for k in ("B", "Hq", "Hkv", "D", "block", "prefix", "n_hi"))
    G = Hq // Hkv
    q, ctx = s["q"], s["ctx_lens"].long()
    dev = q.device
    j = torch.arange(N, device=dev)
    if s["seq_starts"] is None:
        n = torch.ones(B, dtype=torch.long, device=dev)
        token = torch.arange(B, device=dev)[:, None]
    else:
        st = s["seq_starts"].long()
        n = st[1:] - st[:-1]
        token = (st[:-1, None] + j).clamp(max=q.shape[0] - 1)
    live = j < n[:, None]                                                    # [B][N]
    qpos = ctx[:, None] - n[:, None] + j
    qf = q[token].float().view(B, N, Hkv, G, D) * s["scale"]

    def visible(kpos):                                                       # [B][N][keys]
        ok = kpos <= qpos[:, :, None]
        return ok & (kpos > qpos[:, :, None] - s["window"]) if s["window"] else ok

    ppos = torch.arange(P, device=dev)
    prow = s["block_tables"][0, ppos // bs].long()
    kp = s["kcache"][prow, ppos % bs].float().permute(1, 2, 0).contiguous()  # [Hkv][D][P]
    vp = s["vcache"][prow, ppos % bs].float().transpose(0, 1).contiguous()   # [Hkv][P][D]
    sp = torch.matmul(qf.permute(2, 0, 1, 3, 4).reshape(Hkv, B * N * G, D), kp).view(Hkv, B, N, G, P)
    sp = sp.masked_fill(~visible(ppos)[None, :, :, None, :], float("-inf"))
    blk, off = _own_slots(s)
    opos = torch.arange(P, s["max_ctx"], device=dev)
    O = opos.numel()
    inside = (opos < ctx[:, None])[:, :, None, None]
    ko = (s["kcache"][blk, off].float() * inside).permute(0, 2, 3, 1).contiguous()   # [B][Hkv][D][O]
    vo = (s["vcache"][blk, off].float() * inside).transpose(1, 2).contiguous()       # [B][Hkv][O][D]
    so = torch.matmul(qf.permute(0, 2, 1, 3, 4).reshape(B, Hkv, N * G, D), ko).view(B, Hkv, N, G, O)
    so = so.masked_fill(~visible(opos)[:, None, :, None, :], float("-inf"))
    m = so.amax(-1).permute(1, 0, 2, 3)                                      # [Hkv][B][N][G]
    if P:
        m = torch.maximum(m, sp.amax(-1))
    if s["sinks"] is not None:
        sink = s["sinks"].float().view(Hkv, 1, 1, G)
        m = torch.maximum(m, sink)
    m = m.masked_fill(m == float("-inf"), 0.0)
    ep = torch.exp(sp - m[..., None])
    eo = torch.exp(so - m.permute(1, 0, 2, 3)[..., None])
    l = ep.sum(-1) + eo.sum(-1).permute(1, 0, 2, 3)
    if s["sinks"] is not None:
        l = l + torch.exp(sink - m)
    o = torch.matmul(ep.reshape(Hkv, B * N * G, P), vp).view(Hkv, B, N, G, D)
    o = o + torch.matmul(eo.reshape(B, Hkv, N * G, O), vo).view(B, Hkv, N, G, D).permute(1, 0, 2, 3, 4)
    inv = torch.where(l > 0, 1.0 / l, torch.zeros_like(l))
    o = (o * inv[..., None]).permute(1, 2, 0, 3, 4).reshape(B, N, Hq, D)
    if c["op"] == "scored":
        w = (eo * inv.permute(1, 0, 2, 3)[..., None]).sum(dim=(2, 3))        # [B][Hkv][O]
        return o[:, 0].to(q.dtype), w
    return o[live].to(q.dtype), None


def _plain_evict(s):
    """Of every sequence's own tokens and per KV head: the last `recent`, and of the others those with the largest scores
    (ties: the lower position), `keep` in all, copied in order to the pages of dst_tables together with their scores."""
    c = s["case"]
    B, Hkv, bs, P = (c[k] for k in ("B", "Hkv", "block", "prefix"))
    keep, recent, ctx = s["keep"], s["recent"], s["ctx_lens"].long()
    dev = ctx.device
    blk, off = _own_slots(s)
    O = off.numel()
    score = s["scores"][blk, :, off[None, :]].permute(0, 2, 1)               # [B][Hkv][O]
    pos = torch.arange(O, device=dev)
    own_len = ctx - P
    group = (pos < own_len[:, None]).long() + (pos >= own_len[:, None] - recent).long() * (pos < own_len[:, None])
    order = torch.sort(score, dim=-1, descending=True, stable=True).indices
    group = torch.gather(group[:, None, :].expand(B, Hkv, O), 2, order)
    order = torch.gather(order, 2, torch.sort(group, dim=-1, descending=True, stable=True).indices)[..., :keep]
    if O < keep:
        order = torch.nn.functional.pad(order, (0, keep - O), value=O)
    new_own = own_len.clamp(max=keep)
    valid = torch.arange(keep, device=dev) < new_own[:, None]                # [B][keep]
    kept = torch.sort(torch.where(valid[:, None, :], order, O), dim=-1).values
    b, h, i = torch.nonzero(valid[:, None, :].expand(B, Hkv, keep), as_tuple=True)
    src = kept[b, h, i]
    sblk, soff = blk[b, src], off[src]
    dpos = P + i
    dblk, doff = s["dst_tables"][b, dpos // bs].long(), dpos % bs
    for name in ("kcache", "vcache"):
        s[name][dblk, doff, h] = s[name][sblk, soff, h]
    moved = s["scores"][sblk, h, soff]
    # the rows behind the last kept token in its page start at zero
    end = P + new_own
    tail = end[:, None] + torch.arange(bs, device=dev)
    b2, k2 = torch.nonzero((tail // bs == (end[:, None] - 1) // bs) & (new_own[:, None] > 0), as_tuple=True)
    s["scores"][s["dst_tables"][b2, tail[b2, k2] // bs].long(), :, tail[b2, k2] % bs] = 0.0
    s["scores"][dblk, h, doff] = moved
    kept = torch.where(valid[:, None, :], kept + P, -1).to(torch.int32)
    return kept, end.to(torch.int32), s["kcache"], s["vcache"], s["scores"]


# ---------------------------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------------------------------
def work(case):
    own_len, n = _lengths(case, 0)
    Hq, Hkv, D, P, W = (case[k] for k in ("Hq", "Hkv", "D", "prefix", "window"))
    row = 2 * Hkv * D * 2                                  # K and V of one token, bytes
    if case["op"] == "evict":
        kept = sum(min(o, case["keep"]) for o in own_len)
        return {"bytes": 2 * kept * row + 4 * Hkv * (sum(own_len) + 2 * kept), "flops": 0}
    pairs, own_rows, lowest = 0, 0, P
    for o, k in zip(own_len, n):
        for i in range(k):
            pairs += min(P + o - k + i + 1, W) if W else P + o - k + i + 1
        first = max(0, P + o - k + 1 - W) if W else 0      # the first key that one of its queries sees
        lowest = min(lowest, first)
        own_rows += o - max(0, first - P)
    T = sum(n)
    moved = row * (P - lowest + own_rows) + 2 * T * Hq * D * 2
    if case["op"] == "scored":
        moved += 2 * 4 * Hkv * own_rows
    return {"bytes": moved, "flops": 4 * D * Hq * pairs}


# ---------------------------------------------------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    return _exact_evict(s) if case["op"] == "evict" else _exact_attention(s)


def _exact_attention(s):
    """Sequence by sequence: all visible tokens' logits, their softmax with the sink, the weighted sum of the values."""
    c = s["case"]
    Hq, Hkv, D, bs, P, W = (c[k] for k in ("Hq", "Hkv", "D", "block", "prefix", "window"))
    G = Hq // Hkv
    q = s["q"].double()
    out = torch.zeros_like(q)
    scores = s["scores"].double() if c["op"] == "scored" else None
    table = s["block_tables"].cpu().long()
    starts = list(range(c["B"] + 1)) if s["seq_starts"] is None else s["seq_starts"].tolist()
    for b, ctx in enumerate(s["ctx_lens"].tolist()):
        pos = torch.arange(ctx)
        page = torch.where(pos < P, table[0, pos // bs], table[b, pos // bs]).to(q.device)
        off = (pos % bs).to(q.device)
        pos = pos.to(q.device)
        k, v = s["kcache"][page, off].double(), s["vcache"][page, off].double()        # [ctx][Hkv][D]
        t0, t1 = starts[b], starts[b + 1]
        at = torch.arange(ctx - (t1 - t0), ctx, device=q.device)                       # the queries' positions
        hidden = pos[None, :] > at[:, None]
        if W:
            hidden |= pos[None, :] <= at[:, None] - W
        for h in range(Hkv):
            logits = torch.matmul(q[t0:t1, h * G:(h + 1) * G].reshape(-1, D), k[:, h].t().contiguous()) * s["scale"]
            logits = logits.view(t1 - t0, G, ctx).masked_fill(hidden[:, None, :], float("-inf"))
            if s["sinks"] is not None:
                sink = s["sinks"][h * G:(h + 1) * G].double().view(1, G, 1).expand(t1 - t0, G, 1)
                logits = torch.cat([logits, sink], dim=-1)
            p = torch.softmax(logits, dim=-1)[..., :ctx]
            out[t0:t1, h * G:(h + 1) * G] = torch.matmul(p.view(-1, ctx), v[:, h].contiguous()).view(t1 - t0, G, D)
            if scores is not None:
                scores[page[P:], h, off[P:]] += p.sum(dim=(0, 1))[P:]
    return out if scores is None else (out, scores)


def _exact_evict(s):
    c = s["case"]
    bs, P, keep, recent = c["block"], c["prefix"], c["keep"], c["recent"]
    kc, vc, sc = s["kcache"].double(), s["vcache"].double(), s["scores"].double()
    kc0, vc0, sc0 = kc.clone(), vc.clone(), sc.clone()
    table, dst = s["block_tables"].long(), s["dst_tables"].long()
    dev = kc.device
    kept = torch.full((c["B"], c["Hkv"], keep), -1, dtype=torch.int32, device=dev)
    new_lens = []
    for b, ctx in enumerate(s["ctx_lens"].tolist()):
        pos = torch.arange(P, ctx, device=dev)
        page, off = table[b, pos // bs], pos % bs
        m = min(keep, ctx - P)
        to = torch.arange(P, P + m, device=dev)
        to_page, to_off = dst[b, to // bs], to % bs
        new_lens.append(P + m)
        if m:
            sc[to_page[-1], :, (P + m - 1) % bs + 1:] = 0.0
        for h in range(c["Hkv"]):
            rank = sc0[page, h, off]
            rank[ctx - P - min(recent, ctx - P):] = float("inf")
            chosen = torch.argsort(rank, descending=True, stable=True)[:m].sort().values
            # (the last tokens count as infinite, and no finite number of them exceeds keep: ties among them cannot lose one)
            kept[b, h, :m] = (chosen + P).to(torch.int32)
            kc[to_page, to_off, h] = kc0[page[chosen], off[chosen], h]
            vc[to_page, to_off, h] = vc0[page[chosen], off[chosen], h]
            sc[to_page, h, to_off] = sc0[page[chosen], h, off[chosen]]
    return kept, torch.tensor(new_lens, dtype=torch.int32, device=dev), kc, vc, sc
