"""The long-context operators at the ends of what their arguments allow: lengths and windows at the type's limits, weights
far below the largest, infinite and NaN values behind ranges that weigh nothing, workspaces kept over differing batches,
layers whose graphs outlive a buffer.  Oracle and tolerances are those of test_long_context.py."""
import pytest
import torch

from test_long_context import BF16, F16, Cache, _inputs, check, oracle, score_err


# ---------------------------------------------------------------------------------------------------------------------
# lengths and windows
# ---------------------------------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("window", [0, 1, 40, (1 << 31) - 1])
@pytest.mark.parametrize("P", [0, 2500])
def test_gpu_negative_lengths_are_empty(P, window, m355, cuda):
    """A length below zero is an empty context, whatever the window: zeros, and no score moves; the other sequences keep
    their results."""
    c = Cache(3, [P + 70, P + 33, P + 5], 2, 64, 16, F16, prefix=P)
    q, _ = _inputs(c, 3, 16, 1, False)
    want, mag, weights = oracle(c, q, [1] * 3, 0.125, window=window)
    kc, vc, bt, cl = c.device(cuda)
    sc = c.scores.to(cuda)
    for length in (-1, -2, -100, -(1 << 31)):
        lens = cl.clone()
        lens[1] = length
        before = sc.clone()
        st = torch.tensor([0, 1, 2, 3], dtype=torch.int32, device=cuda)
        for got in (m355.shared_prefix_attn(q.to(cuda), kc, vc, bt, lens, prefix_len=P, max_ctx=P + 70, scale=0.125, window=window),
                    m355.shared_prefix_attn(q.to(cuda), kc, vc, bt, lens, prefix_len=P, max_ctx=P + 70, scale=0.125, window=window, seq_starts=st, max_q=1),
                    m355.paged_attn_decode_scored(q.to(cuda), kc, vc, sc, bt, lens, prefix_len=P, max_ctx=P + 70, scale=0.125, window=window)):
            assert (got[1] == 0).all()
            check(got[[0, 2]], want[[0, 2]], mag[[0, 2]], F16, score_err(c, q, 0.125))
        moved = (sc != before).cpu()
        page, off = c.slots(1)
        assert not moved[page[P:], :, off[P:]].any()
        page, off = c.slots(0)
        seen = weights[0].t()[P:] > 1e-6
        assert moved[page[P:], :, off[P:]][seen].all()
    # several tokens of a sequence that is shorter than they are many: the ones in front of it see nothing
    n = [2, 2, 5]
    c = Cache(4, [P + 70, 0, 3], 2, 64, 16, F16, prefix=P)
    q, _ = _inputs(c, 9, 16, 2, False)
    want, mag, _ = oracle(c, q, n, 0.125, window=window)
    kc, vc, bt, cl = c.device(cuda)
    cl[1] = -5
    st = torch.tensor([0, 2, 4, 9], dtype=torch.int32, device=cuda)
    got = m355.shared_prefix_attn(q.to(cuda), kc, vc, bt, cl, prefix_len=P, max_ctx=P + 70, scale=0.125, window=window, seq_starts=st, max_q=5)
    check(got, want, mag, F16, score_err(c, q, 0.125))
    assert (got[2:6] == 0).all()


# ---------------------------------------------------------------------------------------------------------------------
# weights far below the largest
# ---------------------------------------------------------------------------------------------------------------------
# fp16 probabilities: the largest of a row is held as 2^9 or more, so one that falls below the normal range is off by at
# most half of 2^-24 of that, 2^-34 of the largest, on top of the relative half step that test_long_context.py counts.
FP16_LOST = 2.0 ** -34

# sequences, own tokens, new tokens, prefix, position of the dominant key, heads
DOMINATED = [(64, 1500, 1, 0, 7, (4, 2)), (40, 3, 1, 6000, 11, (8, 2)), (3, 900, 1, 0, 899, (8, 2)), (4, 300, 300, 3000, 2999, (8, 2)),
             (2, 256, 256, 1500, 3, (64, 8)), (1, 40, 7, 4096, 4000, (6, 2))]


def _dominated(case, gap, dtype):
    B, own, n, P, at, (Hq, Hkv) = DOMINATED[case]
    c = Cache(900 + case, [P + own] * B, Hkv, 64, 16, dtype, prefix=P)
    c.k[..., 0] = (0.05 * torch.randn(c.k.shape[:3], generator=c.g)).to(dtype)
    c.v = (1 + 0.25 * torch.randn(c.v.shape, generator=c.g)).to(dtype)
    for b in range(B):
        page, off = c.slots(b)
        c.k[page[at], off[at], :, 0] = gap
        c.v[page[at], off[at]] = 0
    c.k_norm = float(c.k.float().norm(dim=-1).max())
    q = torch.zeros((B * n, Hq, 64), dtype=dtype)
    q[..., 0] = 8                                              # scores, at a scale of 1/8, are the keys' first columns
    return c, q, [n] * B


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("case, gap", [(c, g) for c in range(len(DOMINATED)) for g in ((17.5, 20.0) if c == 4 else (12.0, 17.5, 20.0, 22.0))])
def test_gpu_one_key_dominates(case, gap, dtype, m355, cuda):
    """One key whose value is 0, thousands of others 12 to 22 nats below it: what they add up to is the output."""
    c, q, n = _dominated(case, gap, dtype)
    P, B = c.prefix, len(n)
    want, mag, weights = oracle(c, q, n, 0.125)
    rel = score_err(c, q, 0.125)
    lost = FP16_LOST * 2.5 * max(c.ctx) if dtype == F16 else 0.0          # (values lie below 2.5)
    kc, vc, bt, cl = c.device(cuda)
    assert float(c.v.abs().max()) < 2.5
    st = None if n[0] == 1 else torch.arange(0, B * n[0] + 1, n[0], dtype=torch.int32, device=cuda)
    got = m355.shared_prefix_attn(q.to(cuda), kc, vc, bt, cl, prefix_len=P, max_ctx=max(c.ctx), scale=0.125, seq_starts=st, max_q=n[0])
    _check_lost(got, want, mag, dtype, rel, lost)
    if n[0] == 1:
        sc = torch.zeros(c.scores.shape, device=cuda)
        got = m355.paged_attn_decode_scored(q.to(cuda), kc, vc, sc, bt, cl, prefix_len=P, max_ctx=max(c.ctx), scale=0.125)
        _check_lost(got, want, mag, dtype, rel, lost)
        for b in range(B):
            page, off = c.slots(b)
            w = weights[b].t()[P:]
            assert ((sc.cpu().double()[page[P:], :, off[P:]] - w).abs() <= (2 * rel + 2.0 ** -23 * (q.shape[1] // c.Hkv)) * w).all()


def _check_lost(got, want, mag, dtype, rel, lost):
    half = torch.finfo(dtype).eps / 2
    tol = half * want.abs() + (half + 2 * rel) * mag + 2 * torch.finfo(dtype).smallest_normal * half + lost
    err = (got.cpu().double() - want).abs()
    assert (err <= tol).all(), f"worst {float((err / tol).max()):.2f} of the tolerance"


@pytest.mark.gpu
@pytest.mark.parametrize("B,own,n,P,heads", [(1, 700, 1, 0, (4, 2)), (40, 5, 1, 3000, (8, 2)), (1, 300, 300, 1000, (8, 2)), (2, 256, 256, 1500, (64, 8)),
                                             (1, 5000, 1, 0, (33, 1))])
def test_gpu_values_near_the_largest_finite_ones(B, own, n, P, heads, m355, cuda):
    """bfloat16 values of up to 2^126 and scores that grow along the keys by as much as leaves the reference where it was:
    the output is an average of the values, however large its terms were on the way."""
    Hq, Hkv = heads
    c = Cache(950, [P + own] * B, Hkv, 64, 16, BF16, prefix=P)
    for b in range(B):
        page, off = c.slots(b)
        c.k[page, off, :, 0] = (7.5 * torch.arange(c.ctx[b]) / c.ctx[b]).to(BF16)[:, None]     # 2^10.8 from the first to the last
    c.v = (c.v.float().clamp(-4, 4) * 2.0 ** 124).to(BF16)
    c.k_norm = float(c.k.float().norm(dim=-1).max())
    q = torch.zeros((B * n, Hq, 64), dtype=BF16)
    q[..., 0] = 8
    want, mag, _ = oracle(c, q, [n] * B, 0.125)
    kc, vc, bt, cl = c.device(cuda)
    st = None if n == 1 else torch.arange(0, B * n + 1, n, dtype=torch.int32, device=cuda)
    got = m355.shared_prefix_attn(q.to(cuda), kc, vc, bt, cl, prefix_len=P, max_ctx=max(c.ctx), scale=0.125, seq_starts=st, max_q=n)
    check(got, want, mag, BF16, score_err(c, q, 0.125))
    if n == 1:
        got = m355.paged_attn_decode_scored(q.to(cuda), kc, vc, torch.zeros(c.scores.shape, device=cuda), bt, cl, prefix_len=P, max_ctx=max(c.ctx),
                                            scale=0.125)
        check(got, want, mag, BF16, score_err(c, q, 0.125))


# ---------------------------------------------------------------------------------------------------------------------
# infinite and NaN values that weigh almost nothing
# ---------------------------------------------------------------------------------------------------------------------
def _same_nonfinite(got, want, mag, dtype, rel, lost):
    got = got.cpu().double()
    bad = ~want.isfinite()
    assert torch.equal(got.isfinite(), ~bad)
    assert torch.equal(got[bad].isnan(), want[bad].isnan()) and torch.equal(got[got.isinf()], want[want.isinf()])
    zero = torch.zeros_like(want)
    _check_lost(torch.where(bad, zero, got), torch.where(bad, zero, want), torch.where(bad, zero, mag), dtype, rel, lost)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("by", ["key", "sink"])
@pytest.mark.parametrize("case, gap", [(c, g) for c in range(len(DOMINATED)) for g in ((30.0, 110.0) if c == 4 else (14.0, 30.0, 110.0, 250.0))])
def test_gpu_nonfinite_values_of_keys_that_weigh_nothing(case, by, gap, dtype, m355, cuda):
    """Infinite and NaN values of keys 14 to 250 nats below a dominating key, or below the sink, reach every query that sees
    them, as what they are: next to the dominating key, in the same range, in other ranges, in the prefix and behind it."""
    c, q, n = _dominated(case, gap if by == "key" else 0.0, dtype)
    sinks = torch.full((q.shape[1],), gap).to(dtype) if by == "sink" else None
    P, B, at, ctx = c.prefix, len(n), DOMINATED[case][4], c.ctx[0]
    near = at + 1 if at + 1 < ctx else at - 1
    spots = [(near, 1, float("nan")), (near, 2, float("inf")), (ctx // 2, 5, float("-inf")), (ctx // 2, 6, float("nan")), (0, 63, float("inf")),
             (ctx - 1, 33, float("inf")), (max(P - 1, 2), 40, float("-inf")), (ctx // 3, 12, float("inf")), (ctx // 5, 12, float("inf")),
             (ctx // 3, 13, float("inf")), (ctx // 5, 13, float("-inf"))]
    for pos, column, value in spots:
        if pos != at:
            for b in range(B if pos >= P else 1):
                page, off = c.slots(b)
                c.v[page[pos], off[pos], c.Hkv - 1, column] = value            # (the other KV heads stay finite)
    want, mag, _ = oracle(c, q, n, 0.125, sinks)
    assert want.isnan().any() and want.isinf().any() and want.isfinite().any()
    rel = score_err(c, q, 0.125)
    lost = FP16_LOST * 2.5 * max(c.ctx) if dtype == F16 else 0.0
    kc, vc, bt, cl = c.device(cuda)
    st = None if n[0] == 1 else torch.arange(0, B * n[0] + 1, n[0], dtype=torch.int32, device=cuda)
    sk = None if sinks is None else sinks.to(cuda)
    got = m355.shared_prefix_attn(q.to(cuda), kc, vc, bt, cl, prefix_len=P, max_ctx=ctx, scale=0.125, seq_starts=st, max_q=n[0], sinks=sk)
    _same_nonfinite(got, want, mag, dtype, rel, lost)
    if n[0] == 1:
        sc = torch.zeros(c.scores.shape, device=cuda)
        got = m355.paged_attn_decode_scored(q.to(cuda), kc, vc, sc, bt, cl, prefix_len=P, max_ctx=ctx, scale=0.125, sinks=sk)
        _same_nonfinite(got, want, mag, dtype, rel, lost)
        assert sc.isfinite().all()


@pytest.mark.gpu
@pytest.mark.parametrize("window", [0, 700])
def test_gpu_nonfinite_keys_and_queries(window, m355, cuda):
    """A NaN in a key or in a query reaches the rows whose scores it enters, whatever their other weights, and no other."""
    P, n = 2500, [3, 1]
    c = Cache(77, [P + 40, P + 9], 2, 64, 16, F16, prefix=P)
    q, _ = _inputs(c, 4, 16, 3, False)
    rel = score_err(c, q, 0.125)
    want, mag, _ = oracle(c, q, n, 0.125, window=window)
    page, off = c.slots(0)
    c.k[page[P + 38], off[P + 38], 0, 5] = float("nan")          # rows 1 and 2 of the first sequence see it, KV head 0
    c.k[page[P - 660], off[P - 660], 1, 9] = float("nan")        # windowed: rows 0 (and 3) see it, KV head 1; else everyone
    q[3, 15, 7] = float("nan")
    hit = torch.zeros(q.shape[:2], dtype=torch.bool)
    hit[1:3, :8] = True
    for row, pos in ((0, P + 37), (1, P + 38), (2, P + 39), (3, P + 8)):
        if not window or P - 660 > pos - window:
            hit[row, 8:] = True
    hit[3, 15] = True
    kc, vc, bt, cl = c.device(cuda)
    st = torch.tensor([0, 3, 4], dtype=torch.int32, device=cuda)
    got = m355.shared_prefix_attn(q.to(cuda), kc, vc, bt, cl, prefix_len=P, max_ctx=P + 40, scale=0.125, seq_starts=st, max_q=3, window=window).cpu()
    assert got[hit].isnan().all()
    zero = torch.zeros_like(want)
    check(torch.where(hit[..., None], torch.zeros_like(got), got), torch.where(hit[..., None], zero, want), mag, F16, rel)


# ---------------------------------------------------------------------------------------------------------------------
# workspaces
# ---------------------------------------------------------------------------------------------------------------------
def _answer(m355, ws_bytes, T, B, max_q, Hq, Hkv, D, max_ctx, prefix, scored):
    """The call's answer to a workspace of so many bytes: -6 where it is too small, else -3, since it is at an odd address."""
    ptr, L = 0x10000, m355.load()
    blocks = (max_ctx + 15) // 16
    tail = [16, blocks, 16 * Hkv * D, max_ctx, prefix, Hq * D, Hq * D, 0.1, None, 0, ptr + 1, ws_bytes, ptr, None]
    if scored:
        return L.m355_paged_attn_decode_scored(*[ptr] * 6, B, Hq, Hkv, D, 0, blocks, *tail)
    return L.m355_shared_prefix_attn(*[ptr] * 6, T, B, max_q, Hq, Hkv, D, 0, blocks, *tail)


def _need(m355, T, B, max_q, Hq, Hkv, D, max_ctx, prefix, scored):
    if scored:
        return m355.paged_attn_decode_scored_workspace_bytes(B, Hq, Hkv, D, max_ctx, prefix)
    return m355.shared_prefix_attn_workspace_bytes(T, B, max_q, Hq, Hkv, D, max_ctx, prefix)


@pytest.mark.parametrize("scored", [False, True])
def test_a_workspace_for_the_largest_call_serves_every_smaller_one(scored, m355):
    """Fewer tokens, sequences, cached tokens: no call asks for more than the largest one, although the numbers of ranges
    that are best for them do.  Asked for without a prefix, it serves every prefix."""
    import random
    rng = random.Random(5)
    fixed = [((32, 1, 64, 8, 64, 2300, 2048), (31, 1, 2300)), ((32, 1, 64, 8, 64, 2180, 2048), (32, 1, 2116)), ((32, 1, 64, 8, 64, 2116, 2048), (32, 1, 2100)),
             ((96, 1, 32, 8, 128, 21035, 20011), (1, 1, 20012)), ((6, 400, 64, 8, 64, 8612, 8192), (1, 1, 8193)), ((4, 1, 130, 1, 64, 300, 200), (1, 1, 201))]
    pairs = [(big, small) for big, small in fixed if not scored or big[1] == 1]
    for _ in range(3000):
        Hkv = rng.choice([1, 2, 4, 8])
        P = rng.choice([0, rng.randint(1, 200), rng.randint(1, 20000)])
        big = (rng.randint(1, 96), 1 if scored else rng.choice([1, rng.randint(2, 200)]), Hkv * rng.choice([1, 2, 5, 8, 33]), Hkv, rng.choice([64, 128]),
               P + rng.randint(1, rng.choice([100, 1000, 30000])), P)
        pairs.append((big, (rng.randint(1, big[0]), rng.randint(1, big[1]), rng.randint(1, big[5]))))
    for (B, n, Hq, Hkv, D, ctx, P), (b, k, c) in pairs:
        for asked in (P, 0):
            ws = _need(m355, B * n, B, n, Hq, Hkv, D, ctx, asked, scored)
            case = ((B, n, Hq, Hkv, D, ctx, P), (b, k, c), asked, ws)
            assert _answer(m355, ws, B * n, B, n, Hq, Hkv, D, ctx, P, scored) == -3, case
            assert _answer(m355, ws, b * k, b, k, Hq, Hkv, D, c, P, scored) == -3, case
    # one range per sequence leaves nothing to join: a call that is best served by it asks for next to nothing
    assert scored or _need(m355, 4, 4, 1, 64, 8, 64, 233, 200, False) <= 4096


WORKSPACES = [([2000, 7, 300], [1, 1, 1], 0, (64, 8)), ([30, 1, 9], [1, 1, 1], 5000, (16, 2)), ([900, 40], [1, 1], 2100, (8, 2)),
              ([700, 90], [5, 90], 3001, (16, 2)), ([300, 2], [1, 1], 130, (66, 1))]


@pytest.mark.gpu
@pytest.mark.parametrize("case, scored", [(i, s) for i in range(len(WORKSPACES)) for s in (False, True) if not s or max(WORKSPACES[i][1]) == 1])
def test_gpu_results_hold_for_every_workspace(case, scored, m355, cuda):
    """From the least that is accepted to all that is asked for: the same results within the tolerance, nothing written
    behind the bytes that were named, nothing read that the call has not written."""
    own, n, P, (Hq, Hkv) = WORKSPACES[case]
    c = Cache(61, [P + o for o in own], Hkv, 64, 16, F16, prefix=P, n=n)
    T, B, max_ctx = sum(n), len(n), P + max(own)
    q, sk = _inputs(c, T, Hq, 6, True)
    want, mag, weights = oracle(c, q, n, 0.125, sk)
    kc, vc, bt, cl = c.device(cuda)
    need = _need(m355, T, B, max(n), Hq, Hkv, 64, max_ctx, P, scored)
    low, least = 0, need                       # the least that is accepted, by halving
    while least - low > 4:
        mid = (low + least) // 8 * 4
        low, least = (low, mid) if _answer(m355, mid, T, B, max(n), Hq, Hkv, 64, max_ctx, P, scored) == -3 else (mid, least)
    buffer = torch.empty(need + 4096, dtype=torch.uint8, device=cuda)
    st = None if max(n) == 1 else torch.tensor([0] + [sum(n[:i + 1]) for i in range(B)], dtype=torch.int32, device=cuda)
    rel = score_err(c, q, 0.125)
    for part in range(9):
        size = least + (need - least) * part // 8 // 4 * 4
        buffer.fill_(255)
        kw = dict(prefix_len=P, max_ctx=max_ctx, scale=0.125, sinks=sk.to(cuda), workspace=buffer[:size])
        if scored:
            sc = torch.zeros(c.scores.shape, device=cuda)
            got = m355.paged_attn_decode_scored(q.to(cuda), kc, vc, sc, bt, cl, **kw)
            for b in range(B):
                page, off = c.slots(b)
                w = weights[b].t()[P:]
                assert ((sc.cpu().double()[page[P:], :, off[P:]] - w).abs() <= (2 * rel + 2.0 ** -23 * (Hq // Hkv + 2)) * w).all()
        else:
            got = m355.shared_prefix_attn(q.to(cuda), kc, vc, bt, cl, seq_starts=st, max_q=max(n), **kw)
        check(got, want, mag, F16, rel)
        assert (buffer[size:] == 255).all()


# ---------------------------------------------------------------------------------------------------------------------
# refusals
# ---------------------------------------------------------------------------------------------------------------------
def test_several_tokens_need_their_longest_number(m355):
    """Without max_q a packed call would leave all tokens but the sequences' first ones unwritten."""
    c = Cache(1, [20, 30], 2, 64, 16, F16)
    q, st = torch.zeros((5, 8, 64), dtype=F16), torch.tensor([0, 2, 5], dtype=torch.int32)
    with pytest.raises(ValueError, match="max_q"):
        m355.shared_prefix_attn(q, c.k, c.v, c.tables, torch.tensor(c.ctx, dtype=torch.int32), prefix_len=0, max_ctx=32, scale=0.1, seq_starts=st)


def test_validate_eviction_reads_shared_pages_through_row_0():
    """Leading entries of the other rows may be padding or stale: a destination page of the same number is free.  Pages that
    are shared, or hold a sequence's own tokens, or are handed out twice, are not."""
    from gpt_oss_vllm_amd.layer import validate_eviction
    kc = torch.zeros((12, 16, 1, 64), dtype=F16)
    src = torch.tensor([[7, 8, 3, 4], [0, 5, 1, 2], [9, 9, 9, 9]], dtype=torch.int32)     # prefix: pages 7 and 8
    lens = torch.tensor([60, 64, 20], dtype=torch.int32)                                   # the third ends inside the prefix
    dst = torch.tensor([[7, 8, 0], [7, 8, 5], [7, 8, 9]], dtype=torch.int32)
    validate_eviction(src, lens, dst, kc, keep=10, prefix_len=32)
    for row, page, why in ((0, 7, "in use"), (0, 8, "in use"), (1, 3, "in use"), (0, 2, "in use"), (1, 0, "in use"), (0, 12, "outside"), (1, -1, "outside")):
        bad = dst.clone()
        bad[row, 2] = page
        with pytest.raises(ValueError, match=why):
            validate_eviction(src, lens, bad, kc, keep=10, prefix_len=32)
    with pytest.raises(ValueError, match="holds 3"):
        validate_eviction(src, lens, dst, kc, keep=17, prefix_len=32)
    validate_eviction(src[:0], lens[:0], dst[:0], kc, keep=10, prefix_len=32)


def test_evict_tokens_takes_every_layer_or_none(monkeypatch, m355):
    """Caches without scores of their own would keep their old rows under the new lengths."""
    from gpt_oss_vllm_amd import layer
    seen = []
    monkeypatch.setattr(m355, "kv_evict", lambda kc, vc, sc, *a, **kw: seen.append((kc, sc)) or (None, "lens"))
    args = dict(keep=4, recent=1, max_ctx=32)
    for caches, scores in (([(1, 1), (2, 2)], [3]), ([(1, 1)], [3, 4]), ([(1, 1)], [])):
        with pytest.raises(ValueError, match="layers"):
            layer.evict_tokens(caches, scores, None, None, None, **args)
    assert not seen
    assert layer.evict_tokens(iter([(1, 1), (2, 2)]), iter([3, 4]), None, None, None, **args) == "lens" and seen == [(1, 3), (2, 4)]


def test_prefill_refuses_half_a_continuation():
    """Prompts that continue a cache name its tables, lengths and bound; without tables the rest would be ignored and the
    prompt attend to itself alone."""
    from gpt_oss_vllm_amd import layer
    lyr = layer.GptOssDecodeLayer.__new__(layer.GptOssDecodeLayer)
    t = torch.zeros((1, 64))
    for kw in (dict(prefix_len=8), dict(max_ctx=9), dict(ctx_lens=t), dict(block_tables=t), dict(block_tables=t, ctx_lens=t), dict(block_tables=t, max_ctx=8)):
        with pytest.raises(ValueError, match="continue a cache"):
            lyr.prefill(t, None, None, None, None, 1, None, None, None, None, **kw)


def _evict_answer(m355, **kw):
    p = 0x10000
    a = dict(kc=p, vc=p, scores=p, tables=p, ctx=p * 2, dst=p, B=4, Hkv=2, row_bytes=128, num_blocks=9, block_size=16, max_blocks=4,
             max_dst=3, stride=16 * 2 * 128, max_ctx=64, prefix=16, keep=32, recent=4, kept=p, new_lens=p * 3)
    a.update(kw)
    return m355.load().m355_kv_evict(*a.values(), None)


def test_kv_evict_refuses_sizes_that_its_counters_do_not_hold(m355):
    """A list of nearly 2^31 entries (its loops would step past the type's end), rows of more than 2^20 bytes (32 of them are
    counted in 16-byte pieces); refused before anything is launched."""
    for kw in (dict(keep=(1 << 31) - 1), dict(keep=(1 << 30) + 1), dict(row_bytes=1 << 30, stride=16 * 2 << 30), dict(row_bytes=(1 << 20) + 16, stride=1 << 30)):
        assert _evict_answer(m355, **kw) == -2, kw


def test_kv_evict_refuses_new_lengths_over_the_old_ones(m355):
    """Every head of a sequence reads the old length while the first one writes the new: they share no entry (B is 4)."""
    for entries in (-3, -1, 0, 1, 3):
        assert _evict_answer(m355, new_lens=0x20000 + 4 * entries) == -2, entries
        assert b"new_lens" in m355.load().m355_last_error()
    assert _evict_answer(m355, new_lens=0x20000 + 16, B=0) == 0


# ---------------------------------------------------------------------------------------------------------------------
# the decoder layer
# ---------------------------------------------------------------------------------------------------------------------
def test_layer_keeps_a_workspace_that_a_graph_was_captured_with(monkeypatch):
    """A larger workspace replaces the layer's, but one that a captured graph writes to stays allocated; one that no graph
    uses is let go."""
    import weakref

    from gpt_oss_vllm_amd import layer
    lyr = layer.GptOssDecodeLayer.__new__(layer.GptOssDecodeLayer)

    class Calls:
        """Stands for the library: every call is a no-op that hands out what forward() asks of it."""
        FLAG_SKIP_COMBINE = 1
        used = None

        def __getattr__(self, name):
            if name.endswith("workspace_bytes"):
                return lambda *a, **kw: self.need
            if name in ("paged_attn_decode", "paged_attn_decode_scored", "shared_prefix_attn"):
                return lambda *a, **kw: setattr(self, "used", kw["workspace"])
            return lambda *a, **kw: None

    lib = Calls()
    t = torch.zeros((1, 64))
    lyr.__dict__.update(dict.fromkeys("h1 resid qkv resid2 h2 ids wts moe_out moe_ws".split(), t), lib=lib, w=dict.fromkeys("ln1 wqkv wo ln2 router_w w13_q w13_absmax w2_q w2_absmax".split()),
                        T=1, Hq=1, Hkv=1, D=64, FF=1, E=1, k=1, H=64, eps=1e-5, window=0, act_mode=0, q=t.view(1, 1, 64), attn=t.view(1, 1, 64))
    lyr.attn_ws = None
    lyr._captured, lyr._outgrown = False, []
    capturing = [False]
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: capturing[0])

    def step(need, **kw):
        lib.need = need
        lyr.forward(t, *[None] * 9, max_ctx=9, **kw)
        assert lib.used is not None and lib.used.numel() >= need
        return weakref.ref(lib.used), lib.used.data_ptr()

    eager, _ = step(100)
    capturing[0] = True
    first, at = step(200, prefix_len=3)
    capturing[0] = False
    lib.used = None
    assert eager() is None                                        # no graph uses it
    second, _ = step(5000, scores=t)
    lib.used = None
    assert first() is not None and first().data_ptr() == at       # the graph goes on writing there
    step(9000, scores=t)
    lib.used = None
    assert second() is None and first() is not None


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["full", "sliding"])
def test_gpu_layer_graphs_outlive_larger_steps(name, m355, cuda):
    """A plain step, one behind a shared prefix and a scored one, captured one after the other with growing needs, eager steps
    that need still more in between, other tensors allocated and filled: every replay gives the eager result and leaves
    those tensors as they are."""
    from gpt_oss_vllm_amd import layer
    from test_layer_ops import _decoder_layer
    B, bs, P, ctx = 3, 16, 96, 201
    lyr, p = _decoder_layer(name, B)
    Hkv, D = p["Hkv"], p["D"]
    blocks = B * 320
    g = torch.Generator().manual_seed(4)
    bt = torch.randperm(blocks, generator=g).view(B, -1).to(torch.int32).to(cuda)          # 320 pages each: contexts of up to 5120
    kc = torch.randn((blocks, bs, Hkv, D), generator=g).to(F16).to(cuda)
    vc = torch.randn((blocks, bs, Hkv, D), generator=g).to(F16).to(cuda)
    cos, sin = (t.to(cuda) for t in layer.rope_tables(8192))
    x = torch.from_numpy(p["x"]).to(cuda)[:B].contiguous()
    pos = torch.full((B,), ctx - 1, dtype=torch.int32, device=cuda)
    slots = bt[:, (ctx - 1) // bs].long() * bs + (ctx - 1) % bs
    lens = torch.full((B,), ctx, dtype=torch.int32, device=cuda)
    scores = torch.zeros((blocks, Hkv, bs), device=cuda)
    forms = [dict(max_ctx=600), dict(max_ctx=1500, prefix_len=P), dict(max_ctx=3000, prefix_len=P, scores=scores)]

    def step(kw):
        scores.zero_()
        r, m = lyr.forward(x, None, pos, slots, bt, lens, kc, vc, cos, sin, **kw)
        return r, m

    def result(kw):
        r, m = step(kw)
        torch.cuda.synchronize()
        return r.clone(), m.clone(), scores.clone()

    graphs, wants = [], []
    for kw in forms:
        wants.append(result(kw))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step(kw)
        graphs.append(graph)
    others = []
    for turn in range(3):
        result(dict(max_ctx=5120 - 16 * (2 - turn), prefix_len=P, scores=scores))            # needs more than any step before
        others += [torch.full((n,), 7.0, device=cuda) for n in (1 << 10, 1 << 14, 1 << 16, 1 << 18, 1 << 20, 1 << 21) for _ in range(4)]
        for graph, want in zip(graphs, wants):
            lyr.resid2.zero_(), lyr.moe_out.zero_()
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            for got, exp in zip((lyr.resid2, lyr.moe_out, scores), want):
                assert torch.equal(got, exp)
        assert all((t == 7.0).all() for t in others)


# ---------------------------------------------------------------------------------------------------------------------
# forms of the kernels that only larger calls take
# ---------------------------------------------------------------------------------------------------------------------
def _scored_check(m355, cuda, c, q, sk, scale, window, max_ctx=None):
    B, P = len(c.ctx), c.prefix
    want, mag, weights = oracle(c, q, [1] * B, scale, sk, window)
    kc, vc, bt, cl = c.device(cuda)
    sc = c.scores.to(cuda)
    rel = score_err(c, q, scale)
    got = m355.paged_attn_decode_scored(q.to(cuda), kc, vc, sc, bt, cl, max_ctx=max_ctx or max(c.ctx), scale=scale, prefix_len=P,
                                        sinks=None if sk is None else sk.to(cuda), window=window)
    check(got, want, mag, c.dtype, rel)
    exp, tol = c.scores.double().clone(), torch.zeros(c.scores.shape, dtype=torch.float64)
    for b in range(B):
        page, off = c.slots(b)
        w = weights[b].t()[P:]
        exp[page[P:], :, off[P:]] += w
        # G weights of relative error rel and their sum, then a rounded addition
        tol[page[P:], :, off[P:]] = (2 * rel + 2.0 ** -23 * (q.shape[1] // c.Hkv)) * w
    tol += 2.0 ** -23 * exp * (tol > 0)
    assert ((sc.cpu().double() - exp).abs() <= tol).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("window", [0, 900])
def test_gpu_scored_batch_of_wide_heads_behind_a_prefix(dtype, window, m355, cuda):
    """128 rows per workgroup over the prefix, heads of 128, beside scored own tokens."""
    own = [1 + 7 * b % 50 for b in range(40)]
    c = Cache(21, [2500 + o for o in own], 4, 128, 16, dtype, prefix=2500, poison=True, window=window)
    q, sk = _inputs(c, 40, 32, 8, True)
    _scored_check(m355, cuda, c, q, sk, 128 ** -0.5, window)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_gpu_scored_many_sequences(dtype, m355, cuda):
    """More than 16384 rows: several rows per wave in the joining, and the weights in the same launch."""
    own = [1 + 13 * b % 305 for b in range(260)]
    c = Cache(22, [800 + o for o in own], 8, 64, 16, dtype, prefix=800, poison=True)
    q, sk = _inputs(c, 260, 64, 9, True)
    _scored_check(m355, cuda, c, q, sk, 0.125, 0)


@pytest.mark.gpu
@pytest.mark.parametrize("heads, D, dtype", [((72, 1), 64, F16), ((130, 1), 64, BF16), ((72, 1), 128, BF16), ((130, 1), 128, F16), ((144, 2), 64, F16)])
@pytest.mark.parametrize("P, own, block, window", [(0, [400, 9, 65], 16, 0), (300, [1800, 1, 700], 20, 0), (4050, [3, 50, 1], 64, 0), (300, [1800, 1, 700], 16, 500)])
def test_gpu_scored_more_than_64_heads_on_one_kv_head(heads, D, dtype, P, own, block, window, m355, cuda):
    """The weights of such a group are added up 64 heads at a time."""
    c = Cache(23, [P + o for o in own], heads[1], D, block, dtype, prefix=P, poison=True, window=window)
    q, sk = _inputs(c, len(own), heads[0], 10, True)
    _scored_check(m355, cuda, c, q, sk, D ** -0.5, window, max_ctx=c.tables.shape[1] * block)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_gpu_many_sequences_of_wide_heads_on_a_long_prefix(dtype, m355, cuda):
    """More than 16384 rows of 128 columns: two rows per wave in the joining."""
    own = [1 + b % 5 for b in range(600)]
    c = Cache(24, [1500 + o for o in own], 8, 128, 16, dtype, prefix=1500, poison=True)
    q, sk = _inputs(c, 600, 32, 11, True)
    want, mag, _ = oracle(c, q, [1] * 600, 128 ** -0.5, sk)
    kc, vc, bt, cl = c.device(cuda)
    got = m355.shared_prefix_attn(q.to(cuda), kc, vc, bt, cl, prefix_len=1500, max_ctx=max(c.ctx), scale=128 ** -0.5, sinks=sk.to(cuda))
    check(got, want, mag, dtype, score_err(c, q, 128 ** -0.5))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_gpu_prompts_of_many_rows_on_a_long_prefix(dtype, m355, cuda):
    """256 rows per workgroup over the prefix, 128 over the prompts' own tokens."""
    n, P = [300, 260], 4101
    c = Cache(25, [P + k for k in n], 8, 64, 16, dtype, prefix=P, poison=True, n=n)
    q, sk = _inputs(c, sum(n), 64, 12, True)
    want, mag, _ = oracle(c, q, n, 0.125, sk)
    kc, vc, bt, cl = c.device(cuda)
    st = torch.tensor([0, 300, 560], dtype=torch.int32, device=cuda)
    got = m355.shared_prefix_attn(q.to(cuda), kc, vc, bt, cl, prefix_len=P, max_ctx=max(c.ctx), scale=0.125, seq_starts=st, max_q=300, sinks=sk.to(cuda))
    check(got, want, mag, dtype, score_err(c, q, 0.125))


@pytest.mark.gpu
def test_gpu_infinite_values_in_a_long_context(m355, cuda):
    """Values that are infinite all along a context of 60000 tokens, far below the key that dominates: looking for them takes
    milliseconds, not a walk per row."""
    L = 60000
    c = Cache(27, [L, 40], 2, 64, 64, F16)
    c.k[..., 0] = 0
    page, off = c.slots(0)
    c.k[page[L - 1], off[L - 1], :, 0] = 60
    c.v[page[:-1], off[:-1], 0, 5] = float("inf")
    c.v[page[::2], off[::2], 1, 9], c.v[page[1::2], off[1::2], 1, 9] = float("inf"), float("-inf")
    q = torch.zeros((2, 64, 64), dtype=F16)
    q[..., 0] = 8
    kc, vc, bt, cl = c.device(cuda)
    args = (q.to(cuda), kc, vc, bt, cl)
    for run in range(2):
        start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        start.record()
        got = m355.shared_prefix_attn(*args, prefix_len=0, max_ctx=L, scale=0.125, workspace=torch.empty(256, dtype=torch.uint8, device=cuda))
        end.record()
        torch.cuda.synchronize()
    assert start.elapsed_time(end) < 500.0
    got = got.cpu()
    assert (got[0, :32, 5] == float("inf")).all() and got[0, 32:, 9].isnan().all()
    got[0, :32, 5] = got[0, 32:, 9] = 0
    assert got.isfinite().all()


# ---------------------------------------------------------------------------------------------------------------------
# a cache of many gigabytes
# ---------------------------------------------------------------------------------------------------------------------
@pytest.mark.gpu
def test_gpu_offsets_past_32_bits(m355, cuda):
    """Pages 2^30 elements apart, K and V of a page in one allocation: element offsets reach 2^32 and more."""
    P, keep = 40, 33
    c = Cache(26, [P + 30, P + 50], 2, 64, 32, F16, prefix=P, dst=0, spare=4)
    used = sorted(set(c.tables[0, :3].tolist() + c.tables[1, 1:3].tolist()))
    free = [p for p in range(c.n) if p not in used][:3]
    stride = 1 << 30
    big = torch.empty((c.n - 1) * stride + (1 << 20), dtype=F16, device=cuda)
    shape, strides = tuple(c.k.shape), (stride, 2 * 64, 64, 1)
    kc, vc = big.as_strided(shape, strides), big.as_strided(shape, strides, 1 << 19)
    kc.copy_(c.k), vc.copy_(c.v)
    assert (c.n - 1) * stride >= 1 << 32
    q, sk = _inputs(c, 2, 16, 13, True)
    want, mag, weights = oracle(c, q, [1, 1], 0.125, sk)
    _, _, bt, cl = c.device(cuda)
    sc = c.scores.to(cuda)
    rel = score_err(c, q, 0.125)
    kw = dict(prefix_len=P, max_ctx=P + 50, scale=0.125, sinks=sk.to(cuda))
    check(m355.shared_prefix_attn(q.to(cuda), kc, vc, bt, cl, **kw), want, mag, F16, rel)
    check(m355.paged_attn_decode_scored(q.to(cuda), kc, vc, sc, bt, cl, **kw), want, mag, F16, rel)
    # the second sequence's tokens behind the first page, to free pages at the far end
    dst = torch.tensor([[c.tables[0, 0], free[0], free[1]], [c.tables[0, 0], free[2], free[0]]], dtype=torch.int32)[1:]
    lens = cl[1:].contiguous()
    scores = sc.clone()
    kept, new = m355.kv_evict(kc, vc, scores, bt[1:].contiguous(), lens, dst.to(cuda), keep=keep, recent=4, prefix_len=32, max_ctx=P + 50)
    assert new.tolist() == [32 + keep]
    for h in range(2):
        src = kept[0, h].cpu().long()
        page, off = c.tables[1].long()[src // 32], src % 32
        to = torch.arange(32, 32 + keep)
        tp, tf = dst[0].long()[to // 32], to % 32
        for cache, first in ((kc, c.k), (vc, c.v)):
            assert torch.equal(cache.cpu()[tp, tf, h], first[page, off, h])
        own = sc.cpu()[c.tables[1].long()[torch.arange(32, P + 50) // 32], h, torch.arange(32, P + 50) % 32]
        best = torch.argsort(own[:-4], descending=True, stable=True)[:keep - 4].sort().values + 32
        assert torch.equal(src, torch.cat([best, torch.arange(P + 46, P + 50)]))
