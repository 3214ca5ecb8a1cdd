"""Attention over a shared prefix, decode attention that accumulates token weights, eviction by that weight.

The oracle is the formula in 64 bits, sequence by sequence on the CPU.  Tolerances: an output value is off by the rounding
of its type (half a step, eps/2 relative), by the probabilities' rounding to that type before the second product (another
eps/2 of sum p|v|, whatever their signs), and by the scores' own error: a 32-bit sum of D products of up to SMAX in size
shifts an exponent by at most 2^-23 * D * SMAX, and the exponential and its argument's scaling add a few 2^-23 * SMAX.
"""
import numpy as np
import pytest
import torch

F16, BF16 = torch.float16, torch.bfloat16


class Cache:
    """A paged cache on the CPU with its tables; device() gives the GPU tensors."""

    def __init__(self, seed, ctx, Hkv, D, block, dtype, prefix=0, spare=2, max_blocks=None, dst=0, poison=False, n=None, window=0):
        g = torch.Generator().manual_seed(seed)
        self.g, self.ctx, self.Hkv, self.D, self.block, self.dtype, self.prefix = g, list(ctx), Hkv, D, block, dtype, prefix
        B = len(ctx)
        pages = lambda n: (max(n, 0) + block - 1) // block      # noqa: E731
        first = prefix // block
        need = [max(0, pages(c) - first) for c in ctx]
        dst_pages = max(0, pages(dst) - first) if dst else 0
        total = pages(prefix) + sum(need) + B * dst_pages + spare
        ids = torch.randperm(total, generator=g).tolist()
        shared = [ids.pop() for _ in range(pages(prefix))]
        width = max([pages(prefix)] + [pages(c) for c in ctx] + [1])
        rows = []
        for b in range(B):
            row = shared[:first] + [ids.pop() for _ in range(need[b])]
            if b == 0:
                row = row[:first] + shared[first:] + row[len(shared):]
            rows.append(row + [0] * (width - len(row)))
        if max_blocks:
            rows = [r + [0] * (max_blocks - len(r)) for r in rows]
        self.tables = torch.tensor(rows, dtype=torch.int32)
        self.dst = torch.tensor([shared[:first] + [ids.pop() for _ in range(dst_pages)] for _ in range(B)], dtype=torch.int32)
        self.n = total
        self.k = torch.randn((total, block, Hkv, D), generator=g).to(dtype)
        self.v = torch.randn((total, block, Hkv, D), generator=g).to(dtype)
        self.scores = torch.exp(torch.randn((total, Hkv, block), generator=g))
        self.k_norm = float(self.k.float().norm(dim=-1).max())
        if poison:                 # whatever no query sees holds NaN and infinities
            seen = torch.zeros((total, block), dtype=torch.bool)
            for b in range(B):
                first_query = self.ctx[b] - (n[b] if n else 1)
                page, off = self.slots(b, torch.arange(max(0, first_query - window + 1) if window else 0, max(self.ctx[b], 0)))
                seen[page, off] = True
            junk = torch.tensor([float("nan"), float("inf"), float("-inf"), torch.finfo(dtype).min]).to(dtype)
            for t in (self.k, self.v):
                fill = junk[torch.randint(0, 4, t.shape, generator=g)]
                t[~seen] = fill[~seen]

    def slots(self, b, positions=None):
        pos = torch.arange(self.ctx[b]) if positions is None else positions
        page = torch.where(pos < self.prefix, self.tables[0].long()[pos // self.block], self.tables[b].long()[pos // self.block])
        return page, pos % self.block

    def device(self, cuda):
        return self.k.to(cuda), self.v.to(cuda), self.tables.to(cuda), torch.tensor(self.ctx, dtype=torch.int32, device=cuda)


def oracle(c, q, n, scale, sinks=None, window=0):
    """(out [T][Hq][D], sum p|v| of the same shape, own weights: list of [Hkv][ctx]) in 64 bits."""
    T, Hq, D = q.shape
    G = Hq // c.Hkv
    out, mag, weights = torch.zeros((T, Hq, D), dtype=torch.float64), torch.zeros((T, Hq, D), dtype=torch.float64), []
    t = 0
    for b, nb in enumerate(n):
        ctx = c.ctx[b]
        page, off = c.slots(b)
        k, v = c.k[page, off].double(), c.v[page, off].double()
        w = torch.zeros((c.Hkv, max(ctx, 0)), dtype=torch.float64)
        for j in range(nb):
            pos = ctx - nb + j
            lo = max(0, pos - window + 1) if window else 0
            for h in range(Hq):
                if pos < lo:
                    continue
                s = (k[lo:pos + 1, h // G] @ q[t + j, h].double()) * scale
                m = s.max() if sinks is None else torch.maximum(s.max(), sinks[h].double())
                e = torch.exp(s - m)
                den = e.sum() + (0 if sinks is None else torch.exp(sinks[h].double() - m))
                p = e / den
                out[t + j, h] = p @ v[lo:pos + 1, h // G]
                mag[t + j, h] = p @ v[lo:pos + 1, h // G].abs()
                w[h // G, lo:pos + 1] += p
        weights.append(w)
        t += nb
    return out, mag, weights


def score_err(c, q, scale):
    """Relative error of a probability, from the scores' rounding: see the module's docstring."""
    smax = float(scale * q.float().norm(dim=-1).max()) * c.k_norm * 1.4427
    return 2.0 ** -23 * (q.shape[-1] + 8) * max(smax, 1.0)


def check(got, want, mag, dtype, rel):
    half = torch.finfo(dtype).eps / 2
    tiny = torch.finfo(dtype).smallest_normal * half           # (fp16 results below the normal range round by a fixed step)
    tol = half * want.abs() + (half + 2 * rel) * mag + 2 * tiny
    err = (got.cpu().double() - want).abs()
    bad = ~(err <= tol)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} values off, worst {float((err / tol).max()):.2f} of the tolerance"


LAYOUTS = [(64, 8, 64, F16), (8, 2, 128, BF16), (6, 2, 64, BF16), (5, 1, 128, F16), (3, 3, 64, F16), (40, 1, 64, F16), (66, 2, 64, BF16)]

# own lengths, prefix, block, window, sinks
DECODE = [
    ([1], 0, 16, 0, False), ([1, 2, 33], 0, 16, 0, True), ([31, 32, 33, 64, 65], 7, 16, 0, False), ([1, 300], 257, 20, 0, True),
    ([5, 1, 17], 1000, 16, 0, True), ([1, 9], 1, 1, 0, False), ([130, 1, 4], 333, 48, 128, True), ([1, 40], 64, 16, 1, False),
    ([1], 2048, 16, 0, True), ([130], 2050, 16, 0, False), ([1], 4096, 32, 0, False), ([1], 8192, 64, 0, True), ([1, 2], 2300, 16, 0, True), ([3], 5800, 16, 0, True),
    # (the line above: 17 to 65 ranges, also numbers of them that a wave's lane groups do not divide)
    ([2, 700, 90], 31, 128, 600, False), ([0, 3, 0], 50, 16, 0, False), ([1, 2], 300, 16, 5, True),
]


def _inputs(c, T, Hq, seed, sinks):
    g = torch.Generator().manual_seed(seed)
    q = (1.5 * torch.randn((T, Hq, c.D), generator=g)).to(c.dtype)
    return q, torch.randn((Hq,), generator=g).to(c.dtype) if sinks else None


@pytest.mark.gpu
@pytest.mark.parametrize("layout", LAYOUTS, ids=lambda x: f"{x[0]}-{x[1]}-{x[2]}-{str(x[3])[6:]}")
@pytest.mark.parametrize("case", range(len(DECODE)))
def test_gpu_shared_prefix_decode(layout, case, m355, cuda):
    """One token per sequence; everything no query sees is NaN or infinite."""
    Hq, Hkv, D, dtype = layout
    own, P, block, window, sinks = DECODE[case]
    c = Cache(100 + case, [P + o for o in own], Hkv, D, block, dtype, prefix=P, poison=True, window=window)
    q, sk = _inputs(c, len(own), Hq, case, sinks)
    scale = D ** -0.5
    want, mag, _ = oracle(c, q, [1] * len(own), scale, sk, window)
    kc, vc, bt, cl = c.device(cuda)
    for max_ctx in (max(c.ctx), c.tables.shape[1] * block):      # the bound may be loose
        got = m355.shared_prefix_attn(q.to(cuda), kc, vc, bt, cl, prefix_len=P, max_ctx=max(max_ctx, 1), scale=scale,
                                      sinks=None if sk is None else sk.to(cuda), window=window)
        check(got, want, mag, dtype, score_err(c, q, scale))


# own lengths, new tokens, prefix, block, window, sinks
EXTEND = [
    ([3], [3], 0, 16, 0, False), ([5, 1, 9, 4], [2, 1, 6, 0], 40, 16, 0, True), ([20, 33, 1], [20, 33, 1], 100, 32, 0, False),
    ([70, 7], [65, 7], 31, 20, 9, True), ([2, 2, 50], [1, 2, 3], 200, 16, 0, False), ([40, 90], [7, 80], 129, 16, 64, True),
]


@pytest.mark.gpu
@pytest.mark.parametrize("layout", LAYOUTS[:6], ids=lambda x: f"{x[0]}-{x[1]}-{x[2]}-{str(x[3])[6:]}")
@pytest.mark.parametrize("case", range(len(EXTEND)))
def test_gpu_shared_prefix_several_tokens(layout, case, m355, cuda):
    """Sequences with none to many new tokens; q is a strided slice, the cache's pages are strided, rows of q behind the
    last sequence leave the output as it was."""
    Hq, Hkv, D, dtype = layout
    own, n, P, block, window, sinks = EXTEND[case]
    c = Cache(300 + case, [P + o for o in own], Hkv, D, block, dtype, prefix=P, poison=True, n=n, window=window)
    T, extra = sum(n), 3
    q, sk = _inputs(c, T + extra, Hq, case, sinks)
    scale = 0.7 * D ** -0.5
    want, mag, _ = oracle(c, q[:T], n, scale, sk, window)
    kv = torch.stack([c.k, c.v], dim=1).to(cuda)                          # K and V of a page side by side
    fused = torch.full((T + extra, (Hq + 3) * D), 7.0, dtype=dtype, device=cuda)
    fused[:, :Hq * D] = q.view(T + extra, -1).to(cuda)
    _, _, bt, cl = c.device(cuda)
    starts = torch.tensor(np.concatenate([[0], np.cumsum(n)]), dtype=torch.int32, device=cuda)
    out = torch.full((T + extra, Hq + 1, D), -3.0, dtype=dtype, device=cuda)
    got = m355.shared_prefix_attn(fused.view(T + extra, Hq + 3, D)[:, :Hq], kv[:, 0], kv[:, 1], bt, cl, prefix_len=P, max_ctx=max(c.ctx),
                                  scale=scale, seq_starts=starts, max_q=max(n), sinks=None if sk is None else sk.to(cuda), window=window,
                                  out=out[:, :Hq])
    check(got[:T], want, mag, dtype, score_err(c, q, scale))
    assert (out[T:] == -3.0).all() and (out[:, Hq:] == -3.0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
def test_gpu_nonfinite_values_reach_only_who_sees_them(dtype, value, m355, cuda):
    """The last of four drafted tokens of one sequence has a value row that is not finite: only its own query, the others'
    formula is untouched; the same in the last prefix token under a window that only the shorter sequence still sees."""
    c = Cache(5, [90, 100], 2, 64, 16, dtype, prefix=64)
    q, _ = _inputs(c, 8, 8, 3, False)
    n = [4, 4]
    want, mag, _ = oracle(c, q, n, 0.125)
    page, off = c.slots(0)
    c.v[page[89], off[89], 1, 5] = value
    kc, vc, bt, cl = c.device(cuda)
    st = torch.tensor([0, 4, 8], dtype=torch.int32, device=cuda)
    got = m355.shared_prefix_attn(q.to(cuda), kc, vc, bt, cl, prefix_len=64, max_ctx=100, scale=0.125, seq_starts=st, max_q=4).cpu()
    hit = torch.zeros(got.shape, dtype=torch.bool)
    hit[3, 4:, 5] = True
    exp = torch.full((), value).to(dtype)
    assert torch.equal(got[hit].isnan(), exp.expand(4).isnan()) and (exp.isnan() or (got[hit] == exp).all())
    check(torch.where(hit, torch.zeros_like(got), got), torch.where(hit, 0.0, want), mag, dtype, score_err(c, q, 0.125))
    # window 30: queries 86..89 of sequence 0 see prefix tokens 57.. / 60.., sequence 1's (96..99) none
    c = Cache(6, [90, 100], 2, 64, 16, dtype, prefix=64)
    want, mag, _ = oracle(c, q, n, 0.125, window=30)
    page, off = c.slots(0)
    c.v[page[58], off[58], 0, 63] = value
    kc, vc, bt, cl = c.device(cuda)
    got = m355.shared_prefix_attn(q.to(cuda), kc, vc, bt, cl, prefix_len=64, max_ctx=100, scale=0.125, seq_starts=st, max_q=4, window=30).cpu()
    hit = torch.zeros(got.shape, dtype=torch.bool)
    hit[:2, :4, 63] = True
    assert (~got[hit].isfinite()).all()
    check(torch.where(hit, torch.zeros_like(got), got), torch.where(hit, 0.0, want), mag, dtype, score_err(c, q, 0.125))


# behind prefixes so long that they are walked once for all, in ranges that are joined
EXTEND_LONG = [
    ([20, 33, 1], [20, 33, 1], 3001, 32, 0, False), ([40, 90], [7, 80], 2500, 20, 600, True), ([3, 1], [3, 1], 4100, 16, 0, True),
    ([40, 600], [2, 3], 1201, 16, 0, False), ([700, 30, 2], [5, 30, 0], 4000, 48, 0, True), ([300, 260], [300, 260], 4101, 16, 0, True),
]


@pytest.mark.gpu
@pytest.mark.parametrize("layout, case", [(x, i) for x in LAYOUTS[:6] for i in range(len(EXTEND_LONG)) if i < 5 or x[0] == 64],
                         ids=lambda x: f"{x[0]}-{x[1]}-{x[2]}-{str(x[3])[6:]}" if isinstance(x, tuple) else str(x))
def test_gpu_several_tokens_behind_a_long_prefix(layout, case, m355, cuda):
    Hq, Hkv, D, dtype = layout
    own, n, P, block, window, sinks = EXTEND_LONG[case]
    c = Cache(700 + case, [P + o for o in own], Hkv, D, block, dtype, prefix=P, poison=True, n=n, window=window)
    T = sum(n)
    q, sk = _inputs(c, T + 2, Hq, case, sinks)
    scale = D ** -0.5
    want, mag, _ = oracle(c, q[:T], n, scale, sk, window)
    kc, vc, bt, cl = c.device(cuda)
    starts = torch.tensor(np.concatenate([[0], np.cumsum(n)]), dtype=torch.int32, device=cuda)
    out = torch.full((T + 2, Hq, D), -3.0, dtype=dtype, device=cuda)
    got = m355.shared_prefix_attn(q.to(cuda), kc, vc, bt, cl, prefix_len=P, max_ctx=max(c.ctx), scale=scale, seq_starts=starts, max_q=max(n),
                                  sinks=None if sk is None else sk.to(cuda), window=window, out=out)
    check(got[:T], want, mag, dtype, score_err(c, q, scale))
    assert (out[T:] == -3.0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_gpu_many_sequences_on_a_long_prefix(dtype, m355, cuda):
    own = [1 + b % 5 for b in range(515)]
    c = Cache(41, [1500 + o for o in own], 8, 64, 16, dtype, prefix=1500, poison=True)
    q, sk = _inputs(c, len(own), 64, 9, True)
    want, mag, _ = oracle(c, q, [1] * len(own), 0.125, sk)
    kc, vc, bt, cl = c.device(cuda)
    got = m355.shared_prefix_attn(q.to(cuda), kc, vc, bt, cl, prefix_len=1500, max_ctx=max(c.ctx), scale=0.125, sinks=sk.to(cuda))
    check(got, want, mag, dtype, score_err(c, q, 0.125))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
def test_gpu_nonfinite_values_behind_a_long_prefix(dtype, value, m355, cuda):
    """An infinite or NaN value of a drafted token, and of a prefix token at a window's end, where the prefix is walked once for
    all: they reach the rows that see them and no other."""
    P, n = 4096, [4, 4]
    c = Cache(15, [P + 26, P + 36], 2, 64, 16, dtype, prefix=P)
    q, _ = _inputs(c, 8, 8, 3, False)
    for window, (pos, head, column), rows, heads in ((0, (P + 25, 1, 5), [3], slice(4, 8)), (3990, (P + 25 - 3990, 0, 63), [0, 1, 2], slice(0, 4))):
        want, mag, _ = oracle(c, q, n, 0.125, window=window)
        page, off = c.slots(0)
        kept = c.v[page[pos], off[pos], head, column].clone()
        c.v[page[pos], off[pos], head, column] = value
        kc, vc, bt, cl = c.device(cuda)
        c.v[page[pos], off[pos], head, column] = kept
        st = torch.tensor([0, 4, 8], dtype=torch.int32, device=cuda)
        got = m355.shared_prefix_attn(q.to(cuda), kc, vc, bt, cl, prefix_len=P, max_ctx=max(c.ctx), scale=0.125, seq_starts=st, max_q=4,
                                      window=window).cpu()
        hit = torch.zeros(got.shape, dtype=torch.bool)
        hit[rows, heads, column] = True
        assert (~got[hit].isfinite()).all()
        check(torch.where(hit, torch.zeros_like(got), got), torch.where(hit, 0.0, want), mag, dtype, score_err(c, q, 0.125))


@pytest.mark.gpu
@pytest.mark.parametrize("P", [9, 5000])
@pytest.mark.parametrize("heads", [(8, 2), (64, 2)])
def test_gpu_more_tokens_than_announced_and_empty_contexts(P, heads, m355, cuda):
    """Tokens behind max_q of their sequence keep what the output held; a query without a key to see gets zeros, with and
    without sinks; nothing else changes."""
    c = Cache(31, [P + 40, P + 3], heads[1], 64, 16, F16, prefix=P, n=[40, 3])
    q, _ = _inputs(c, 43, heads[0], 1, False)
    sk = torch.randn((heads[0],), generator=torch.Generator().manual_seed(2)).to(F16)
    kc, vc, bt, cl = c.device(cuda)
    st = torch.tensor([0, 40, 43], dtype=torch.int32, device=cuda)
    full = m355.shared_prefix_attn(q.to(cuda), kc, vc, bt, cl, prefix_len=P, max_ctx=P + 40, scale=0.125, seq_starts=st, max_q=40)
    out = torch.full_like(full, 5.0)
    m355.shared_prefix_attn(q.to(cuda), kc, vc, bt, cl, prefix_len=P, max_ctx=P + 40, scale=0.125, seq_starts=st, max_q=6, out=out)
    assert (out[6:40] == 5.0).all()
    want, mag, _ = oracle(c, q, [40, 3], 0.125)
    for got in (full, torch.cat([out[:6], full[6:40], out[40:]])):
        check(got, want, mag, F16, score_err(c, q, 0.125))
    for sinks in (None, sk.to(cuda)):
        none = m355.shared_prefix_attn(q[:2].to(cuda), kc, vc, bt, torch.zeros_like(cl), prefix_len=P, max_ctx=P + 40, scale=0.125, sinks=sinks)
        assert (none == 0).all()


SCORED = [([1], 0, 16, 0, False), ([1, 2, 33], 0, 16, 0, True), ([31, 300, 65], 7, 16, 0, False), ([700, 5], 64, 20, 0, True),
          ([260, 900], 0, 64, 200, True), ([3, 40], 33, 16, 2, False), ([0, 4], 48, 16, 0, False), ([1500], 1, 128, 0, False),
          ([2000, 3], 3000, 16, 0, True), ([33, 2100], 15, 16, 700, False), ([200, 150, 7], 50, 20, 90, True)]


@pytest.mark.gpu
@pytest.mark.parametrize("layout", LAYOUTS, ids=lambda x: f"{x[0]}-{x[1]}-{x[2]}-{str(x[3])[6:]}")
@pytest.mark.parametrize("case", range(len(SCORED)))
def test_gpu_scored_decode(layout, case, m355, cuda):
    """Output and accumulated weights; two steps in a row add up; no other score moves; the same bits on another run."""
    Hq, Hkv, D, dtype = layout
    own, P, block, window, sinks = SCORED[case]
    c = Cache(500 + case, [P + o for o in own], Hkv, D, block, dtype, prefix=P, poison=True, window=window)
    q, sk = _inputs(c, len(own), Hq, case, sinks)
    scale = D ** -0.5
    want, mag, weights = oracle(c, q, [1] * len(own), scale, sk, window)
    kc, vc, bt, cl = c.device(cuda)
    rel = score_err(c, q, scale)
    steps = [c.scores.to(cuda), c.scores.to(cuda)]
    for sc in steps:
        for step in (1, 2):
            got = m355.paged_attn_decode_scored(q.to(cuda), kc, vc, sc, bt, cl, max_ctx=max(c.ctx), scale=scale, prefix_len=P,
                                                sinks=None if sk is None else sk.to(cuda), window=window)
            check(got, want, mag, dtype, rel)
            exp, tol = c.scores.double().clone(), torch.zeros(c.scores.shape, dtype=torch.float64)
            for b in range(len(own)):
                page, off = c.slots(b)
                w = weights[b].t()[P:]                                              # [own][Hkv]
                exp[page[P:], :, off[P:]] += step * w
                # every step: G weights of relative error rel and their sums, then a rounded addition
                tol[page[P:], :, off[P:]] = step * (2 * rel + 2.0 ** -23 * (Hq // Hkv)) * w
            tol += 2 * 2.0 ** -23 * exp * (tol > 0)
            err = (sc.cpu().double() - exp).abs()
            assert (err <= tol).all(), f"scores off by up to {float((err - tol).max()):.3g} over the tolerance"
    assert torch.equal(*steps)


EVICT = [([1], 0, 16, 4, 1), ([5, 6, 7], 0, 16, 6, 2), ([100, 300, 129], 32, 16, 64, 10), ([1000, 17], 0, 20, 33, 33),
         ([700, 300], 64, 64, 256, 0), ([4, 2], 16, 16, 1, 0), ([3000, 64], 0, 128, 1025, 100), ([0, 9], 48, 16, 8, 3),
         ([1024, 1025], 0, 16, 500, 1), ([17000, 16384], 64, 64, 3333, 128), ([66000, 1], 0, 128, 4097, 5),
         ([3000, 2001], 40, 20, 700, 7), ([40001, 19000], 0, 64, 10000, 77),
         ([30000, 17], 0, 64, 100, 9), ([70000, 5], 0, 128, 60, 3), ([900, 1000], 32, 16, 520, 40),
         ([4096, 4097, 513], 16, 16, 1500, 64), ([4096, 2050, 1025], 0, 64, 100, 100), ([1100] * 172, 0, 20, 40, 4), ([4000, 600] * 87, 0, 64, 700, 9),
         ([6000, 17001], 40, 20, 700, 7), ([5003, 30], 30, 10, 300, 5), ([7007, 4098], 24, 12, 6001, 1)]


def evict_oracle(c, keep, recent):
    kept, lens = torch.full((len(c.ctx), c.Hkv, keep), -1, dtype=torch.int32), []
    for b, ctx in enumerate(c.ctx):
        n = ctx - c.prefix
        m = min(max(n, 0), keep)
        lens.append(c.prefix + m if n > 0 else ctx)
        page, off = c.slots(b)
        for h in range(c.Hkv):
            s = c.scores[page, h, off].tolist()[c.prefix:]
            last = list(range(max(0, n - recent), n)) if n > keep else []
            rest = [i for i in range(max(n, 0)) if i not in set(last)]
            rest.sort(key=lambda i: (-float("inf") if s[i] != s[i] else s[i], s[i] == s[i], -i), reverse=True)
            pick = sorted(rest[:m - len(last)] + last)
            kept[b, h, :m] = torch.tensor(pick, dtype=torch.int32) + c.prefix
    return kept, lens


def _scores_at(c, kind):
    s = c.scores
    if kind == "ties":
        s = torch.randint(0, 3, s.shape, generator=c.g).float()
    elif kind == "special":
        pool = torch.tensor([float("nan"), float("inf"), -float("inf"), 0.0, -0.0, 1e-42, -1.0, 3.4e38, 1.0])
        s = pool[torch.randint(0, len(pool), s.shape, generator=c.g)]
    elif kind == "close":            # differ in the last bits only
        s = (torch.full(s.shape, 0x3f800000, dtype=torch.int32) + torch.randint(0, 700, s.shape, generator=c.g, dtype=torch.int32)).view(torch.float32)
    c.scores = s.contiguous()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["plain", "ties", "special", "close"])
@pytest.mark.parametrize("case", range(len(EVICT)))
def test_gpu_kv_evict(case, kind, m355, cuda):
    """Kept positions, lengths, moved rows and scores, bit for bit; everything else in the cache stays as it was."""
    own, P, block, keep, recent = EVICT[case]
    Hkv, D, dtype = [(8, 64, F16), (2, 128, BF16), (3, 64, F16)][case % 3]
    c = Cache(700 + case, [P + o for o in own], Hkv, D, block, dtype, prefix=P, dst=P + keep)
    _scores_at(c, kind)
    kept, lens = evict_oracle(c, keep, recent)
    exp = [c.k.clone(), c.v.clone(), c.scores.clone()]
    for b in range(len(own)):
        m = lens[b] - P
        if m <= 0:
            continue
        to = torch.arange(P, P + m)
        tp, tf = c.dst[b].long()[to // block], to % block
        exp[2][tp[-1], :, (P + m - 1) % block + 1:] = 0.0
        for h in range(Hkv):
            page, off = c.slots(b, kept[b, h, :m].long())
            exp[0][tp, tf, h], exp[1][tp, tf, h], exp[2][tp, h, tf] = c.k[page, off, h], c.v[page, off, h], c.scores[page, h, off]
    kc, vc, bt, cl = c.device(cuda)
    dst = c.dst.to(cuda)
    sc = torch.empty(c.scores.numel() + 1, device=cuda)[case % 2:][:c.scores.numel()].view(c.scores.shape)    # (4-byte aligned, too)
    sc.copy_(c.scores)
    for _ in range(2):                          # the source pages stay: a second call does the same again
        got_kept, got_lens = m355.kv_evict(kc, vc, sc, bt, cl, dst, keep=keep, recent=recent, prefix_len=P, max_ctx=max(c.ctx))
        assert torch.equal(got_kept.cpu(), kept)
        assert got_lens.tolist() == lens
        for got, want in zip((kc, vc, sc), exp):
            assert torch.equal(got.cpu().view(torch.int16 if got.element_size() == 2 else torch.int32),
                               want.view(torch.int16 if want.element_size() == 2 else torch.int32))


# ---------------------------------------------------------------------------------------------------------------------
# refusals: checked before anything is launched, so they run without a GPU (the addresses are never dereferenced)
# ---------------------------------------------------------------------------------------------------------------------
PTR = 0x10000


def _attn_args(L, **kw):
    a = dict(q=PTR, kc=PTR, vc=PTR, tables=PTR, ctx=PTR, starts=None, T=4, B=4, max_q=1, Hq=16, Hkv=2, D=64, dtype=0, num_blocks=9,
             block_size=16, max_blocks=4, block_stride=16 * 2 * 64, max_ctx=64, prefix=20, q_stride=1024, o_stride=1024, scale=0.125,
             sinks=None, window=0, ws=PTR, ws_bytes=1 << 40, out=PTR)
    a.update(kw)
    return list(a.values()) + [None]


@pytest.mark.parametrize("bad,code", [
    (dict(q=None), -1), (dict(out=None), -1), (dict(tables=None), -1), (dict(dtype=2), -2), (dict(D=96), -2), (dict(D=0), -2), (dict(Hq=15), -2),
    (dict(Hkv=0), -2), (dict(T=-1), -2), (dict(B=-1), -2), (dict(T=5), -2), (dict(max_q=0), -2), (dict(block_size=0), -2),
    (dict(num_blocks=0), -2), (dict(max_blocks=3), -2), (dict(max_ctx=0), -2), (dict(prefix=-1), -2), (dict(window=-1), -2),
    (dict(block_stride=16 * 2 * 64 - 8), -2), (dict(block_stride=16 * 2 * 64 + 4), -2), (dict(q_stride=1016), -2), (dict(q_stride=1028), -2),
    (dict(o_stride=1000), -2), (dict(q=PTR + 8), -3), (dict(kc=PTR + 2), -3), (dict(ws=None), -6), (dict(ws_bytes=100), -6), (dict(ws=PTR + 4), -3),
    (dict(max_ctx=(1 << 30) + 1, max_blocks=1 << 27), -2), (dict(T=1 << 27, B=1 << 27), -2),
])
def test_shared_prefix_attn_refuses(bad, code, m355):
    L = m355.load()
    assert L.m355_shared_prefix_attn(*_attn_args(L, **bad)) == code
    assert b"m355_shared_prefix_attn" in L.m355_last_error()
    args = _attn_args(L, **bad)
    if args[5] is None and not {"T", "max_q"} & set(bad):        # the scored form has no seq_starts, T and max_q
        scored = args[:3] + [PTR] + args[3:5] + [args[7]] + args[9:]
        assert L.m355_paged_attn_decode_scored(*scored) == code
        assert b"m355_paged_attn_decode_scored" in L.m355_last_error()


def test_shared_prefix_attn_accepts_empty(m355):
    L = m355.load()
    assert L.m355_shared_prefix_attn(*_attn_args(L, T=0, starts=PTR)) == 0
    assert L.m355_shared_prefix_attn(*_attn_args(L, T=0, B=0)) == 0
    assert L.m355_paged_attn_decode_scored(PTR, PTR, PTR, None, PTR, PTR, 4, 16, 2, 64, 0, 9, 16, 4, 2048, 64, 0, 1024, 1024, 0.1, None, 0, PTR,
                                           1 << 40, PTR, None) == -1
    assert m355.shared_prefix_attn_workspace_bytes(0, 4, 1, 16, 2, 64, 100, 0) == 0
    for prefix in (0, 1, 64, 100, 200):
        assert m355.paged_attn_decode_scored_workspace_bytes(4, 16, 2, 64, 100, prefix) >= m355.shared_prefix_attn_workspace_bytes(4, 4, 1, 16, 2, 64, 100, prefix) > 0


@pytest.mark.parametrize("bad,code", [
    (dict(kc=None), -1), (dict(kept=None), -1), (dict(B=-1), -2), (dict(Hkv=0), -2), (dict(row_bytes=24), -2), (dict(row_bytes=0), -2),
    (dict(num_blocks=0), -2), (dict(max_blocks=3), -2), (dict(max_dst=1), -2), (dict(prefix=8), -2), (dict(prefix=-16), -2), (dict(keep=0), -2),
    (dict(recent=-1), -2), (dict(recent=33), -2), (dict(stride=16 * 2 * 128 - 16), -2), (dict(stride=16 * 2 * 128 + 8), -2), (dict(kc=PTR + 8), -3),
    (dict(max_ctx=(1 << 30) + 1, max_blocks=1 << 27), -2), (dict(B=1 << 29), -2), (dict(new_lens=PTR * 2), -2),
])
def test_kv_evict_refuses(bad, code, m355):
    L = m355.load()
    a = dict(kc=PTR, vc=PTR, scores=PTR, tables=PTR, ctx=PTR * 2, dst=PTR, B=4, Hkv=2, row_bytes=128, num_blocks=9, block_size=16, max_blocks=4,
             max_dst=3, stride=16 * 2 * 128, max_ctx=64, prefix=16, keep=32, recent=4, kept=PTR, new_lens=PTR * 3)
    assert L.m355_kv_evict(*dict(a, B=0).values(), None) == 0
    a.update(bad)
    assert L.m355_kv_evict(*a.values(), None) == code
    assert b"m355_kv_evict" in L.m355_last_error()


def test_wrappers_refuse_cpu_tensors(m355):
    c = Cache(1, [20, 30], 2, 64, 16, F16, dst=16)
    cl = torch.tensor(c.ctx, dtype=torch.int32)
    q = torch.zeros((2, 8, 64), dtype=F16)
    with pytest.raises(m355.Mi355LibraryError, match="GPU tensor"):
        m355.shared_prefix_attn(q, c.k, c.v, c.tables, cl, prefix_len=0, max_ctx=32, scale=0.1)
    with pytest.raises(m355.Mi355LibraryError, match="GPU tensor"):
        m355.paged_attn_decode_scored(q, c.k, c.v, c.scores, c.tables, cl, max_ctx=32, scale=0.1)
    with pytest.raises(m355.Mi355LibraryError, match="GPU tensor"):
        m355.kv_evict(c.k, c.v, c.scores, c.tables, cl, c.dst, keep=16, recent=1, max_ctx=32)


# ---------------------------------------------------------------------------------------------------------------------
# the three together, through the decoder layer
# ---------------------------------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("name,P", [("full", 112), ("full", 117), ("sliding", 112), ("sliding", 150)])
def test_gpu_layer_serves_sequences_on_a_shared_prefix(name, P, m355, cuda):
    """A 201-token text whose first P tokens are cached once: three sequences continue it with prompts of different lengths
    (packed, one pass over the shared pages), then take the next token in a decode step; every row against transformers'
    decoder layer.  The decode step adds up the tokens' weights, the caches are trimmed, and another step on the trimmed
    cache equals the formula over the kept tokens."""
    from gpt_oss_vllm_amd import layer
    from test_layer_ops import _decoder_layer, _g
    B, bs, S = 3, 16, 201
    lyr, p = _decoder_layer(name, B)
    Hkv, D = p["Hkv"], p["D"]
    want = _g(f"layer_decoder_rows.{name}.npy")
    x = torch.from_numpy(p["x"]).to(cuda)
    pages = (S + 3 + bs - 1) // bs
    first = P // bs
    n = (pages - first) * (2 * B) + pages + 2
    ids = torch.randperm(n, generator=torch.Generator().manual_seed(P)).tolist()
    shared = [ids.pop() for _ in range(pages)]
    tables = [shared] + [shared[:first] + [ids.pop() for _ in range(pages - first)] for _ in range(B - 1)]
    bt = torch.tensor(tables, dtype=torch.int32, device=cuda)
    # (pages that nobody has written hold NaN)
    kc = torch.full((n, bs, Hkv, D), float("nan"), dtype=F16, device=cuda)
    vc = torch.full_like(kc, float("nan"))
    cos, sin = (t.to(cuda) for t in layer.rope_tables(512))
    slot = lambda b, t: tables[0 if t < P else b][t // bs] * bs + t % bs      # noqa: E731
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=cuda)           # noqa: E731
    i64 = lambda v: torch.tensor(v, dtype=torch.int64, device=cuda)           # noqa: E731
    # the shared tokens, once
    r, m = lyr.prefill(x[:P].contiguous(), None, i32(range(P)), i64([slot(0, t) for t in range(P)]), i32([0, P]), P, kc, vc, cos, sin)
    tol = 5e-3 * np.abs(want).max()
    assert np.abs((r.float() + m.float()).cpu().numpy() - want[:P]).max() <= tol
    # the sequences' own prompts: up to 200, 171 and 160 tokens of the text
    ends = [200, 171, 160]
    toks = [(b, t) for b in range(B) for t in range(P, ends[b])]
    starts = np.concatenate([[0], np.cumsum([e - P for e in ends])])
    r, m = lyr.prefill(torch.stack([x[t] for _, t in toks]), None, i32([t for _, t in toks]), i64([slot(b, t) for b, t in toks]), i32(starts),
                       max(ends) - P, kc, vc, cos, sin, block_tables=bt, ctx_lens=i32(ends), max_ctx=max(ends), prefix_len=P)
    got = (r.float() + m.float()).cpu().numpy()
    assert np.abs(got - want[[t for _, t in toks]]).max() <= tol
    # the next token of each, twice over the same cache: without and with the weights added up
    step = lambda pos, where, tb, ctx, **kw: lyr.forward(torch.stack([x[t] for t in ends]), None, i32(pos), i64(where), tb, i32(ctx), kc, vc,  # noqa: E731
                                                         cos, sin, max_ctx=tb.shape[1] * bs, **kw)
    scores = torch.zeros((n, Hkv, bs), device=cuda)
    where = [slot(b, e) for b, e in enumerate(ends)]
    outs = []
    for sc in (None, scores):
        r, m = step(ends, where, bt, [e + 1 for e in ends], prefix_len=P, scores=sc)
        outs.append((r.float() + m.float()).cpu().numpy())
        assert np.abs(outs[-1] - want[ends]).max() <= tol
    # the weights of a KV head's queries add up to their number, less what the prefix and the sinks took
    total = torch.stack([scores[bt[b].long()].sum(dim=(0, 2)) for b in range(B)]).cpu()
    assert (total > 0).all() and (total < p["Hq"] // Hkv * (1 + 1e-5)).all()
    if P % bs:
        with pytest.raises(m355.Mi355LibraryError, match="multiple of block_size"):
            layer.evict_tokens([(kc, vc)], [scores], bt, i32([e + 1 for e in ends]), bt, keep=20, recent=5, max_ctx=S, prefix_len=P)
        return
    # trim: of every sequence's own tokens 20 remain, 5 of them the last
    keep, recent = 20, 5
    dst = [shared[:first] + [ids.pop() for _ in range((keep + 1 + bs - 1) // bs)] for _ in range(B)]
    dt = i32(dst)
    ctx = i32([e + 1 for e in ends])
    layer.validate_eviction(bt, ctx, dt, kc, keep=keep, prefix_len=P)
    with pytest.raises(ValueError, match="in use"):
        layer.validate_eviction(bt, ctx, bt, kc, keep=keep, prefix_len=P)
    c = Cache.__new__(Cache)                     # the oracle's view of the cache before the call
    c.ctx, c.prefix, c.block, c.Hkv, c.scores, c.tables = [e + 1 for e in ends], P, bs, Hkv, scores.cpu().clone(), bt.cpu()
    kept, lens = evict_oracle(c, keep, recent)
    kept_d, lens_d = m355.kv_evict(kc, vc, scores, bt, ctx, dt, keep=keep, recent=recent, max_ctx=S, prefix_len=P)
    assert torch.equal(kept_d.cpu(), kept) and lens_d.tolist() == lens == [P + keep] * B
    # the step after that: positions go on, slots follow the trimmed lengths.  Against the same layer's formula: the
    # attention over the kept rows in 64 bits on the layer's own q, then the layer's projection
    where = [dst[b][(P + keep) // bs] * bs + (P + keep) % bs for b in range(B)]
    before = scores.clone()
    step([e + 1 for e in ends], where, dt, [P + keep + 1] * B, prefix_len=P, scores=scores)
    c.ctx, c.tables, c.k, c.v, c.D = [P + keep + 1] * B, dt.cpu(), kc.cpu(), vc.cpu(), D
    c.k_norm = float(torch.nan_to_num(c.k.float()).norm(dim=-1).max())
    ref, mag, weights = oracle(c, lyr.q.cpu(), [1] * B, D ** -0.5, lyr.w["sinks"].cpu(), lyr.window)
    check(lyr.attn, ref, mag, F16, score_err(c, lyr.q.cpu(), D ** -0.5))
    moved = scores - before
    for b in range(B):
        page, off = c.slots(b)
        w = weights[b].t()[P:].float()
        assert torch.allclose(moved.cpu()[page[P:], :, off[P:]], w, rtol=1e-3, atol=1e-6)


@pytest.mark.gpu
def test_gpu_capture_and_replay(m355, cuda):
    """Both attentions and the eviction in one captured graph on a stream of its own, replayed with other contents, with eager
    work between the replays, through one workspace; the results of an eager call every time."""
    P, keep = 48, 40
    c = Cache(77, [P + o for o in (300, 41, 7)], 8, 64, 16, F16, prefix=P, dst=P + keep)
    kc, vc, bt, cl = c.device(cuda)
    dst, q = c.dst.to(cuda), torch.empty((3, 64, 64), dtype=F16, device=cuda)
    sc0 = c.scores.to(cuda)
    need = max(m355.shared_prefix_attn_workspace_bytes(3, 3, 1, 64, 8, 64, 350, P), m355.paged_attn_decode_scored_workspace_bytes(3, 64, 8, 64, 350, P))
    ws = torch.empty(need, dtype=torch.uint8, device=cuda)
    kept, lens = torch.empty((3, 8, keep), dtype=torch.int32, device=cuda), torch.empty(3, dtype=torch.int32, device=cuda)
    outs = [torch.empty_like(q) for _ in range(2)]
    caches = [kc.clone(), vc.clone(), sc0.clone()]

    def run():
        m355.shared_prefix_attn(q, caches[0], caches[1], bt, cl, prefix_len=P, max_ctx=350, scale=0.125, workspace=ws, out=outs[0])
        m355.paged_attn_decode_scored(q, caches[0], caches[1], caches[2], bt, cl, prefix_len=P, max_ctx=350, scale=0.125, workspace=ws, out=outs[1])
        m355.kv_evict(*caches, bt, cl, dst, keep=keep, recent=3, prefix_len=P, max_ctx=350, kept=kept, new_lens=lens)

    def load(seed, ctx):
        q.copy_((1.5 * torch.randn(q.shape, generator=torch.Generator().manual_seed(seed))).to(F16))
        cl.copy_(torch.tensor([P + o for o in ctx], dtype=torch.int32))
        for t, s in zip(caches, (kc, vc, sc0)):
            t.copy_(s)

    load(0, (300, 41, 7))
    c.tables = None
    side = torch.cuda.Stream(device=cuda)
    side.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        run()
        torch.cuda.synchronize()
        with torch.cuda.graph(g, stream=side):
            run()
    torch.cuda.synchronize()
    for seed, ctx in ((1, (300, 41, 7)), (2, (256, 40, 1)), (3, (0, 41, 7)), (4, (290, 13, 8))):
        load(seed, ctx)
        run()
        torch.cuda.synchronize()
        want = [t.clone() for t in outs + caches + [kept, lens]]
        load(seed, ctx)
        for t in outs + [kept, lens]:
            t.zero_()
        ws.fill_(255)                    # NaN patterns: nothing is read that the call has not written
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        for got, exp in zip(outs + caches + [kept, lens], want):
            assert torch.equal(got, exp)


@pytest.mark.gpu
def test_gpu_two_streams_and_two_graphs_of_joined_ranges(m355, cuda):
    """Long prefixes and long lists (ranges that are joined, rows that a second launch copies), on two streams at once and as
    two captured graphs replayed at once, each with a workspace of its own: the results of calls one after the other."""
    P, keep, own = 4096, 700, (2000, 900, 7)
    sides = []
    for seed in (1, 2):
        c = Cache(80 + seed, [P + o for o in own], 4, 64, 16, F16, prefix=P, dst=P + keep)
        kc, vc, bt, cl = c.device(cuda)
        q = (1.5 * torch.randn((3, 32, 64), generator=torch.Generator().manual_seed(seed))).to(F16).to(cuda)
        need = max(m355.shared_prefix_attn_workspace_bytes(3, 3, 1, 32, 4, 64, P + 2000, P), m355.paged_attn_decode_scored_workspace_bytes(3, 32, 4, 64, P + 2000, P))
        sides.append(dict(first=[kc, vc, c.scores.to(cuda)], caches=[kc.clone(), vc.clone(), c.scores.to(cuda)], bt=bt, cl=cl, dst=c.dst.to(cuda),
                          q=q, ws=torch.empty(need, dtype=torch.uint8, device=cuda), outs=[torch.empty_like(q) for _ in range(2)],
                          kept=torch.empty((3, 4, keep), dtype=torch.int32, device=cuda), lens=torch.empty(3, dtype=torch.int32, device=cuda),
                          stream=torch.cuda.Stream(device=cuda)))

    def run(s):
        k, v, sc = s["caches"]
        m355.shared_prefix_attn(s["q"], k, v, s["bt"], s["cl"], prefix_len=P, max_ctx=P + 2000, scale=0.125, workspace=s["ws"], out=s["outs"][0])
        m355.paged_attn_decode_scored(s["q"], k, v, sc, s["bt"], s["cl"], prefix_len=P, max_ctx=P + 2000, scale=0.125, workspace=s["ws"], out=s["outs"][1])
        m355.kv_evict(k, v, sc, s["bt"], s["cl"], s["dst"], keep=keep, recent=9, prefix_len=P, max_ctx=P + 2000, kept=s["kept"], new_lens=s["lens"])

    def reset(s):
        for t, f in zip(s["caches"], s["first"]):
            t.copy_(f)
        for t in s["outs"] + [s["kept"], s["lens"]]:
            t.zero_()
        s["ws"].fill_(255)

    def results(s):
        return [t.clone() for t in s["outs"] + s["caches"] + [s["kept"], s["lens"]]]

    want = []
    for s in sides:
        reset(s)
        run(s)
        torch.cuda.synchronize()
        want.append(results(s))
    graphs = []
    for s in sides:
        s["stream"].wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s["stream"]):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=s["stream"]):
                run(s)
            graphs.append(g)
    torch.cuda.synchronize()
    for turn in range(4):
        for s in sides:
            reset(s)
        torch.cuda.synchronize()
        for s, g in zip(sides, graphs):
            with torch.cuda.stream(s["stream"]):
                run(s) if turn % 2 else g.replay()
        torch.cuda.synchronize()
        for s, w in zip(sides, want):
            for got, exp in zip(results(s), w):
                assert torch.equal(got, exp)


@pytest.mark.gpu
def test_gpu_equals_the_paged_decode_kernel(m355, cuda):
    """Without a prefix the new entry point computes what m355_paged_attn_decode_ex computes, and a batch whose rows name the
    shared pages gives the same with and without prefix_len."""
    P = 320
    c = Cache(88, [P + o for o in (1, 200, 33, 90)], 8, 64, 16, F16, prefix=P)
    q, sk = _inputs(c, 4, 64, 5, True)
    kc, vc, bt, cl = c.device(cuda)
    args = (q.to(cuda), kc, vc, bt, cl)
    kw = dict(max_ctx=max(c.ctx), scale=0.125, sinks=sk.to(cuda))
    want, mag, _ = oracle(c, q, [1] * 4, 0.125, sk)
    for got in (m355.paged_attn_decode(*args, **kw), m355.shared_prefix_attn(*args, prefix_len=0, **kw),
                m355.shared_prefix_attn(*args, prefix_len=P, **kw), m355.shared_prefix_attn(*args, prefix_len=P - 5, **kw)):
        check(got, want, mag, F16, score_err(c, q, 0.125))


@pytest.mark.gpu
def test_gpu_bad_pages_stay_inside_the_cache(m355, cuda):
    """Table entries far outside the cache are clamped: sequences with sound tables keep their results, nothing else in the
    pool is written."""
    c = Cache(99, [64, 50], 2, 64, 16, F16, dst=16)
    q, _ = _inputs(c, 2, 8, 1, False)
    kc, vc, bt, cl = c.device(cuda)
    want, mag, _ = oracle(c, q, [1, 1], 0.125)
    bad = bt.clone()
    bad[1] = torch.tensor([1 << 30, -5, -(1 << 31), c.n], dtype=torch.int32)
    sc = c.scores.to(cuda)
    for got in (m355.shared_prefix_attn(q.to(cuda), kc, vc, bad, cl, prefix_len=0, max_ctx=64, scale=0.125),
                m355.paged_attn_decode_scored(q.to(cuda), kc, vc, sc, bad, cl, max_ctx=64, scale=0.125)):
        check(got[:1], want[:1], mag[:1], F16, score_err(c, q, 0.125))
    page, off = c.slots(0)
    rest = torch.ones((c.n, 16), dtype=torch.bool)
    rest[page, off] = False
    assert torch.equal(sc.cpu().transpose(1, 2)[rest], c.scores.transpose(1, 2)[rest])
    dst = torch.full((2, 1), 1 << 20, dtype=torch.int32, device=cuda)
    before = [t.clone() for t in (kc, vc, sc)]
    _, lens = m355.kv_evict(kc, vc, sc, bad, cl, dst, keep=16, recent=2, max_ctx=64)
    assert lens.tolist() == [16, 16] and all(torch.equal(a, b) for a, b in zip((kc, vc, sc), before))


@pytest.mark.gpu
def test_gpu_wrappers_refuse(m355, cuda):
    c = Cache(1, [20, 30], 2, 64, 16, F16, dst=16)
    kc, vc, bt, cl = c.device(cuda)
    sc, q = c.scores.to(cuda), torch.zeros((2, 8, 64), dtype=F16, device=cuda)
    call = lambda **kw: m355.shared_prefix_attn(*[kw.pop(n, d) for n, d in (("q", q), ("kc", kc), ("vc", vc), ("bt", bt), ("cl", cl))],      # noqa: E731
                                                **dict(dict(prefix_len=0, max_ctx=32, scale=0.1), **kw))
    for kw, err in ((dict(q=q.float()), TypeError), (dict(q=q.bfloat16()), TypeError), (dict(kc=kc.bfloat16()), TypeError),
                    (dict(q=q[..., :32].contiguous()), ValueError), (dict(q=q.transpose(0, 1)), ValueError), (dict(kc=kc.transpose(0, 1)), ValueError),
                    (dict(kc=kc[:, :, :, ::2], vc=vc[:, :, :, ::2]), ValueError), (dict(kc=torch.stack([kc, kc], 1)[:, 0]), ValueError),
                    (dict(bt=bt.long()), TypeError), (dict(cl=cl[:1]), ValueError), (dict(sinks=torch.zeros(7, dtype=F16, device=cuda)), ValueError),
                    (dict(sinks=torch.zeros(8, dtype=BF16, device=cuda)), TypeError), (dict(seq_starts=cl), ValueError),
                    (dict(out=torch.zeros((2, 8, 32), dtype=F16, device=cuda)), ValueError), (dict(bt=bt.cpu()), m355.Mi355LibraryError),
                    (dict(workspace=torch.zeros(16, dtype=torch.uint8, device=cuda)), m355.Mi355LibraryError), (dict(max_ctx=1000), m355.Mi355LibraryError)):
        with pytest.raises(err):
            call(**kw)
    for bad in (sc[:, :1], sc.half(), sc.transpose(0, 1)):
        with pytest.raises((ValueError, TypeError)):
            m355.paged_attn_decode_scored(q, kc, vc, bad, bt, cl, max_ctx=32, scale=0.1)
        with pytest.raises((ValueError, TypeError)):
            m355.kv_evict(kc, vc, bad, bt, cl, c.dst.to(cuda), keep=16, recent=1, max_ctx=32)
    with pytest.raises(ValueError):
        m355.kv_evict(kc, vc, sc, bt, cl, c.dst[:1].to(cuda), keep=16, recent=1, max_ctx=32)
    with pytest.raises(m355.Mi355LibraryError, match="new_lens"):
        m355.kv_evict(kc, vc, sc, bt, cl, c.dst.to(cuda), keep=16, recent=1, max_ctx=32, new_lens=cl)
    assert m355.shared_prefix_attn(q[:0], kc, vc, bt[:0], cl[:0], prefix_len=0, max_ctx=32, scale=0.1).shape == (0, 8, 64)
