// Eviction from a paged KV cache by accumulated attention weight: per (sequence, KV head) the last tokens and, of the
// others, those with the largest scores are kept and copied, in order, to other pages.
//
// kv_select: a workgroup per (sequence, KV head) finds the c-th largest score by radix selection (11, 11 and 10 bits of an
// order-preserving integer image of the score, histograms in LDS; the first digit reaches into the mantissa, so that scores of
// one magnitude spread over bins), then lists in order the positions above it and the first of those equal to it.  kv_move: a
// 16-byte piece of a row per lane; reads and writes are whole rows.  A few rows are copied by the selection's workgroup itself.
// What bounds them: the copy by memory (412 MB in 87 us, 4.7 TB/s, of the 5.2 TB/s of a plain copy); a selection by its chain of
// barriers and LDS passes, and over long lists by what one CU reads (16 heads of 300 tokens 7 us, 256 of 4096 11 us, 24 of 65536
// 36 us, of which 10 us for reading and the first histogram, 5 us for the second digit, 3 us for listing the limit's bin, 2 us
// for the low digits, 9 us for counting and writing; 66 us when the keys were read again for every pass).
#include "common.h"

#include <type_traits>

namespace m355 {

constexpr int EV_THREADS = 256;
// Up to so many bytes of K per head, the selection's workgroup copies the kept rows itself, without a second launch.  Measured,
// kernels in one launch / two, us: rows of 128 bytes, 128 of 300 tokens, 16 heads 8.4 / 10.1; of 1000 tokens, 256 heads, 128 rows
// 11.7 / 13.4, 512 rows 20.2 / 21.7; 16 heads, 512 rows 12.3 / 10.8; of 9000 tokens, 32 heads, 512 rows 18.8 / 19.0, 1024 rows
// 24.1 / 19.7.  At the limit few heads lose 1.5 us on the GPU, less than the 2.5 us of the host's time that the second launch
// costs (which a captured graph does not pay); many heads still gain.  The rule does not look at their number.
constexpr int64_t EV_ONE_LAUNCH = 65536;

struct EvictArgs {
    unsigned char *kc, *vc;
    float* scores;
    const int32_t *tables, *ctx_lens, *dst_tables;
    int B, Hkv, row_bytes, num_blocks, block_size, max_blocks, max_dst_blocks;
    int64_t block_stride;
    uint32_t page_mul;
    int page_shift;
    int max_ctx, prefix_len, keep, recent;
    int32_t *kept, *new_lens;
};

// position / block_size
__device__ __forceinline__ int page_of(const EvictArgs& a, int pos) { return (int)(((uint64_t)(uint32_t)pos * a.page_mul) >> a.page_shift); }

// Scores in order: NaN first, then -inf .. inf, both zeros alike.
__device__ __forceinline__ uint32_t score_key(float s) {
    if (s != s) return 0u;
    const uint32_t u = __builtin_bit_cast(uint32_t, s + 0.0f);
    return u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
}

// What a selection works on, and the part of it that needs no selection: lengths, the last tokens, the filler.
struct Selection {
    int cand, c;   // c of the first cand own tokens are to be found
    int32_t* kept;
    const int32_t* table;
};
template <int THREADS>
__device__ __forceinline__ bool begin_selection(const EvictArgs& a, int hk, int b, Selection& s) {
    const int tid = threadIdx.x;
    const int ctx = min(max(a.ctx_lens[b], 0), a.max_ctx), n = ctx - a.prefix_len;
    const int m = min(max(n, 0), a.keep);
    s.kept = a.kept + ((int64_t)b * a.Hkv + hk) * a.keep;
    s.table = a.tables + (int64_t)b * a.max_blocks;
    if (hk == 0 && tid == 0) a.new_lens[b] = n > 0 ? a.prefix_len + m : ctx;
    for (int i = m + tid; i < a.keep; i += THREADS) s.kept[i] = -1;
    if (n <= a.keep) {
        for (int i = tid; i < m; i += THREADS) s.kept[i] = a.prefix_len + i;
        return false;
    }
    s.cand = n - a.recent, s.c = a.keep - a.recent;   // cand > c: there is something to leave out
    for (int i = tid; i < a.recent; i += THREADS) s.kept[s.c + i] = a.prefix_len + s.cand + i;
    return s.c > 0;
}
__device__ __forceinline__ uint32_t key_at(const EvictArgs& a, const Selection& s, int hk, int i) {
    const int pos = a.prefix_len + min(i, s.cand - 1), page = page_of(a, pos), blk = min(max(s.table[page], 0), a.num_blocks - 1);
    return score_key(a.scores[((int64_t)blk * a.Hkv + hk) * a.block_size + (pos - page * a.block_size)]);
}

// f(step, key) for the wave's steps [0, steps) (token first + 64 step), EV_GROUP page numbers and then scores on their way
// at a time.  Steps behind the last one come with step = -1.
constexpr int EV_GROUP = 8;
template <typename F>
__device__ __forceinline__ void each_key(const EvictArgs& a, const Selection& s, int hk, int first, int steps, F f) {
    for (int j0 = 0; j0 < steps; j0 += EV_GROUP) {
        int off[EV_GROUP], blk[EV_GROUP];
        float score[EV_GROUP];
#pragma unroll
        for (int j = 0; j < EV_GROUP; j++) {
            const int pos = a.prefix_len + min(first + 64 * (j0 + j), s.cand - 1), page = page_of(a, pos);
            off[j] = pos - page * a.block_size;
            blk[j] = s.table[page];
        }
#pragma unroll
        for (int j = 0; j < EV_GROUP; j++)
            score[j] = a.scores[((int64_t)min(max(blk[j], 0), a.num_blocks - 1) * a.Hkv + hk) * a.block_size + off[j]];
#pragma unroll
        for (int j = 0; j < EV_GROUP; j++) f(j0 + j < steps ? j0 + j : -1, score_key(score[j]));
    }
}

__device__ __forceinline__ bool aligned_scores(const EvictArgs& a) { return (reinterpret_cast<uintptr_t>(a.scores) & 15) == 0; }

// Copies up to `rows` of the m kept rows from entry i0 on; a thread has EV_AHEAD 16-byte pieces of K and of V on their way.
constexpr int EV_ROWS = 32, EV_AHEAD = 2;
template <int THREADS>
__device__ __forceinline__ void move_rows(const EvictArgs& a, int hk, int b, int m, int i0, int rows) {
    const int tid = threadIdx.x;
    const int32_t* kept = a.kept + ((int64_t)b * a.Hkv + hk) * a.keep;
    const int32_t* table = a.tables + (int64_t)b * a.max_blocks;
    const int32_t* dst = a.dst_tables + (int64_t)b * a.max_dst_blocks;
    const int pieces = a.row_bytes / 16, items = min(rows, m - i0) * pieces;
    for (int w0 = tid; w0 < items; w0 += THREADS * EV_AHEAD) {
        int64_t src[EV_AHEAD], put[EV_AHEAD], score_src[EV_AHEAD], score_put[EV_AHEAD];   // (put < 0: dropped)
        u32x4_t k[EV_AHEAD], v[EV_AHEAD];
        int from[EV_AHEAD], fb[EV_AHEAD], tb[EV_AHEAD];
#pragma unroll
        for (int u = 0; u < EV_AHEAD; u++)   // (clamped: no access leaves the table, whatever became of the scores)
            from[u] = min(max(kept[i0 + min(w0 + u * THREADS, items - 1) / pieces], 0), a.max_ctx - 1);
#pragma unroll
        for (int u = 0; u < EV_AHEAD; u++) {
            fb[u] = table[page_of(a, from[u])];
            tb[u] = dst[page_of(a, a.prefix_len + i0 + min(w0 + u * THREADS, items - 1) / pieces)];
        }
#pragma unroll
        for (int u = 0; u < EV_AHEAD; u++) {
            const int w = min(w0 + u * THREADS, items - 1), off = w % pieces * 16, to = a.prefix_len + i0 + w / pieces;
            const int fo = from[u] - page_of(a, from[u]) * a.block_size, ro = to - page_of(a, to) * a.block_size;
            const int f = min(max(fb[u], 0), a.num_blocks - 1);
            src[u] = f * a.block_stride + ((int64_t)fo * a.Hkv + hk) * a.row_bytes + off;
            k[u] = *reinterpret_cast<const u32x4_t*>(a.kc + src[u]);
            v[u] = *reinterpret_cast<const u32x4_t*>(a.vc + src[u]);
            const bool ok = w0 + u * THREADS < items && tb[u] >= 0 && tb[u] < a.num_blocks;
            put[u] = ok ? tb[u] * a.block_stride + ((int64_t)ro * a.Hkv + hk) * a.row_bytes + off : -1;
            score_src[u] = ((int64_t)f * a.Hkv + hk) * a.block_size + fo;
            score_put[u] = ok && off == 0 ? ((int64_t)tb[u] * a.Hkv + hk) * a.block_size + ro : -1;
        }
#pragma unroll
        for (int u = 0; u < EV_AHEAD; u++) {
            if (put[u] < 0) continue;
            __builtin_nontemporal_store(k[u], reinterpret_cast<u32x4_t*>(a.kc + put[u]));   // (nobody reads them soon)
            __builtin_nontemporal_store(v[u], reinterpret_cast<u32x4_t*>(a.vc + put[u]));
            if (score_put[u] >= 0) a.scores[score_put[u]] = a.scores[score_src[u]];
        }
    }
    if (i0 == 0 && m > 0) {   // the rest of the last page
        const int end = a.prefix_len + m, tp = page_of(a, end - 1), tb = dst[tp];
        if (tb >= 0 && tb < a.num_blocks)
            for (int i = end - tp * a.block_size + tid; i < a.block_size; i += THREADS)
                a.scores[((int64_t)tb * a.Hkv + hk) * a.block_size + i] = 0.f;
    }
}
// The selection's own workgroup copies what it has listed.
template <int THREADS>
__device__ __forceinline__ void move_listed(const EvictArgs& a, int hk, int b) {
    __syncthreads();
    const int n = min(max(a.ctx_lens[b], 0), a.max_ctx) - a.prefix_len, m = min(max(n, 0), a.keep);
    move_rows<THREADS>(a, hk, b, m, 0, m);
}

// The bin of the left-th largest of the values counted in hist[0 .. bins); left becomes its rank within that bin.  Called by
// all threads behind a barrier; ends with one.
template <int THREADS, int BINS>
__device__ __forceinline__ int find_bin(const int* hist, int& left) {
    constexpr int PER = (BINS + THREADS - 1) / THREADS;   // bins per thread, the topmost ones first
    __shared__ int wave_sum_of[THREADS / 64], found[2];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    int mine = 0;
#pragma unroll
    for (int i = 0; i < PER; i++)
        if (tid * PER + i < BINS) mine += hist[BINS - 1 - (tid * PER + i)];
    int incl = mine;
#pragma unroll
    for (int o = 1; o < 64; o *= 2) {
        const int v = __shfl_up(incl, o, 64);
        if (lane >= o) incl += v;
    }
    if (lane == 63) wave_sum_of[wave] = incl;
    __syncthreads();
    int above = incl - mine;   // values in the bins above this thread's
    for (int w = 0; w < wave; w++) above += wave_sum_of[w];
    if (above < left && above + mine >= left) {   // exactly one thread
#pragma unroll
        for (int i = 0; i < PER; i++) {
            const int bin = BINS - 1 - (tid * PER + i), h = hist[bin];
            if (above + h >= left) {
                found[0] = bin;
                found[1] = left - above;
                break;
            }
            above += h;
        }
    }
    __syncthreads();
    left = found[1];
    const int bin = found[0];
    __syncthreads();
    return bin;
}
template <int THREADS>
__device__ __forceinline__ void clear_bins(int* hist, int bins) {
    for (int i = threadIdx.x; i < bins; i += THREADS) hist[i] = 0;
    __syncthreads();
}
__device__ __forceinline__ int lanes_below(uint64_t votes) {
    return (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(votes >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)votes, 0));
}

// Lists in order the candidates above `limit` and the first `left` equal to it.  Each wave looks after a run of consecutive
// tokens, 64 of them at a time, so that positions come out in order from ballots alone; each(f) calls f(token, above, equal)
// for the wave's steps.  Nothing is written behind entry c, whatever another stream does to the scores between the passes.
template <int THREADS, typename EACH>
__device__ __forceinline__ void list_kept(const EvictArgs& a, int32_t* kept, int c, int left, EACH each) {
    __shared__ int wave_gt[THREADS / 64], wave_eq[THREADS / 64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int gt = 0, eq = 0;
    each([&](int, bool above, bool equal) {
        gt += __popcll(__ballot(above));
        eq += __popcll(__ballot(equal));
    });
    if (lane == 0) {
        wave_gt[wave] = gt;
        wave_eq[wave] = eq;
    }
    __syncthreads();
    int at = 0, seen = 0;   // kept before this wave; equal ones seen before it
    for (int w = 0; w < wave; w++) {
        at += wave_gt[w];
        seen += wave_eq[w];
    }
    at += min(seen, left);
    each([&](int i, bool above, bool equal) {
        const uint64_t eqs = __ballot(equal);
        const bool take = above || (equal && seen + lanes_below(eqs) < left);
        seen += __popcll(eqs);
        const uint64_t takes = __ballot(take);
        if (take && at + lanes_below(takes) < c) kept[at + lanes_below(takes)] = a.prefix_len + i;
        at += __popcll(takes);
    });
}

// Up to THREADS * ITEMS own tokens, their keys in registers (ITEMS = 0: any number, keys are read again for every pass).
template <int THREADS, int ITEMS>
__device__ __forceinline__ void select_kept(const EvictArgs& a, int hk, int b) {
    __shared__ int hist[2048];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    Selection s;
    if (!begin_selection<THREADS>(a, hk, b, s)) return;
    const int steps = (s.cand + THREADS - 1) / THREADS, first = wave * steps * 64 + lane;   // lane's token of step j: first + 64 j
    uint32_t key[ITEMS ? ITEMS : 1];
#pragma unroll
    for (int j = 0; j < ITEMS; j++)
        if (j < steps) key[j] = key_at(a, s, hk, first + 64 * j);
    auto each = [&](auto f) {   // f(token, key, is it a candidate) for every step of the wave
        if constexpr (ITEMS > 0) {
#pragma unroll
            for (int j = 0; j < ITEMS; j++)
                if (j < steps) f(first + 64 * j, key[j], first + 64 * j < s.cand);
        } else {
            each_key(a, s, hk, first, steps, [&](int j, uint32_t k) { f(first + 64 * j, k, j >= 0 && first + 64 * j < s.cand); });
        }
    };
    int left = s.c;
    clear_bins<THREADS>(hist, 2048);
    each([&](int, uint32_t k, bool in) {
        if (in) atomicAdd(&hist[k >> 21], 1);
    });
    __syncthreads();
    uint32_t limit = find_bin<THREADS, 2048>(hist, left);
    clear_bins<THREADS>(hist, 2048);
    each([&](int, uint32_t k, bool in) {
        if (in && k >> 21 == limit) atomicAdd(&hist[k >> 10 & 2047], 1);
    });
    __syncthreads();
    limit = limit << 11 | find_bin<THREADS, 2048>(hist, left);
    clear_bins<THREADS>(hist, 1024);
    each([&](int, uint32_t k, bool in) {
        if (in && k >> 10 == limit) atomicAdd(&hist[k & 1023], 1);
    });
    __syncthreads();
    limit = limit << 10 | find_bin<THREADS, 1024>(hist, left);
    list_kept<THREADS>(a, s.kept, s.c, left, [&](auto f) { each([&](int i, uint32_t k, bool in) { f(i, in && k > limit, in && k == limit); }); });
}
template <int THREADS, int ITEMS, bool MOVE>
__global__ __launch_bounds__(THREADS) void kv_select_kernel(EvictArgs a) {
    const int hk = blockIdx.x % a.Hkv, b = blockIdx.x / a.Hkv;
    select_kept<THREADS, ITEMS>(a, hk, b);
    if (MOVE) move_listed<THREADS>(a, hk, b);
}

// Exclusive prefix sum over the wave, and its total.
template <int CTRL, int ROW_MASK = 0xf>
__device__ __forceinline__ int dpp_add(int v) { return v + __builtin_amdgcn_update_dpp(0, v, CTRL, ROW_MASK, 0xf, false); }
__device__ __forceinline__ int wave_scan(int v, int& total) {
    int s = dpp_add<0x111>(v);     // row_shr:1, 2, 4, 8: inclusive sums within 16 lanes
    s = dpp_add<0x112>(s);
    s = dpp_add<0x114>(s);
    s = dpp_add<0x118>(s);
    s = dpp_add<0x142, 0xa>(s);    // row_bcast15 into rows 1 and 3
    s = dpp_add<0x143, 0xc>(s);    // row_bcast31 into rows 2 and 3
    total = __builtin_amdgcn_readlane(s, 63);
    return s - v;
}

// Up to N own tokens: the upper halves of their keys stay in LDS, eight tokens to a lane's 16 bytes, 512 to a wave's block.
// Once the limit's upper half is known, only the few keys that share it are needed whole: each wave lists its own ones in
// order and reads them once more, all together, so that their lower halves are at hand wherever the wave comes across them
// again.  Where equal scores make them too many for the lists, they are read again each time.
constexpr int EV_LONG = 65536, EV_LIST = 256;
template <int N>
__device__ __forceinline__ void select_kept_long(const EvictArgs& a, int hk, int b) {
    constexpr int THREADS = 1024, WAVES = THREADS / 64;
    __shared__ __attribute__((aligned(16))) uint16_t upper[N];
    __shared__ uint16_t list_at[WAVES][EV_LIST], list_low[WAVES][EV_LIST];
    __shared__ int hist[2048], too_many, wave_gt[WAVES], wave_eq[WAVES];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    Selection s;
    if (!begin_selection<THREADS>(a, hk, b, s)) return;
    const int blocks = (s.cand + WAVES * 512 - 1) / (WAVES * 512), run = wave * blocks * 512;   // this wave's first token
    if (tid == 0) too_many = 0;
    clear_bins<THREADS>(hist, 2048);
    {
        // pages of a multiple of 8 (4) tokens: a lane's eight (twice four) scores lie side by side (own tokens start on a page)
        const int side = !aligned_scores(a) ? 1 : a.block_size % 8 == 0 ? 8 : a.block_size % 4 == 0 ? 4 : 1;
        for (int q0 = 0; q0 < blocks; q0 += 4) {
            float sc[4][8];
            auto load = [&](auto parts_c) {   // parts of 8 / parts tokens
                constexpr int PARTS = decltype(parts_c)::value, W = 8 / PARTS;
                int off[4][PARTS], blk[4][PARTS];
#pragma unroll
                for (int q = 0; q < 4; q++)
#pragma unroll
                    for (int h = 0; h < PARTS; h++) {
                        const int i = min(run + (q0 + q) * 512 + lane * 8 + h * W, (s.cand - 1) & ~(W - 1)), pos = a.prefix_len + i;
                        const int page = page_of(a, pos);
                        off[q][h] = pos - page * a.block_size;
                        blk[q][h] = s.table[page];
                    }
#pragma unroll
                for (int q = 0; q < 4; q++)
#pragma unroll
                    for (int e = 0; e < 8; e += 4) {
                        const int h = e / W;
                        const float4_t x = *reinterpret_cast<const float4_t*>(
                            a.scores + ((int64_t)min(max(blk[q][h], 0), a.num_blocks - 1) * a.Hkv + hk) * a.block_size + off[q][h] + e % W);
#pragma unroll
                        for (int c = 0; c < 4; c++) sc[q][e + c] = x[c];
                    }
            };
            if (side == 8) {
                load(std::integral_constant<int, 1>{});
            } else if (side == 4) {
                load(std::integral_constant<int, 2>{});
            } else {
#pragma unroll
                for (int q = 0; q < 4; q++)
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        const int pos = a.prefix_len + min(run + (q0 + q) * 512 + lane * 8 + e, s.cand - 1), page = page_of(a, pos);
                        const int blk = min(max(s.table[page], 0), a.num_blocks - 1);
                        sc[q][e] = a.scores[((int64_t)blk * a.Hkv + hk) * a.block_size + (pos - page * a.block_size)];
                    }
            }
#pragma unroll
            for (int q = 0; q < 4; q++) {
                if (q0 + q >= blocks) break;
                const int i = run + (q0 + q) * 512 + lane * 8;
                u32x4_t packed;
#pragma unroll
                for (int e = 0; e < 8; e += 2) {
                    const uint32_t k0 = score_key(sc[q][e]), k1 = score_key(sc[q][e + 1]);
                    packed[e / 2] = k0 >> 16 | (k1 & 0xffff0000u);
                    if (i + e < s.cand) atomicAdd(&hist[k0 >> 21], 1);
                    if (i + e + 1 < s.cand) atomicAdd(&hist[k1 >> 21], 1);
                }
                if (i < s.cand) *reinterpret_cast<u32x4_t*>(upper + i) = packed;   // (N is a multiple of 8)
            }
        }
    }
    __syncthreads();
    auto each = [&](auto f) {   // f(first token, eight upper halves, how many of them are candidates) for the wave's blocks
        for (int q = 0; q < blocks; q++) {
            const int i = run + q * 512 + lane * 8;
            const u32x4_t u = *reinterpret_cast<const u32x4_t*>(upper + min(i, (s.cand - 1) & ~7));
            f(i, u, min(max(s.cand - i, 0), 8));
        }
    };
    auto half = [](u32x4_t u, int e) { return e & 1 ? u[e / 2] >> 16 : u[e / 2] & 0xffffu; };
    auto equal_to = [&](u32x4_t u, uint32_t t, int n) {
        uint32_t m = 0;
#pragma unroll
        for (int e = 0; e < 8; e++) m |= half(u, e) == t ? 1u << e : 0u;
        return m & ((1u << n) - 1);
    };
    int left = s.c;
    uint32_t top = find_bin<THREADS, 2048>(hist, left);
    clear_bins<THREADS>(hist, 32);
    each([&](int, u32x4_t u, int n) {
#pragma unroll
        for (int e = 0; e < 8; e++)
            if (e < n && half(u, e) >> 5 == top) atomicAdd(&hist[half(u, e) & 31], 1);
    });
    __syncthreads();
    top = top << 5 | find_bin<THREADS, 32>(hist, left);
    int mine = 0;   // of this wave's keys, how many have the limit's upper half
    each([&](int i, u32x4_t u, int n) {
        const uint32_t eq = equal_to(u, top, n);
        if (!__any(eq != 0)) return;
        int total, at = mine + wave_scan(__popc(eq), total);
        for (uint32_t m = eq; m; m &= m - 1, at++)
            if (at < EV_LIST) list_at[wave][at] = (uint16_t)(i - run + __builtin_ctz(m));
        mine += total;
    });
    if (mine > EV_LIST) too_many = 1;
    __syncthreads();
    const bool listed = !too_many;
    if (listed)
        for (int e = lane; e < mine; e += 64) list_low[wave][e] = (uint16_t)key_at(a, s, hk, run + list_at[wave][e]);
    __syncthreads();
    auto each_low = [&](auto f) {   // f(lower half) of every key whose upper half is the limit's
        if (listed) {
            for (int e = lane; e < mine; e += 64) f((uint32_t)list_low[wave][e]);
        } else {
            each([&](int i, u32x4_t u, int n) {
                for (uint32_t m = equal_to(u, top, n); m; m &= m - 1) f(key_at(a, s, hk, i + __builtin_ctz(m)) & 0xffffu);
            });
        }
    };
    clear_bins<THREADS>(hist, 256);
    each_low([&](uint32_t l) { atomicAdd(&hist[l >> 8], 1); });
    __syncthreads();
    uint32_t low = find_bin<THREADS, 256>(hist, left);
    clear_bins<THREADS>(hist, 256);
    each_low([&](uint32_t l) {
        if (l >> 8 == low) atomicAdd(&hist[l & 255], 1);
    });
    __syncthreads();
    low = low << 8 | find_bin<THREADS, 256>(hist, left);

    // f(first token, mask of the eight that lie above the limit, mask of those equal to it)
    auto judged = [&](auto f) {
        int met = 0;
        each([&](int i, u32x4_t u, int n) {
            uint32_t above = 0, equal = 0;
#pragma unroll
            for (int e = 0; e < 8; e++) above |= half(u, e) > top ? 1u << e : 0u;
            above &= (1u << n) - 1;
            const uint32_t eq = equal_to(u, top, n);
            if (__any(eq != 0)) {
                int total, at = met + wave_scan(__popc(eq), total);
                for (uint32_t m = eq; m; m &= m - 1, at++) {
                    const int e = __builtin_ctz(m);
                    const uint32_t l = listed ? (uint32_t)list_low[wave][at] : key_at(a, s, hk, i + e) & 0xffffu;
                    above |= l > low ? 1u << e : 0u;
                    equal |= l == low ? 1u << e : 0u;
                }
                met += total;
            }
            f(i, above, equal);
        });
    };
    int gt = 0, eq = 0;
    judged([&](int, uint32_t above, uint32_t equal) {
        gt += __popc(above);
        eq += __popc(equal);
    });
    int gt_all, eq_all;
    wave_scan(gt, gt_all), wave_scan(eq, eq_all);
    if (lane == 0) {
        wave_gt[wave] = gt_all;
        wave_eq[wave] = eq_all;
    }
    __syncthreads();
    int at = 0, seen = 0;   // kept before this wave; equal ones seen before it
    for (int w = 0; w < wave; w++) {
        at += wave_gt[w];
        seen += wave_eq[w];
    }
    at += min(seen, left);
    judged([&](int i, uint32_t above, uint32_t equal) {
        if (__any(equal != 0)) {   // the first `left` equal ones
            int total, rank = seen + wave_scan(__popc(equal), total);
            for (uint32_t m = equal; m; m &= m - 1, rank++)
                if (rank < left) above |= m & -m;
            seen += total;
        }
        int total;
        int to = at + wave_scan(__popc(above), total);
#pragma unroll
        for (int e = 0; e < 8; e++)
            if (above >> e & 1) {
                if (to < s.c) s.kept[to] = a.prefix_len + i + e;   // (see list_kept)
                to++;
            }
        at += total;
    });
}
template <int N, bool MOVE>
__global__ __launch_bounds__(1024) void kv_select_long_kernel(EvictArgs a) {
    const int hk = blockIdx.x % a.Hkv, b = blockIdx.x / a.Hkv;
    select_kept_long<N>(a, hk, b);
    if (MOVE) move_listed<1024>(a, hk, b);
}

// A workgroup per (sequence, KV head, EV_ROWS kept tokens).
__global__ __launch_bounds__(EV_THREADS) void kv_move_kernel(EvictArgs a, int chunks) {
    const int hk = blockIdx.x % a.Hkv, chunk = blockIdx.x / a.Hkv % chunks, b = blockIdx.x / a.Hkv / chunks;
    move_rows<EV_THREADS>(a, hk, b, a.new_lens[b] - a.prefix_len, chunk * EV_ROWS, EV_ROWS);
}

}  // namespace m355

using namespace m355;

extern "C" int m355_kv_evict(void* kcache, void* vcache, float* scores, const int32_t* block_tables, const int32_t* ctx_lens,
                             const int32_t* dst_tables, int B, int Hkv, int row_bytes, int num_blocks, int block_size, int max_blocks,
                             int max_dst_blocks, int64_t block_stride_bytes, int max_ctx, int prefix_len, int keep, int recent,
                             int32_t* kept, int32_t* new_lens, m355_stream_t stream) {
    if (B == 0) return 0;
    if (!kcache || !vcache || !scores || !block_tables || !ctx_lens || !dst_tables || !kept || !new_lens)
        return fail(-1, "m355_kv_evict: null pointer");
    // (keep: the loops over a list step past it; row_bytes: EV_ROWS rows' pieces are counted in 32 bits)
    if (B < 0 || Hkv <= 0 || row_bytes <= 0 || row_bytes % 16 || row_bytes > (1 << 20) || num_blocks <= 0 || block_size <= 0 || max_blocks <= 0 ||
        max_dst_blocks <= 0 || keep > (1 << 30) || max_ctx <= 0 || max_ctx > (1 << 30) || prefix_len < 0 || keep <= 0 || recent < 0 || recent > keep)
        return fail(-2, "m355_kv_evict: unsupported shape B=%d Hkv=%d row_bytes=%d num_blocks=%d block_size=%d max_blocks=%d max_dst_blocks=%d "
                        "max_ctx=%d prefix_len=%d keep=%d recent=%d (need row_bytes %% 16 == 0, at most 2^20, 0 < keep <= 2^30, 0 <= recent <= keep)",
                    B, Hkv, row_bytes, num_blocks, block_size, max_blocks, max_dst_blocks, max_ctx, prefix_len, keep, recent);
    if (prefix_len % block_size) return fail(-2, "m355_kv_evict: prefix_len %d must be a multiple of block_size %d (its last page stays shared)", prefix_len, block_size);
    if ((int64_t)max_blocks * block_size < max_ctx)
        return fail(-2, "m355_kv_evict: max_ctx %d exceeds max_blocks*block_size %lld", max_ctx, (long long)max_blocks * block_size);
    const int64_t most = max_ctx > prefix_len ? (max_ctx - prefix_len < keep ? max_ctx - prefix_len : keep) : 0;   // rows that a head may keep
    if ((int64_t)max_dst_blocks * block_size < prefix_len + most && most > 0)
        return fail(-2, "m355_kv_evict: prefix_len + keep of %lld tokens exceed max_dst_blocks*block_size %lld", (long long)(prefix_len + most),
                    (long long)max_dst_blocks * block_size);
    if (block_stride_bytes < (int64_t)block_size * Hkv * row_bytes || block_stride_bytes % 16)
        return fail(-2, "m355_kv_evict: a page stride of %lld bytes (need at least block_size*Hkv*row_bytes, a multiple of 16)", (long long)block_stride_bytes);
    if (!aligned(kcache, 16) || !aligned(vcache, 16)) return fail(-3, "m355_kv_evict: caches must be 16-byte aligned");
    if (new_lens < ctx_lens + B && ctx_lens < new_lens + B) return fail(-2, "m355_kv_evict: new_lens must not overlap ctx_lens");
    const int64_t chunks = (most + EV_ROWS - 1) / EV_ROWS;
    if ((int64_t)B * Hkv * (chunks + 1) >= (1ll << 30)) return fail(-2, "m355_kv_evict: unsupported size B=%d Hkv=%d keep=%d", B, Hkv, keep);
    uint32_t page_mul;
    int page_shift;
    divide_by(block_size, page_mul, page_shift);
    EvictArgs a{(unsigned char*)kcache, (unsigned char*)vcache, scores, block_tables, ctx_lens, dst_tables, B, Hkv, row_bytes, num_blocks,
                block_size, max_blocks, max_dst_blocks, block_stride_bytes, page_mul, page_shift, max_ctx, prefix_len, keep, recent, kept, new_lens};
    hipStream_t st = (hipStream_t)stream;
    const int64_t own = max_ctx - (int64_t)prefix_len;
    const bool move = most * row_bytes <= EV_ONE_LAUNCH;
    const int wgs = B * Hkv;
#define M355_EV(KERNEL, THREADS, ...)                                  \
    if (move) KERNEL<__VA_ARGS__, true><<<wgs, THREADS, 0, st>>>(a);   \
    else KERNEL<__VA_ARGS__, false><<<wgs, THREADS, 0, st>>>(a)
    // Keys in registers, eight to each of 512 threads, several workgroups per CU; four to each of 1024 if two of those per CU hold
    // all heads (256 heads of up to 4096 tokens 10.6 us, with 512 threads 13.3; 664 of 1000 26.6 and 16.5; 632 of 3300 29.8 and
    // 18.4).  In LDS beyond: 12.3, 33 and 36.5 us on these.
    if (own <= 4096 && own > 1024 && wgs <= 512) { M355_EV(kv_select_kernel, 1024, 1024, 4); }
    else if (own <= 4096) { M355_EV(kv_select_kernel, 512, 512, 8); }
    else if (own <= 16384) { M355_EV(kv_select_long_kernel, 1024, 16384); }
    else if (own <= EV_LONG) { M355_EV(kv_select_long_kernel, 1024, EV_LONG); }
    else { M355_EV(kv_select_kernel, 1024, 1024, 0); }
#undef M355_EV
    M355_LAUNCH_CHECK("kv_select_kernel");
    if (chunks && !move) {
        kv_move_kernel<<<(int)(B * Hkv * chunks), EV_THREADS, 0, st>>>(a, (int)chunks);
        M355_LAUNCH_CHECK("kv_move_kernel");
    }
    return 0;
}
