// Eviction from a paged KV cache by accumulated attention weight: per (sequence, KV head) the last tokens and, of the
// others, those with the largest scores are kept and copied, in order, to other pages.
//
// Two launches.  kv_select: a workgroup per (sequence, KV head) finds the c-th largest score by radix selection (11, 11 and
// 10 bits of an order-preserving integer image of the score, histograms in LDS; the first digit reaches into the mantissa,
// so that scores of one magnitude spread over bins), then lists in order the positions above it and the first of those
// equal to it.  kv_move: a 16-byte piece of a row per lane; reads and writes are whole rows.
#include "common.h"

namespace m355 {

constexpr int EV_THREADS = 256;

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

// Each wave looks after a run of consecutive tokens, 64 of them at a time, so that kept positions come out in order from
// ballots alone.  ITEMS: keys per lane that stay in registers (0: they are read again for every pass).
constexpr int EV_BINS = 2048;
template <int THREADS, int ITEMS>
__global__ __launch_bounds__(THREADS) void kv_select_kernel(EvictArgs a) {
    constexpr int WAVES = THREADS / 64;
    __shared__ int hist[EV_BINS];
    __shared__ int wave_sum_of[WAVES], wave_gt[WAVES], wave_eq[WAVES];
    __shared__ uint32_t sh_prefix;
    __shared__ int sh_left;
    const int hk = blockIdx.x % a.Hkv, b = blockIdx.x / a.Hkv, tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int ctx = min(max(a.ctx_lens[b], 0), a.max_ctx), n = ctx - a.prefix_len;
    int32_t* kept = a.kept + ((int64_t)b * a.Hkv + hk) * a.keep;
    const int m = min(max(n, 0), a.keep);
    if (hk == 0 && tid == 0) a.new_lens[b] = n > 0 ? a.prefix_len + m : ctx;
    for (int i = m + tid; i < a.keep; i += THREADS) kept[i] = -1;
    if (n <= a.keep) {
        for (int i = tid; i < m; i += THREADS) kept[i] = a.prefix_len + i;
        return;
    }
    const int32_t* table = a.tables + (int64_t)b * a.max_blocks;
    const int cand = n - a.recent, c = a.keep - a.recent;   // cand > c: there is something to leave out
    for (int i = tid; i < a.recent; i += THREADS) kept[c + i] = a.prefix_len + cand + i;
    if (c == 0) return;
    const int steps = (cand + THREADS - 1) / THREADS, first = wave * steps * 64 + lane;   // lane's token of step j: first + 64 j
    auto score_at = [&](int i, int page, int blk) {
        const int pos = a.prefix_len + min(i, cand - 1);
        return a.scores[((int64_t)min(max(blk, 0), a.num_blocks - 1) * a.Hkv + hk) * a.block_size + (pos - page * a.block_size)];
    };
    uint32_t key[ITEMS ? ITEMS : 1];
    if constexpr (ITEMS > 0) {
        constexpr int G = ITEMS < 16 ? ITEMS : 16;   // page numbers, then scores on their way at a time
#pragma unroll
        for (int j0 = 0; j0 < ITEMS; j0 += G) {
            if (j0 >= steps) break;
            int page[G], blk[G];
#pragma unroll
            for (int j = 0; j < G; j++) {
                page[j] = page_of(a, a.prefix_len + min(first + 64 * (j0 + j), cand - 1));
                blk[j] = table[page[j]];
            }
#pragma unroll
            for (int j = 0; j < G; j++) key[j0 + j] = score_key(score_at(first + 64 * (j0 + j), page[j], blk[j]));
        }
    }
    auto each = [&](auto f) {   // f(token, key, is it a candidate) for every step of the wave
        if constexpr (ITEMS > 0) {
#pragma unroll
            for (int j = 0; j < ITEMS; j++)
                if (j < steps) f(first + 64 * j, key[j], first + 64 * j < cand);
        } else {
            for (int j = 0; j < steps; j++) {
                const int i = first + 64 * j;
                const int page = page_of(a, a.prefix_len + min(i, cand - 1));
                f(i, score_key(score_at(i, page, table[page])), i < cand);
            }
        }
    };
    uint32_t prefix = 0;   // the leading bits of the c-th largest key, found so far
    int left = c;          // how many of the keys with those leading bits are wanted
#pragma unroll
    for (int pass = 0; pass < 3; pass++) {
        const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, width = pass == 2 ? 10 : 11;
        for (int i = tid; i < EV_BINS; i += THREADS) hist[i] = 0;
        __syncthreads();
        each([&](int, uint32_t k, bool in) {
            if (in && (pass == 0 || (k >> (shift + width)) == (prefix >> (shift + width)))) atomicAdd(&hist[(k >> shift) & ((1 << width) - 1)], 1);
        });
        __syncthreads();
        // the bin of the left-th largest: thread t looks after PER bins, the topmost ones first
        constexpr int PER = EV_BINS / THREADS;
        int mine = 0;
#pragma unroll
        for (int i = 0; i < PER; i++) mine += hist[EV_BINS - 1 - (tid * PER + i)];
        int incl = mine;
#pragma unroll
        for (int o = 1; o < 64; o *= 2) {
            const int v = __shfl_up(incl, o, 64);
            if (lane >= o) incl += v;
        }
        if (lane == 63) wave_sum_of[wave] = incl;
        __syncthreads();
        int above = incl - mine;   // keys in the bins above this thread's
        for (int w = 0; w < wave; w++) above += wave_sum_of[w];
        if (above < left && above + mine >= left) {   // exactly one thread
#pragma unroll
            for (int i = 0; i < PER; i++) {
                const int bin = EV_BINS - 1 - (tid * PER + i), h = hist[bin];
                if (above < left && above + h >= left) {
                    sh_prefix = prefix | ((uint32_t)bin << shift);
                    sh_left = left - above;
                    break;
                }
                above += h;
            }
        }
        __syncthreads();
        prefix = sh_prefix;
        left = sh_left;
    }
    // prefix is the c-th largest key: all above it and the first `left` equal to it
    int gt = 0, eq = 0;
    each([&](int, uint32_t k, bool in) {
        gt += __popcll(__ballot(in && k > prefix));
        eq += __popcll(__ballot(in && k == prefix));
    });
    if (lane == 0) {
        wave_gt[wave] = gt;
        wave_eq[wave] = eq;
    }
    __syncthreads();
    int at = 0, equal = 0;   // kept before this wave; equal ones seen before it
    for (int w = 0; w < wave; w++) {
        at += wave_gt[w];
        equal += wave_eq[w];
    }
    at += min(equal, left);
    auto below = [](uint64_t votes) { return (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(votes >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)votes, 0)); };
    each([&](int i, uint32_t k, bool in) {
        bool take = in && k > prefix;
        const uint64_t eqs = __ballot(in && k == prefix);
        if (eqs && equal < left) take |= in && k == prefix && equal + below(eqs) < left;
        equal += __popcll(eqs);
        const uint64_t takes = __ballot(take);
        if (take) kept[at + below(takes)] = a.prefix_len + i;
        at += __popcll(takes);
    });
}

// A workgroup per (sequence, KV head, EV_ROWS kept tokens).
constexpr int EV_ROWS = 64;
__global__ __launch_bounds__(EV_THREADS) void kv_move_kernel(EvictArgs a, int chunks) {
    const int hk = blockIdx.x % a.Hkv, chunk = blockIdx.x / a.Hkv % chunks, b = blockIdx.x / a.Hkv / chunks, tid = threadIdx.x;
    const int m = a.new_lens[b] - a.prefix_len;
    const int32_t* kept = a.kept + ((int64_t)b * a.Hkv + hk) * a.keep;
    const int32_t* table = a.tables + (int64_t)b * a.max_blocks;
    const int32_t* dst = a.dst_tables + (int64_t)b * a.max_dst_blocks;
    const int pieces = a.row_bytes / 16, i0 = chunk * EV_ROWS, rows = min(EV_ROWS, m - i0);
    for (int w = tid; w < rows * pieces; w += EV_THREADS) {
        const int i = i0 + w / pieces, off = (w % pieces) * 16;
        const int from = kept[i], to = a.prefix_len + i;
        const int fp = page_of(a, from), tp = page_of(a, to);
        const int fb = min(max(table[fp], 0), a.num_blocks - 1), tb = dst[tp];
        if (tb < 0 || tb >= a.num_blocks) continue;
        const int64_t src = fb * a.block_stride + ((int64_t)(from - fp * a.block_size) * a.Hkv + hk) * a.row_bytes + off;
        const int64_t put = tb * a.block_stride + ((int64_t)(to - tp * a.block_size) * a.Hkv + hk) * a.row_bytes + off;
        *reinterpret_cast<u32x4_t*>(a.kc + put) = *reinterpret_cast<const u32x4_t*>(a.kc + src);
        *reinterpret_cast<u32x4_t*>(a.vc + put) = *reinterpret_cast<const u32x4_t*>(a.vc + src);
        if (off == 0)
            a.scores[((int64_t)tb * a.Hkv + hk) * a.block_size + (to - tp * a.block_size)] =
                a.scores[((int64_t)fb * a.Hkv + hk) * a.block_size + (from - fp * a.block_size)];
    }
    if (chunk == 0 && m > 0) {   // the rest of the last page
        const int end = a.prefix_len + m, tp = page_of(a, end - 1), tb = dst[tp];
        if (tb >= 0 && tb < a.num_blocks)
            for (int i = end - tp * a.block_size + tid; i < a.block_size; i += EV_THREADS)
                a.scores[((int64_t)tb * a.Hkv + hk) * a.block_size + i] = 0.f;
    }
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
    if (B < 0 || Hkv <= 0 || row_bytes <= 0 || row_bytes % 16 || num_blocks <= 0 || block_size <= 0 || max_blocks <= 0 || max_dst_blocks <= 0 ||
        max_ctx <= 0 || max_ctx > (1 << 30) || prefix_len < 0 || keep <= 0 || recent < 0 || recent > keep)
        return fail(-2, "m355_kv_evict: unsupported shape B=%d Hkv=%d row_bytes=%d num_blocks=%d block_size=%d max_blocks=%d max_dst_blocks=%d "
                        "max_ctx=%d prefix_len=%d keep=%d recent=%d (need row_bytes %% 16 == 0, keep > 0, 0 <= recent <= keep)",
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
    if (new_lens == ctx_lens) return fail(-2, "m355_kv_evict: new_lens must not be ctx_lens");
    const int64_t chunks = (most + EV_ROWS - 1) / EV_ROWS;
    if ((int64_t)B * Hkv * (chunks + 1) >= (1ll << 30)) return fail(-2, "m355_kv_evict: unsupported size B=%d Hkv=%d keep=%d", B, Hkv, keep);
    uint32_t page_mul;
    int page_shift;
    divide_by(block_size, page_mul, page_shift);
    EvictArgs a{(unsigned char*)kcache, (unsigned char*)vcache, scores, block_tables, ctx_lens, dst_tables, B, Hkv, row_bytes, num_blocks,
                block_size, max_blocks, max_dst_blocks, block_stride_bytes, page_mul, page_shift, max_ctx, prefix_len, keep, recent, kept, new_lens};
    hipStream_t st = (hipStream_t)stream;
    const int64_t own = max_ctx - (int64_t)prefix_len;
    if (own <= 1024) kv_select_kernel<256, 4><<<B * Hkv, 256, 0, st>>>(a);
    else if (own <= 16384) kv_select_kernel<1024, 16><<<B * Hkv, 1024, 0, st>>>(a);
    else if (own <= 65536) kv_select_kernel<1024, 64><<<B * Hkv, 1024, 0, st>>>(a);
    else kv_select_kernel<1024, 0><<<B * Hkv, 1024, 0, st>>>(a);
    M355_LAUNCH_CHECK("kv_select_kernel");
    if (chunks) {
        kv_move_kernel<<<(int)(B * Hkv * chunks), EV_THREADS, 0, st>>>(a, (int)chunks);
        M355_LAUNCH_CHECK("kv_move_kernel");
    }
    return 0;
}
