// Eviction from a paged KV cache by accumulated attention weight: per (sequence, KV head) the last tokens and, of the
// others, those with the largest scores are kept and copied, in order, to other pages.
//
// Two launches.  kv_select: a workgroup per (sequence, KV head) finds the c-th largest score by radix selection (8 bits of
// an order-preserving integer image of the score at a time, histogram in LDS), then lists in order the positions above it
// and the first of those equal to it.  kv_move: a 16-byte piece of a row per lane; reads and writes are whole rows.
#include "common.h"

namespace m355 {

constexpr int EV_THREADS = 256;

struct EvictArgs {
    unsigned char *kc, *vc;
    float* scores;
    const int32_t *tables, *ctx_lens, *dst_tables;
    int B, Hkv, row_bytes, num_blocks, block_size, max_blocks, max_dst_blocks;
    int64_t block_stride;
    int max_ctx, prefix_len, keep, recent;
    int32_t *kept, *new_lens;
};

// Scores in order: NaN first, then -inf .. inf, both zeros alike.
__device__ __forceinline__ uint32_t score_key(float s) {
    if (s != s) return 0u;
    const uint32_t u = __builtin_bit_cast(uint32_t, s + 0.0f);
    return u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
}

// Exclusive prefix sum of a flag over the workgroup's threads, and the total.
__device__ __forceinline__ int wg_rank(bool flag, int* part, int& total) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const uint64_t mask = __ballot(flag);
    const int below = __popcll(mask & ((1ull << lane) - 1));
    __syncthreads();
    if (lane == 0) part[wave] = __popcll(mask);
    __syncthreads();
    int base = 0;
    total = 0;
    for (int w = 0; w < EV_THREADS / 64; w++) {
        if (w < wave) base += part[w];
        total += part[w];
    }
    return base + below;
}

__global__ __launch_bounds__(EV_THREADS) void kv_select_kernel(EvictArgs a) {
    __shared__ int hist[256];
    __shared__ int part[EV_THREADS / 64];
    __shared__ uint32_t sh_prefix;
    __shared__ int sh_left;
    const int hk = blockIdx.x % a.Hkv, b = blockIdx.x / a.Hkv, tid = threadIdx.x;
    const int ctx = min(max(a.ctx_lens[b], 0), a.max_ctx), n = ctx - a.prefix_len;
    int32_t* kept = a.kept + ((int64_t)b * a.Hkv + hk) * a.keep;
    const int m = min(max(n, 0), a.keep);
    if (hk == 0 && tid == 0) a.new_lens[b] = n > 0 ? a.prefix_len + m : ctx;
    for (int i = m + tid; i < a.keep; i += EV_THREADS) kept[i] = -1;
    if (n <= a.keep) {
        for (int i = tid; i < m; i += EV_THREADS) kept[i] = a.prefix_len + i;
        return;
    }
    const int32_t* table = a.tables + (int64_t)b * a.max_blocks;
    const int cand = n - a.recent, c = a.keep - a.recent;   // cand > c: there is something to leave out
    auto key_of = [&](int i) {
        const int pos = a.prefix_len + i, page = pos / a.block_size;
        const int blk = min(max(table[page], 0), a.num_blocks - 1);
        return score_key(a.scores[((int64_t)blk * a.Hkv + hk) * a.block_size + (pos - page * a.block_size)]);
    };
    uint32_t prefix = 0;   // the leading bits of the c-th largest key, found so far
    int left = c;          // how many of the keys with those leading bits are wanted
    if (c > 0) {
        for (int shift = 24; shift >= 0; shift -= 8) {
            for (int i = tid; i < 256; i += EV_THREADS) hist[i] = 0;
            __syncthreads();
            for (int i = tid; i < cand; i += EV_THREADS) {
                const uint32_t k = key_of(i);
                if (shift == 24 || (k >> (shift + 8)) == (prefix >> (shift + 8))) atomicAdd(&hist[(k >> shift) & 255], 1);
            }
            __syncthreads();
            if (tid == 0) {
                int bin = 255, l = left;
                while (bin > 0 && hist[bin] < l) l -= hist[bin--];
                sh_prefix = prefix | ((uint32_t)bin << shift);
                sh_left = l;
            }
            __syncthreads();
            prefix = sh_prefix;
            left = sh_left;
            __syncthreads();
        }
        int done = 0, equal = 0;   // kept so far; of those equal to the c-th largest, seen so far
        for (int i0 = 0; i0 < cand; i0 += EV_THREADS) {
            const int i = i0 + tid;
            const uint32_t k = i < cand ? key_of(i) : 0u;
            const bool eq = i < cand && k == prefix;
            int total;
            const int er = equal + wg_rank(eq, part, total);
            equal += total;
            const bool take = i < cand && (k > prefix || (eq && er < left));
            const int at = done + wg_rank(take, part, total);
            if (take) kept[at] = a.prefix_len + i;
            done += total;
        }
    }
    for (int i = tid; i < a.recent; i += EV_THREADS) kept[c + i] = a.prefix_len + cand + i;
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
        const int fp = from / a.block_size, tp = to / a.block_size;
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
        const int end = a.prefix_len + m, tp = (end - 1) / a.block_size, tb = dst[tp];
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
    EvictArgs a{(unsigned char*)kcache, (unsigned char*)vcache, scores, block_tables, ctx_lens, dst_tables, B, Hkv, row_bytes, num_blocks,
                block_size, max_blocks, max_dst_blocks, block_stride_bytes, max_ctx, prefix_len, keep, recent, kept, new_lens};
    hipStream_t st = (hipStream_t)stream;
    kv_select_kernel<<<B * Hkv, EV_THREADS, 0, st>>>(a);
    M355_LAUNCH_CHECK("kv_select_kernel");
    if (chunks) {
        kv_move_kernel<<<(int)(B * Hkv * chunks), EV_THREADS, 0, st>>>(a, (int)chunks);
        M355_LAUNCH_CHECK("kv_move_kernel");
    }
    return 0;
}
