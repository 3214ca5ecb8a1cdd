// Attention of new tokens over a paged KV cache whose first `prefix_len` tokens are the same for the whole batch, computed
// once for all, and its single-token form that accumulates every cached token's attention weight.
//
//   o[t][h] = sum_j p_j v_j,   p_j = exp(s_j) / (sum_i exp(s_i) + exp(sink_h)),   s_j = scale * q[t][h] . k_j
//
// over the keys j <= pos(t), j > pos(t) - window, of sequence b(t), whose last n_b positions are its new tokens.  Key j of
// sequence b lies in page block_tables[j < prefix_len ? 0 : b][j / block_size].
//
// The softmax splits over the keys: a workgroup walks one range of keys with a running maximum m and denominator l per
// query row and leaves (m, l, unnormalised o); a merge joins the ranges with the factors exp(m_range - m).  The rows of one
// KV head, (token, query head of the group), are one list: over the prefix the rows of ALL sequences share every K and V
// row that is fetched, over a sequence's own tokens its own rows do.
//   S^T[key][row] = K Q^T    v_mfma_f32_32x32x16: A = K rows from LDS, B = the wave's 32 query rows in registers; a lane
//                            holds one row's scores of 16 keys (lane ^ 32 the other 16).
//   O^T[d][row] += V^T P^T   the probabilities, rounded to the cache's type where they sit (the matrix core takes 16-bit
//                            operands; o and l stay fp32), are the B operand; V^T comes from LDS through the transposing read.
//
// What bounds it.  Own tokens: memory (32 sequences of 2500 tokens, 8 KV heads of 64: 164 MB in 35 us, 4.7 TB/s; a plain copy
// of the card: 5.2).  A walk over a prefix: the chain of one wave per SIMD, products, exponentials and LDS reads behind one
// another (1.0 us per 64 keys of 128 rows, D 64, where the matrix cores need 0.25), so that two workgroups per CU get 1.6 times
// as much done; matrix cores busy for 13 % of the busy CUs' cycles, vector instructions 40 %, waves waiting half of the time (32
// tokens on 8192).  Many rows: vector instructions (about 90 per 32 keys and 32 rows, 16 of them exponentials; 59 % of the busy
// cycles) and products (8; 34 %) almost one after the other, with two waves per SIMD (6 prompts of 150 to 420 tokens behind 8192,
// 226 GFLOP: 317 us, 0.71 PFLOP/s of the 1.2 that a large product reaches).  Tried without gain: 64 keys at a time, a K tile's
// fragments read a tile ahead, four or five tiles in LDS instead of three.  Few tokens: launches (7 us for one, 10 for the ranges
// and their joining).
// Registers: the walks over prefix and own tokens, their two loops and both endings are one kernel.  Heads of 128 use all 256
// vector registers that two waves per SIMD leave and spill 5 to 14 more, the 256-row form 3; every form keeps 48 to 124
// scalar registers in vector lanes.  What that costs has not been measured apart.
#include "common.h"

#include <algorithm>
#include <cmath>
#include <type_traits>

namespace m355 {

constexpr int SA_THREADS = 256;
constexpr int SA_WAVES = SA_THREADS / 64;
constexpr int SA_PAGES = 256;     // entries of a wave's slice of the page table
constexpr float SA_NONE = -0x1p127f;   // "maximum" of a row that has seen no key: below every score, and finite

typedef __bf16 bf16_t;
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x16_t __attribute__((ext_vector_type(16)));
typedef unsigned short ushort2_t __attribute__((ext_vector_type(2)));
typedef float f32x2_t __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
typedef const u32x4_t __attribute__((address_space(3))) sa_lds_u4_t;
typedef __attribute__((address_space(3))) void sa_lds_void_t;
typedef const __attribute__((address_space(1))) void sa_glb_void_t;

struct SharedAttnArgs {
    const void *q, *kc, *vc, *sinks;
    const int32_t *tables, *ctx_lens, *starts;   // starts null: token t is sequence t's only one
    int B, T, Hq, Hkv, G, num_blocks, block_size, max_blocks;
    uint32_t page_mul;
    int page_shift;
    int64_t block_stride, q_stride, o_stride;
    int prefix_len, max_ctx, max_q, window;
    int folded;                                  // prefix tokens that the own walks take along (prefix_len is then 0)
    int direct;                                  // one range in all: its workgroups write the output themselves
    float scale2;                                // |scale| * log2(e): scores are in the units of exp2
    uint32_t q_sign;                             // flips q's signs when scale is negative
    int np, sp, ns, so;                          // ranges over the prefix / the own tokens, and their lengths
    float *part_o, *part_ml;                     // [np + ns][T * Hq][D], [np + ns][T * Hq][2]
    float *logits, *scores;                      // scored form: [B][Hq][lstride], the caller's [num_blocks][Hkv][block_size]
    int lstride;
    void* out;
};

// key / block_size
__device__ __forceinline__ int page_of(const SharedAttnArgs& a, int key) {
    return (int)(((uint64_t)(uint32_t)key * a.page_mul) >> a.page_shift);
}
// What a sequence's row range and positions are.  Everything is clamped to what the arguments allow.
__device__ __forceinline__ int context_of(const SharedAttnArgs& a, int b) { return min(max(a.ctx_lens[b], 0), a.max_ctx); }
struct SeqSpan {
    int t0, n, ctx;   // first token, number of tokens, cached tokens
};
__device__ __forceinline__ SeqSpan seq_span(const SharedAttnArgs& a, int b) {
    SeqSpan s;
    s.ctx = context_of(a, b);
    if (!a.starts) {
        s.t0 = b;
        s.n = 1;
    } else {
        s.t0 = min(max(a.starts[b], 0), a.T);
        s.n = min(max(a.starts[b + 1], s.t0), a.T) - s.t0;
    }
    return s;
}
// The sequence of a token: the last one that starts at or before it; -1 behind the last sequence.
__device__ __forceinline__ int seq_of(const SharedAttnArgs& a, int token) {
    if (!a.starts) return token;
    if (token >= a.starts[a.B]) return -1;
    int lo = 0, hi = a.B - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (a.starts[mid] <= token) lo = mid;
        else hi = mid - 1;
    }
    return a.starts[lo] <= token ? lo : -1;
}
// (positions may be negative and a window as large as the type: no difference is formed that leaves it)
__device__ __forceinline__ int window_lo(const SharedAttnArgs& a, int pos) {
    return a.window > 0 && pos >= a.window ? pos - a.window + 1 : 0;
}

// Wave-wide minimum with DPP only (lanes that a step leaves out combine with themselves).
template <int CTRL, int ROW_MASK = 0xf>
__device__ __forceinline__ int dpp_min(int v) { return min(v, __builtin_amdgcn_update_dpp(v, v, CTRL, ROW_MASK, 0xf, false)); }
__device__ __forceinline__ int wave_min_i(int v) {
    v = dpp_min<0xB1>(v);          // quad_perm [1,0,3,2]
    v = dpp_min<0x4E>(v);          // quad_perm [2,3,0,1]
    v = dpp_min<0x141>(v);         // row_half_mirror
    v = dpp_min<0x140>(v);         // row_mirror: every lane holds its 16 lanes' minimum
    v = dpp_min<0x142, 0xa>(v);    // row_bcast15 into rows 1 and 3
    v = dpp_min<0x143, 0xc>(v);    // row_bcast31 into rows 2 and 3
    return __builtin_amdgcn_readlane(v, 63);
}

template <typename E>
__device__ __forceinline__ f32x16_t mma(u32x4_t a, u32x4_t b, f32x16_t c) {
    if constexpr (sizeof(E) == 2 && __is_same(E, half_t))
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8_t, a), __builtin_bit_cast(half8_t, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
}

// Which 16-bit elements of a fragment are infinite or NaN: all exponent bits set.  `plus` / `minus` receive 1 where the
// element is +inf / -inf (both where it is NaN), `clean` the element or 0.
template <typename E>
__device__ __forceinline__ bool split_nonfinite(u32x4_t v, u32x4_t& clean, u32x4_t& plus, u32x4_t& minus) {
    constexpr uint32_t EXP = __is_same(E, half_t) ? 0x7c00u : 0x7f80u, ONE = __is_same(E, half_t) ? 0x3c00u : 0x3f80u;
    bool any = false;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        uint32_t c = 0, p = 0, n = 0;
#pragma unroll
        for (int sh = 0; sh < 32; sh += 16) {
            const uint32_t e = (v[i] >> sh) & 0xffffu;
            const bool bad = (e & EXP) == EXP, nan = bad && (e & 0x7fffu) != EXP;
            any |= bad;
            c |= (bad ? 0u : e) << sh;
            p |= (bad && (nan || e < 0x8000u) ? ONE : 0u) << sh;
            n |= (bad && (nan || e >= 0x8000u) ? ONE : 0u) << sh;
        }
        clean[i] = c, plus[i] = p, minus[i] = n;
    }
    return any;
}

// Two probabilities rounded to the cache's type (to nearest even), packed; `sum` takes them on as they were rounded.
template <typename E>
__device__ __forceinline__ uint32_t pack_p(float p0, float p1, float& sum) {
    if constexpr (__is_same(E, half_t)) {
        const half2_t ph = __builtin_convertvector(f32x2_t{p0, p1}, half2_t);
        sum = __builtin_amdgcn_fdot2(ph, half2_t{(half_t)1.0f, (half_t)1.0f}, sum, false);
        return __builtin_bit_cast(uint32_t, ph);
    } else {
        const bf16x2_t ph = __builtin_convertvector(f32x2_t{p0, p1}, bf16x2_t);
        sum = __builtin_amdgcn_fdot2_f32_bf16(ph, bf16x2_t{(bf16_t)1.0f, (bf16_t)1.0f}, sum, false);
        return __builtin_bit_cast(uint32_t, ph);
    }
}

// 16-byte chunk c of a tile's row `key` lies at chunk c ^ k_swz (K) or c ^ v_swz (V) of that row: the 32 rows read together
// (K: one chunk of each; V: the transposing read's 4 rows x 64 bytes) then cover every bank.
template <int D>
__device__ __forceinline__ int k_swz(int key) { return D == 64 ? (key >> 1) & 7 : key & 15; }
template <int D>
__device__ __forceinline__ int v_swz(int key) { return (D == 64 ? (key >> 1) & 1 : key & 3) << 2; }

// V^T fragments through the transposing read.  In assembly, waiting for them in the same block: for the builtin the compiler
// waits until every load into LDS in flight has landed, the coming tiles' among them.  `at`: LDS addresses of the 32-column
// pieces, OFF: the 16 keys' offset in the tile; fragment dt is o[2 dt], o[2 dt + 1] (keys + 0 .. 7, + 8 .. 15).
template <int OFF, int ROW>
__device__ __forceinline__ void read_v4(uint32_t a0, uint32_t a1, u32x2_t (&o)[4]) {
    asm volatile(
        "ds_read_b64_tr_b16 %0, %4 offset:%6\n\t"
        "ds_read_b64_tr_b16 %1, %4 offset:%7\n\t"
        "ds_read_b64_tr_b16 %2, %5 offset:%6\n\t"
        "ds_read_b64_tr_b16 %3, %5 offset:%7\n\t"
        "s_waitcnt lgkmcnt(0)"
        : "=&v"(o[0]), "=&v"(o[1]), "=&v"(o[2]), "=&v"(o[3])
        : "v"(a0), "v"(a1), "i"(OFF), "i"(OFF + 8 * ROW)
        : "memory");
}
template <int OFF, int ROW>
__device__ __forceinline__ void read_v8(uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, u32x2_t (&o)[8]) {
    asm volatile(
        "ds_read_b64_tr_b16 %0, %8 offset:%12\n\t"
        "ds_read_b64_tr_b16 %1, %8 offset:%13\n\t"
        "ds_read_b64_tr_b16 %2, %9 offset:%12\n\t"
        "ds_read_b64_tr_b16 %3, %9 offset:%13\n\t"
        "ds_read_b64_tr_b16 %4, %10 offset:%12\n\t"
        "ds_read_b64_tr_b16 %5, %10 offset:%13\n\t"
        "ds_read_b64_tr_b16 %6, %11 offset:%12\n\t"
        "ds_read_b64_tr_b16 %7, %11 offset:%13\n\t"
        "s_waitcnt lgkmcnt(0)"
        : "=&v"(o[0]), "=&v"(o[1]), "=&v"(o[2]), "=&v"(o[3]), "=&v"(o[4]), "=&v"(o[5]), "=&v"(o[6]), "=&v"(o[7])
        : "v"(a0), "v"(a1), "v"(a2), "v"(a3), "i"(OFF), "i"(OFF + 8 * ROW)
        : "memory");
}

// A factor between reference points that never underflows to 0: an infinite or NaN value behind it stays what it is.
__device__ __forceinline__ float factor(float from, float to) { return from == to ? 1.0f : fmaxf(__builtin_amdgcn_exp2f(from - to), 0x1p-149f); }

// The ranges of one row, lane i looking after range i0 + i: does the row see a key of it (else nothing was written), and
// its (m, l).
struct RangeStat {
    bool live;
    float m, l;
};
__device__ __forceinline__ RangeStat range_stat(const SharedAttnArgs& a, int i, int64_t r, int pos, int lo) {
    const int beg = i < a.np ? i * a.sp : a.prefix_len + (i - a.np) * a.so;
    const int end = i < a.np ? min(beg + a.sp, a.prefix_len) : beg + a.so;
    RangeStat s{i < a.np + a.ns && max(beg, lo) < min(end, pos + 1), SA_NONE, 0.f};
    if (s.live) {
        const float* ml = a.part_ml + (i * (int64_t)a.T * a.Hq + r) * 2;
        s.m = ml[0];
        s.l = ml[1];
    }
    return s;
}
template <typename E>
__device__ __forceinline__ void start_with_sink(const SharedAttnArgs& a, int head, float& m, float& den) {
    m = SA_NONE;
    den = 0.f;
    if (a.sinks) {   // one more logit in the denominator
        const float sk = (float)reinterpret_cast<const E*>(a.sinks)[head] * 1.44269504088896341f;
        m = sk > SA_NONE ? sk : SA_NONE;
        den = sk == -INFINITY ? 0.f : sk == sk ? 1.0f : sk;   // (a NaN stays one)
    }
}
// One step of the running (m, den) over the ranges of N neighbouring lanes: returns this lane's factor (0: its range was not
// written).
template <int N>
__device__ __forceinline__ float join_stats(const RangeStat& s, float& m_run, float& den, float& back) {
    float top = s.m;
#pragma unroll
    for (int o = 1; o < N; o *= 2) top = fmaxf(top, __shfl_xor(top, o, 64));
    const float m_new = fmaxf(m_run, top);
    back = factor(m_run, m_new);
    const float f = s.live ? factor(s.m, m_new) : 0.f;
    float part = f * s.l;   // (not written: l is 0)
#pragma unroll
    for (int o = 1; o < N; o *= 2) part += __shfl_xor(part, o, 64);
    den = den * back + part;
    m_run = m_new;
    return f;
}
__device__ __forceinline__ float inverse(float den) { return den > 0.f ? 1.0f / den : den == 0.f ? 0.f : den; }
// Four columns of a row's output (of any alignment).
template <typename E>
__device__ __forceinline__ void put_out(const SharedAttnArgs& a, int token, int head, int D, int c, float4_t num, float inv) {
    E* out = reinterpret_cast<E*>(a.out) + token * a.o_stride + head * D + 4 * c;
#pragma unroll
    for (int i = 0; i < 4; i++) out[i] = (E)(num[i] * inv);
}

// Adds the weights of a sequence's own tokens that its only range has left logits of (from position 0 on); fin: every head's
// maximum and inverse denominator.
__device__ __forceinline__ void add_weights(const SharedAttnArgs& a, int b, int hk, const float (*fin)[2]) {
    const int ctx = context_of(a, b), lo = max(window_lo(a, ctx - 1), a.folded);
    const float* x = a.logits + ((int64_t)b * a.Hq + hk * a.G) * a.lstride;
    for (int rel = lo / 4 * 4 + 4 * (int)threadIdx.x; rel < ctx; rel += 4 * SA_THREADS) {
        float* slot[4];
        float old[4];
#pragma unroll
        for (int u = 0; u < 4; u++) {
            const int key = rel + u;
            slot[u] = nullptr;
            if (key >= ctx || key < lo) continue;
            const int page = page_of(a, key), blk = a.tables[(int64_t)b * a.max_blocks + page];
            if (blk < 0 || blk >= a.num_blocks) continue;   // no score is written outside the cache
            slot[u] = a.scores + ((int64_t)blk * a.Hkv + hk) * a.block_size + (key - page * a.block_size);
            old[u] = *slot[u];
        }
        float4_t w = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
        for (int g = 0; g < a.G; g++) {
            const float4_t v = *reinterpret_cast<const float4_t*>(x + (int64_t)g * a.lstride + rel);
#pragma unroll
            for (int u = 0; u < 4; u++) w[u] += __builtin_amdgcn_exp2f(v[u] - fin[g][0]) * fin[g][1];
        }
#pragma unroll
        for (int u = 0; u < 4; u++)
            if (slot[u]) *slot[u] = old[u] + w[u];
    }
}

// Shape of a workgroup's walk.  RW = 4: every wave holds 32 * QT rows, tiles of 64 keys are shared, NS of them in LDS or on
// their way.  RW = 1: one set of 32 rows, the waves take tiles of 32 keys in turn, each in LDS of its own; a tile is read
// into registers whole, and the next one requested into its place before the softmax.
template <int D, int RW>
struct Walk {
    static constexpr int KT = RW == 4 ? 64 : 32;
    static constexpr int STAGE = 2 * KT * D * 2;                             // bytes: K rows, V rows
    static constexpr int NS = RW == 1 ? 1 : D == 64 ? 3 : 2;
    static constexpr int NI = KT * D * 2 / 1024 / (RW == 4 ? SA_WAVES : 1);  // load instructions of a wave for K (as many for V)
    static constexpr int TILES = NS * STAGE * (RW == 4 ? 1 : SA_WAVES);
    static constexpr int LDS = TILES + SA_WAVES * SA_PAGES * 4;              // and every wave's slice of the page table
};

// The pages of a walk as one list: those of the first `folded` tokens from row 0 of the block tables, then the row's own from
// the page of token `folded` on (which is a second entry for that page if the folded tokens end inside it).
__device__ __forceinline__ int split_page(const SharedAttnArgs& a, int folded) { return folded > page_of(a, folded) * a.block_size ? 1 : 0; }
// A wave's slice of that list from entry `from` on.  Entries behind the row's end repeat its last one, and an entry outside
// the cache is clamped: no access leaves either, whatever the table holds.
template <int D, int RW>
__device__ __forceinline__ void fetch_pages(const SharedAttnArgs& a, unsigned char* smem, const int32_t* table, int from, int folded) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int32_t* pages = reinterpret_cast<int32_t*>(smem + Walk<D, RW>::TILES) + wave * SA_PAGES;
    const int extra = split_page(a, folded), shared_pages = page_of(a, folded) + extra;
    int raw[SA_PAGES / 64];
#pragma unroll
    for (int i = 0; i < SA_PAGES / 64; i++) {
        const int entry = from + 64 * i + lane;
        raw[i] = entry < shared_pages ? a.tables[min(entry, a.max_blocks - 1)] : table[min(entry - extra, a.max_blocks - 1)];
    }
#pragma unroll
    for (int i = 0; i < SA_PAGES / 64; i++) pages[64 * i + lane] = min(max(raw[i], 0), a.num_blocks - 1);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
}

// One workgroup: the rows [row0, row_end) of KV head hk (at most 32 * RW * QT) over the keys [kbeg, kend) of `table`, of
// which those from kfloor on may be read, the first `folded` through row 0.  pos / lo: position and lowest visible key of this
// lane's row(s).  The waves' slices of the page list start with entry pages_from (fetch_pages).  direct: no other range has keys
// of these rows, so the output is written here.
template <typename E, int D, int RW, int QT, bool SCORED>
__device__ __forceinline__ void attend(const SharedAttnArgs& a, unsigned char* smem, int hk, int row0, int row_end, const int (&pos)[QT],
                                       const int (&lo)[QT], const int32_t* table, int pages_from, int kbeg, int kend, int kfloor,
                                       int split, int own_b, int own_k0, int folded, bool direct) {
    typedef Walk<D, RW> W;
    constexpr int KT = W::KT, ROW = D * 2, STEPS = D / 16, DT = D / 32, NI = W::NI, AHEAD = RW == 1 ? 1 : W::NS - 1;
    constexpr int VH = RW == 4 && DT == 4 ? 1 : 2;   // V fragments of how many 16-key halves are held at a time
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int qi = lane & 31, hh = lane >> 5;
    int token[QT], head[QT];
    bool mine[QT];
    u32x4_t qf[QT][STEPS];   // B operand of step s: Q[row][16 s + 8 hh ..]
    int pos_min = INT32_MAX, lo_max = 0;
#pragma unroll
    for (int t = 0; t < QT; t++) {
        const int r = row0 + (RW == 4 ? 32 * (wave * QT + t) : 0) + qi, row = min(r, row_end - 1);
        mine[t] = r < row_end;
        token[t] = row / a.G;
        head[t] = hk * a.G + row % a.G;
        const E* qrow = reinterpret_cast<const E*>(a.q) + token[t] * a.q_stride + head[t] * D + 8 * hh;
#pragma unroll
        for (int s = 0; s < STEPS; s++) {
            qf[t][s] = *reinterpret_cast<const u32x4_t*>(qrow + 16 * s);
            qf[t][s] ^= a.q_sign;   // (a negative scale: scale2 is its magnitude)
        }
        pos_min = min(pos_min, wave_min_i(pos[t]));
        lo_max = max(lo_max, -wave_min_i(-lo[t]));
    }

    unsigned char* tiles = smem + (RW == 4 ? 0 : wave * W::NS * W::STAGE);
    const uint32_t tiles_at = (uint32_t)(uintptr_t)(sa_lds_void_t*)tiles;
    // what this lane loads: chunk `lchunk` of row lrow of the 1024 bytes of each load instruction
    constexpr int RPI = 1024 / ROW, LPR = 64 / RPI;
    const int lrow = lane / LPR, lchunk = lane % LPR;
    auto key_of = [&](int t) { return kbeg + KT * (RW == 4 ? t : wave + SA_WAVES * t); };   // first key of this wave's tile t
    const int nt_all = (kend - kbeg + KT - 1) / KT, nt = RW == 4 ? nt_all : (nt_all - wave + SA_WAVES - 1) / SA_WAVES;
    // The wave's slice of the page table, in LDS: look-ups then do not queue behind the rows' loads (which return in order)
    const int32_t* pages = reinterpret_cast<const int32_t*>(smem + W::TILES) + wave * SA_PAGES;
    // keys outside re-read the nearest one: they are masked below, and rows nobody may see are never read
    auto readable = [&](int key) { return max(min(key, kend - 1), kfloor); };
    const int extra = split_page(a, folded);
    auto entry_of = [&](int key) { return page_of(a, key) + (key >= folded ? extra : 0); };
    auto stage = [&](int t) {
        const int k_first = key_of(t);
        if (entry_of(readable(k_first + KT - 1)) >= pages_from + SA_PAGES) {   // (uniform; a tile spans at most KT + 1 < SA_PAGES pages)
            pages_from = entry_of(readable(k_first));
            fetch_pages<D, RW>(a, smem, table, pages_from, folded);
        }
        const int key = readable(k_first + (lane & (KT - 1))), page = page_of(a, key);   // lane l looks up key l
        const int64_t off = pages[entry_of(key) - pages_from] * a.block_stride + ((int64_t)(key - page * a.block_size) * a.Hkv + hk) * D;
        unsigned char* dst = tiles + (t % W::NS) * W::STAGE + (RW == 4 ? wave * NI * 1024 : 0);
        int64_t src[NI];
#pragma unroll
        for (int i = 0; i < NI; i++) {
            const int row = ((RW == 4 ? wave * NI : 0) + i) * RPI + lrow;
            const uint32_t lo32 = __shfl((int)(uint32_t)off, row, 64), hi32 = __shfl((int)(off >> 32), row, 64);
            src[i] = (int64_t)(((uint64_t)hi32 << 32) | lo32);
        }
#pragma unroll
        for (int i = 0; i < NI; i++) {
            const int row = ((RW == 4 ? wave * NI : 0) + i) * RPI + lrow;
            __builtin_amdgcn_global_load_lds((sa_glb_void_t*)(reinterpret_cast<const E*>(a.kc) + src[i] + ((lchunk ^ k_swz<D>(row)) << 3)),
                                             (sa_lds_void_t*)(dst + i * 1024), 16, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < NI; i++) {
            const int row = ((RW == 4 ? wave * NI : 0) + i) * RPI + lrow;
            __builtin_amdgcn_global_load_lds((sa_glb_void_t*)(reinterpret_cast<const E*>(a.vc) + src[i] + ((lchunk ^ v_swz<D>(row)) << 3)),
                                             (sa_lds_void_t*)(dst + KT * ROW + i * 1024), 16, 0, 0);
        }
    };

    // A fragment of S^T step s: chunk 2 s + hh of key qi's row
    uint32_t kat[STEPS];
#pragma unroll
    for (int s = 0; s < STEPS; s++) kat[s] = qi * ROW + (((2 * s + hh) ^ k_swz<D>(qi)) << 4);
    // V^T: lane 4 ga + gc of a 16-lane group supplies key 4 hh + ga, columns 4 gc .. of its 16; lane i receives column i
    const int ga = (lane & 15) >> 2, gc = lane & 3, vkey = 4 * hh + ga;
    uint32_t vat[DT];
#pragma unroll
    for (int dt = 0; dt < DT; dt++)
        vat[dt] = KT * ROW + vkey * ROW + (((4 * dt + 2 * ((lane >> 4) & 1) + (gc >> 1)) ^ v_swz<D>(vkey)) << 4) + 8 * (gc & 1);

    float m_run[QT], l_run[QT];   // reference point of the exponents; this lane's half of the denominator
    f32x16_t o[QT][DT];
#pragma unroll
    for (int t = 0; t < QT; t++) {
        m_run[t] = SA_NONE;
        l_run[t] = 0.f;
#pragma unroll
        for (int dt = 0; dt < DT; dt++)
#pragma unroll
            for (int i = 0; i < 16; i++) o[t][dt][i] = 0.f;
    }

    // 32 keys from k0 on, whose rows lie at LDS address `base` (K; V behind the tile's K rows).  EDGE: some row does not see
    // some of them.  RW = 1: tile t_next is requested as soon as this one has been read.
    auto step = [&](auto edge_c, int k0, uint32_t base, int t_next) {
        constexpr bool EDGE = decltype(edge_c)::value;
        const f32x16_t zero = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        f32x16_t x[QT];
#pragma unroll
        for (int s = 0; s < STEPS; s++) {
            const u32x4_t kf = *reinterpret_cast<sa_lds_u4_t*>(base + kat[s]);
#pragma unroll
            for (int q = 0; q < QT; q++) x[q] = mma<E>(kf, qf[q][s], s ? x[q] : zero);
        }
        u32x2_t vf[VH][2 * DT];   // (the reads run while the matrix cores form the scores)
        if constexpr (DT == 2) {
            read_v4<0, ROW>(base + vat[0], base + vat[1], vf[0]);
            read_v4<16 * ROW, ROW>(base + vat[0], base + vat[1], vf[1]);
        } else {
            read_v8<0, ROW>(base + vat[0], base + vat[1], base + vat[2], base + vat[3], vf[0]);
            if constexpr (VH == 2) read_v8<16 * ROW, ROW>(base + vat[0], base + vat[1], base + vat[2], base + vat[3], vf[1]);
        }
        if constexpr (RW == 1) {   // (those reads have returned, and K's before them)
            if (t_next < nt) stage(t_next);
        }
        // register i of a lane: key k0 + (i & 3) + 8 (i >> 2) + 4 hh
        uint32_t seen[QT];   // (EDGE) bit i: this row sees register i's key
#pragma unroll
        for (int q = 0; q < QT; q++) {
            if constexpr (EDGE) {
                seen[q] = 0;
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    const int key = k0 + (i & 3) + 8 * (i >> 2) + 4 * hh;
                    const bool ok = key < kend && key <= pos[q] && key >= lo[q];
                    x[q][i] = ok ? x[q][i] : -INFINITY;
                    seen[q] |= ok ? 1u << i : 0u;
                }
            }
            if constexpr (SCORED) {
                if (own_k0 >= 0 && mine[q]) {
                    float* dst = a.logits + ((int64_t)own_b * a.Hq + head[q]) * a.lstride + (k0 - own_k0) + 4 * hh;
#pragma unroll
                    for (int i4 = 0; i4 < 4; i4++)
                        *reinterpret_cast<float4_t*>(dst + 8 * i4) =
                            float4_t{x[q][4 * i4], x[q][4 * i4 + 1], x[q][4 * i4 + 2], x[q][4 * i4 + 3]} * a.scale2;
                }
            }
        }
        // The exponents' reference follows the running maximum lazily: probabilities are formed against the old one, and only
        // if one of them exceeds LIMIT (seen on the packed 16-bit values, whose order is that of whole numbers) do the maximum,
        // the rescaling and the probabilities take another turn: a few times per row instead of a maximum per tile.  The
        // denominator carries the same factor.  fp16 ends at 2^-24 below and 65504 above, so its reference is put 2^LIFT below the
        // maximum: a row's largest probability is held as 2^9 to 2^16, and one that falls out of the normal range is off by at
        // most 2^-34 of the largest (2^-25 with the maximum itself as the reference, which lost thousands of keys 18 nats below
        // one that dominates).  A higher lift leaves less room before the next turn: 2^9 costs nothing, 2^10 1 %, 2^11 4 % (32
        // tokens on 8192, drafted tokens, prompts).  bf16 has the exponents of fp32, its values too: there the reference lies
        // above the maximum, so that no probability exceeds 2^-16 and 65536 of them times the largest finite value still add up
        // to a finite sum.
        uint32_t pb[QT][8];
        float sum[QT];
        auto exponentials = [&] {
            ushort2_t top = {0, 0};
#pragma unroll
            for (int q = 0; q < QT; q++) {
                sum[q] = l_run[q];
#pragma unroll
                for (int i = 0; i < 16; i += 2) {
                    const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(x[q][i], a.scale2, -m_run[q]));
                    const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(x[q][i + 1], a.scale2, -m_run[q]));
                    float rounded = sum[q];
                    pb[q][i >> 1] = pack_p<E>(p0, p1, rounded);
                    // (the accumulated weights are fp32: their denominator sums the unrounded terms)
                    sum[q] = SCORED ? sum[q] + (p0 + p1) : rounded;
                    top = __builtin_elementwise_max(top, __builtin_bit_cast(ushort2_t, pb[q][i >> 1]));
                }
            }
            return top;
        };
        const ushort2_t top = exponentials();
        constexpr uint16_t LIMIT = __is_same(E, half_t) ? 0x7bffu : 0x3780u;   // 65504, 2^-16
        constexpr float LIFT = __is_same(E, half_t) ? 9.f : -28.f;
        if (__any(top[0] > LIMIT || top[1] > LIMIT)) {
#pragma unroll
            for (int q = 0; q < QT; q++) {
                float mx = fmaxf(fmaxf(x[q][0], x[q][1]), x[q][2]);
#pragma unroll
                for (int i = 3; i < 15; i += 2) mx = fmaxf(fmaxf(mx, x[q][i]), x[q][i + 1]);
                mx = fmaxf(cross_half_max(fmaxf(mx, x[q][15])) * a.scale2 - LIFT, m_run[q]);
                const float alpha = __builtin_amdgcn_exp2f(m_run[q] - mx);   // (0 for the first key)
                m_run[q] = mx;
                l_run[q] *= alpha;
#pragma unroll
                for (int dt = 0; dt < DT; dt++)
#pragma unroll
                    for (int i = 0; i < 16; i++) o[q][dt][i] *= alpha;
            }
            exponentials();
        }
#pragma unroll
        for (int q = 0; q < QT; q++) l_run[q] = sum[q];
        // element j of half s2 is key 16 s2 + 8 (j >> 2) + 4 hh + (j & 3)
#pragma unroll
        for (int s2 = 0; s2 < 2; s2++) {
            if constexpr (VH == 1) {
                if (s2 == 1) read_v8<16 * ROW, ROW>(base + vat[0], base + vat[1], base + vat[2], base + vat[3], vf[0]);
            }
#pragma unroll
            for (int dt = 0; dt < DT; dt++) {
                const u32x2_t v0 = vf[VH == 2 ? s2 : 0][2 * dt], v1 = vf[VH == 2 ? s2 : 0][2 * dt + 1];
                u32x4_t av = {v0[0], v0[1], v1[0], v1[1]};
                if constexpr (EDGE) {
                    // 0 * inf is NaN: an infinite or NaN value of a token that some row does not see must not reach that row.
                    // Such values are taken out of the product and counted instead, per row that sees them.
                    u32x4_t clean, plus, minus;
                    if (__any(split_nonfinite<E>(av, clean, plus, minus))) {
                        constexpr uint32_t ONE = __is_same(E, half_t) ? 0x3c00u : 0x3f80u;
                        av = clean;
#pragma unroll
                        for (int q = 0; q < QT; q++) {
                            u32x4_t ones;
#pragma unroll
                            for (int j = 0; j < 4; j++)
                                ones[j] = (seen[q] >> (8 * s2 + 2 * j) & 1 ? ONE : 0u) | (seen[q] >> (8 * s2 + 2 * j + 1) & 1 ? ONE << 16 : 0u);
#pragma unroll
                            for (int sign = 0; sign < 2; sign++) {
                                const f32x16_t count = mma<E>(sign ? minus : plus, ones, zero);
#pragma unroll
                                for (int i = 0; i < 16; i++)
                                    if (count[i] > 0.f) o[q][dt][i] += sign ? -INFINITY : INFINITY;
                            }
                        }
                    }
                }
#pragma unroll
                for (int q = 0; q < QT; q++) {
                    const u32x4_t pv = {pb[q][4 * s2], pb[q][4 * s2 + 1], pb[q][4 * s2 + 2], pb[q][4 * s2 + 3]};
                    o[q][dt] = mma<E>(av, pv, o[q][dt]);
                }
            }
        }
    };

#pragma unroll
    for (int t = 0; t < AHEAD; t++)
        if (t < nt) stage(t);
    // Tiles from t on as long as they are of the kind asked for; returns the next one.  (Two loops instead of a branch in one:
    // across such a branch the compiler copies the outputs.)  Only tiles at a range's ends, a window's or a query's are EDGE.
    auto is_edge = [&](int t) {   // (uniform over the wave)
        const int k0 = key_of(t);
        return k0 + KT > kend || k0 + KT - 1 > pos_min || k0 < lo_max;
    };
    auto tiles_of_kind = [&](auto edge_c, int t) {
        constexpr bool EDGE = decltype(edge_c)::value;
        for (; t < nt && is_edge(t) == EDGE; t++) {
            // This tile has landed: of the requests after it, those of AHEAD - 1 tiles may still be under way (behind the last
            // request: none).  RW = 4: on every wave, and nobody reads the buffer that is filled next.
            if (AHEAD > 1 && t + AHEAD <= nt) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"i"((AHEAD - 1) * 2 * NI) : "memory");
            else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
            if (RW == 4) asm volatile("s_barrier" ::: "memory");
            if (RW == 4 && t + AHEAD < nt) stage(t + AHEAD);
            const int k0 = key_of(t);
            const uint32_t base = tiles_at + (t % W::NS) * W::STAGE;
#pragma unroll 1
            for (int sub = 0; sub < KT && (!EDGE || k0 + sub < kend); sub += 32) step(edge_c, k0 + sub, base + sub * ROW, t + 1);
        }
        return t;
    };
    for (int t = 0; t < nt;) {
        t = tiles_of_kind(std::true_type{}, t);
        t = tiles_of_kind(std::false_type{}, t);
    }

    // The outputs go through LDS (in place of the tiles), so that whole rows are stored: straight from the accumulators a
    // store would touch 32 rows with 32 bytes each.  16-byte chunk c of row r lies at chunk c ^ (r & 15).
    const int64_t rows = (int64_t)a.T * a.Hq;
    constexpr int CH = D / 4;   // 16-byte chunks, and lanes, per row
    auto put = [&](unsigned char* at, const f32x16_t(&acc)[DT]) {
#pragma unroll
        for (int dt = 0; dt < DT; dt++)
#pragma unroll
            for (int i4 = 0; i4 < 4; i4++)
                *reinterpret_cast<float4_t*>(at + qi * D * 4 + (((8 * dt + 2 * i4 + hh) ^ (qi & 15)) << 4)) =
                    float4_t{acc[dt][4 * i4], acc[dt][4 * i4 + 1], acc[dt][4 * i4 + 2], acc[dt][4 * i4 + 3]};
    };
    // An output may be NaN only because an infinite value met a probability that rounds to 0: then the values of its column
    // that the row sees are looked through once more (tiles that are seen in part count them in the walk).  What all the
    // wave's rows see is looked through once, several keys at a time, the rest row by row: 65536 keys take some ms, and only
    // where an output is NaN.
    auto settle = [&](unsigned char* at, const f32x16_t(&acc)[DT], float l, int row_pos, int row_lo) {
        float z[4] = {0.f, 0.f, 0.f, 0.f};   // (0 times an infinity or NaN: one instruction per value)
#pragma unroll
        for (int dt = 0; dt < DT; dt++)
#pragma unroll
            for (int i = 0; i < 16; i++) z[i & 3] = __builtin_fmaf(acc[dt][i], 0.f, z[i & 3]);
        if (__builtin_expect(!__any((z[0] + z[1]) + (z[2] + z[3]) != 0.f), 1)) return;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        const int c = lane % CH;
        // bit e (e + 4): column 4 c + e holds a value that is +inf or NaN (-inf or NaN), keys from, from + by, .. upto
        auto look = [&](int from, int upto, int by) {
            constexpr int AT_ONCE = 4;
            uint32_t found = 0;
            for (int key0 = from; key0 <= upto && found != 0xffu; key0 += AT_ONCE * by) {
                u32x2_t raw[AT_ONCE];
#pragma unroll
                for (int u = 0; u < AT_ONCE; u++) {
                    const int key = min(key0 + u * by, upto), page = page_of(a, key);
                    const int blk = min(max(key < folded ? a.tables[page] : table[page], 0), a.num_blocks - 1);
                    const int64_t off = blk * a.block_stride + ((int64_t)(key - page * a.block_size) * a.Hkv + hk) * D + 4 * c;
                    raw[u] = *reinterpret_cast<const u32x2_t*>(reinterpret_cast<const E*>(a.vc) + off);
                }
#pragma unroll
                for (int u = 0; u < AT_ONCE; u++) {
                    u32x4_t clean, p, m;
                    if (!split_nonfinite<E>(u32x4_t{raw[u][0], raw[u][1], 0u, 0u}, clean, p, m)) continue;
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        found |= (p[e / 2] >> 16 * (e & 1) & 0xffffu) != 0 ? 1u << e : 0u;
                        found |= (m[e / 2] >> 16 * (e & 1) & 0xffffu) != 0 ? 16u << e : 0u;
                    }
                }
            }
            return found;
        };
        const int all_first = max(kfloor, lo_max), all_last = min(kend - 1, pos_min);
        int seen = (int)look(all_first + lane / CH, all_last, 64 / CH);
#pragma unroll
        for (int st = CH; st < 64; st *= 2) seen |= __shfl_xor(seen, st, 64);
#pragma unroll 1
        for (int i = 0; i < 32 * CH / 64; i++) {
            const int r = i * (64 / CH) + lane / CH;
            const int first = max(kfloor, __shfl(row_lo, r, 64)), last = min(kend - 1, __shfl(row_pos, r, 64));
            const float lr = __shfl(l, r, 64);
            float4_t* to = reinterpret_cast<float4_t*>(at + r * D * 4 + ((c ^ (r & 15)) << 4));
            float4_t v = *to;
            bool asked[4], any = false;
#pragma unroll
            for (int e = 0; e < 4; e++) any |= asked[e] = lr == lr && v[e] != v[e];   // (l is NaN where a score is)
            if (!any) continue;
            uint32_t found = (uint32_t)seen;
            if (all_first > all_last) {
                found |= look(first, last, 1);
            } else {
                found |= look(first, all_first - 1, 1);
                found |= look(all_last + 1, last, 1);
            }
#pragma unroll
            for (int e = 0; e < 4; e++)
                if (asked[e] && (found >> e & 1) != (found >> (e + 4) & 1)) v[e] = found >> e & 1 ? INFINITY : -INFINITY;
            *to = v;
        }
    };
    auto get = [&](const unsigned char* at, int r, int c) { return *reinterpret_cast<const float4_t*>(at + r * D * 4 + ((c ^ (r & 15)) << 4)); };
    if constexpr (RW == 4) {
        static_assert(SA_WAVES * 32 * D * 4 <= W::TILES);
        unsigned char* at = smem + wave * 32 * D * 4;
        __syncthreads();   // every wave is done with the tiles
#pragma unroll
        for (int q = 0; q < QT; q++) {
            put(at, o[q]);
            const float l = cross_half_sum(l_run[q]);
            settle(at, o[q], l, pos[q], lo[q]);
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            const int first = row0 + 32 * (wave * QT + q), c = lane % CH;
            if (direct) {
                float m, den, back;
                start_with_sink<E>(a, head[q], m, den);
                const float f = join_stats<1>(RangeStat{true, m_run[q], l}, m, den, back), inv = inverse(den);
#pragma unroll
                for (int i = 0; i < 32 * CH / 64; i++) {
                    const int r32 = i * (64 / CH) + lane / CH, rr = first + r32;
                    const float fr = __shfl(f, r32, 64), ir = __shfl(inv, r32, 64);
                    const float4_t v = get(at, r32, c);
                    if (rr < row_end) put_out<E>(a, rr / a.G, hk * a.G + rr % a.G, D, c, fr * v, ir);
                }
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                continue;
            }
#pragma unroll
            for (int i = 0; i < 32 * CH / 64; i++) {
                const int r32 = i * (64 / CH) + lane / CH, rr = first + r32;
                const float4_t v = get(at, r32, c);
                if (rr < row_end) *reinterpret_cast<float4_t*>(a.part_o + (split * rows + (int64_t)(rr / a.G) * a.Hq + hk * a.G + rr % a.G) * D + 4 * c) = v;
            }
            if (mine[q] && hh == 0) {
                const int64_t r = split * rows + (int64_t)token[q] * a.Hq + head[q];
                a.part_ml[r * 2] = m_run[q];
                a.part_ml[r * 2 + 1] = l;
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        }
    } else {
        static_assert(QT == 1 && 32 * D * 4 <= W::STAGE);
        __shared__ float wm[SA_WAVES][32], wl[SA_WAVES][32];
        put(tiles, o[0]);   // (each wave in place of its own tile)
        const float lsum = cross_half_sum(l_run[0]);
        settle(tiles, o[0], lsum, pos[0], lo[0]);
        if (hh == 0) {
            wm[wave][qi] = m_run[0];
            wl[wave][qi] = lsum;
        }
        __syncthreads();
        const int nrows = min(32, row_end - row0);
        if constexpr (SCORED) {
            if (direct) {   // (the rows are one token's, all of the KV head's)
                __shared__ float fin[32][2];
                if (tid < nrows) {
                    float m = wm[0][tid], l = 0.f, m_all, den, back;
#pragma unroll
                    for (int w = 1; w < SA_WAVES; w++) m = fmaxf(m, wm[w][tid]);
#pragma unroll
                    for (int w = 0; w < SA_WAVES; w++) l += factor(wm[w][tid], m) * wl[w][tid];
                    start_with_sink<E>(a, hk * a.G + tid, m_all, den);
                    join_stats<1>(RangeStat{true, m, l}, m_all, den, back);
                    fin[tid][0] = m_all;
                    fin[tid][1] = inverse(den);
                }
                __syncthreads();   // (and the waves' logits)
                add_weights(a, own_b, hk, fin);
            }
        }
        for (int i = tid; i < nrows * CH; i += SA_THREADS) {
            const int r32 = i / CH, c = i % CH;
            float m = wm[0][r32];
#pragma unroll
            for (int w = 1; w < SA_WAVES; w++) m = fmaxf(m, wm[w][r32]);
            float4_t tot = {0.f, 0.f, 0.f, 0.f};
            float l = 0.f;
#pragma unroll
            for (int w = 0; w < SA_WAVES; w++) {
                const float f = factor(wm[w][r32], m);   // (nothing seen at all: 1 * 0)
                tot += f * get(smem + w * W::NS * W::STAGE, r32, c);
                l += f * wl[w][r32];
            }
            const int rr = row0 + r32;
            if (direct) {
                float m_all, den, back;
                start_with_sink<E>(a, hk * a.G + rr % a.G, m_all, den);
                const float f = join_stats<1>(RangeStat{true, m, l}, m_all, den, back);
                put_out<E>(a, rr / a.G, hk * a.G + rr % a.G, D, c, f * tot, inverse(den));
                continue;
            }
            const int64_t r = split * rows + (int64_t)(rr / a.G) * a.Hq + hk * a.G + rr % a.G;
            *reinterpret_cast<float4_t*>(a.part_o + r * D + 4 * c) = tot;
            if (c == 0) {
                a.part_ml[r * 2] = m;
                a.part_ml[r * 2 + 1] = l;
            }
        }
    }
}

// The shared tokens: a workgroup per (row set, range, KV head).  All tokens' rows, in order.
template <typename E, int D, int RW, int QT, bool SCORED>
__device__ __forceinline__ void prefix_part(const SharedAttnArgs& a, unsigned char* smem, int id) {
    constexpr int ROWS = 32 * RW * QT;
    __shared__ int ends[SA_WAVES][2];
    const int hk = id % a.Hkv, unit = id / a.Hkv, split = unit % a.np, row0 = unit / a.np * ROWS;
    const int row_end = min(a.T * a.G, row0 + ROWS), pages_from = page_of(a, split * a.sp);
    fetch_pages<D, RW>(a, smem, a.tables, pages_from, 0);   // (needs nothing that is still to be looked up)
    const int tid = threadIdx.x, wave = tid >> 6, qi = tid & 31;
    int pos[QT], lo[QT], pos_max = -1, lo_min = INT32_MAX;
#pragma unroll
    for (int t = 0; t < QT; t++) {
        const int row = min(row0 + (RW == 4 ? 32 * (wave * QT + t) : 0) + qi, row_end - 1);
        const int token = row / a.G, b = seq_of(a, token);
        pos[t] = -1;
        if (b >= 0) {
            const SeqSpan s = seq_span(a, b);
            pos[t] = s.ctx - s.n + (token - s.t0);
        }
        lo[t] = window_lo(a, pos[t]);
        pos_max = max(pos_max, pos[t]);
        if (pos[t] >= 0) lo_min = min(lo_min, lo[t]);
    }
    // the range's keys that any row of the workgroup sees
    pos_max = -wave_min_i(-pos_max), lo_min = wave_min_i(lo_min);
    if (RW == 4) {
        if ((tid & 63) == 0) {
            ends[wave][0] = lo_min;
            ends[wave][1] = pos_max;
        }
        __syncthreads();
        for (int w = 0; w < SA_WAVES; w++) {
            lo_min = min(lo_min, ends[w][0]);
            pos_max = max(pos_max, ends[w][1]);
        }
    }
    const int kbeg = max(split * a.sp, lo_min), kend = min(min(split * a.sp + a.sp, a.prefix_len), pos_max + 1);
    if (kbeg >= kend) return;   // (the merge leaves out a range that a row does not see)
    attend<E, D, RW, QT, SCORED>(a, smem, hk, row0, row_end, pos, lo, a.tables, pages_from, kbeg, kend, kbeg, split, 0, -1, 0, false);
}

// The sequences' own tokens: a workgroup per (sequence, row set of the longest sequence, range, KV head).
template <typename E, int D, int RW, bool SCORED>
__device__ __forceinline__ void own_part(const SharedAttnArgs& a, unsigned char* smem, int id, int row_sets) {
    const int hk = id % a.Hkv, unit = id / a.Hkv, split = unit % a.ns;
    const int b = unit / a.ns / row_sets, set = unit / a.ns % row_sets;
    const int32_t* table = a.tables + (int64_t)b * a.max_blocks;
    const int k0 = a.prefix_len + split * a.so, folded = a.folded;
    const int pages_from = page_of(a, k0) + (k0 >= folded ? split_page(a, folded) : 0);
    fetch_pages<D, RW>(a, smem, table, pages_from, folded);
    const SeqSpan s = seq_span(a, b);
    const int row0 = s.t0 * a.G + set * 32 * RW, row_end = min((s.t0 + min(s.n, a.max_q)) * a.G, row0 + 32 * RW);
    if (row0 >= row_end) return;
    const int tid = threadIdx.x, wave = tid >> 6, qi = tid & 31;
    const int row = min(row0 + (RW == 4 ? 32 * wave : 0) + qi, row_end - 1);
    const int pos0 = s.ctx - s.n - s.t0;                       // position of token t is pos0 + t
    const int pos[1] = {pos0 + row / a.G}, lo[1] = {window_lo(a, pos[0])};
    const int kbeg = max(k0, window_lo(a, pos0 + row0 / a.G));
    int kend = min(k0 + a.so, pos0 + (row_end - 1) / a.G + 1);
    const bool direct = a.direct;
    if (kbeg >= kend && !direct) return;
    kend = max(kend, kbeg);   // (direct: rows that see nothing are written all the same)
    // (scored: the logits are addressed from the range's start in steps of a tile, so the walk starts on one)
    const int start = SCORED ? k0 + (kbeg - k0) / 32 * 32 : kbeg;
    attend<E, D, RW, 1, SCORED>(a, smem, hk, row0, row_end, pos, lo, table, pages_from, start, kend, kbeg, a.np + split, b,
                                SCORED ? a.prefix_len : -1, folded, direct);
}

// Both in one launch: the prefix (bound by the matrix cores when there are many rows) and the own tokens (bound by memory)
// run beside one another.
template <typename E, int D, int RWP, int QT, int RWO, bool SCORED>
__global__ __launch_bounds__(SA_THREADS, D == 64 && QT == 1 ? 3 : 2) void shared_attn_kernel(SharedAttnArgs a, int prefix_wgs, int row_sets) {
    constexpr int LP = Walk<D, RWP>::LDS, LO = Walk<D, RWO>::LDS;
    __shared__ __attribute__((aligned(16))) unsigned char smem[LP > LO ? LP : LO];
    if ((int)blockIdx.x < prefix_wgs) prefix_part<E, D, RWP, QT, SCORED>(a, smem, blockIdx.x);
    else own_part<E, D, RWO, SCORED>(a, smem, blockIdx.x - prefix_wgs, row_sets);
}

// Joins a row's ranges, LANES lanes per (token, query head): each looks after one range's (m, l), then they take the ranges'
// outputs on, D / 4 lanes to a range's row.  LANES = 64: a wave's whole width on one row, LANES / (D / 4) ranges at a time,
// for few rows with many ranges.  LANES = D / 4: several rows per wave, for many rows (waves beyond what the chip holds at
// once cost another round of memory latency: 109000 rows of 3 ranges took 57 us a wave each, 20 us this way, and 2048 rows of
// 34 ranges 6 us and 14).
template <typename E, int D, int LANES>
__device__ __forceinline__ void merge_part(const SharedAttnArgs& a, int id) {
    constexpr int LPR = D / 4, GROUPS = LANES / LPR, ROWS = SA_THREADS / LANES;
    constexpr int AHEAD = LANES == 64 ? 8 : 4;   // ranges whose rows are requested at a time
    const int lane = threadIdx.x % LANES, base = (threadIdx.x & 63) - lane, group = lane / LPR, col = lane % LPR * 4;
    const int hk = id % a.Hkv, row_asked = id / a.Hkv * ROWS + (int)threadIdx.x / LANES;   // (a KV head's rows stay on their chiplet)
    const int row = min(row_asked, a.T * a.G - 1);
    const int token = row / a.G, head = hk * a.G + row % a.G;
    const int b = seq_of(a, token);
    const SeqSpan s = seq_span(a, max(b, 0));
    const int pos = s.ctx - s.n + (token - s.t0), lo = window_lo(a, pos), n = a.np + a.ns;
    const int64_t rows = (int64_t)a.T * a.Hq, r = (int64_t)token * a.Hq + head;
    float m_run, den;
    start_with_sink<E>(a, head, m_run, den);
    float4_t num = {0.f, 0.f, 0.f, 0.f};
    for (int i0 = 0; i0 < n; i0 += LANES) {   // (every lane of the wave goes along: the sums below span its rows' lanes)
        float back;
        const float f = join_stats<LANES>(range_stat(a, i0 + lane, r, pos, lo), m_run, den, back);
        num *= back;
        const int cnt = min(LANES, n - i0);
        auto take = [&](auto ahead, int j0) {   // (all lanes go along: any of them may be asked for its factor)
            constexpr int N = decltype(ahead)::value;
            float4_t v[N];
#pragma unroll
            for (int u = 0; u < N; u++)
                v[u] = *reinterpret_cast<const float4_t*>(a.part_o + ((i0 + min(j0 + u * GROUPS + group, cnt - 1)) * rows + r) * D + col);
#pragma unroll
            for (int u = 0; u < N; u++) {
                const int j = j0 + u * GROUPS + group;
                const float fj = __shfl(f, base + min(j, cnt - 1), 64);
                if (j < cnt && fj != 0.f) num += fj * v[u];   // (what was not written may be anything)
            }
        };
        for (int j0 = 0; j0 < cnt; j0 += AHEAD * GROUPS) {
            if (cnt - j0 > 2 * GROUPS) take(std::integral_constant<int, AHEAD>{}, j0);
            else take(std::integral_constant<int, 2>{}, j0);
        }
    }
#pragma unroll
    for (int st = LPR; st < LANES; st *= 2)
#pragma unroll
        for (int c = 0; c < 4; c++) num[c] += __shfl_xor(num[c], st, 64);
    // rows behind the last sequence, and tokens behind the longest one that was announced, leave the output as it was
    if (group || row_asked >= a.T * a.G || b < 0 || token - s.t0 >= a.max_q) return;
    put_out<E>(a, token, head, D, lane % LPR, num, inverse(den));
}

// Adds the own tokens' weights, summed over the group's query heads: a workgroup per (sequence, KV head, SA_SCORE_KEYS
// tokens), which joins the heads' (m, l) once more for itself instead of waiting for another launch.  The logits that the walk
// leaves behind and this reads are 4 bytes per key and query head beside 4 D per key and KV head of K and V: 20 of 205 MB twice
// for 32 sequences of 2500 tokens, D 64, where the walk takes 47 us with them, 35 without, and this launch 10.
constexpr int SA_SCORE_KEYS = 4 * SA_THREADS;
template <typename E>
__device__ __forceinline__ void score_part(const SharedAttnArgs& a, int id, int pieces) {
    constexpr int HEADS = 64, AHEAD = 8;
    __shared__ float fin[HEADS][2];
    const int hk = id % a.Hkv, piece = id / a.Hkv % pieces, b = id / a.Hkv / pieces, tid = threadIdx.x;
    const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int ctx = context_of(a, b), lo = window_lo(a, ctx - 1), first = a.prefix_len + piece * SA_SCORE_KEYS;
    if (first >= ctx || first + SA_SCORE_KEYS <= lo) return;
    const int rel = piece * SA_SCORE_KEYS + 4 * tid;
    const bool some = a.prefix_len + rel < ctx;
    const float* x = a.logits + ((int64_t)b * a.Hq + hk * a.G) * a.lstride + rel;
    // the first heads' logits, the scores so far: on their way while the heads' (m, l) are joined
    float4_t ahead[AHEAD];
#pragma unroll
    for (int g = 0; g < AHEAD; g++)
        if (some && g < a.G) ahead[g] = *reinterpret_cast<const float4_t*>(x + (int64_t)g * a.lstride);
    float *slot[4], *slots = nullptr;   // (slots: all four side by side)
    float old[4];
    {
        const int key = a.prefix_len + rel, page = page_of(a, key), off = key - page * a.block_size;
        if (key + 3 < ctx && key >= lo && off + 3 < a.block_size) {
            const int blk = a.tables[(int64_t)b * a.max_blocks + page];
            float* to = a.scores + ((int64_t)min(max(blk, 0), a.num_blocks - 1) * a.Hkv + hk) * a.block_size + off;
            if (blk >= 0 && blk < a.num_blocks && (reinterpret_cast<uintptr_t>(to) & 15) == 0) {
                slots = to;
                const float4_t v = *reinterpret_cast<const float4_t*>(to);
#pragma unroll
                for (int u = 0; u < 4; u++) old[u] = v[u];
            }
        }
    }
#pragma unroll
    for (int u = 0; u < 4; u++) {
        const int key = a.prefix_len + rel + u;
        slot[u] = nullptr;
        if (slots) continue;
        if (key >= ctx || key < lo) continue;
        const int page = page_of(a, key), blk = a.tables[(int64_t)b * a.max_blocks + page];
        if (blk < 0 || blk >= a.num_blocks) continue;   // no score is written outside the cache
        slot[u] = a.scores + ((int64_t)blk * a.Hkv + hk) * a.block_size + (key - page * a.block_size);
        old[u] = *slot[u];
    }
    float4_t w = {0.f, 0.f, 0.f, 0.f};
    for (int g0 = 0; g0 < a.G; g0 += HEADS) {
        const int heads = min(HEADS, a.G - g0);
        if (g0) __syncthreads();
        for (int g = wave; g < heads; g += SA_WAVES) {
            const int head = hk * a.G + g0 + g;
            float m, den, back;
            start_with_sink<E>(a, head, m, den);
            for (int i0 = 0; i0 < a.np + a.ns; i0 += 64) join_stats<64>(range_stat(a, i0 + lane, (int64_t)b * a.Hq + head, ctx - 1, lo), m, den, back);
            if (lane == 0) {
                fin[g][0] = m;
                fin[g][1] = inverse(den);
            }
        }
        __syncthreads();
        auto take = [&](float4_t v, int g) {
#pragma unroll
            for (int u = 0; u < 4; u++) w[u] += __builtin_amdgcn_exp2f(v[u] - fin[g][0]) * fin[g][1];
        };
        if (some && g0 == 0) {
#pragma unroll
            for (int g = 0; g < AHEAD; g++)
                if (g < heads) take(ahead[g], g);
        }
        if (some) {
#pragma unroll 4
            for (int g = g0 ? 0 : AHEAD; g < heads; g++) take(*reinterpret_cast<const float4_t*>(x + (int64_t)(g0 + g) * a.lstride), g);
        }
    }
    if (slots) *reinterpret_cast<float4_t*>(slots) = float4_t{old[0], old[1], old[2], old[3]} + w;
#pragma unroll
    for (int u = 0; u < 4; u++)
        if (slot[u]) *slot[u] = old[u] + w[u];
}

template <typename E, int D, int LANES>
__global__ __launch_bounds__(SA_THREADS) void shared_join_kernel(SharedAttnArgs a, int merge_wgs, int pieces) {
    if ((int)blockIdx.x < merge_wgs) merge_part<E, D, LANES>(a, blockIdx.x);
    else score_part<E>(a, blockIdx.x - merge_wgs, pieces);
}

// ---------------------------------------------------------------------------------------------------------------------
// Into how many ranges a walk over `keys` keys is cut, for `units` (row set, KV head) pairs.  More ranges fill the 256 CUs
// and even them out; each costs its workgroups' start and the writing and reading of its rows' outputs.  In ns, fitted to
// sweeps of 1 to 64 ranges over prefixes of 8192 and 20011 keys, 32 to 2500 tokens, and own contexts of 512 to 65536:
//   7000 + len * max(alone, share * c) + start * c + merge * n + uneven   c: workgroups per CU, whole ones until there are four
// alone: ns per key of one workgroup on a CU, share: of all of a CU's workgroups together.  A few workgroups over a whole
// number per CU cost arithmetic (`tiles`) little, memory another round.  `beside`: time of memory-bound work of the same
// launch, which runs in the shadow of one workgroup per CU, but behind a second one.  uneven = 0.4 * alone * len / c for own
// tokens, whose sequences differ in length: on a CU with few long ranges, the prefix's (`others`) among them, their sums differ
// more (8 sequences of 500 to 65536 tokens, D 128: 16 ranges 153 us, 32 ranges 118; 32 of 1000 to 4096: 2 ranges 73 us, 4
// ranges 71.5; but 64 of up to 1024: 1 range 34 us, 2 ranges 37).
struct CutCost {
    bool tiles;
    double alone, share, start, uneven, merge, beside, others;
};
// Cost of ranges of `len` keys.
static double cut_cost(int64_t keys, int64_t units, const CutCost& w, int64_t len) {
    const int64_t used = (keys + len - 1) / len;
    const double c = (double)(units * used) / 256, whole = c <= 1 ? 1 : c < 4 ? ceil(c - (w.tiles ? 0.125 : 0)) : c;
    const double per_key = w.share * whole;
    const double behind = c <= 1 ? 0 : c < 2 ? c - 1 : 1;
    return 7000 + len * (per_key > w.alone ? per_key : w.alone) + w.start * c + w.merge * used +
           w.uneven * w.alone * len / (c + w.others < 1 ? 1 : c + w.others) + 0.5 * behind * w.beside;
}
static double cut_keys(int64_t keys, int64_t units, const CutCost& w, int64_t most, int& n, int& len) {
    n = 0, len = 128;
    if (keys <= 0) return 0;
    double best = 0;
    for (int64_t k = 1; k <= 1024 && (k == 1 || k <= most) && (k == 1 || (k - 1) * 128 < keys); k += k < 16 ? 1 : k / 8) {
        const int64_t l = ((keys + k - 1) / k + 127) / 128 * 128;
        const double t = cut_cost(keys, units, w, l);
        if (n == 0 || t < best) best = t, n = (int)((keys + l - 1) / l), len = (int)l;
    }
    return best;
}
struct SharedAttnPlan {
    int np, sp, ns, so, lstride;
    bool direct;                 // one range, which takes the prefix along
    int prefix_rows, own_rows;   // rows per workgroup: 32 (RW = 1), 128 or 256 (RW = 4)
    int64_t units;               // an upper bound of every launch's workgroups and row numbers
    size_t part_floats, bytes;   // the workspace: ranges' outputs, then (scored) logits; of both
    size_t least;                // a workspace of so many bytes will do
};
// The cheapest plan that makes do with a workspace of `budget` bytes (at least `least`, which no smaller call exceeds: a
// workspace that was made for the largest call serves all of them, with fewer ranges where the best number does not fit).
static SharedAttnPlan plan_shared_attn(int T, int B, int max_q, int Hq, int Hkv, int D, int max_ctx, int prefix_len, int window, bool scored,
                                       size_t budget) {
    SharedAttnPlan p;
    max_q = max_q < T ? max_q : T;
    const int64_t G = Hq / Hkv, P = prefix_len < max_ctx ? prefix_len : max_ctx, own = max_ctx - P, R = T * G;
    // Rows per workgroup.  32: the four waves share the keys (4 tokens of 8 heads on 8192 keys 13.4 us, with 128 rows 15.8); 128:
    // they share the tiles; 256 (D 64, many rows): every fragment read from LDS serves two row sets (512 tokens of 64 heads on
    // 8192 keys 120 us, with 128 rows 134; 600 tokens 144 and 147, 1700 tokens 331 and 341).
    p.prefix_rows = R <= 32 ? 32 : D == 64 && R * Hkv >= 32768 && !scored ? 256 : 128;
    p.own_rows = max_q * G > 32 && !scored ? 128 : 32;
    const double merge = (double)T * Hq * D * 4 / 2500;
    const bool d64 = D <= 64;
    const int64_t prefix_units = Hkv * ((R + p.prefix_rows - 1) / p.prefix_rows);
    auto cost = [&](bool own_keys, int rows, double beside) {
        CutCost w{true, 36, 21.7, 1300, 0, merge, beside, 0};                   // 256 rows
        if (rows == 128) w.alone = d64 ? 18 : 33, w.share = d64 ? 11.2 : 20;
        if (rows == 32) w.tiles = false, w.alone = d64 ? 14 : 28, w.share = d64 ? 13 : 26;
        if (rows == 32 && own_keys) w.start = d64 ? 1300 : 4000, w.uneven = 0.4, w.others = (double)p.np * prefix_units / 256;
        return w;
    };
    const int64_t own_units = Hkv * (int64_t)B * ((max_q * G + p.own_rows - 1) / p.own_rows);
    const size_t rows = (size_t)T * Hq, range = rows * (D + 2);   // floats that a range leaves behind
    auto logits_of = [&](int64_t keys) { return scored ? rows * (size_t)((keys + 127) / 128 * 128) : (size_t)0; };
    auto cut = [&](int64_t most_p, int64_t most_s) {
        const double prefix = cut_keys(P, prefix_units, cost(false, p.prefix_rows, p.own_rows == 32 ? (double)own * B * Hkv * D * 4 / 5000 : 0), most_p, p.np, p.sp);
        return prefix + cut_keys(own, own_units, cost(true, p.own_rows, 0), most_s, p.ns, p.so) - (P && own > 0 ? 7000 : 0);
    };
    p.least = scored ? (2 * range + logits_of(own) + 4) * sizeof(float) : 256;
    double t = cut(1024, 1024);
    const size_t room = budget / sizeof(float) > logits_of(own) ? budget / sizeof(float) - logits_of(own) : 0;
    const int64_t fit = (int64_t)(room / 4 * 4 / range);   // ranges that there is room for
    const bool ranges = fit >= (P > 0) + (own > 0);
    if (ranges && p.np + p.ns > fit) {   // (as many for the prefix as its share of the best plan)
        const int64_t most_p = P ? (own > 0 ? std::min<int64_t>(std::max<int64_t>(p.np * fit / (p.np + p.ns), 1), fit - 1) : fit) : 0;
        t = cut(most_p, fit - most_p);
    }
    // One range per sequence, which takes the prefix along, instead: every sequence reads the prefix again (from the L2s), but
    // no outputs are left to be joined, nor is there a second launch (about 3000 ns of the host's time, and a base of 5500 for 7000).
    // Fitted to 31 pairs, among them (us of kernels, ranges and joining / one range): 4 sequences of 200 + 33 tokens 9.6 / 7.2,
    // 16 of 500 + 100 13.1 / 9.5, 32 of 1500 + 60 14.7 / 15.7, 32 of 8192 + 512 22.9 / 58.9; 45 prompts of 42 to 81 tokens
    // behind 9 92 / 35, 24 of 200 to 300 behind 512 282 / 160, 6 of 150 to 420 behind 8192 364 / 410.
    auto one_range = [&](int64_t keys_prefix, int64_t keys_own) {
        CutCost w = cost(true, p.own_rows, 0);
        const int64_t keys = keys_prefix + keys_own;
        w.merge = w.others = 0;
        const double uneven = p.own_rows == 32 ? w.uneven * w.alone * keys_own : 0, c = (double)own_units / 256;
        if (p.own_rows == 32) w.alone = d64 ? 6 : 10, w.share = (w.alone * keys_prefix + w.share * keys_own) / keys;
        w.uneven = 0;
        return cut_cost(keys, own_units, w, (keys + 127) / 128 * 128) + uneven / (c < 1 ? 1 : c) - (p.own_rows == 32 ? 1500 : 0);
    };
    // (scored: one row set; 32 of 200 + 100 to 300 tokens 17.2 / 13.5, 64 of 500 to 1000 44.1 / 37.8, 9 of 2278 + 20 19.5 / 32.6)
    auto take_one_range = [&] {
        p.direct = true;
        p.np = 0, p.ns = 1, p.so = (int)((max_ctx + 127) / 128 * 128);
        p.prefix_rows = p.own_rows;   // (no kernel with more LDS and registers than the own walks use)
    };
    p.direct = false;
    if ((!scored || (G <= 32 && logits_of(max_ctx) * sizeof(float) <= budget)) && (!ranges || one_range(P, own) < t + 3000)) take_one_range();
    if (window > 0 && !scored && !p.direct) {   // (a row set sees its queries' positions and the window in front of the first)
        const int64_t seen = (int64_t)window + (p.own_rows == 32 ? max_q : 128 / G + 1);
        if (seen < max_ctx && one_range(0, seen) < t + 3000) take_one_range();
    }
    p.part_floats = p.direct ? 0 : ((size_t)(p.np + p.ns) * range + 3) / 4 * 4;   // (the logits behind it are stored 16 bytes at a time)
    p.lstride = (int)(((p.direct ? max_ctx : own) + 127) / 128 * 128);
    p.bytes = (p.part_floats + logits_of(p.direct ? max_ctx : own)) * sizeof(float);
    p.units = (int64_t)Hq * T * (p.np + 1) + (int64_t)Hkv * B * (p.ns * (max_q * G / 32 + 1) + own / SA_SCORE_KEYS + 1);
    return p;
}

template <typename E, int D>
static int launch_shared_attn(SharedAttnArgs& a, const SharedAttnPlan& p, bool scored, hipStream_t st) {
    const int rows = a.T * a.G, sets = (a.max_q * a.G + p.own_rows - 1) / p.own_rows;
    const int np_wgs = a.Hkv * a.np * ((rows + p.prefix_rows - 1) / p.prefix_rows), grid = np_wgs + a.Hkv * a.ns * a.B * sets;
#define M355_SA(RWP, QT, RWO, SCORED) shared_attn_kernel<E, D, RWP, QT, RWO, SCORED><<<grid, SA_THREADS, 0, st>>>(a, np_wgs, sets)
    if (grid) {
        if (scored && p.prefix_rows == 32) M355_SA(1, 1, 1, true);
        else if (scored) M355_SA(4, 1, 1, true);
        else if (p.prefix_rows == 32) M355_SA(1, 1, 1, false);
        else if (p.prefix_rows == 128 && p.own_rows == 32) M355_SA(4, 1, 1, false);
        else if (p.prefix_rows == 128) M355_SA(4, 1, 4, false);
        else if constexpr (D == 64) {
            if (p.own_rows == 32) M355_SA(4, 2, 1, false);
            else M355_SA(4, 2, 4, false);
        }
        M355_LAUNCH_CHECK("shared_attn_kernel");
    }
#undef M355_SA
    if (a.direct) return 0;
    const bool many = (int64_t)rows * a.Hkv > 16384;   // twice the waves that the chip holds at once
    const int per = SA_THREADS / (many ? D / 4 : 64), merge_wgs = a.Hkv * ((rows + per - 1) / per);
    const int pieces = scored ? (a.max_ctx - a.prefix_len + SA_SCORE_KEYS - 1) / SA_SCORE_KEYS : 0, join_grid = merge_wgs + a.Hkv * a.B * pieces;
    if (many) shared_join_kernel<E, D, D / 4><<<join_grid, SA_THREADS, 0, st>>>(a, merge_wgs, pieces);
    else shared_join_kernel<E, D, 64><<<join_grid, SA_THREADS, 0, st>>>(a, merge_wgs, pieces);
    M355_LAUNCH_CHECK("shared_join_kernel");
    return 0;
}

// What a workspace is asked to hold: twice the ranges of the best plan (up to 32 MB more) and of the best ones for fewer tokens
// (down to single ones, by factors of four), since a call with fewer tokens or a shorter context often wants more of them, and
// it is made once for the largest call.  By the model, 0.3 % of 300000 random pairs of a largest and a smaller call then take
// another plan than with all the memory they want, 0.15 % at a cost of more than 15 %.
static size_t shared_attn_workspace(int T, int B, int max_q, int Hq, int Hkv, int D, int max_ctx, int prefix_len, bool scored) {
    size_t need = 0;
    auto ask = [&](int t, int b, int n) {
        const SharedAttnPlan p = plan_shared_attn(t, b, n, Hq, Hkv, D, max_ctx, prefix_len, 0, scored, SIZE_MAX);
        need = std::max({need, p.least, p.bytes + std::min<size_t>(p.part_floats * sizeof(float), 32 << 20)});
    };
    for (int t = T; t > 0; t /= 4) ask(t, std::min(B, t), std::min(max_q, t));
    if (max_q > 1)
        for (int t = std::min(T, B); t > 0; t /= 4) ask(t, t, 1);
    return need;
}

// What both entry points check and set up alike.  Returns 0 with `a` and `p` filled in.
static int setup_shared_attn(const char* who, SharedAttnArgs& a, SharedAttnPlan& p, const void* q, const void* kc, const void* vc,
                             const int32_t* tables, const int32_t* ctx_lens, const int32_t* starts, int T, int B, int max_q, int Hq,
                             int Hkv, int D, int dtype, int num_blocks, int block_size, int max_blocks, int64_t block_stride,
                             int max_ctx, int prefix_len, int64_t q_stride, int64_t o_stride, float scale, const void* sinks,
                             int window, bool scored, void* workspace, size_t ws_bytes, void* out) {
    if (!q || !kc || !vc || !tables || !ctx_lens || !out) return fail(-1, "%s: null pointer", who);
    if (dtype != M355_DTYPE_F16 && dtype != M355_DTYPE_BF16) return fail(-2, "%s: unknown type %d", who, dtype);
    if (T < 0 || B < 0 || max_q <= 0 || Hkv <= 0 || Hq <= 0 || Hq % Hkv || (D != 64 && D != 128) || num_blocks <= 0 || block_size <= 0 ||
        max_blocks <= 0 || max_ctx <= 0 || prefix_len < 0 || window < 0)
        return fail(-2, "%s: unsupported shape T=%d B=%d max_q=%d Hq=%d Hkv=%d D=%d num_blocks=%d block_size=%d max_blocks=%d max_ctx=%d "
                        "prefix_len=%d window=%d (need D == 64 or 128, Hq a multiple of Hkv)",
                    who, T, B, max_q, Hq, Hkv, D, num_blocks, block_size, max_blocks, max_ctx, prefix_len, window);
    if (!starts && T != B) return fail(-2, "%s: %d tokens for %d sequences and no seq_starts", who, T, B);
    if ((int64_t)max_blocks * block_size < max_ctx)
        return fail(-2, "%s: max_ctx %d exceeds max_blocks*block_size %lld", who, max_ctx, (long long)max_blocks * block_size);
    if (block_stride < (int64_t)block_size * Hkv * D || block_stride % 8)
        return fail(-2, "%s: a page stride of %lld elements (need at least block_size*Hkv*D, a multiple of 8)", who, (long long)block_stride);
    if (q_stride < (int64_t)Hq * D || o_stride < (int64_t)Hq * D || q_stride % 8)
        return fail(-2, "%s: token strides must cover the heads, q's be a multiple of 8 elements", who);
    if (!aligned(q, 16) || !aligned(kc, 16) || !aligned(vc, 16)) return fail(-3, "%s: q and caches must be 16-byte aligned", who);
    p = plan_shared_attn(T, B, max_q, Hq, Hkv, D, max_ctx, prefix_len, window, scored, ws_bytes);
    if (max_ctx > (1 << 30) || p.units >= (1ll << 30))
        return fail(-2, "%s: unsupported size T=%d B=%d max_q=%d Hq=%d max_ctx=%d", who, T, B, max_q, Hq, max_ctx);
    if (!workspace || ws_bytes < p.least || ws_bytes < p.bytes)
        return fail(-6, "%s: workspace of %zu bytes needed, %zu given", who, std::max(p.least, p.bytes), ws_bytes);
    if (!aligned(workspace, 16)) return fail(-3, "%s: the workspace must be 16-byte aligned", who);
    a = SharedAttnArgs{};
    a.q = q, a.kc = kc, a.vc = vc, a.sinks = sinks, a.tables = tables, a.ctx_lens = ctx_lens, a.starts = starts;
    a.B = B, a.T = T, a.Hq = Hq, a.Hkv = Hkv, a.G = Hq / Hkv, a.num_blocks = num_blocks, a.block_size = block_size, a.max_blocks = max_blocks;
    divide_by(block_size, a.page_mul, a.page_shift);
    a.block_stride = block_stride, a.q_stride = q_stride, a.o_stride = o_stride;
    a.prefix_len = prefix_len < max_ctx ? prefix_len : max_ctx, a.max_ctx = max_ctx, a.max_q = max_q < T ? max_q : T, a.window = window;
    // (never 0: a masked score, -inf, times 0 would be NaN; 1e-30 times any score is nothing)
    a.scale2 = fmaxf(fabsf(scale) * 1.44269504088896341f, 1e-30f);
    a.q_sign = scale < 0.f ? 0x80008000u : 0u;
    a.np = p.np, a.sp = p.sp, a.ns = p.ns, a.so = p.so;
    a.direct = p.direct;
    if (p.direct) a.folded = a.prefix_len, a.prefix_len = 0;
    if (!p.direct) {
        a.part_o = reinterpret_cast<float*>(workspace);
        a.part_ml = a.part_o + (size_t)(p.np + p.ns) * T * Hq * D;
    }
    a.out = out;
    return 0;
}

}  // namespace m355

using namespace m355;

extern "C" size_t m355_shared_prefix_attn_workspace_bytes(int T, int B, int max_q, int Hq, int Hkv, int D, int max_ctx, int prefix_len) {
    if (T <= 0 || B <= 0 || max_q <= 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv || D <= 0 || max_ctx <= 0 || prefix_len < 0) return 0;
    return shared_attn_workspace(T, B, max_q, Hq, Hkv, D, max_ctx, prefix_len, false);
}

extern "C" size_t m355_paged_attn_decode_scored_workspace_bytes(int B, int Hq, int Hkv, int D, int max_ctx, int prefix_len) {
    if (B <= 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv || D <= 0 || max_ctx <= 0 || prefix_len < 0) return 0;
    return shared_attn_workspace(B, B, 1, Hq, Hkv, D, max_ctx, prefix_len, true);
}

extern "C" int m355_shared_prefix_attn(const void* q, const void* kcache, const void* vcache, const int32_t* block_tables,
                                       const int32_t* ctx_lens, const int32_t* seq_starts, int T, int B, int max_q, int Hq, int Hkv, int D,
                                       int dtype, int num_blocks, int block_size, int max_blocks, int64_t block_stride, int max_ctx,
                                       int prefix_len, int64_t q_stride, int64_t o_stride, float scale, const void* sinks, int window,
                                       void* workspace, size_t ws_bytes, void* out, m355_stream_t stream) {
    if (T == 0 || B == 0) return 0;
    SharedAttnArgs a;
    SharedAttnPlan p;
    if (int rc = setup_shared_attn("m355_shared_prefix_attn", a, p, q, kcache, vcache, block_tables, ctx_lens, seq_starts, T, B, max_q, Hq,
                                   Hkv, D, dtype, num_blocks, block_size, max_blocks, block_stride, max_ctx, prefix_len, q_stride, o_stride,
                                   scale, sinks, window, false, workspace, ws_bytes, out))
        return rc;
    hipStream_t st = (hipStream_t)stream;
    if (dtype == M355_DTYPE_F16) return D == 64 ? launch_shared_attn<half_t, 64>(a, p, false, st) : launch_shared_attn<half_t, 128>(a, p, false, st);
    return D == 64 ? launch_shared_attn<bf16_t, 64>(a, p, false, st) : launch_shared_attn<bf16_t, 128>(a, p, false, st);
}

extern "C" int m355_paged_attn_decode_scored(const void* q, const void* kcache, const void* vcache, float* scores,
                                             const int32_t* block_tables, const int32_t* ctx_lens, int B, int Hq, int Hkv, int D, int dtype,
                                             int num_blocks, int block_size, int max_blocks, int64_t block_stride, int max_ctx,
                                             int prefix_len, int64_t q_stride, int64_t o_stride, float scale, const void* sinks, int window,
                                             void* workspace, size_t ws_bytes, void* out, m355_stream_t stream) {
    if (B == 0) return 0;
    if (!scores) return fail(-1, "m355_paged_attn_decode_scored: null pointer");
    SharedAttnArgs a;
    SharedAttnPlan p;
    if (int rc = setup_shared_attn("m355_paged_attn_decode_scored", a, p, q, kcache, vcache, block_tables, ctx_lens, nullptr, B, B, 1, Hq, Hkv,
                                   D, dtype, num_blocks, block_size, max_blocks, block_stride, max_ctx, prefix_len, q_stride, o_stride, scale,
                                   sinks, window, true, workspace, ws_bytes, out))
        return rc;
    a.logits = reinterpret_cast<float*>(workspace) + p.part_floats;
    a.lstride = p.lstride;
    a.scores = scores;
    hipStream_t st = (hipStream_t)stream;
    if (dtype == M355_DTYPE_F16) return D == 64 ? launch_shared_attn<half_t, 64>(a, p, true, st) : launch_shared_attn<half_t, 128>(a, p, true, st);
    return D == 64 ? launch_shared_attn<bf16_t, 64>(a, p, true, st) : launch_shared_attn<bf16_t, 128>(a, p, true, st);
}
