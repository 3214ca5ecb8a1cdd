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
#include "common.h"

namespace m355 {

constexpr int SA_THREADS = 256;
constexpr int SA_WAVES = SA_THREADS / 64;
constexpr int SA_KT = 32;   // keys per tile

typedef __bf16 bf16_t;
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x16_t __attribute__((ext_vector_type(16)));
typedef short sa_short4_t __attribute__((ext_vector_type(4)));
typedef short sa_short8_t __attribute__((ext_vector_type(8)));
typedef const u32x4_t __attribute__((address_space(3))) sa_lds_u4_t;
typedef __attribute__((address_space(3))) sa_short4_t sa_lds_s4_t;

struct SharedAttnArgs {
    const void *q, *kc, *vc, *sinks;
    const int32_t *tables, *ctx_lens, *starts;   // starts null: token t is sequence t's only one
    int B, T, Hq, Hkv, G, num_blocks, block_size, max_blocks;
    uint32_t page_mul;
    int page_shift;
    int64_t block_stride, q_stride, o_stride;
    int prefix_len, max_ctx, max_q, window;
    float scale2;                                // scale * log2(e): scores are in the units of exp2
    int np, sp, ns, so;                          // ranges over the prefix / the own tokens, and their lengths
    float *part_o, *part_ml;                     // [np + ns][T * Hq][D], [np + ns][T * Hq][2]
    float *logits, *final_ml, *scores;           // scored form: [B][Hq][lstride], [B * Hq][2], the caller's [num_blocks][Hkv][block_size]
    int lstride;
    void* out;
};

// key / block_size for 0 <= key < 2^31: multiplication by a rounded-up reciprocal, exact in that range
__device__ __forceinline__ int page_of(const SharedAttnArgs& a, int key) {
    return (int)(((uint64_t)(uint32_t)key * a.page_mul) >> a.page_shift);
}
// element offset of a key's row of KV head hk; a table entry outside the cache is clamped (no access leaves the cache)
__device__ __forceinline__ int64_t key_row(const SharedAttnArgs& a, const int32_t* table, int key, int hk, int D) {
    const int page = page_of(a, key);
    const int blk = min(max(table[page], 0), a.num_blocks - 1);
    return blk * a.block_stride + ((int64_t)(key - page * a.block_size) * a.Hkv + hk) * D;
}

// What a sequence's row range and positions are.  Everything is clamped to what the arguments allow.
struct SeqSpan {
    int t0, n, ctx;   // first token, number of tokens, cached tokens
};
__device__ __forceinline__ SeqSpan seq_span(const SharedAttnArgs& a, int b) {
    SeqSpan s;
    s.ctx = min(a.ctx_lens[b], a.max_ctx);
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
__device__ __forceinline__ int window_lo(const SharedAttnArgs& a, int pos) {
    return a.window > 0 ? max(pos - a.window + 1, 0) : 0;
}

__device__ __forceinline__ float swap_half(float v) {   // the value that lane ^ 32 holds
    return __shfl_xor(v, 32, 64);
}
__device__ __forceinline__ int wave_min_i(int v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = min(v, __shfl_xor(v, o, 64));
    return __builtin_amdgcn_readfirstlane(v);
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

// Where a 16-byte chunk of a K row and of a V row lies in its LDS tile: XOR-swizzled so that the 32 rows read together
// (K: one chunk of each; V: the transposing read's 4 rows x 64 bytes) cover every bank.
template <int D>
__device__ __forceinline__ uint32_t k_at(int key, int chunk) {
    return key * (D * 2) + ((chunk ^ (D == 64 ? (key >> 1) & 7 : key & 15)) << 4);
}
template <int D>
__device__ __forceinline__ uint32_t v_at(int key, int chunk) {
    return key * (D * 2) + ((chunk ^ ((D == 64 ? (key >> 1) & 1 : key & 3) << 2)) << 4);
}

constexpr int lds_bytes(int D, int RW) { return (RW == 4 ? 1 : SA_WAVES) * 2 * SA_KT * D * 2; }

// One workgroup: the rows [row0, row_end) of KV head hk (at most 32 * RW) over the keys [kbeg, kend) of `table`, of which
// those from kfloor on may be read.
// RW = 4: the waves hold 32 rows each and share the tiles.  RW = 1: one set of 32 rows; the waves take the tiles in turn,
// each in LDS of its own, and are joined at the end.  pos / lo: position and lowest visible key of this lane's row.
template <typename E, int D, int RW, bool SCORED>
__device__ __forceinline__ void attend(const SharedAttnArgs& a, unsigned char* smem, int hk, int row0, int row_end, int pos, int lo,
                                       const int32_t* table, int kbeg, int kend, int kfloor, int split, int own_b, int own_k0) {
    constexpr int TILE = SA_KT * D * 2;   // bytes of one K (or V) tile
    constexpr int STEPS = D / 16, DT = D / 32;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int qi = lane & 31, hh = lane >> 5;
    const int row = min(row0 + (RW == 4 ? 32 * wave : 0) + qi, row_end - 1);
    const int token = row / a.G, head = hk * a.G + row % a.G;

    u32x4_t qf[STEPS];   // B operand of step s: Q[row][16 s + 8 hh ..]
    {
        const E* qrow = reinterpret_cast<const E*>(a.q) + token * a.q_stride + head * D + 8 * hh;
#pragma unroll
        for (int s = 0; s < STEPS; s++) qf[s] = *reinterpret_cast<const u32x4_t*>(qrow + 16 * s);
    }
    const int pos_min = wave_min_i(pos), lo_max = -wave_min_i(-lo);
    unsigned char* kt = smem + (RW == 4 ? 0 : wave * 2 * TILE);
    unsigned char* vt = kt + TILE;
    const int dg = (lane >> 4) & 1, ga = (lane & 15) >> 2, gc = lane & 3;

    float m_run = -INFINITY, l_run = 0.f;
    f32x16_t o[DT];
#pragma unroll
    for (int dt = 0; dt < DT; dt++)
#pragma unroll
        for (int i = 0; i < 16; i++) o[dt][i] = 0.f;

    for (int k0 = kbeg + (RW == 4 ? 0 : wave * SA_KT); k0 < kend; k0 += (RW == 4 ? SA_KT : SA_WAVES * SA_KT)) {
        constexpr int CH = D / 8;                            // 16-byte chunks per row
        constexpr int N = SA_KT * CH / (RW == 4 ? SA_THREADS : 64);
        u32x4_t kr[N], vr[N];
        const int first = RW == 4 ? tid : lane;
#pragma unroll
        for (int i = 0; i < N; i++) {
            const int c = first + i * (RW == 4 ? SA_THREADS : 64);
            // keys outside re-read the nearest one: they are masked below, and rows nobody may see are never read
            const int64_t at = key_row(a, table, max(min(k0 + c / CH, kend - 1), kfloor), hk, D) + (c % CH) * 8;
            kr[i] = *reinterpret_cast<const u32x4_t*>(reinterpret_cast<const E*>(a.kc) + at);
            vr[i] = *reinterpret_cast<const u32x4_t*>(reinterpret_cast<const E*>(a.vc) + at);
        }
        if (RW == 4) __syncthreads();   // the previous tile has been read
#pragma unroll
        for (int i = 0; i < N; i++) {
            const int c = first + i * (RW == 4 ? SA_THREADS : 64);
            *reinterpret_cast<u32x4_t*>(kt + k_at<D>(c / CH, c % CH)) = kr[i];
            *reinterpret_cast<u32x4_t*>(vt + v_at<D>(c / CH, c % CH)) = vr[i];
        }
        if (RW == 4) {
            __syncthreads();
        } else {   // (LDS serves a wave's instructions in order; the fence keeps the compiler's order)
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
        }
        f32x16_t x;
#pragma unroll
        for (int i = 0; i < 16; i++) x[i] = 0.f;
#pragma unroll
        for (int s = 0; s < STEPS; s++) x = mma<E>(*(sa_lds_u4_t*)(kt + k_at<D>(qi, 2 * s + hh)), qf[s], x);
        // register i: key k0 + (i & 3) + 8 (i >> 2) + 4 hh
#pragma unroll
        for (int i = 0; i < 16; i++) x[i] *= a.scale2;
        const bool edge = k0 + SA_KT > kend || k0 + SA_KT - 1 > pos_min || k0 < lo_max;   // (uniform over the wave)
        if (edge) {
#pragma unroll
            for (int i = 0; i < 16; i++) {
                const int key = k0 + (i & 3) + 8 * (i >> 2) + 4 * hh;
                x[i] = (key < kend && key <= pos && key >= lo) ? x[i] : -INFINITY;
            }
        }
        if constexpr (SCORED) {
            if (own_k0 >= 0 && row0 + qi < row_end) {
                float* dst = a.logits + ((int64_t)own_b * a.Hq + head) * a.lstride + (k0 - own_k0) + 4 * hh;
#pragma unroll
                for (int i4 = 0; i4 < 4; i4++)
                    *reinterpret_cast<float4_t*>(dst + 8 * i4) = float4_t{x[4 * i4], x[4 * i4 + 1], x[4 * i4 + 2], x[4 * i4 + 3]};
            }
        }
        float mx = x[0];
#pragma unroll
        for (int i = 1; i < 16; i++) mx = fmaxf(mx, x[i]);
        mx = fmaxf(mx, swap_half(mx));
        const float m_new = fmaxf(m_run, mx);
        const float m_use = m_new == -INFINITY ? 0.f : m_new;   // nothing visible so far: every term is 0
        const float alpha = __builtin_amdgcn_exp2f(m_run - m_use);
        float sum = 0.f;
        E pf[2][8];
#pragma unroll
        for (int i = 0; i < 16; i++) {
            const float p = __builtin_amdgcn_exp2f(x[i] - m_use);
            sum += p;
            pf[i >> 3][i & 7] = (E)p;
        }
        sum += swap_half(sum);
        l_run = l_run * alpha + sum;
        m_run = m_new;
#pragma unroll
        for (int dt = 0; dt < DT; dt++)
#pragma unroll
            for (int i = 0; i < 16; i++) o[dt][i] *= alpha;
        // element j of step s2 is key 16 s2 + 8 (j >> 2) + 4 hh + (j & 3)
#pragma unroll
        for (int s2 = 0; s2 < 2; s2++) {
            u32x4_t pb;
            __builtin_memcpy(&pb, pf[s2], 16);
#pragma unroll
            for (int dt = 0; dt < DT; dt++) {
                // lane 4 ga + gc of a 16-lane group supplies key 4 hh + ga, columns 4 gc ..; lane i receives column i
                const int key = 16 * s2 + 4 * hh + ga, chunk = 4 * dt + 2 * dg + (gc >> 1);
                const sa_short4_t v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((sa_lds_s4_t*)(vt + v_at<D>(key, chunk) + 8 * (gc & 1)));
                const sa_short4_t v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((sa_lds_s4_t*)(vt + v_at<D>(key + 8, chunk) + 8 * (gc & 1)));
                const sa_short8_t av8 = {v0[0], v0[1], v0[2], v0[3], v1[0], v1[1], v1[2], v1[3]};
                u32x4_t av = __builtin_bit_cast(u32x4_t, av8);
                if (edge) {
                    // 0 * inf is NaN: an infinite or NaN value of a token that some row does not see must not reach that row.
                    // Such values are taken out of the product and counted instead, per row that sees them.
                    u32x4_t clean, plus, minus;
                    if (__any(split_nonfinite<E>(av, clean, plus, minus))) {
                        constexpr uint32_t ONE = __is_same(E, half_t) ? 0x3c00u : 0x3f80u;
                        u32x4_t seen;
#pragma unroll
                        for (int j = 0; j < 4; j++)
                            seen[j] = (x[8 * s2 + 2 * j] != -INFINITY ? ONE : 0u) | (x[8 * s2 + 2 * j + 1] != -INFINITY ? ONE << 16 : 0u);
                        f32x16_t up, down;
#pragma unroll
                        for (int i = 0; i < 16; i++) up[i] = down[i] = 0.f;
                        up = mma<E>(plus, seen, up);
                        down = mma<E>(minus, seen, down);
#pragma unroll
                        for (int i = 0; i < 16; i++) {
                            if (up[i] > 0.f) o[dt][i] += INFINITY;
                            if (down[i] > 0.f) o[dt][i] -= INFINITY;
                        }
                        av = clean;
                    }
                }
                o[dt] = mma<E>(av, pb, o[dt]);
            }
        }
        if (RW != 4) {
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
        }
    }

    const int64_t rows = (int64_t)a.T * a.Hq;
    if constexpr (RW == 4) {
        if (row0 + 32 * wave + qi < row_end) {
            const int64_t r = split * rows + (int64_t)token * a.Hq + head;
#pragma unroll
            for (int dt = 0; dt < DT; dt++)
#pragma unroll
                for (int i4 = 0; i4 < 4; i4++)
                    *reinterpret_cast<float4_t*>(a.part_o + r * D + 32 * dt + 8 * i4 + 4 * hh) =
                        float4_t{o[dt][4 * i4], o[dt][4 * i4 + 1], o[dt][4 * i4 + 2], o[dt][4 * i4 + 3]};
            if (hh == 0) {
                a.part_ml[r * 2] = m_run;
                a.part_ml[r * 2 + 1] = l_run;
            }
        }
    } else {
        __shared__ float wm[SA_WAVES][32], wl[SA_WAVES][32];
        float* po = reinterpret_cast<float*>(smem) + wave * 32 * D;   // takes the place of the wave's tiles (same size)
#pragma unroll
        for (int dt = 0; dt < DT; dt++)
#pragma unroll
            for (int i4 = 0; i4 < 4; i4++)
                *reinterpret_cast<float4_t*>(po + qi * D + 32 * dt + 8 * i4 + 4 * hh) =
                    float4_t{o[dt][4 * i4], o[dt][4 * i4 + 1], o[dt][4 * i4 + 2], o[dt][4 * i4 + 3]};
        if (hh == 0) {
            wm[wave][qi] = m_run;
            wl[wave][qi] = l_run;
        }
        __syncthreads();
        const int nrows = min(32, row_end - row0);
        for (int i = tid; i < nrows * (D / 4); i += SA_THREADS) {
            const int r32 = i / (D / 4), d = (i % (D / 4)) * 4;
            float m = wm[0][r32];
#pragma unroll
            for (int w = 1; w < SA_WAVES; w++) m = fmaxf(m, wm[w][r32]);
            float4_t tot = {0.f, 0.f, 0.f, 0.f};
            float l = 0.f;
            if (m > -INFINITY) {
#pragma unroll
                for (int w = 0; w < SA_WAVES; w++) {
                    const float f = __builtin_amdgcn_exp2f(wm[w][r32] - m);
                    tot += f * *reinterpret_cast<const float4_t*>(reinterpret_cast<const float*>(smem) + (w * 32 + r32) * D + d);
                    l += f * wl[w][r32];
                }
            }
            const int rr = row0 + r32;
            const int64_t r = split * rows + (int64_t)(rr / a.G) * a.Hq + hk * a.G + rr % a.G;
            *reinterpret_cast<float4_t*>(a.part_o + r * D + d) = tot;
            if (d == 0) {
                a.part_ml[r * 2] = m;
                a.part_ml[r * 2 + 1] = l;
            }
        }
    }
}

// The shared tokens: a workgroup per (row set, range, KV head).  All tokens' rows, in order.
template <typename E, int D, int RW>
__global__ __launch_bounds__(SA_THREADS) void shared_prefix_kernel(SharedAttnArgs a) {
    __shared__ __attribute__((aligned(16))) unsigned char smem[lds_bytes(D, RW)];
    __shared__ int ends[SA_WAVES][2];
    const int hk = blockIdx.x % a.Hkv, unit = blockIdx.x / a.Hkv, split = unit % a.np, row0 = unit / a.np * 32 * RW;
    const int row_end = min(a.T * a.G, row0 + 32 * RW);
    const int tid = threadIdx.x, wave = tid >> 6, qi = tid & 31;
    const int row = min(row0 + (RW == 4 ? 32 * wave : 0) + qi, row_end - 1);
    const int token = row / a.G, b = seq_of(a, token);
    int pos = -1;
    if (b >= 0) {
        const SeqSpan s = seq_span(a, b);
        pos = s.ctx - s.n + (token - s.t0);
    }
    const int lo = window_lo(a, pos);
    // the range's keys that any row of the workgroup sees
    const int pos_max = -wave_min_i(-pos), lo_min = wave_min_i(pos >= 0 ? lo : INT32_MAX);
    if ((tid & 63) == 0) {
        ends[wave][0] = lo_min;
        ends[wave][1] = pos_max;
    }
    __syncthreads();
    int kbeg = split * a.sp, kend = min(kbeg + a.sp, a.prefix_len), first = INT32_MAX, last = -1;
    for (int w = 0; w < SA_WAVES; w++) {
        first = min(first, ends[w][0]);
        last = max(last, ends[w][1]);
    }
    kbeg = max(kbeg, first);
    kend = min(kend, last + 1);
    if (kbeg >= kend) return;   // (the merge leaves out a range that a row does not see)
    attend<E, D, RW, false>(a, smem, hk, row0, row_end, pos, lo, a.tables, kbeg, kend, kbeg, split, 0, -1);
}

// The sequences' own tokens: a workgroup per (sequence, row set of the longest sequence, range, KV head).
template <typename E, int D, int RW, bool SCORED>
__global__ __launch_bounds__(SA_THREADS) void own_tokens_kernel(SharedAttnArgs a, int row_sets) {
    __shared__ __attribute__((aligned(16))) unsigned char smem[lds_bytes(D, RW)];
    const int hk = blockIdx.x % a.Hkv, unit = blockIdx.x / a.Hkv, split = unit % a.ns;
    const int b = unit / a.ns / row_sets, set = unit / a.ns % row_sets;
    const SeqSpan s = seq_span(a, b);
    const int row0 = s.t0 * a.G + set * 32 * RW, row_end = min((s.t0 + s.n) * a.G, row0 + 32 * RW);
    if (row0 >= row_end) return;
    const int tid = threadIdx.x, wave = tid >> 6, qi = tid & 31;
    const int row = min(row0 + (RW == 4 ? 32 * wave : 0) + qi, row_end - 1);
    const int pos0 = s.ctx - s.n - s.t0;                       // position of token t is pos0 + t
    const int pos = pos0 + row / a.G, lo = window_lo(a, pos);
    const int k0 = a.prefix_len + split * a.so;
    const int kbeg = max(k0, window_lo(a, pos0 + row0 / a.G));
    const int kend = min(k0 + a.so, pos0 + (row_end - 1) / a.G + 1);
    if (kbeg >= kend) return;
    // (scored: the logits are addressed from the range's start in steps of a tile, so the walk starts on one)
    const int aligned = SCORED ? k0 + (kbeg - k0) / SA_KT * SA_KT : kbeg;
    attend<E, D, RW, SCORED>(a, smem, hk, row0, row_end, pos, lo, a.tables + (int64_t)b * a.max_blocks, aligned, kend, kbeg,
                             a.np + split, b, SCORED ? a.prefix_len : -1);
}

// Joins the ranges of one (token, query head).  One wave; a lane holds D / 64 columns.
template <typename E, int D>
__global__ __launch_bounds__(64) void shared_merge_kernel(SharedAttnArgs a) {
    const int head = blockIdx.x % a.Hq, token = blockIdx.x / a.Hq, lane = threadIdx.x;
    const int b = seq_of(a, token);
    if (b < 0) return;   // behind the last sequence: left as it was
    const SeqSpan s = seq_span(a, b);
    if (token - s.t0 >= a.max_q) return;
    const int pos = s.ctx - s.n + (token - s.t0), lo = window_lo(a, pos);
    const int64_t rows = (int64_t)a.T * a.Hq, r = (int64_t)token * a.Hq + head;
    auto live = [&](int i) {   // does this row see a key of range i?
        const int beg = i < a.np ? i * a.sp : a.prefix_len + (i - a.np) * a.so;
        const int end = i < a.np ? min(beg + a.sp, a.prefix_len) : beg + a.so;
        return max(beg, lo) < min(end, pos + 1);
    };
    float m = -INFINITY;
    for (int i = 0; i < a.np + a.ns; i++)
        if (live(i)) m = fmaxf(m, a.part_ml[(i * rows + r) * 2]);
    float den = 0.f, num[D / 64] = {};
    if (a.sinks) {
        const float sk = (float)reinterpret_cast<const E*>(a.sinks)[head] * 1.44269504088896341f;
        m = fmaxf(m, sk);
        if (sk != -INFINITY) den = __builtin_amdgcn_exp2f(sk - m);
    }
    for (int i = 0; i < a.np + a.ns; i++) {
        if (!live(i)) continue;
        const float l = a.part_ml[(i * rows + r) * 2 + 1];
        if (l == 0.f) continue;
        const float f = __builtin_amdgcn_exp2f(a.part_ml[(i * rows + r) * 2] - m);
        den += f * l;
#pragma unroll
        for (int c = 0; c < D / 64; c++) num[c] += f * a.part_o[(i * rows + r) * D + c * 64 + lane];
    }
    const float inv = den > 0.f ? 1.0f / den : (den == 0.f ? 0.f : den);   // (a NaN stays one)
#pragma unroll
    for (int c = 0; c < D / 64; c++) reinterpret_cast<E*>(a.out)[token * a.o_stride + head * D + c * 64 + lane] = (E)(num[c] * inv);
    if (a.final_ml && lane == 0) {
        a.final_ml[r * 2] = m == -INFINITY ? 0.f : m;
        a.final_ml[r * 2 + 1] = inv;
    }
}

// Adds the own tokens' weights, summed over the group's query heads: a workgroup per (sequence, KV head, 256 tokens).
__global__ __launch_bounds__(SA_THREADS) void score_add_kernel(SharedAttnArgs a, int pieces) {
    const int piece = blockIdx.x % pieces, hk = blockIdx.x / pieces % a.Hkv, b = blockIdx.x / pieces / a.Hkv;
    const int rel = piece * SA_THREADS + threadIdx.x, key = a.prefix_len + rel;
    const int ctx = min(a.ctx_lens[b], a.max_ctx);
    if (key >= ctx || key < window_lo(a, ctx - 1)) return;
    float w = 0.f;
    for (int g = 0; g < a.G; g++) {
        const int64_t r = (int64_t)b * a.Hq + hk * a.G + g;
        w += __builtin_amdgcn_exp2f(a.logits[r * a.lstride + rel] - a.final_ml[r * 2]) * a.final_ml[r * 2 + 1];
    }
    const int page = page_of(a, key), blk = a.tables[(int64_t)b * a.max_blocks + page];
    if (blk < 0 || blk >= a.num_blocks) return;   // no score is written outside the cache
    a.scores[((int64_t)blk * a.Hkv + hk) * a.block_size + (key - page * a.block_size)] += w;
}

// ---------------------------------------------------------------------------------------------------------------------
struct SharedAttnPlan {
    int np, sp, ns, so, lstride;
    bool wide_prefix, wide_own;   // 128 rows per workgroup (RW = 4) instead of 32
    int64_t units;   // an upper bound of every launch's workgroups and row numbers
    size_t part_floats, logit_floats, bytes;
};
static SharedAttnPlan plan_shared_attn(int T, int B, int max_q, int Hq, int Hkv, int D, int max_ctx, int prefix_len, bool scored) {
    SharedAttnPlan p;
    max_q = max_q < T ? max_q : T;
    const int64_t G = Hq / Hkv, P = prefix_len < max_ctx ? prefix_len : max_ctx, own = max_ctx - P;
    p.wide_prefix = T * G > 32;
    p.wide_own = max_q * G > 32 && !scored;
    // ranges: enough workgroups for the chip, none shorter than 256 keys
    auto cut = [](int64_t keys, int64_t units, int& n, int& len) {
        n = 0, len = 256;
        if (keys <= 0) return;
        int64_t want = (1024 + units - 1) / units;
        int64_t l = (keys + want - 1) / want;
        l = (l + 127) / 128 * 128;
        if (l < 256) l = 256;
        len = (int)l;
        n = (int)((keys + l - 1) / l);
    };
    cut(P, (int64_t)Hkv * ((T * G + (p.wide_prefix ? 127 : 31)) / (p.wide_prefix ? 128 : 32)), p.np, p.sp);
    cut(own, (int64_t)Hkv * B * ((max_q * G + (p.wide_own ? 127 : 31)) / (p.wide_own ? 128 : 32)), p.ns, p.so);
    const size_t rows = (size_t)T * Hq;
    p.part_floats = ((size_t)(p.np + p.ns) * rows * (D + 2) + 3) / 4 * 4;   // (the logits behind it are stored 16 bytes at a time)
    p.lstride = (int)((own + 127) / 128 * 128);
    p.logit_floats = scored ? rows * ((size_t)p.lstride + 2) : 0;
    p.bytes = (p.part_floats + p.logit_floats) * sizeof(float);
    p.units = (int64_t)Hq * T * (p.np + 1) + (int64_t)Hkv * B * (p.ns * (max_q * G / 32 + 1) + own / SA_THREADS + 1);
    return p;
}

template <typename E, int D>
static int launch_shared_attn(SharedAttnArgs& a, const SharedAttnPlan& p, bool scored, hipStream_t st) {
    const int rows = a.T * a.G;
    if (a.np) {
        if (p.wide_prefix)
            shared_prefix_kernel<E, D, 4><<<a.Hkv * a.np * ((rows + 127) / 128), SA_THREADS, 0, st>>>(a);
        else
            shared_prefix_kernel<E, D, 1><<<a.Hkv * a.np * ((rows + 31) / 32), SA_THREADS, 0, st>>>(a);
        M355_LAUNCH_CHECK("shared_prefix_kernel");
    }
    if (a.ns) {
        const int per = p.wide_own ? 128 : 32, sets = (a.max_q * a.G + per - 1) / per;
        const int grid = a.Hkv * a.ns * a.B * sets;
        if (scored)
            own_tokens_kernel<E, D, 1, true><<<grid, SA_THREADS, 0, st>>>(a, sets);
        else if (p.wide_own)
            own_tokens_kernel<E, D, 4, false><<<grid, SA_THREADS, 0, st>>>(a, sets);
        else
            own_tokens_kernel<E, D, 1, false><<<grid, SA_THREADS, 0, st>>>(a, sets);
        M355_LAUNCH_CHECK("own_tokens_kernel");
    }
    shared_merge_kernel<E, D><<<a.Hq * a.T, 64, 0, st>>>(a);
    M355_LAUNCH_CHECK("shared_merge_kernel");
    if (scored && a.ns) {
        const int pieces = (a.max_ctx - a.prefix_len + SA_THREADS - 1) / SA_THREADS;
        score_add_kernel<<<a.Hkv * a.B * pieces, SA_THREADS, 0, st>>>(a, pieces);
        M355_LAUNCH_CHECK("score_add_kernel");
    }
    return 0;
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
    p = plan_shared_attn(T, B, max_q, Hq, Hkv, D, max_ctx, prefix_len, scored);
    if (max_ctx > (1 << 30) || p.units >= (1ll << 30))
        return fail(-2, "%s: unsupported size T=%d B=%d max_q=%d Hq=%d max_ctx=%d", who, T, B, max_q, Hq, max_ctx);
    if (!workspace || ws_bytes < p.bytes) return fail(-6, "%s: workspace of %zu bytes needed, %zu given", who, p.bytes, ws_bytes);
    if (!aligned(workspace, 16)) return fail(-3, "%s: the workspace must be 16-byte aligned", who);
    a = SharedAttnArgs{};
    a.q = q, a.kc = kc, a.vc = vc, a.sinks = sinks, a.tables = tables, a.ctx_lens = ctx_lens, a.starts = starts;
    a.B = B, a.T = T, a.Hq = Hq, a.Hkv = Hkv, a.G = Hq / Hkv, a.num_blocks = num_blocks, a.block_size = block_size, a.max_blocks = max_blocks;
    int sh = 0;
    while ((1ll << sh) < block_size) sh++;
    a.page_mul = (uint32_t)(((1ull << (31 + sh)) + block_size - 1) / block_size);
    a.page_shift = 31 + sh;
    a.block_stride = block_stride, a.q_stride = q_stride, a.o_stride = o_stride;
    a.prefix_len = prefix_len < max_ctx ? prefix_len : max_ctx, a.max_ctx = max_ctx, a.max_q = max_q < T ? max_q : T, a.window = window;
    a.scale2 = scale * 1.44269504088896341f;
    a.np = p.np, a.sp = p.sp, a.ns = p.ns, a.so = p.so;
    a.part_o = reinterpret_cast<float*>(workspace);
    a.part_ml = a.part_o + (size_t)(p.np + p.ns) * T * Hq * D;
    a.out = out;
    return 0;
}

}  // namespace m355

using namespace m355;

extern "C" size_t m355_shared_prefix_attn_workspace_bytes(int T, int B, int max_q, int Hq, int Hkv, int D, int max_ctx, int prefix_len) {
    if (T <= 0 || B <= 0 || max_q <= 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv || D <= 0 || max_ctx <= 0 || prefix_len < 0) return 0;
    return plan_shared_attn(T, B, max_q, Hq, Hkv, D, max_ctx, prefix_len, false).bytes;
}

extern "C" size_t m355_paged_attn_decode_scored_workspace_bytes(int B, int Hq, int Hkv, int D, int max_ctx, int prefix_len) {
    if (B <= 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv || D <= 0 || max_ctx <= 0 || prefix_len < 0) return 0;
    return plan_shared_attn(B, B, 1, Hq, Hkv, D, max_ctx, prefix_len, true).bytes;
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
    a.logits = a.part_o + p.part_floats;
    a.lstride = p.lstride;
    a.final_ml = a.logits + (size_t)B * Hq * p.lstride;
    a.scores = scores;
    hipStream_t st = (hipStream_t)stream;
    if (dtype == M355_DTYPE_F16) return D == 64 ? launch_shared_attn<half_t, 64>(a, p, true, st) : launch_shared_attn<half_t, 128>(a, p, true, st);
    return D == 64 ? launch_shared_attn<bf16_t, 64>(a, p, true, st) : launch_shared_attn<bf16_t, 128>(a, p, true, st);
}
