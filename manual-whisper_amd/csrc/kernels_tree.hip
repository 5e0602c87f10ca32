// Attention of trees of drafted tokens over a K/V cache in pages, for gfx950.
//
// For row (node) i of request b and query head h:  out = sum_j p_j V[j],  p = softmax_j(scale * q . K[j])  over the keys that
// the row sees: all of the request's `kept` cached tokens, and of its own step's nodes (at positions kept ..) those whose
// bit is set in the row's mask, or without a mask the nodes up to itself.  A row that sees nothing is zero.
//
// Bound: the K/V rows of a request are read once per K/V head for all nodes and all query heads of its group, so a step with
// few columns (nodes x heads per K/V head) is bound by HBM.  With some hundred columns the matrix products, the exponents and the
// LDS reads of a tile each come near the time that its rows take to arrive, and none of them alone sets the pace.
//
// One workgroup takes one work unit (a stretch of a request's keys), one K/V head and up to 128 query columns.  Keys are on
// the row index of the matrix instructions, so that a lane's scores belong to one query column: S^T = K Q^T, then
// O^T = V^T P^T with P straight from the registers of S (its 4-key groups are the k-slots of the second product) and
// V^T by transposing LDS reads.  Tiles of 64 keys go global -> registers -> LDS, the next tile's loads in flight behind the
// current tile's products.  The softmax is online: one running reference and sum per column.
// A request that is cut into several units leaves its partial results (fp32, with maximum and sum) in the workspace and a
// second launch joins them.
//
// Measured (rows; K/V heads x head_dim; K/V read; this kernel, then the join; medians of 498 launches in a graph, three input sets in
// turn.  Further down "a where it is b" compares builds of one session by their smallest times, which lie up to 8 % lower):
//   8 requests of 1 row, 207 k tokens of 8 x 128 bf16, 32 heads       849 MB           135 us (6.3 TB/s)                5.5 us
//   16 trees of 8, 2.5 k tokens of 20 x 64 fp16, 20 heads              13 MB           9.8 us (latency: seven tiles)     no cut
//   32 trees of 20..61, 80 k tokens of 8 x 128 bf16, 32 heads         329 MB, 51 GF   120 us (2.7 TB/s, 428 TFLOP/s)   14.5 us
//   24 chains of 3..16, 138 k tokens of 8 x 128 e4m3, 64 heads        282 MB, 34 GF   104 us (2.7 TB/s, 328 TFLOP/s)   15.9 us
// The wide trees' workgroups do not divide evenly over the CUs (23 % of the CU time is idle), 63 MB of partial results are written
// and read, and 20 % of the products are padding.  Loads alone take 83 us, everything but the loads 80.
#include "mw_kernels.h"

#include <type_traits>

namespace mw {

namespace {

typedef __bf16 bf16;
typedef __bf16 bf8v __attribute__((ext_vector_type(8)));
typedef short short4v __attribute__((ext_vector_type(4)));
typedef short short8v __attribute__((ext_vector_type(8)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.4426950408889634f;
constexpr int KT = 64;                                       // keys of a tile

// Weights are 2^(score - reference).  When a column's reference moves it goes kLow below the largest score, and it stays until a
// score is more than kGap above it (positive: gap > 0 says that a column has seen a key).  fp16 holds full precision from 2^-14 to
// 2^15, so its weights are kept high: the largest is 2^10 .. 2^14, and one is rounded by more than half a step of the type only
// where it is below 2^-24 of the largest, then by at most 2^-35 of it.  (With the largest near 1 a long cache beside one dominant
// key loses its weights: 20 k tokens of e^-18 each came out as nothing.)
template <typename T> struct Mat;
template <> struct Mat<f16> {
    static __device__ __forceinline__ float4v mma32(short8v a, short8v b, float4v c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8, a), __builtin_bit_cast(half8, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ float4v mma16(short4v a, short4v b, float4v c) {
        return __builtin_amdgcn_mfma_f32_16x16x16f16(__builtin_bit_cast(half4, a), __builtin_bit_cast(half4, b), c, 0, 0, 0);
    }
    static constexpr unsigned kExp = 0x7c007c00u;            // exponents of a pair of values
    static constexpr float kLow = 10.f, kGap = 14.f;
};
template <> struct Mat<bf16> {
    static __device__ __forceinline__ float4v mma32(short8v a, short8v b, float4v c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf8v, a), __builtin_bit_cast(bf8v, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ float4v mma16(short4v a, short4v b, float4v c) {
        return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(a, b, c, 0, 0, 0);
    }
    static constexpr unsigned kExp = 0x7f807f80u;
    static constexpr float kLow = 0.f, kGap = 6.f;           // (the range of fp32)
};
// eight values with 0 in the place of infinities and NaN (all bits of the exponent set); `any`: whether there were some
template <typename T> __device__ __forceinline__ u32x4 finite_only(u32x4 u, bool& any) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const unsigned e = u[i] & Mat<T>::kExp;
        const bool lo = (e & 0xffffu) == (Mat<T>::kExp & 0xffffu), hi = (e >> 16) == (Mat<T>::kExp >> 16);
        u[i] &= (lo ? 0xffff0000u : 0xffffffffu) & (hi ? 0x0000ffffu : 0xffffffffu);
        any = any || lo || hi;
    }
    return u;
}
template <typename T> __device__ __forceinline__ short bits_of(float x) { return __builtin_bit_cast(short, (T)x); }       // nearest even

// largest of three, a NaN passed over (of values that vector instructions made; written out, since the compiler first copies every
// operand to quiet a NaN)
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
    return r;
}
__device__ __forceinline__ int exponent(float x) { return (int)(__float_as_uint(x) >> 23 & 0xffu); }               // the field
__device__ __forceinline__ float column_max(float v) {       // over the four lanes that share a query column
    v = fmaxf(v, __shfl_xor(v, 16));
    return fmaxf(v, __shfl_xor(v, 32));
}
__device__ __forceinline__ float column_sum(float v) {
    v += __shfl_xor(v, 16);
    return v + __shfl_xor(v, 32);
}
// LDS images of a tile: rows of K are D + 8 values apart, rows of V D + 16, so that the rows that one instruction reads (16
// pieces of 16 bytes of K, 8 of 32 bytes of V) start in different banks and every address is one register and a constant.
template <int D> __device__ __forceinline__ int k_at(int row, int chunk) { return row * (D + 8) + chunk * 8; }
template <int D> __device__ __forceinline__ int v_at(int row, int col) { return row * (D + 16) + col; }
// Order of a phase of N operands from LDS (READS reads each) with M matrix instructions each: AHEAD operands first, then one
// operand after the products of another.
template <int N, int M, int AHEAD, int READS> __device__ __forceinline__ void interleave() {
    constexpr int A = AHEAD < N ? AHEAD : N;
    __builtin_amdgcn_sched_group_barrier(0x100, A * READS, 0);
#pragma unroll
    for (int i = 0; i < N - A; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, M, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, READS, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x008, A * M, 0);
}
// 8 e4m3 codes -> 8 values of T (exact, NaN included: two codes an instruction)
template <typename T> __device__ __forceinline__ u32x4 widen8(unsigned a, unsigned b) {
    if constexpr (__is_same(T, f16))
        return u32x4{__builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, 1.f, false)),
                     __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, 1.f, true)),
                     __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, 1.f, false)),
                     __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, 1.f, true))};
    else
        return u32x4{__builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 1.f, false)),
                     __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 1.f, true)),
                     __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 1.f, false)),
                     __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 1.f, true))};
}

// LDS of a workgroup: K and V of a tile (at the end: partial results of waves that split the keys), K's and V's row scales.
template <bool KV8, int D> struct Shared {
    short tiles[KT * (2 * D + 24)] __attribute__((aligned(16)));
    float scales[2][KV8 ? KT : 4] __attribute__((aligned(16)));
    int page_ok[4] __attribute__((aligned(16)));             // per 16 keys: the page exists
    int bad_v;                                               // V rows of this step held an infinity or a NaN
    float red_m[4][32], red_l[4][32];
};
// What a workgroup works on: keys key0 .. key1 of request b for K/V head g, query columns col0 .. of `cols`
struct Work { int b, unit, pieces, g, row0, nodes, cols, col0, kept, key0, key1; };

// T: type of q, of the products and of out.  KV8: the cache holds e4m3 codes with a scale per row; the codes go to the matrix
// cores as they are, K's scale multiplies the score and V's the weight.  QT: 16-column query tiles per wave.  WK: waves that
// share the columns and split a tile's keys; 4 / WK groups of waves hold different columns.
template <typename T, bool KV8, int D, int QT, int WK>
__device__ __forceinline__ void attend(const TreeAttnParams& p, int group, const Work& w, Shared<KV8, D>& lds) {
    constexpr int NK = 4 / WK;                               // 16-key tiles of a wave
    constexpr int EPL = KV8 ? 16 : 8;                        // values of a 16-byte load
    constexpr int CPR = D / EPL, RPL = 64 / CPR, NI = 16 / RPL;               // lanes of a row, rows of a load, loads of 16 rows
    constexpr int ND = D / 16;
    short* const ldsK = lds.tiles;
    short* const ldsV = lds.tiles + KT * (D + 8);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int fr = lane & 15, fg = lane >> 4;
    const int wq = wave / WK, wk = wave % WK;
    const int key0 = w.key0, key1 = w.key1, kept = w.kept;
    const int n_tiles = key1 > key0 ? (key1 - key0 + KT - 1) / KT : 0;
    const bool active = w.col0 + wq * QT * 16 < w.cols;      // wave-uniform; a wave without columns only helps with the staging

    // ---- the query columns of this wave
    short8v qf[QT][D / 32];
    int node[QT];
#pragma unroll
    for (int qs = 0; qs < QT; ++qs) {
        const int c = min(w.col0 + (wq * QT + qs) * 16 + fr, w.cols - 1);
        node[qs] = c / group;
        const short* src = static_cast<const short*>(p.q) + (long)(w.row0 + node[qs]) * p.q_row + (long)(w.g * group + c - node[qs] * group) * p.q_head;
#pragma unroll
        for (int s = 0; s < D / 32; ++s) qf[qs][s] = *reinterpret_cast<const short8v*>(src + s * 32 + fg * 8);
    }
    const float to_log2 = p.scale * kLog2e;                  // exponents of two: weight = exp2((s - max) * scale * log2 e)

    // ---- staging.  Wave w moves keys 16 w .. 16 w + 15 of a tile: one run of 16, so one page, whose address is scalar.  A lane
    // adds offsets that are the same for every tile.
    const int ch = lane % CPR, srow = lane / CPR;
    const int* const pages = p.table + (long)w.b * p.table_stride;
    const int page_mask = (1 << p.c.page_shift) - 1;
    constexpr int ES = KV8 ? 1 : 2;                          // bytes of a value
    unsigned lane_off[NI];
#pragma unroll
    for (int i = 0; i < NI; ++i) lane_off[i] = ((unsigned)(srow + RPL * i) * (unsigned)p.c.token_stride + ch * EPL) * ES;
    const char* const kbase = static_cast<const char*>(p.c.k) + (long)w.g * p.c.head_stride * ES;
    const char* const vbase = static_cast<const char*>(p.c.v) + (long)w.g * p.c.head_stride * ES;
    u32x4 rk[NI], rv[NI];
    int pg = -1;                                             // page of the rows to be loaded next
    bool ok = false;                                         // the page of the loaded rows exists
    float rscale = 0.f;
    // What is loaded here and in load_tile is looked at one tile later: a comparison here would wait for every load in flight.
    auto load_page = [&](int kv0) { pg = pages[min(kv0 + 16 * wave, key1 - 1) >> p.c.page_shift]; };
    auto load_tile = [&](int kv0) {
        const int id = __builtin_amdgcn_readfirstlane(pg);
        ok = (unsigned)id < (unsigned)p.c.n_pages;
        const unsigned page = ok ? id : 0, place = (kv0 + 16 * wave) & page_mask;
        const long off = ((long)page * (unsigned)p.c.page_stride + (long)place * (unsigned)p.c.token_stride) * ES;
        // at most 16 columns: the rows are read once, and a step moves more than the caches hold
        auto row16 = [&](const char* at) {
            if constexpr (QT == 1) return __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(at));
            else return *reinterpret_cast<const u32x4*>(at);
        };
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            rk[i] = row16(kbase + off + lane_off[i]);
            rv[i] = row16(vbase + off + lane_off[i]);
        }
        if constexpr (KV8)                                   // lanes 0..15: K's scales of the 16 rows, 16..31: V's
            rscale = (lane & 16 ? p.c.vs : p.c.ks)[(((long)page * p.c.heads + w.g) << p.c.page_shift) + place + (lane & 15)];
    };
    auto store_tile = [&](int it) {
        const int kv0 = key0 + it * KT;
        bool bad = false;
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            const int row = 16 * wave + srow + RPL * i;
            if constexpr (KV8) {
                *reinterpret_cast<u32x4*>(&ldsK[k_at<D>(row, 2 * ch)]) = widen8<T>(rk[i][0], rk[i][1]);
                *reinterpret_cast<u32x4*>(&ldsK[k_at<D>(row, 2 * ch + 1)]) = widen8<T>(rk[i][2], rk[i][3]);
            } else {
                *reinterpret_cast<u32x4*>(&ldsK[k_at<D>(row, ch)]) = rk[i];
            }
            u32x4 lo = rv[i], hi = rv[i];
            if constexpr (KV8) {
                lo = widen8<T>(rv[i][0], rv[i][1]);
                hi = widen8<T>(rv[i][2], rv[i][3]);
            }
            if (kv0 + KT > min(kept, key1) || !ok) {                    // (uniform) tiles with rows of this step, or behind the last key
                // V's infinities and NaN are held back here, kept tokens' too: in the product they would reach rows that do not see them
                // (0 times NaN is NaN).  The rows that do get them at the end.  What lies behind the last key may be anything.
                const u32x4 none = {0, 0, 0, 0};
                if (kv0 + row >= key1 || !ok) lo = hi = none;
                lo = finite_only<T>(lo, bad);
                if constexpr (KV8) hi = finite_only<T>(hi, bad);
            }
            *reinterpret_cast<u32x4*>(&ldsV[v_at<D>(row, EPL * ch)]) = lo;
            if constexpr (KV8) *reinterpret_cast<u32x4*>(&ldsV[v_at<D>(row, EPL * ch + 8)]) = hi;
        }
        if (lane == 0) lds.page_ok[wave] = ok;
        if (bad) lds.bad_v = 1;
        if constexpr (KV8) {
            if (lane < 32) {
                const bool there = ok && kv0 + 16 * wave + (lane & 15) < key1;
                lds.scales[lane >> 4][16 * wave + (lane & 15)] = !there ? 0.f : lane < 16 ? rscale * to_log2 : rscale;
            }
        }
    };

    float4v o[ND][QT];                                       // O^T: rows of 16 head dims, columns of 16 queries
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int qs = 0; qs < QT; ++qs) o[d][qs] = float4v{0, 0, 0, 0};
    // a column's weights are 2^(s - ref); `gap`: what an exponent may reach before ref rises (-inf: no key seen yet)
    float ref[QT], gap[QT], l[QT];
#pragma unroll
    for (int qs = 0; qs < QT; ++qs) { ref[qs] = 0.f; gap[qs] = -INFINITY; l[qs] = 0.f; }
    // e4m3: weights are p_j times V's row scale relative to a power of two above every scale that the column has seen so far, so
    // that they stay within fp16's range whatever the scales are; the accumulators are multiplied by it at the end.  `vexp`: the
    // largest exponent field of those scales, so that the power of two is 2^(vexp - 126)
    int vexp[QT];
#pragma unroll
    for (int qs = 0; qs < QT; ++qs) vexp[qs] = 0;
    // which of the 64 keys from node `first` on (negative: kept tokens before it) the row of node `n` sees
    auto visible = [&](int n, int first) -> unsigned long long {
        if (first <= -64) return ~0ull;
        if (!p.mask) {
            const int c = n - first + 1;
            return c <= 0 ? 0ull : c >= 64 ? ~0ull : (1ull << c) - 1;
        }
        const unsigned* words = p.mask + (long)(w.row0 + n) * p.mask_words;
        auto word = [&](int i) -> unsigned long long { return i < p.mask_words ? words[i] : 0u; };
        if (first < 0) return ((word(0) | word(1) << 32) << -first) | ((1ull << -first) - 1);
        const int i = first >> 5, sh = first & 31;
        const unsigned long long x = (word(i) | word(i + 1) << 32) >> sh;
        return sh ? x | word(i + 2) << (64 - sh) : x;
    };
    if (tid == 0) lds.bad_v = 0;
    if (n_tiles > 0) {
        load_page(key0);
        load_tile(key0);
        load_page(key0 + KT);
    }
    // the queries are here before the first product: a wait for them inside the loop would be one for all loads in flight
#pragma unroll
    for (int qs = 0; qs < QT; ++qs)
#pragma unroll
        for (int s = 0; s < D / 32; ++s) asm volatile("" : "+v"(qf[qs][s]));
    for (int it = 0; it < n_tiles; ++it) {
        const int kv0 = key0 + it * KT;
        __syncthreads();                                     // the previous tile has been read
        store_tile(it);
        __syncthreads();
        if (it + 1 < n_tiles) {
            load_tile(kv0 + KT);
            load_page(kv0 + 2 * KT);
        }
        __builtin_amdgcn_sched_barrier(0);                   // phases stay apart: mixed, their operands do not fit the registers
        if (!active) continue;
        // ---- S^T
        float4v sc[NK][QT];
#pragma unroll
        for (int i = 0; i < NK; ++i) {
            const int krow = (wk * NK + i) * 16 + fr;
#pragma unroll
            for (int qs = 0; qs < QT; ++qs) sc[i][qs] = float4v{0, 0, 0, 0};
#pragma unroll
            for (int s = 0; s < D / 32; ++s) {
                const short8v kf = *reinterpret_cast<const short8v*>(&ldsK[k_at<D>(krow, s * 4 + fg)]);
#pragma unroll
                for (int qs = 0; qs < QT; ++qs) sc[i][qs] = Mat<T>::mma32(kf, qf[qs][s], sc[i][qs]);
            }
        }
        // six operands on their way to the products throughout (left alone, the scheduler waits for every second one)
        interleave<NK * (D / 32), QT, 6, 1>();
        __builtin_amdgcn_sched_barrier(0);
        // ---- the keys that a column does not see
        const int4 there = *reinterpret_cast<const int4*>(lds.page_ok);
        const bool edge = kv0 + KT > kept || kv0 + KT > key1 || !(there.x && there.y && there.z && there.w);
        // ---- exponents of the weights: score * scale * log2 e (e4m3: times K's row scale) - ref
#pragma unroll
        for (int i = 0; i < NK; ++i) {
            float4v by = float4v{to_log2, to_log2, to_log2, to_log2};
            if constexpr (KV8) by = *reinterpret_cast<const float4v*>(&lds.scales[0][(wk * NK + i) * 16 + 4 * fg]);      // (all of it)
#pragma unroll
            for (int qs = 0; qs < QT; ++qs)
#pragma unroll
                for (int r = 0; r < 4; ++r) sc[i][qs][r] = fmaf(sc[i][qs][r], by[r], -ref[qs]);
        }
        if (edge) {
            const int first = kv0 - kept, limit = key1 - kv0;                 // node of the tile's first key (may be negative)
            unsigned long long exist = limit >= 64 ? ~0ull : (1ull << limit) - 1;
            if (!there.x) exist &= ~0xffffull;
            if (!there.y) exist &= ~0xffff0000ull;
            if (!there.z) exist &= ~0xffff00000000ull;
            if (!there.w) exist &= ~0xffff000000000000ull;
#pragma unroll
            for (int qs = 0; qs < QT; ++qs) {
                const unsigned long long sees = visible(node[qs], first) & exist;
#pragma unroll
                for (int i = 0; i < NK; ++i)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (!(sees >> ((wk * NK + i) * 16 + 4 * fg + r) & 1)) sc[i][qs][r] = -INFINITY;
            }
        }
        // ---- online softmax.  A column's reference rises only when an exponent exceeds kGap, so that weights stay below 2^kGap
        // and the lanes of a column need not agree on a maximum in every tile.
        bool lift = false;
        float top[QT];
#pragma unroll
        for (int qs = 0; qs < QT; ++qs) {
            top[qs] = -INFINITY;
#pragma unroll
            for (int i = 0; i < NK; ++i) top[qs] = max3(max3(top[qs], sc[i][qs][0], sc[i][qs][1]), sc[i][qs][2], sc[i][qs][3]);
            lift = lift || top[qs] > gap[qs];
        }
        float big[QT];                                       // e4m3: V's largest row scale in this tile among the keys that a column sees
        if constexpr (KV8) {
            if (kv0 + KT > kept) {
#pragma unroll
                for (int qs = 0; qs < QT; ++qs) {
                    big[qs] = 0.f;
#pragma unroll
                    for (int i = 0; i < NK; ++i) {
                        const float4v s4 = *reinterpret_cast<const float4v*>(&lds.scales[1][(wk * NK + i) * 16 + 4 * fg]);
#pragma unroll
                        for (int r = 0; r < 4; ++r) big[qs] = fmaxf(big[qs], sc[i][qs][r] == -INFINITY ? 0.f : s4[r]);
                    }
                    big[qs] = column_max(big[qs]);
                }
            } else {                                         // kept tokens: every column sees all of them (0 where there is none)
                float all = 0.f;
#pragma unroll
                for (int i = 0; i < NK; ++i) {
                    const float4v s4 = *reinterpret_cast<const float4v*>(&lds.scales[1][(wk * NK + i) * 16 + 4 * fg]);
                    all = fmaxf(all, fmaxf(fmaxf(s4[0], s4[1]), fmaxf(s4[2], s4[3])));
                }
                all = column_max(all);
#pragma unroll
                for (int qs = 0; qs < QT; ++qs) big[qs] = all;
            }
#pragma unroll
            for (int qs = 0; qs < QT; ++qs) lift = lift || exponent(big[qs]) > vexp[qs];
        }
        if (__any(lift)) {                                   // wave-uniform; a column moves for what it sees itself only
#pragma unroll
            for (int qs = 0; qs < QT; ++qs) {
                float f = 1.f;
                if constexpr (KV8) {
                    const int now = max(exponent(big[qs]), vexp[qs]);
                    f = __builtin_ldexpf(1.f, vexp[qs] - now);
                    vexp[qs] = now;
                }
                const float up = column_max(top[qs]);
                const bool rises = up > gap[qs];
                const float to = ref[qs] + (rises ? up - Mat<T>::kLow : 0.f), d = to - ref[qs];
                const float alpha = gap[qs] > 0.f ? __builtin_amdgcn_exp2f(-d) : 1.f;
                if (rises) gap[qs] = Mat<T>::kGap;
                ref[qs] = to;
#pragma unroll
                for (int i = 0; i < NK; ++i)
#pragma unroll
                    for (int r = 0; r < 4; ++r) sc[i][qs][r] -= d;
                l[qs] *= alpha;
#pragma unroll
                for (int d = 0; d < ND; ++d) { o[d][qs][0] *= alpha * f; o[d][qs][1] *= alpha * f; o[d][qs][2] *= alpha * f; o[d][qs][3] *= alpha * f; }
            }
        }
        auto weigh = [&](auto some_unseen) {
            constexpr bool EDGE = decltype(some_unseen)::value;
#pragma unroll
            for (int i = 0; i < NK; ++i) {
                float4v vs4 = float4v{1, 1, 1, 1};
                if constexpr (KV8) {
                    vs4 = *reinterpret_cast<const float4v*>(&lds.scales[1][(wk * NK + i) * 16 + 4 * fg]);
                    if constexpr (!EDGE)                     // kept tokens only so far: the columns' references are the same
#pragma unroll
                        for (int r = 0; r < 4; ++r) vs4[r] = __builtin_ldexpf(vs4[r], 126 - vexp[0]);
                }
#pragma unroll
                for (int qs = 0; qs < QT; ++qs)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const float e = __builtin_amdgcn_exp2f(sc[i][qs][r]);
                        l[qs] += e;                          // of this lane's keys; the column's sum is formed at the end
                        if constexpr (!KV8) sc[i][qs][r] = e;
                        else if constexpr (!EDGE) sc[i][qs][r] = e * vs4[r];
                        else sc[i][qs][r] = e == 0.f ? 0.f : e * __builtin_ldexpf(vs4[r], 126 - vexp[qs]);        // whatever the scale of an unseen key
                    }
            }
        };
        if (KV8 && edge) weigh(std::true_type{});
        else weigh(std::false_type{});
        __builtin_amdgcn_sched_barrier(0);
        // ---- O^T += V^T P^T.  The weights are rounded once to T (half a step of T, for fp16 down to 2^-24 of the largest); the sum
        // above is of the unrounded ones.
        const short* const vt = ldsV;
        {
            typedef short4v __attribute__((address_space(3)))* lds4;
            if constexpr (NK == 1) {
                short4v pf[QT];
#pragma unroll
                for (int qs = 0; qs < QT; ++qs)
                    pf[qs] = short4v{bits_of<T>(sc[0][qs][0]), bits_of<T>(sc[0][qs][1]), bits_of<T>(sc[0][qs][2]), bits_of<T>(sc[0][qs][3])};
#pragma unroll
                for (int d = 0; d < ND; ++d) {
                    const short4v vf = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(vt + v_at<D>(wk * 16 + 4 * fg + (fr >> 2), d * 16 + 4 * (fr & 3))));
#pragma unroll
                    for (int qs = 0; qs < QT; ++qs) o[d][qs] = Mat<T>::mma16(vf, pf[qs], o[d][qs]);
                }
            } else {
                short8v pf[QT][NK / 2 ? NK / 2 : 1];
#pragma unroll
                for (int qs = 0; qs < QT; ++qs)
#pragma unroll
                    for (int s = 0; s < NK / 2; ++s)
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            pf[qs][s][r] = bits_of<T>(sc[2 * s][qs][r]);
                            pf[qs][s][4 + r] = bits_of<T>(sc[2 * s + 1][qs][r]);
                        }
#pragma unroll
                for (int d = 0; d < ND; ++d)
#pragma unroll
                    for (int s = 0; s < NK / 2; ++s) {       // element j of step s is key 32 s + 16 (j >> 2) + 4 fg + (j & 3) of the wave's
                        const int krow = wk * NK * 16 + 32 * s + 4 * fg + (fr >> 2);
                        const short4v lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(vt + v_at<D>(krow, d * 16 + 4 * (fr & 3))));
                        const short4v hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(vt + v_at<D>(krow + 16, d * 16 + 4 * (fr & 3))));
                        const short8v vf = short8v{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
#pragma unroll
                        for (int qs = 0; qs < QT; ++qs) o[d][qs] = Mat<T>::mma32(vf, pf[qs][s], o[d][qs]);
                    }
            }
            interleave<NK == 1 ? ND : ND * NK / 2, QT, 4, NK == 1 ? 1 : 2>();
        }
    }

    // ---- join the waves that split the keys, then normalise and store, or leave the partial result to the second launch
    float m[QT];                                             // the references, -inf for columns that saw nothing
#pragma unroll
    for (int qs = 0; qs < QT; ++qs) m[qs] = gap[qs] > 0.f ? ref[qs] : -INFINITY;
#pragma unroll
    for (int qs = 0; qs < QT; ++qs) {
        l[qs] = column_sum(l[qs]);
        if constexpr (KV8)
#pragma unroll
            for (int d = 0; d < ND; ++d)
#pragma unroll
                for (int r = 0; r < 4; ++r) o[d][qs][r] = __builtin_ldexpf(o[d][qs][r], vexp[qs] - 126);
    }
    constexpr int DW = ND / WK;                              // 16-dim tiles of the result that a wave ends up with
    const int d0 = WK > 1 ? wk * DW : 0;
    if constexpr (WK > 1) {
        if (fg == 0)
#pragma unroll
            for (int qs = 0; qs < QT; ++qs) { lds.red_m[wave][qs * 16 + fr] = m[qs]; lds.red_l[wave][qs * 16 + fr] = l[qs]; }
        float* const ex = reinterpret_cast<float*>(lds.tiles);
#pragma unroll
        for (int qs = 0; qs < QT; ++qs) {
            __syncthreads();                                 // the tile's memory is free; all maxima are there
            float all = -INFINITY, sum = 0.f;
#pragma unroll
            for (int k = 0; k < WK; ++k) all = fmaxf(all, lds.red_m[wq * WK + k][qs * 16 + fr]);
            const float ref = all == -INFINITY ? 0.f : all;
#pragma unroll
            for (int k = 0; k < WK; ++k) sum += lds.red_l[wq * WK + k][qs * 16 + fr] * __builtin_amdgcn_exp2f(lds.red_m[wq * WK + k][qs * 16 + fr] - ref);
            const float f = __builtin_amdgcn_exp2f(m[qs] - ref);
            m[qs] = all; l[qs] = sum;
            // a wave's O as [16 columns][D] floats, chunks of four exchanged by the column; then wave k of the group adds up
            // the head dims [k D / WK, ...) of all of its waves, in wave order
#pragma unroll
            for (int d = 0; d < ND; ++d)
                *reinterpret_cast<float4v*>(&ex[(wave * 16 + fr) * D + ((d * 4 + fg) ^ fr) * 4]) =
                    float4v{o[d][qs][0] * f, o[d][qs][1] * f, o[d][qs][2] * f, o[d][qs][3] * f};
            __syncthreads();
#pragma unroll
            for (int d = 0; d < DW; ++d) {
                float4v sum4 = float4v{0, 0, 0, 0};
#pragma unroll
                for (int k = 0; k < WK; ++k) {
                    const float4v x = *reinterpret_cast<const float4v*>(&ex[((wq * WK + k) * 16 + fr) * D + (((d0 + d) * 4 + fg) ^ fr) * 4]);
#pragma unroll
                    for (int r = 0; r < 4; ++r) sum4[r] += x[r];
                }
                o[d][qs] = sum4;
            }
        }
    }
    if constexpr (WK == 1) __syncthreads();
    if (lds.bad_v) {                                         // (written before the last barrier)
        // from the first tile that store_tile held something back in: kept tokens share it with the step's rows
        for (int key = max(key0, min(kept, key1) & ~(KT - 1)); key < key1; ++key) {
            const int pgid = pages[key >> p.c.page_shift];
            if (pgid < 0 || pgid >= p.c.n_pages) continue;
            const long at = (long)pgid * p.c.page_stride + w.g * p.c.head_stride + (long)(key & page_mask) * p.c.token_stride;
#pragma unroll
            for (int qs = 0; qs < QT; ++qs) {
                if (!(visible(node[qs], key - kept) & 1)) continue;
#pragma unroll
                for (int d = 0; d < DW; ++d)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const long e = at + (d0 + d) * 16 + 4 * fg + r;
                        float x;
                        if constexpr (KV8) x = (static_cast<const uint8_t*>(p.c.v)[e] & 0x7f) == 0x7f ? __uint_as_float(0x7fc00000u) : 0.f;
                        else x = (float)static_cast<const T*>(p.c.v)[e];
                        if (!(fabsf(x) < INFINITY)) o[d][qs][r] += x;
                    }
            }
        }
    }
#pragma unroll
    for (int qs = 0; qs < QT; ++qs) {
        const int c = w.col0 + (wq * QT + qs) * 16 + fr;
        if (c >= w.cols) continue;
        if (w.pieces <= 1) {
            const float inv = l[qs] == 0.f ? 0.f : 1.f / l[qs];               // (a NaN sum stays NaN)
            short* dst = static_cast<short*>(p.out) + (long)(w.row0 + node[qs]) * p.out_row + (long)(w.g * group + c - node[qs] * group) * p.out_head;
#pragma unroll
            for (int d = 0; d < DW; ++d)
                *reinterpret_cast<short4v*>(dst + (d0 + d) * 16 + 4 * fg) =
                    short4v{bits_of<T>(o[d][qs][0] * inv), bits_of<T>(o[d][qs][1] * inv), bits_of<T>(o[d][qs][2] * inv), bits_of<T>(o[d][qs][3] * inv)};
        } else {
            const long slot = ((long)w.unit * p.c.heads + w.g) * (p.max_nodes * group) + c;
            float* po = p.workspace + slot * D;
#pragma unroll
            for (int d = 0; d < DW; ++d) *reinterpret_cast<float4v*>(po + (d0 + d) * 16 + 4 * fg) = o[d][qs];
            if (fg == 0 && wk == 0) {
                float* ml = p.workspace + (long)p.n_units * p.c.heads * (p.max_nodes * group) * D + slot * 2;
                ml[0] = m[qs]; ml[1] = l[qs];
            }
        }
    }
}

// Workgroup -> (unit, K/V head, column block): the blocks of one (unit, head) are 8 ids apart, on the same XCD, so that its K/V
// rows come from that XCD's L2 after the first of them.  False: nothing to do.
__device__ __forceinline__ bool find_work(const TreeAttnParams& p, int n_blocks, int group, int block, Work& w) {
    const int pair = blockIdx.x / (8 * n_blocks) * 8 + (blockIdx.x & 7), cb = (blockIdx.x >> 3) % n_blocks;
    w.unit = pair / p.c.heads; w.g = pair - w.unit * p.c.heads;
    if (w.unit >= p.n_units) return false;
    int4 u = reinterpret_cast<const int4*>(p.units)[w.unit];
    if (u.w > 1 && !p.workspace) {                           // no room for partial results: the first unit takes the whole request
        if (u.y > 0) return false;
        u.z = 0x7fffffff; u.w = 1;
    }
    w.b = u.x; w.pieces = u.w;
    if (w.b < 0 || w.b >= p.batch) return false;
    w.row0 = max(0, p.row_start[w.b]);
    w.nodes = min(min(p.row_start[w.b + 1], p.rows) - w.row0, p.max_nodes);
    w.cols = w.nodes * group;
    w.col0 = cb * block;
    if (w.col0 >= w.cols) return false;
    w.kept = max(0, p.kept[w.b]);
    // keys: the unit's, none behind the last one that a row of this block can see
    const int last_node = p.mask ? w.nodes - 1 : min(w.nodes - 1, (w.col0 + block - 1) / group);
    w.key0 = max(0, u.y) & ~(KT - 1);
    w.key1 = (int)min((long)min(u.z, p.max_pages << p.c.page_shift), (long)w.kept + last_node + 1);
    return true;
}
// At most 16 columns a workgroup: a stream of K/V through the compute units; registers are held down for more workgroups on each
// (8 requests of 1 row over 207 k tokens of 8 x 128 e4m3: 84 us with four, 87 with three).
template <typename T, bool KV8, int D>
__global__ __launch_bounds__(256, D == 64 || KV8 ? 4 : 3) void tree_attn_narrow_kernel(TreeAttnParams p, int n_blocks, int group) {
    __shared__ Shared<KV8, D> lds;
    Work w;
    if (find_work(p, n_blocks, group, 16, w)) attend<T, KV8, D, 1, 4>(p, group, w, lds);
}
// Up to 128 columns a workgroup; how the four waves share columns and keys goes by the columns that this request has left: a wave
// without columns would only stage.  (Both launches of the wide trees, where it was 142 us: a wave of 64 columns reads half as much
// LDS per product but spills, 250; eight waves of 256 columns read a request's rows once, but one workgroup per CU waits at its
// barriers, 155; eight of 16 columns each 164; queries in LDS and two tiles in flight 156.)
template <typename T, bool KV8, int D>
__global__ __launch_bounds__(256, 2) void tree_attn_wide_kernel(TreeAttnParams p, int n_blocks, int group) {
    __shared__ Shared<KV8, D> lds;
    Work w;
    if (!find_work(p, n_blocks, group, 128, w)) return;
    const int left = w.cols - w.col0;
    if (left <= 32) attend<T, KV8, D, 2, 4>(p, group, w, lds);
    else if (left <= 64) attend<T, KV8, D, 2, 2>(p, group, w, lds);
    else attend<T, KV8, D, 2, 1>(p, group, w, lds);
}

// Rows of requests that were cut: the units' partial results, weighted by their maxima.  D / 4 lanes hold a (row, query head),
// four head dims each.  SHARE: a workgroup per pair whose groups of lanes take the units in turn and are joined through LDS;
// else every group has a pair of its own.  Bound by the bytes of the partial results (63 MB of wide trees in 14.5 us, 67 MB of
// chains in 15.9: 4.3 TB/s); four loads ahead of a group that is alone with its pair (eight: 16.1 and 15.3 us), eight of one that shares.
template <typename T, int D, bool SHARE>
__global__ __launch_bounds__(256) void tree_join_kernel(TreeAttnParams p, int group) {
    constexpr int LANES = D / 4, GROUPS = 256 / LANES, AHEAD = SHARE ? 8 : 4, STEP = SHARE ? GROUPS : 1;
    __shared__ float red_m[GROUPS], red_l[GROUPS];
    __shared__ __attribute__((aligned(16))) float red_o[SHARE ? GROUPS : 1][D];
    const int mine = threadIdx.x / LANES, d = (threadIdx.x % LANES) * 4;
    const long id = SHARE ? blockIdx.x : (long)blockIdx.x * GROUPS + mine;
    const int h = (int)(id % p.heads);
    const long bi = id / p.heads;
    const int b = (int)(bi / p.max_nodes), i = (int)(bi - (long)b * p.max_nodes);
    if (b >= p.batch) return;
    const int u0 = p.unit_start[b], n = p.unit_start[b + 1] - u0, r0 = p.row_start[b], row = r0 + i;
    if (n < 2 || u0 < 0 || u0 + n > p.n_units || r0 < 0 || row >= p.row_start[b + 1] || row >= p.rows) return;
    const int g = h / group;
    const long cols = (long)p.max_nodes * group, step = p.c.heads * cols;               // slots from one unit to the next
    const long first = ((long)u0 * p.c.heads + g) * cols + (long)i * group + (h - g * group);
    const float* const po = p.workspace;
    const float* const ml = p.workspace + (long)p.n_units * step * D;
    float m = -INFINITY, l = 0.f;
    float4v acc = float4v{0, 0, 0, 0};
    auto add = [&](float um, float ul, float4v x) {
        const float mn = fmaxf(m, um), ref = mn == -INFINITY ? 0.f : mn;
        const float fo = __builtin_amdgcn_exp2f(m - ref), fu = __builtin_amdgcn_exp2f(um - ref);
        m = mn;
        l = l * fo + ul * fu;
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[r] = acc[r] * fo + x[r] * fu;
    };
    for (int u = SHARE ? mine : 0; u < n; u += STEP * AHEAD) {
        float um[AHEAD], ul[AHEAD];
        float4v x[AHEAD];
#pragma unroll
        for (int a = 0; a < AHEAD; ++a) {
            const long slot = first + min(u + a * STEP, n - 1) * step;
            const float2 two = *reinterpret_cast<const float2*>(ml + slot * 2);
            um[a] = two.x; ul[a] = two.y;
            x[a] = *reinterpret_cast<const float4v*>(po + slot * D + d);
        }
#pragma unroll
        for (int a = 0; a < AHEAD; ++a)
            if (u + a * STEP < n) add(um[a], ul[a], x[a]);
    }
    if constexpr (SHARE) {
        if (d == 0) { red_m[mine] = m; red_l[mine] = l; }
        *reinterpret_cast<float4v*>(&red_o[mine][d]) = acc;
        __syncthreads();
        if (mine) return;
        m = -INFINITY; l = 0.f; acc = float4v{0, 0, 0, 0};
#pragma unroll
        for (int k = 0; k < GROUPS; ++k) add(red_m[k], red_l[k], *reinterpret_cast<const float4v*>(&red_o[k][d]));
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    *reinterpret_cast<short4v*>(static_cast<short*>(p.out) + (long)row * p.out_row + (long)h * p.out_head + d) =
        short4v{bits_of<T>(acc[0] * inv), bits_of<T>(acc[1] * inv), bits_of<T>(acc[2] * inv), bits_of<T>(acc[3] * inv)};
}

template <typename T, bool KV8, int D>
hipError_t launch_tree_t(const TreeAttnParams& p, hipStream_t s) {
    const int group = p.heads / p.c.heads;
    const long cols = (long)p.max_nodes * group;
    // 24 chains over 138 k tokens, 8 K/V heads of 128, narrow / wide: 16 columns 115 / 127 us bf16, 73 / 94 us e4m3; 24 columns, two
    // narrow blocks that read the rows twice, 166 / 131 and 106 / 96 us
    const int block = cols <= 16 ? 16 : 128;
    const int n_blocks = (int)((cols + block - 1) / block);
    const long pairs = ((long)p.n_units * p.c.heads + 7) / 8 * 8;
    const unsigned grid = (unsigned)(pairs * n_blocks);
    const hipError_t e = launch(block == 16 ? tree_attn_narrow_kernel<T, KV8, D> : tree_attn_wide_kernel<T, KV8, D>, grid, 256, s, p, n_blocks, group);
    if (e == hipSuccess && p.n_units > p.batch) {
        // few rows have few waves: a workgroup shares a row's units then (8 requests of 1 row, 32 heads, up to 80 units: 15.5 ->
        // 5.1 us); for many rows with a pair on every group of lanes it is faster without (32 trees, 8 units at most: 44 us shared)
        const long pairs = (long)p.batch * p.max_nodes * p.heads, groups = 256 / (D / 4);
        if (pairs <= 4096) return launch(tree_join_kernel<T, D, true>, (unsigned)pairs, 256, s, p, group);
        return launch(tree_join_kernel<T, D, false>, (unsigned)((pairs + groups - 1) / groups), 256, s, p, group);
    }
    return e;
}

}  // namespace

// Partial results of every unit; none where there are no more units than requests (no request is cut then).
long tree_attn_workspace(int n_units, int batch, int kv_heads, int group, int max_nodes, int dim) {
    return n_units > batch ? (long)n_units * kv_heads * max_nodes * group * (dim + 2) * 4 : 0;
}

hipError_t launch_tree_attention(const TreeAttnParams& p, hipStream_t s) {
    if (!p.n_units || !p.batch || !p.max_nodes) return hipSuccess;
    const bool kv8 = p.c.ks != nullptr;
    if (p.dim == 64) {
        if (p.bf16) { if (kv8) return launch_tree_t<bf16, true, 64>(p, s); else return launch_tree_t<bf16, false, 64>(p, s); }
        else { if (kv8) return launch_tree_t<f16, true, 64>(p, s); else return launch_tree_t<f16, false, 64>(p, s); }
    } else {
        if (p.bf16) { if (kv8) return launch_tree_t<bf16, true, 128>(p, s); else return launch_tree_t<bf16, false, 128>(p, s); }
        else { if (kv8) return launch_tree_t<f16, true, 128>(p, s); else return launch_tree_t<f16, false, 128>(p, s); }
    }
}

}  // namespace mw
