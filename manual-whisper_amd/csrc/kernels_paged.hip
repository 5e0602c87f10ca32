// Operators of drafted decoding over a K/V cache in pages, for gfx950: the plan of a step (block tables, slot map, tree
// masks, work units), the write of K/V rows into pages, acceptance of a tree of drafted tokens against the logits, and the
// compaction of the accepted rows.  The attention over the pages is in kernels_tree.hip.
//
// All of them are bound by HBM or, at the sizes of one decode step, by the latency of a launch: each is one launch (accept:
// two), nothing is allocated, nothing waits for the host, and every index that comes from device memory is checked
// against its buffer before it is used.
//
// Times are medians of launches in a graph, three input sets in turn; "a where it is b" compares builds of one session by their
// smallest times, which lie lower, by a third for the smallest launches.
#include "mw_kernels.h"

#include <algorithm>

namespace mw {

namespace {

// -------------------------------------------------------------------------------------------- plan
// Every workgroup computes the prefix sums over the requests for itself (at most 2048 requests, a few KB that stay in L2)
// and then does its share of the rows, new pages, returned pages, tree masks and units: one launch without any exchange
// between workgroups.  A page popped from a stack entry that this very step pushes is looked up in the table of the request
// that gives it back, so pops never wait for pushes.  Bound by latency: round trips to memory and the scans' barriers.  Sums go
// through a wave by DPP and across waves once (with shuffles and a search per row: 13.4 us where it is 8.2).  16 trees of 8 nodes
// 8.0 us (3 KB), 256 chains of 166 k rows in all 7.9 us (2 MB).
constexpr int kPlanThreads = 1024, kPlanWaves = kPlanThreads / 64;
constexpr int kPlanPer = kPlanMaxBatch / kPlanThreads;       // requests per thread of the prefix sums
constexpr unsigned kFull = 1u << 30;                         // sums of counts stop here: above every capacity, and two of them fit 32 bits

__device__ __forceinline__ unsigned sat_add(unsigned a, unsigned b) { return min(a + b, kFull); }
template <int CTRL, int ROWS> __device__ __forceinline__ unsigned scan_step(unsigned v) {
    return sat_add(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xf, false));
}
__device__ __forceinline__ unsigned wave_scan(unsigned v) {  // inclusive, over 64 lanes: within rows of 16, then across them
    v = scan_step<0x111, 0xf>(v);
    v = scan_step<0x112, 0xf>(v);
    v = scan_step<0x114, 0xf>(v);
    v = scan_step<0x118, 0xf>(v);
    v = scan_step<0x142, 0xa>(v);
    return scan_step<0x143, 0xc>(v);
}
// Exclusive prefixes of N counts over the workgroup's threads, and their totals.  `ws`: LDS of its own for this call.
template <int N> __device__ __forceinline__ void block_scan(unsigned (&v)[N], unsigned (&total)[N], unsigned (*ws)[kPlanWaves]) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int k = 0; k < N; ++k) {
        const unsigned inc = wave_scan(v[k]);
        if (lane == 63) ws[k][wave] = inc;
        const unsigned before = (unsigned)__shfl_up((int)inc, 1);
        v[k] = lane ? before : 0u;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < N; ++k) {
        const unsigned w = wave_scan(lane < kPlanWaves ? ws[k][lane] : 0u);
        total[k] = (unsigned)__shfl((int)w, kPlanWaves - 1);
        const unsigned before = (unsigned)__shfl((int)w, max(wave - 1, 0));
        v[k] = sat_add(v[k], wave ? before : 0u);
    }
}
// number of entries of the ascending array a[0..n) that are <= x
__device__ __forceinline__ int count_le(const int* a, int n, int x) {
    int lo = 0, hi = n;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (a[mid] <= x) lo = mid + 1; else hi = mid;
    }
    return lo;
}

__global__ __launch_bounds__(kPlanThreads) void paged_plan_kernel(PlanParams p) {
    __shared__ unsigned ws[4][kPlanWaves];
    __shared__ unsigned long long lens[kPlanWaves];
    __shared__ int start[kPlanMaxBatch + 1];                 // first row of each request
    __shared__ int gend[kPlanMaxBatch];                      // new pages wanted up to and including each request
    __shared__ int bend[kPlanMaxBatch];                      // pages given back up to and including each request
    __shared__ int kept_of[kPlanMaxBatch], held_of[kPlanMaxBatch];
    __shared__ int uend[kPlanMaxBatch + 1];                  // units before each request (the last workgroup's)
    __shared__ unsigned char state[kPlanMaxBatch];           // 1 = valid, 2 = admitted
    __shared__ unsigned anc[32 * kPlanMaxWords][kPlanMaxWords + 1];
    __shared__ int jump[32 * kPlanMaxWords];
    const int tid = threadIdx.x, B = p.batch;
    const int page = 1 << p.page_shift;

    // ---- prefix sums over the requests
    int kept[kPlanPer], fresh[kPlanPer], held[kPlanPer];
    unsigned rows[1] = {0}, total_rows[1];
    const int n_free = min(max(p.n_free_in[0], 0), p.n_pages);
#pragma unroll
    for (int i = 0; i < kPlanPer; ++i) {
        const int b = tid * kPlanPer + i;
        kept[i] = b < B ? p.kept[b] : 0;
        fresh[i] = b < B ? p.fresh[b] : 0;
        held[i] = b < B ? min(max(p.pages_in[b], 0), p.max_pages) : 0;
        rows[0] = sat_add(rows[0], min((unsigned)max(fresh[i], 0), kFull));
    }
    block_scan<1>(rows, total_rows, ws);
    int need[kPlanPer];
    unsigned grow[kPlanPer], back[kPlanPer], both[2] = {0, 0}, total[2];
    bool valid[kPlanPer];
#pragma unroll
    for (int i = 0; i < kPlanPer; ++i) {
        const int b = tid * kPlanPer + i;
        if (b < B) { start[b] = (int)rows[0]; kept_of[b] = kept[i]; held_of[b] = held[i]; }
        rows[0] = sat_add(rows[0], min((unsigned)max(fresh[i], 0), kFull));
        const long pages = ((long)kept[i] + fresh[i] + page - 1) >> p.page_shift;
        valid[i] = b < B && kept[i] >= 0 && fresh[i] >= 0 && pages <= p.max_pages && rows[0] <= (unsigned)p.rows &&
                   (!p.parents || fresh[i] <= 32 * p.mask_words);
        need[i] = valid[i] ? (int)pages : 0;
        grow[i] = valid[i] && need[i] > held[i] ? need[i] - held[i] : 0;
        back[i] = valid[i] && need[i] < held[i] ? held[i] - need[i] : 0;
        both[0] = sat_add(both[0], grow[i]); both[1] = sat_add(both[1], back[i]);
    }
    if (tid == 0) start[B] = (int)total_rows[0];
    block_scan<2>(both, total, ws + 1);
    const unsigned stack = min(n_free + total[1], (unsigned)p.n_pages);      // pages to be had in this step: no more than there are
    unsigned used = 0;                                       // growing requests are admitted up to some point and none behind it
    unsigned long long len_sum = 0;
    int len[kPlanPer];
#pragma unroll
    for (int i = 0; i < kPlanPer; ++i) {
        const int b = tid * kPlanPer + i;
        both[0] = sat_add(both[0], grow[i]); both[1] = sat_add(both[1], back[i]);
        const bool admitted = valid[i] && (grow[i] == 0 || both[0] <= stack);
        if (b < B) {
            gend[b] = (int)both[0]; bend[b] = (int)both[1];
            state[b] = (valid[i] ? 1 : 0) | (admitted ? 2 : 0);
            if (blockIdx.x == 0) {
                p.row_start[b] = start[b];
                p.admitted[b] = admitted;
                p.pages_out[b] = admitted ? need[i] : held[i];
            }
        }
        if (admitted && grow[i]) used = both[0];
        len[i] = admitted && fresh[i] > 0 ? kept[i] + fresh[i] : 0;
        len_sum += (unsigned)len[i];
    }
    // largest `used`, sum of the lengths
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        used = max(used, (unsigned)__shfl_xor((int)used, d));
        len_sum += __shfl_xor(len_sum, d);
    }
    if ((tid & 63) == 0) { ws[3][tid >> 6] = used; lens[tid >> 6] = len_sum; }
    __syncthreads();
    if (blockIdx.x == 0 && tid == 0) {
        for (int w = 1; w < kPlanWaves; ++w) used = max(used, ws[3][w]);
        p.row_start[B] = start[B];
        p.n_free_out[0] = (int)(stack - used);
    }

    // page on top of entry `e` of the stack as this step's pushes leave it
    auto stack_page = [&](int e) -> int {
        if (e < n_free) return p.free_list[e];
        const int k = e - n_free, b = min(count_le(bend, B, k), B - 1);
        const int first = held_of[b] - (bend[b] - (b ? bend[b - 1] : 0));                // what request b keeps
        return p.table[(long)b * p.table_stride + first + (k - (b ? bend[b - 1] : 0))];
    };
    // page `n` of admitted request b, old or new
    auto page_of = [&](int b, int n) -> int {
        const int h = held_of[b];
        if (n < h) return p.table[(long)b * p.table_stride + n];
        return stack_page((int)stack - 1 - ((b ? gend[b - 1] : 0) + (n - h)));
    };
    auto slot_of = [&](int b, int place) -> long {
        const int pg = page_of(b, place >> p.page_shift);
        return pg >= 0 ? ((long)pg << p.page_shift) + (place & (page - 1)) : -1;
    };
    const long threads = (long)gridDim.x * kPlanThreads, me = (long)blockIdx.x * kPlanThreads + tid;

    // ---- trees: a workgroup per request.  Ancestors by pointer doubling: node i starts with {i} and its parent; a round adds
    // the ancestors that its jump target has gathered and jumps on from there: log2(depth) rounds, all nodes at once.
    if (p.parents && (int)blockIdx.x < B && (state[blockIdx.x] & 1)) {
        const int b = blockIdx.x, n = start[b + 1] - start[b], W = p.mask_words;
        const long r = start[b] + tid;
        if (tid < n) {
            int up = p.parents[r];
            if (up < 0 || up >= tid) up = -1;                // a parent is an earlier node of the same tree
            jump[tid] = up;
            for (int w = 0; w < W; ++w) anc[tid][w] = (tid >> 5) == w ? 1u << (tid & 31) : 0u;
            p.slots[r] = (state[b] & 2) ? slot_of(b, kept_of[b] + tid) : -1;
        }
        bool more = true;
        while (more) {
            __syncthreads();
            unsigned add[kPlanMaxWords];
            int next = -1;
            if (tid < n && jump[tid] >= 0) {
                const int j = jump[tid];
                next = jump[j];
#pragma unroll
                for (int w = 0; w < kPlanMaxWords; ++w) add[w] = w < W ? anc[j][w] : 0u;
            }
            __syncthreads();
            if (tid < n && jump[tid] >= 0) {
#pragma unroll
                for (int w = 0; w < kPlanMaxWords; ++w)
                    if (w < W) anc[tid][w] |= add[w];
                jump[tid] = next;
            }
            more = __syncthreads_or(tid < n && next >= 0);
        }
        if (tid < n) {
            int depth = -1;
            for (int w = 0; w < W; ++w) { p.mask[r * W + w] = anc[tid][w]; depth += __popc(anc[tid][w]); }
            p.positions[r] = kept_of[b] + depth;
        }
    }

    // ---- rows of chains; in a step of trees the rows that belong to none of them
    for (long r = me; r < p.rows; r += threads) {
        long slot = -1;
        int pos = -1;
        if (r < start[B]) {
            const int b = count_le(start, B + 1, (int)r) - 1;
            if (state[b] & 1) {
                if (p.parents) continue;
                pos = kept_of[b] + (int)r - start[b];
            }
            if (state[b] & 2) slot = slot_of(b, pos);
        }
        p.slots[r] = slot;
        p.positions[r] = pos;
        if (p.parents)
            for (int w = 0; w < p.mask_words; ++w) p.mask[r * p.mask_words + w] = 0;
    }
    // ---- new pages into the tables, returned pages onto the stack
    const long grown = min(total[0], stack);
    for (long k = me; k < grown; k += threads) {
        const int b = min(count_le(gend, B, (int)k), B - 1);
        if (!(state[b] & 2)) continue;
        p.table[(long)b * p.table_stride + held_of[b] + ((int)k - (b ? gend[b - 1] : 0))] = stack_page((int)stack - 1 - (int)k);
    }
    for (long k = me; k < (long)stack - n_free; k += threads) p.free_list[n_free + k] = stack_page(n_free + (int)k);

    // ---- work units of the attention
    if (p.units && blockIdx.x == gridDim.x - 1) {
        unsigned long long total_len = 0;
        for (int w = 0; w < kPlanWaves; ++w) total_len += lens[w];
        unsigned long long most = p.chunk_units ? (total_len + p.chunk_units - 1) / p.chunk_units : total_len;
        most = max((most + 63) / 64 * 64, ((unsigned long long)p.chunk_min + 63) / 64 * 64);
        unsigned cnt[kPlanPer], sum[1] = {0}, total_units[1];
#pragma unroll
        for (int i = 0; i < kPlanPer; ++i) {
            cnt[i] = fresh[i] > 0 ? max((unsigned)(((unsigned long long)(unsigned)len[i] + most - 1) / most), 1u) : 0u;
            sum[0] += cnt[i];
        }
        block_scan<1>(sum, total_units, ws);
#pragma unroll
        for (int i = 0; i < kPlanPer; ++i) {
            const int b = tid * kPlanPer + i;
            if (b < B) { uend[b] = (int)sum[0]; p.unit_start[b] = (int)sum[0]; }
            sum[0] += cnt[i];
        }
        if (tid == 0) { uend[B] = (int)total_units[0]; p.unit_start[B] = (int)total_units[0]; }
        __syncthreads();
        for (int u = tid; u < B + p.chunk_units; u += kPlanThreads) {
            int4 unit = make_int4(-1, -1, -1, -1);
            if (u < uend[B]) {
                const int b = count_le(uend, B + 1, u) - 1, n = uend[b + 1] - uend[b];
                const int l = (state[b] & 2) ? kept_of[b] + (start[b + 1] - start[b]) : 0;
                const long each = (((long)l + n - 1) / n + 63) / 64 * 64, first = (u - uend[b]) * each;
                unit = make_int4(b, (int)min(first, (long)l), (int)min(first + each, (long)l), n);
            }
            reinterpret_cast<int4*>(p.units)[u] = unit;
        }
    }
}

// -------------------------------------------------------------------------------------------- write
// One thread moves 8 values of one (row, head): 16 bytes of K and of V in; the same bytes out, or 8 codes each.  HBM-bound:
// every byte is touched once.  The row scale of an e4m3 cache needs the row's largest magnitude: a butterfly over the
// D / 8 lanes that hold the row; a quotient is a product and one correction (divided out it is 30 us where it is now 26).
// 128 rows of 20 heads of 64: 2.1 us, the launch.  19 k bf16 rows of 8 heads of 128 to e4m3: 26.2 us, 107 MB that become 123 at the
// memory (scales are 4 bytes here and there): 4.7 TB/s, nearly a large copy's rate (4.9).
template <bool BF> __device__ __forceinline__ void to_f32x8(uint4 u, float (&f)[8]) {
    const unsigned w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (BF) {
            f[2 * i] = __uint_as_float(w[i] << 16);
            f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        } else {
            f[2 * i] = (float)__builtin_bit_cast(f16, (unsigned short)w[i]);
            f[2 * i + 1] = (float)__builtin_bit_cast(f16, (unsigned short)(w[i] >> 16));
        }
    }
}
template <bool BF, int LPR> __device__ __forceinline__ uint2 quant8(uint4 u, float& scale) {
    float f[8];
    to_f32x8<BF>(u, f);
    unsigned big = 0;                                        // magnitudes compare like their bits, NaN above infinity
#pragma unroll
    for (int i = 0; i < 8; ++i) big = max(big, __float_as_uint(f[i]) & 0x7fffffffu);
#pragma unroll
    for (int d = 1; d < LPR; d <<= 1) big = max(big, (unsigned)__shfl_xor((int)big, d));
    // a row with an infinity or a NaN has no scale: it comes back as NaN throughout
    scale = big >= 0x7f800000u ? __uint_as_float(0x7fc00000u) : __uint_as_float(big) / 448.f;
    if (scale > 0x1p-100f) {                                 // quotients to the last bit: a product and one correction
        const float inv = 1.f / scale;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float q = f[i] * inv;
            f[i] = fmaf(fmaf(-q, scale, f[i]), inv, q);
        }
    } else {
        const float by = scale > 0.f ? scale : 1.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = f[i] / by;
    }
    return make_uint2(pack4_e4m3(f[0], f[1], f[2], f[3]), pack4_e4m3(f[4], f[5], f[6], f[7]));
}

template <bool BF, bool KV8, int D>
__global__ __launch_bounds__(256) void paged_write_kernel(PagedCacheView c, const unsigned short* __restrict__ k, const unsigned short* __restrict__ v,
                                                          long k_row, long k_head, long v_row, long v_head, const long* __restrict__ slots,
                                                          long n) {
    constexpr int LPR = D / 8;
    const long id = (long)blockIdx.x * 256 + threadIdx.x;
    const long pair = id / LPR;                              // (row, head); the lanes of a pair stay together
    if (pair >= n) return;
    const int ch = (int)(id % LPR);
    const long row = pair / c.heads;
    const int h = (int)(pair - row * c.heads);
    const long slot = slots[row];
    const long pg = slot >> c.page_shift;
    if (slot < 0 || pg >= c.n_pages) return;                 // (all lanes of the pair)
    const int off = (int)(slot & ((1L << c.page_shift) - 1));
    const uint4 uk = *reinterpret_cast<const uint4*>(k + row * k_row + h * k_head + ch * 8);
    const uint4 uv = *reinterpret_cast<const uint4*>(v + row * v_row + h * v_head + ch * 8);
    const long dst = pg * c.page_stride + h * c.head_stride + off * c.token_stride + ch * 8;
    if constexpr (KV8) {
        float sk, sv;
        const uint2 ck = quant8<BF, LPR>(uk, sk), cv = quant8<BF, LPR>(uv, sv);
        *reinterpret_cast<uint2*>(static_cast<uint8_t*>(c.k) + dst) = ck;
        *reinterpret_cast<uint2*>(static_cast<uint8_t*>(c.v) + dst) = cv;
        if (ch == 0) {
            const long s = ((pg * c.heads + h) << c.page_shift) + off;
            c.ks[s] = sk; c.vs[s] = sv;
        }
    } else {
        *reinterpret_cast<uint4*>(static_cast<unsigned short*>(c.k) + dst) = uk;
        *reinterpret_cast<uint4*>(static_cast<unsigned short*>(c.v) + dst) = uv;
    }
}

// -------------------------------------------------------------------------------------------- accept
// Arg-max of every row: HBM-bound, the logits once.  A row is cut into parts so that few rows still fill the chip; a thread
// keeps its best (value, id) and looks at the suppressed ids only where a value would become its best.  Four loads of 16 bytes
// ahead (eight: 9.2 us where it is 8.2, for parts of 4096 fp32).  1102 rows of 128000 bf16: 44.6 us, 282 MB, 6.3 TB/s; 128 rows of
// 51866 fp32: 10.3 us, 27 MB, of which half is the first load's latency and the reduction's.
struct Best { float v; int i; };
__device__ __forceinline__ Best better(Best a, Best b) {     // larger value, lower id on ties
    return b.v > a.v || (b.v == a.v && b.i < a.i) ? b : a;
}
template <typename T> __device__ __forceinline__ float logit_f32(T x);
template <> __device__ __forceinline__ float logit_f32<float>(float x) { return x; }
template <> __device__ __forceinline__ float logit_f32<f16>(f16 x) { return (float)x; }
template <> __device__ __forceinline__ float logit_f32<unsigned short>(unsigned short x) { return __uint_as_float((unsigned)x << 16); }

template <typename T>
__global__ __launch_bounds__(256) void accept_scan_kernel(const T* __restrict__ logits, long stride, int V, const uint8_t* __restrict__ suppress,
                                                          int parts, int per, float* __restrict__ part_v, int* __restrict__ part_i) {
    constexpr int VEC = 16 / (int)sizeof(T);
    const long row = blockIdx.x / parts;
    const int part = (int)(blockIdx.x - row * parts);
    const T* x = logits + row * stride;
    const int v0 = part * per, v1 = min(V, v0 + per);
    Best best{-INFINITY, 0x7fffffff};
    auto take = [&](float f, int i) {
        if (f > best.v && !(suppress && suppress[i])) best = Best{f, i};
    };
    // the aligned middle in vectors of 16 bytes, the ends one by one
    const int lead = (int)(((16 - (reinterpret_cast<uintptr_t>(x + v0) & 15)) & 15) / sizeof(T));
    const int a0 = min(v1, v0 + lead), nvec = (v1 - a0) / VEC;
    if (v0 + (int)threadIdx.x < a0) take(logit_f32<T>(x[v0 + threadIdx.x]), v0 + threadIdx.x);
    typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
    const u32x4* body = reinterpret_cast<const u32x4*>(x + a0);
    constexpr int AHEAD = 4;
    for (int j0 = threadIdx.x; j0 < nvec; j0 += 256 * AHEAD) {
        u32x4 u[AHEAD];                                      // read once: nothing is gained by keeping them in the caches
#pragma unroll
        for (int a = 0; a < AHEAD; ++a) u[a] = __builtin_nontemporal_load(body + min(j0 + 256 * a, nvec - 1));
#pragma unroll
        for (int a = 0; a < AHEAD; ++a) {
            const int j = j0 + 256 * a;
            float f[VEC];
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                if constexpr (sizeof(T) == 4) f[i] = __uint_as_float(u[a][i]);
                else f[i] = logit_f32<T>(__builtin_bit_cast(T, (unsigned short)(u[a][i >> 1] >> (16 * (i & 1)))));
            }
            float m = f[0];
#pragma unroll
            for (int i = 1; i < VEC; ++i) m = fmaxf(m, f[i]);
            if (j < nvec && m > best.v) {
#pragma unroll
                for (int i = 0; i < VEC; ++i) take(f[i], a0 + j * VEC + i);
            }
        }
    }
    const int tail = a0 + nvec * VEC + threadIdx.x;
    if (tail < v1) take(logit_f32<T>(x[tail]), tail);
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) best = better(best, Best{__shfl_xor(best.v, d), __shfl_xor(best.i, d)});
    __shared__ Best wb[4];
    if ((threadIdx.x & 63) == 0) wb[threadIdx.x >> 6] = best;
    __syncthreads();
    if (threadIdx.x == 0) {
        best = better(better(wb[0], wb[1]), better(wb[2], wb[3]));
        part_v[row * parts + part] = best.v;
        part_i[row * parts + part] = best.i;
    }
}

// The path of every tree: next[i] = the lowest child of i whose token is the arg-max of i's row, all nodes at once; then
// one thread follows next[] from the root.  Bound by the latency of three dependent loads: 3.9 us for 16 trees of 8, 4.6 us for
// 48 of up to 45.
__global__ __launch_bounds__(256) void accept_walk_kernel(AcceptParams p, int parts, const float* __restrict__ part_v, const int* __restrict__ part_i) {
    __shared__ int next[kAcceptMaxNodes], ids[kAcceptMaxNodes];
    __shared__ int count;
    const int b = blockIdx.x;
    const int r0 = max(0, p.row_start[b]), r1 = min(p.rows, p.row_start[b + 1]);
    const int n = max(0, min(r1 - r0, p.depth));
    for (int i = threadIdx.x; i < max(0, r1 - r0); i += 256) {
        Best best{-INFINITY, 0x7fffffff};
        const long at = (long)(r0 + i) * parts;
        for (int k0 = 0; k0 < parts; k0 += 8) {
            Best x[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) x[k] = Best{part_v[at + min(k0 + k, parts - 1)], part_i[at + min(k0 + k, parts - 1)]};
#pragma unroll
            for (int k = 0; k < 8; ++k) best = better(best, x[k]);
        }
        const int id = best.i == 0x7fffffff ? 0 : best.i;    // nothing to choose from: the lowest id
        p.best[r0 + i] = id;
        if (i < n) { ids[i] = id; next[i] = 0x7fffffff; }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += 256) {
        const int up = p.parents[r0 + i];
        if (up >= 0 && up < i && p.tokens[r0 + i] == ids[up]) atomicMin(&next[up], i);      // LDS; the lowest wins whatever the order
    }
    __syncthreads();
    int* path = p.path + (long)b * p.depth;
    int* out = p.out_tokens + (long)b * p.depth;
    if (threadIdx.x == 0) {
        int m = 0;
        for (int i = 0; i < n; i = next[i]) { path[m] = i; out[m] = ids[i]; ++m; }          // next[] ascends: it ends
        count = m;
        p.count[b] = m;
    }
    __syncthreads();
    for (int i = count + (int)threadIdx.x; i < p.depth; i += 256) { path[i] = -1; out[i] = -1; }
}

// -------------------------------------------------------------------------------------------- compact
// A workgroup owns up to 64 pieces of 16 bytes of a layer's token rows (heads of K, heads of V, and the row scales as pieces
// of 4) and moves them for every accepted node: HBM-bound, 16 bytes in and out per piece.  A path ascends and path[i] >= i, so
// what move i overwrites is only ever read by moves before it: a batch of moves is read as a whole, then written.  Pieces of 64
// keep a workgroup's moves of 16 nodes in flight at once (256 pieces and node after node: 83 us where it is 51).  64 trees of up to
// 60 nodes, 48 layers of 8 heads of 128 e4m3: 52.6 us, 213 MB in and out, 4.0 TB/s; 16 trees of 8, 32 layers of 20 heads of 64: 6.5 us, 14 MB.
constexpr int kCompactPieces = 64, kCompactPer = 4;
template <typename V> __device__ __forceinline__ void move_pieces(char* const* column, int pieces, const long* src, const long* dst, int moves, long layer_off) {
    // item e = (move, piece), neighbours in a row side by side; kCompactPer items per thread are in flight
    const unsigned inv = (1u << 20) / pieces + 1;            // e / pieces = e * inv >> 20, exact for e < 1024 and pieces <= 64
    const int per = 256 * kCompactPer / pieces;
    for (int j0 = 0; j0 < moves; j0 += per) {
        const int items = min(moves - j0, per) * pieces;
        V v[kCompactPer];
        char* to[kCompactPer];
#pragma unroll
        for (int a = 0; a < kCompactPer; ++a) {
            const int e = threadIdx.x + 256 * a, j = (int)(e * inv >> 20);
            if (e >= items) continue;
            char* const at = column[e - j * pieces] + layer_off;
            v[a] = *reinterpret_cast<const V*>(at + src[j0 + j]);
            to[a] = at + dst[j0 + j];
        }
        __syncthreads();
#pragma unroll
        for (int a = 0; a < kCompactPer; ++a)
            if ((int)threadIdx.x + 256 * a < items) *reinterpret_cast<V*>(to[a]) = v[a];
    }
}
__global__ __launch_bounds__(256) void paged_compact_kernel(PagedCacheView c, long layer_stride, long scale_layer_stride, int esize, int dim,
                                                            const int* __restrict__ table, long table_stride, int max_pages,
                                                            const int* __restrict__ kept, const int* __restrict__ path, int path_cols,
                                                            const int* __restrict__ count, int layers) {
    typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
    __shared__ char* column[kCompactPieces];                 // where piece e of token 0 of page 0 lies
    __shared__ long src[2][256], dst[2][256];                // byte offsets of up to 256 moves; [1]: of the scales
    __shared__ int wsum[4];
    const int b = blockIdx.z;
    const int m = min(max(count[b], 0), path_cols), kept_b = kept[b];
    const int per_row = dim * esize / 16;                    // pieces of a (head, token) row
    const int all = 2 * c.heads * per_row, scale_blocks = c.ks ? (2 * c.heads + kCompactPieces - 1) / kCompactPieces : 0;
    const bool scales = (int)blockIdx.x >= (int)gridDim.x - scale_blocks;
    const int first = (scales ? blockIdx.x - (gridDim.x - scale_blocks) : blockIdx.x) * kCompactPieces;
    const int pieces = min((scales ? 2 * c.heads : all) - first, kCompactPieces);
    const int page = 1 << c.page_shift;
    for (int e = threadIdx.x; e < pieces; e += 256) {
        const int q = first + e;
        if (scales) {
            const int which = q / c.heads, h = q - which * c.heads;
            column[e] = reinterpret_cast<char*>((which ? c.vs : c.ks) + (long)h * page);
        } else {
            const int which = q / (c.heads * per_row), rest = q - which * c.heads * per_row, h = rest / per_row;
            column[e] = static_cast<char*>(which ? c.v : c.k) + h * c.head_stride * esize + (rest - h * per_row) * 16;
        }
    }
    auto page_of = [&](long place) -> int {
        const long n = place >> c.page_shift;
        if (place < 0 || n >= max_pages) return -1;
        const int pg = table[b * table_stride + n];
        return pg >= 0 && pg < c.n_pages ? pg : -1;
    };
    for (int i0 = 0; i0 < m; i0 += 256) {
        const int i = i0 + threadIdx.x, node = i < m ? path[(long)b * path_cols + i] : -1;
        const long from = (long)kept_b + node, to = (long)kept_b + i;
        const int ps = node > i ? page_of(from) : -1, pd = node > i ? page_of(to) : -1;
        const bool move = ps >= 0 && pd >= 0;
        // the moves in path order, without the nodes that lie in their place already
        const unsigned long long ball = __ballot(move);
        const int before = __popcll(ball & ((1ull << (threadIdx.x & 63)) - 1)), wave = threadIdx.x >> 6;
        __syncthreads();                                     // the previous batch is done with src and dst
        if ((threadIdx.x & 63) == 0) wsum[wave] = __popcll(ball);
        __syncthreads();
        int base = 0;
        for (int w = 0; w < wave; ++w) base += wsum[w];
        if (move) {
            const int os = (int)(from & (page - 1)), od = (int)(to & (page - 1));
            src[0][base + before] = (ps * c.page_stride + os * c.token_stride) * esize;
            dst[0][base + before] = (pd * c.page_stride + od * c.token_stride) * esize;
            src[1][base + before] = (((long)ps * c.heads << c.page_shift) + os) * 4;
            dst[1][base + before] = (((long)pd * c.heads << c.page_shift) + od) * 4;
        }
        const int moves = wsum[0] + wsum[1] + wsum[2] + wsum[3];
        __syncthreads();
        // workgroups of a request take the layers in turn: finding the moves is four round trips to memory, once for all of them
        for (int layer = blockIdx.y; layer < layers; layer += gridDim.y) {
            if (scales) move_pieces<unsigned>(column, pieces, src[1], dst[1], moves, layer * scale_layer_stride * 4);
            else move_pieces<u32x4>(column, pieces, src[0], dst[0], moves, layer * layer_stride * esize);
        }
    }
}

}  // namespace

hipError_t launch_paged_plan(const PlanParams& p, hipStream_t s) {
    // a row per thread (256 chains of 166 k rows: 7.2 us; 2 rows 8.2, 4 rows 9.8, 8 rows 13.8), up to what runs side by side; one
    // workgroup per tree
    long wgs = (p.rows + kPlanThreads - 1) / kPlanThreads;
    wgs = wgs < 1 ? 1 : wgs > 512 ? 512 : wgs;
    if (p.parents && wgs < p.batch) wgs = p.batch;
    return launch(paged_plan_kernel, (unsigned)wgs, kPlanThreads, s, p);
}

hipError_t launch_paged_write(const PagedCacheView& c, int dim, int bf16, const void* k, const void* v, long k_row, long k_head, long v_row,
                        long v_head, const long* slots, long rows, hipStream_t s) {
    const long pairs = rows * c.heads, threads = pairs * (dim / 8);
    if (!threads) return hipSuccess;
    const unsigned grid = (unsigned)((threads + 255) / 256);
    const unsigned short *kk = static_cast<const unsigned short*>(k), *vv = static_cast<const unsigned short*>(v);
#define MW_WRITE(BF, KV8, D) return launch(paged_write_kernel<BF, KV8, D>, grid, 256, s, c, kk, vv, k_row, k_head, v_row, v_head, slots, pairs)
    if (!c.ks) { if (dim == 64) MW_WRITE(false, false, 64); else MW_WRITE(false, false, 128); }       // 16-bit values are copied as they are
    else if (bf16) { if (dim == 64) MW_WRITE(true, true, 64); else MW_WRITE(true, true, 128); }
    else { if (dim == 64) MW_WRITE(false, true, 64); else MW_WRITE(false, true, 128); }
#undef MW_WRITE
}

// Parts of a row: about 6144 workgroups, but none with less than 4096 values, the 16 KB (fp32) that its threads have in flight at
// once.  128 rows of 51866 fp32: 13 parts of 4096 8.2 us, 7 of 8192 9.8, 26 of 2048 9.7; 1102 rows of 128000 bf16: 6 parts 42.7 us,
// 2 45.9, 8 42.4 with a slower second launch.
int accept_parts(long rows, int vocab) {
    const long want = rows > 0 ? (6144 + rows - 1) / rows : 1, most = (vocab + 4095) / 4096;
    const long n = want < most ? want : most;
    return n < 1 ? 1 : n > kAcceptMaxParts ? kAcceptMaxParts : (int)n;
}

hipError_t launch_tree_accept(const AcceptParams& p, hipStream_t s) {
    const int parts = accept_parts(p.rows, p.vocab);
    const int per = ((p.vocab + parts - 1) / parts + 7) / 8 * 8;
    float* pv = static_cast<float*>(p.workspace);
    int* pi = reinterpret_cast<int*>(pv + (long)p.rows * parts);
    if (p.rows > 0) {
        const unsigned grid = (unsigned)((long)p.rows * parts);
        hipError_t e;
        if (p.dtype == 0) e = launch(accept_scan_kernel<float>, grid, 256, s, static_cast<const float*>(p.logits), p.stride, p.vocab, p.suppress, parts, per, pv, pi);
        else if (p.dtype == 1) e = launch(accept_scan_kernel<f16>, grid, 256, s, static_cast<const f16*>(p.logits), p.stride, p.vocab, p.suppress, parts, per, pv, pi);
        else e = launch(accept_scan_kernel<unsigned short>, grid, 256, s, static_cast<const unsigned short*>(p.logits), p.stride, p.vocab, p.suppress, parts, per, pv, pi);
        if (e != hipSuccess) return e;
    }
    return launch(accept_walk_kernel, (unsigned)p.batch, 256, s, p, parts, pv, pi);
}

hipError_t launch_paged_compact(const PagedCacheView& c, int layers, long layer_stride, long scale_layer_stride, int dim, const int* table,
                          long table_stride, int max_pages, const int* kept, const int* path, int path_cols, const int* count, int batch,
                          hipStream_t s) {
    const int esize = c.ks ? 1 : 2;
    const int blocks = (2 * c.heads * (dim * esize / 16) + kCompactPieces - 1) / kCompactPieces +
                       (c.ks ? (2 * c.heads + kCompactPieces - 1) / kCompactPieces : 0);
    // Layers a workgroup takes.  64 requests with trees of 60 nodes, 48 layers, 3 blocks: 8192 workgroups at most (2 layers each)
    // 55 us, 2048 (5 layers) 63 us; short paths are over before the next workgroup is found: 16 requests with trees of 8, 32
    // layers, 5 blocks: 7.3 us with 2 layers each, 8.6 with one.
    const long share = std::max(((long)blocks * batch * layers + 8191) / 8192, (long)(16 + path_cols - 1) / path_cols);
    const int groups = (int)((layers + share - 1) / share);
    return launch(paged_compact_kernel, dim3(blocks, groups, batch), 256, s, c, layer_stride, scale_layer_stride, esize, dim, table, table_stride, max_pages,
                  kept, path, path_cols, count, layers);
}

}  // namespace mw
