// Operators of drafted decoding over a K/V cache in pages, for gfx950: the plan of a step (block tables, slot map, tree
// masks, work units), the write of K/V rows into pages, acceptance of a tree of drafted tokens against the logits, and the
// compaction of the accepted rows.  The attention over the pages is in kernels_tree.hip.
//
// All of them are bound by HBM or, at the sizes of one decode step, by the latency of a launch: each is one launch (accept:
// two), nothing is allocated, nothing waits for the host, and every index that comes from device memory is checked
// against its buffer before it is used.
#include "mw_kernels.h"

namespace mw {

namespace {

// -------------------------------------------------------------------------------------------- plan
// Every workgroup computes the prefix sums over the requests for itself (at most 2048 requests, a few KB that stay in L2)
// and then does its share of the rows, new pages, returned pages, tree masks and units: one launch without any exchange
// between workgroups.  A page popped from a stack entry that this very step pushes is looked up in the table of the request
// that gives it back, so pops never wait for pushes.
constexpr int kPlanThreads = 1024;
constexpr int kPlanPer = kPlanMaxBatch / kPlanThreads;       // requests per thread of the prefix sums

__device__ __forceinline__ long wave_scan(long v) {          // inclusive, over 64 lanes
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const long o = __shfl_up(v, d);
        if (lane >= d) v += o;
    }
    return v;
}
// Exclusive prefix of `v` over the 1024 threads; `total` receives the sum.  `ws`: 17 longs of LDS.
__device__ __forceinline__ long block_scan(long v, long* ws, long& total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const long inc = wave_scan(v);
    __syncthreads();                                         // ws may still be read by the previous scan
    if (lane == 63) ws[wave] = inc;
    __syncthreads();
    long before = 0, sum = 0;
#pragma unroll
    for (int w = 0; w < kPlanThreads / 64; ++w) {
        const long x = ws[w];
        if (w < wave) before += x;
        sum += x;
    }
    total = sum;
    return before + inc - v;
}
__device__ __forceinline__ int sat32(long v) { return v > 0x7fffffffL ? 0x7fffffff : (int)v; }
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
    __shared__ long ws[17];
    __shared__ int start[kPlanMaxBatch + 1];                 // first row of each request
    __shared__ int gend[kPlanMaxBatch];                      // new pages wanted up to and including each request
    __shared__ int bend[kPlanMaxBatch];                      // pages given back up to and including each request
    __shared__ int uend[kPlanMaxBatch + 1];                  // units before each request (the last workgroup's)
    __shared__ unsigned char state[kPlanMaxBatch];           // 1 = valid, 2 = admitted
    __shared__ unsigned anc[32 * kPlanMaxWords][kPlanMaxWords + 1];
    __shared__ int jump[32 * kPlanMaxWords];
    const int tid = threadIdx.x, B = p.batch;
    const int page = 1 << p.page_shift;

    // ---- prefix sums over the requests
    long kept[kPlanPer], fresh[kPlanPer];
    int held[kPlanPer];
    long sum = 0;
#pragma unroll
    for (int i = 0; i < kPlanPer; ++i) {
        const int b = tid * kPlanPer + i;
        kept[i] = b < B ? p.kept[b] : 0;
        fresh[i] = b < B ? p.fresh[b] : 0;
        held[i] = b < B ? min(max(p.pages_in[b], 0), p.max_pages) : 0;
        sum += fresh[i] > 0 ? fresh[i] : 0;
    }
    long total_rows;
    long at = block_scan(sum, ws, total_rows);
    long grow[kPlanPer], back[kPlanPer], need[kPlanPer];
    bool valid[kPlanPer];
    long gsum = 0, bsum = 0;
#pragma unroll
    for (int i = 0; i < kPlanPer; ++i) {
        const int b = tid * kPlanPer + i;
        if (b < B) start[b] = sat32(at);
        at += fresh[i] > 0 ? fresh[i] : 0;
        need[i] = (kept[i] + fresh[i] + page - 1) >> p.page_shift;
        valid[i] = b < B && kept[i] >= 0 && fresh[i] >= 0 && need[i] <= p.max_pages && at <= p.rows &&
                   (!p.parents || fresh[i] <= 32 * p.mask_words);
        grow[i] = valid[i] && need[i] > held[i] ? need[i] - held[i] : 0;
        back[i] = valid[i] && need[i] < held[i] ? held[i] - need[i] : 0;
        gsum += grow[i]; bsum += back[i];
    }
    if (tid == 0) start[B] = sat32(total_rows);
    long total_grow, total_back;
    long gat = block_scan(gsum, ws, total_grow);
    long bat = block_scan(bsum, ws, total_back);
    const int n_free = min(max(p.n_free_in[0], 0), p.n_pages);
    const long stack = n_free + total_back;                  // pages to be had in this step
    long used = 0, len_sum = 0;
    long len[kPlanPer];
#pragma unroll
    for (int i = 0; i < kPlanPer; ++i) {
        const int b = tid * kPlanPer + i;
        gat += grow[i]; bat += back[i];
        const bool admitted = valid[i] && (grow[i] == 0 || gat <= stack);
        if (b < B) {
            gend[b] = sat32(gat); bend[b] = sat32(bat);
            state[b] = (valid[i] ? 1 : 0) | (admitted ? 2 : 0);
            if (blockIdx.x == 0) {
                p.row_start[b] = start[b];
                p.admitted[b] = admitted;
                p.pages_out[b] = admitted ? (int)need[i] : held[i];
            }
        }
        if (admitted) used += grow[i];
        len[i] = admitted && fresh[i] > 0 ? kept[i] + fresh[i] : 0;
        len_sum += len[i];
    }
    long total_used, total_len;
    block_scan(used, ws, total_used);
    block_scan(len_sum, ws, total_len);
    if (blockIdx.x == 0 && tid == 0) {
        p.row_start[B] = start[B];
        p.n_free_out[0] = (int)min(stack - total_used, (long)p.n_pages);
    }
    __syncthreads();

    // page on top of entry `e` of the stack as this step's pushes leave it
    auto stack_page = [&](long e) -> int {
        if (e < n_free) return p.free_list[e];
        const int k = sat32(e - n_free), b = min(count_le(bend, B, k), B - 1);
        const int first = (int)((p.kept[b] + (long)p.fresh[b] + page - 1) >> p.page_shift);
        return p.table[(long)b * p.table_stride + first + (k - (b ? bend[b - 1] : 0))];
    };
    // page `n` of admitted request b, old or new
    auto page_of = [&](int b, int n) -> int {
        const int h = min(max(p.pages_in[b], 0), p.max_pages);
        if (n < h) return p.table[(long)b * p.table_stride + n];
        return stack_page(stack - 1 - ((b ? gend[b - 1] : 0) + (n - h)));
    };
    const long threads = (long)gridDim.x * kPlanThreads, me = (long)blockIdx.x * kPlanThreads + tid;

    // ---- rows: slots, and positions of chains
    for (long r = me; r < p.rows; r += threads) {
        long slot = -1;
        int pos = -1;
        bool masked = p.parents != nullptr;                  // no tree is going to write this row's mask
        if (r < start[B]) {
            const int b = count_le(start, B + 1, (int)r) - 1;
            const int i = (int)r - start[b];
            const int kb = p.kept[b];
            if (state[b] & 1) { pos = kb + i; masked = false; }
            if (state[b] & 2) {
                const int place = kb + i;
                const int pg = page_of(b, place >> p.page_shift);
                slot = pg >= 0 ? ((long)pg << p.page_shift) + (place & (page - 1)) : -1;
            }
        }
        p.slots[r] = slot;
        if (!p.parents || masked) p.positions[r] = pos;
        if (masked)
            for (int w = 0; w < p.mask_words; ++w) p.mask[r * p.mask_words + w] = 0;
    }
    // ---- new pages into the tables, returned pages onto the stack
    const long grown = total_grow < stack ? total_grow : stack;
    for (long k = me; k < grown; k += threads) {
        const int b = min(count_le(gend, B, (int)k), B - 1);
        if (!(state[b] & 2)) continue;
        const int h = min(max(p.pages_in[b], 0), p.max_pages);
        p.table[(long)b * p.table_stride + h + ((int)k - (b ? gend[b - 1] : 0))] = stack_page(stack - 1 - k);
    }
    for (long k = me; k < total_back; k += threads)
        if (n_free + k < p.n_pages) p.free_list[n_free + k] = stack_page(n_free + k);

    // ---- trees: ancestors by pointer doubling.  Node i starts with {i} and its parent; a round adds the ancestors that its
    // jump target has gathered and jumps on from there: log2(depth) rounds, all nodes at once.
    if (p.parents && (int)blockIdx.x < B && (state[blockIdx.x] & 1)) {
        const int b = blockIdx.x, n = start[b + 1] - start[b], W = p.mask_words;
        if (tid < n) {
            int up = p.parents[start[b] + tid];
            if (up < 0 || up >= tid) up = -1;                // a parent is an earlier node of the same tree
            jump[tid] = up;
            for (int w = 0; w < W; ++w) anc[tid][w] = (tid >> 5) == w ? 1u << (tid & 31) : 0u;
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
            const long r = start[b] + tid;
            for (int w = 0; w < W; ++w) { p.mask[r * W + w] = anc[tid][w]; depth += __popc(anc[tid][w]); }
            p.positions[r] = p.kept[b] + depth;
        }
    }

    // ---- work units of the attention
    if (p.units && blockIdx.x == gridDim.x - 1) {
        long most = p.chunk_units ? (total_len + p.chunk_units - 1) / p.chunk_units : total_len;
        most = (most + 63) / 64 * 64;
        const long least = ((long)p.chunk_min + 63) / 64 * 64;
        most = most > least ? most : least;
        long cnt[kPlanPer], csum = 0;
#pragma unroll
        for (int i = 0; i < kPlanPer; ++i) {
            const long c = (len[i] + most - 1) / most;
            cnt[i] = fresh[i] > 0 ? (c > 1 ? c : 1) : 0;
            csum += cnt[i];
        }
        long total_units;
        long uat = block_scan(csum, ws, total_units);
#pragma unroll
        for (int i = 0; i < kPlanPer; ++i) {
            const int b = tid * kPlanPer + i;
            if (b < B) { uend[b] = sat32(uat); p.unit_start[b] = sat32(uat); }
            uat += cnt[i];
        }
        if (tid == 0) { uend[B] = sat32(total_units); p.unit_start[B] = sat32(total_units); }
        __syncthreads();
        for (int u = tid; u < B + p.chunk_units; u += kPlanThreads) {
            int4 unit = make_int4(-1, -1, -1, -1);
            if (u < uend[B]) {
                const int b = count_le(uend, B + 1, u) - 1, n = uend[b + 1] - uend[b];
                const long l = (state[b] & 2) ? p.kept[b] + (long)p.fresh[b] : 0;
                const long each = ((l + n - 1) / n + 63) / 64 * 64;
                const long first = (u - uend[b]) * each;
                unit = make_int4(b, (int)min(first, l), (int)min(first + each, l), n);
            }
            reinterpret_cast<int4*>(p.units)[u] = unit;
        }
    }
}

// -------------------------------------------------------------------------------------------- write
// One thread moves 8 values of one (row, head): 16 bytes of K and of V in; the same bytes out, or 8 codes each.  HBM-bound:
// every byte is touched once.  The row scale of an e4m3 cache needs the row's largest magnitude: a butterfly over the
// D / 8 lanes that hold the row.
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
    const float by = scale > 0.f ? scale : 1.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = f[i] / by;
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
// keeps its best (value, id) and looks at the suppressed ids only where a value would become its best.
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
    const uint4* body = reinterpret_cast<const uint4*>(x + a0);
    for (int j = threadIdx.x; j < nvec; j += 256) {
        const uint4 u = body[j];
        const T* e = reinterpret_cast<const T*>(&u);
        float m = logit_f32<T>(e[0]);
#pragma unroll
        for (int i = 1; i < VEC; ++i) m = fmaxf(m, logit_f32<T>(e[i]));
        if (m > best.v) {
#pragma unroll
            for (int i = 0; i < VEC; ++i) take(logit_f32<T>(e[i]), a0 + j * VEC + i);
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
// one thread follows next[] from the root.
__global__ __launch_bounds__(256) void accept_walk_kernel(AcceptParams p, int parts, const float* __restrict__ part_v, const int* __restrict__ part_i) {
    __shared__ int next[kAcceptMaxNodes], ids[kAcceptMaxNodes];
    __shared__ int count;
    const int b = blockIdx.x;
    const int r0 = max(0, p.row_start[b]), r1 = min(p.rows, p.row_start[b + 1]);
    const int n = max(0, min(r1 - r0, p.depth));
    for (int i = threadIdx.x; i < max(0, r1 - r0); i += 256) {
        Best best{-INFINITY, 0x7fffffff};
        for (int k = 0; k < parts; ++k) best = better(best, Best{part_v[(long)(r0 + i) * parts + k], part_i[(long)(r0 + i) * parts + k]});
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
// A thread owns 16 bytes of a (layer, head, K or V) column and moves them for every accepted node: HBM-bound, 16 bytes in
// and out per piece.  A path ascends and path[i] >= i, so a row that is written is never one that is still to be read:
// the reads of eight nodes are issued together.
__global__ __launch_bounds__(256) void paged_compact_kernel(PagedCacheView c, long layer_stride, long scale_layer_stride, int esize, int dim,
                                                            const int* __restrict__ table, long table_stride, int max_pages,
                                                            const int* __restrict__ kept, const int* __restrict__ path, int path_cols,
                                                            const int* __restrict__ count) {
    constexpr int PER = 8;
    __shared__ int src[256], dst[256];                       // slots of up to 256 moves; -1: nothing to move
    __shared__ int n_moves;
    const int b = blockIdx.z, layer = blockIdx.y;
    const int m = min(max(count[b], 0), path_cols);
    const int per_row = dim * esize / 16;                    // pieces of a (head, token) row
    const int pieces = 2 * c.heads * per_row, scales = c.ks ? 2 * c.heads : 0;
    const int id = blockIdx.x * 256 + threadIdx.x;
    const int page = 1 << c.page_shift;
    auto slot_of = [&](long place) -> int {
        const long n = place >> c.page_shift;
        if (place < 0 || n >= max_pages) return -1;
        const int pg = table[b * table_stride + n];
        return pg >= 0 && pg < c.n_pages ? (int)((pg << c.page_shift) + (place & (page - 1))) : -1;
    };
    for (int i0 = 0; i0 < m; i0 += 256) {
        __syncthreads();
        if (threadIdx.x == 0) n_moves = 0;
        __syncthreads();
        const int i = i0 + threadIdx.x;
        int s = -1, d = -1;
        if (i < m) {
            const int node = path[(long)b * path_cols + i];
            if (node > i) { s = slot_of((long)kept[b] + node); d = slot_of((long)kept[b] + i); }
        }
        const bool move = s >= 0 && d >= 0;
        // the moves in path order, without the nodes that lie in their place already
        const unsigned long long ball = __ballot(move);
        const int before = __popcll(ball & ((1ull << (threadIdx.x & 63)) - 1));
        __shared__ int wsum[4];
        if ((threadIdx.x & 63) == 0) wsum[threadIdx.x >> 6] = __popcll(ball);
        __syncthreads();
        int base = 0;
        for (int w = 0; w < (int)(threadIdx.x >> 6); ++w) base += wsum[w];
        if (move) { src[base + before] = s; dst[base + before] = d; }
        if (threadIdx.x == 0) n_moves = wsum[0] + wsum[1] + wsum[2] + wsum[3];
        __syncthreads();
        const int moves = n_moves;
        if (id < pieces) {
            const int which = id / (c.heads * per_row), rest = id - which * c.heads * per_row;
            const int h = rest / per_row, piece = rest - h * per_row;
            char* base_p = static_cast<char*>(which ? c.v : c.k) + (layer * layer_stride + h * c.head_stride) * esize + piece * 16;
            for (int j0 = 0; j0 < moves; j0 += PER) {
                uint4 u[PER];
                char* to[PER];
#pragma unroll
                for (int j = 0; j < PER; ++j) {
                    const int jj = min(j0 + j, moves - 1), sl = src[jj], dl = dst[jj];
                    const char* from = base_p + ((long)(sl >> c.page_shift) * c.page_stride + (sl & (page - 1)) * c.token_stride) * esize;
                    to[j] = base_p + ((long)(dl >> c.page_shift) * c.page_stride + (dl & (page - 1)) * c.token_stride) * esize;
                    u[j] = *reinterpret_cast<const uint4*>(from);
                }
#pragma unroll
                for (int j = 0; j < PER; ++j)
                    if (j0 + j < moves) *reinterpret_cast<uint4*>(to[j]) = u[j];
            }
        } else if (id < pieces + scales) {
            const int which = (id - pieces) / c.heads, h = (id - pieces) - which * c.heads;
            float* s32 = (which ? c.vs : c.ks) + layer * scale_layer_stride;
            for (int j = 0; j < moves; ++j) {
                const int sl = src[j], dl = dst[j];
                s32[(((long)(dl >> c.page_shift) * c.heads + h) << c.page_shift) + (dl & (page - 1))] =
                    s32[(((long)(sl >> c.page_shift) * c.heads + h) << c.page_shift) + (sl & (page - 1))];
            }
        }
    }
}

}  // namespace

void launch_paged_plan(const PlanParams& p, hipStream_t s) {
    long wgs = (p.rows + 2 * kPlanThreads - 1) / (2 * kPlanThreads);
    wgs = wgs < 1 ? 1 : wgs > 512 ? 512 : wgs;
    if (p.parents && wgs < p.batch) wgs = p.batch;           // one workgroup per tree
    paged_plan_kernel<<<(unsigned)wgs, kPlanThreads, 0, s>>>(p);
}

void launch_paged_write(const PagedCacheView& c, int dim, int bf16, const void* k, const void* v, long k_row, long k_head, long v_row,
                        long v_head, const long* slots, long rows, hipStream_t s) {
    const long pairs = rows * c.heads, threads = pairs * (dim / 8);
    if (!threads) return;
    const unsigned grid = (unsigned)((threads + 255) / 256);
    const unsigned short *kk = static_cast<const unsigned short*>(k), *vv = static_cast<const unsigned short*>(v);
#define MW_WRITE(BF, KV8, D) paged_write_kernel<BF, KV8, D><<<grid, 256, 0, s>>>(c, kk, vv, k_row, k_head, v_row, v_head, slots, pairs)
    if (!c.ks) { if (dim == 64) MW_WRITE(false, false, 64); else MW_WRITE(false, false, 128); }       // 16-bit values are copied as they are
    else if (bf16) { if (dim == 64) MW_WRITE(true, true, 64); else MW_WRITE(true, true, 128); }
    else { if (dim == 64) MW_WRITE(false, true, 64); else MW_WRITE(false, true, 128); }
#undef MW_WRITE
}

// Parts of a row: enough workgroups for every CU several times over, none with less than 4096 values.
int accept_parts(long rows, int vocab) {
    const long want = rows > 0 ? (2048 + rows - 1) / rows : 1, most = (vocab + 4095) / 4096;
    const long n = want < most ? want : most;
    return n < 1 ? 1 : n > kAcceptMaxParts ? kAcceptMaxParts : (int)n;
}

void launch_tree_accept(const AcceptParams& p, hipStream_t s) {
    const int parts = accept_parts(p.rows, p.vocab);
    const int per = ((p.vocab + parts - 1) / parts + 7) / 8 * 8;
    float* pv = static_cast<float*>(p.workspace);
    int* pi = reinterpret_cast<int*>(pv + (long)p.rows * parts);
    if (p.rows > 0) {
        const unsigned grid = (unsigned)((long)p.rows * parts);
        if (p.dtype == 0) accept_scan_kernel<float><<<grid, 256, 0, s>>>(static_cast<const float*>(p.logits), p.stride, p.vocab, p.suppress, parts, per, pv, pi);
        else if (p.dtype == 1) accept_scan_kernel<f16><<<grid, 256, 0, s>>>(static_cast<const f16*>(p.logits), p.stride, p.vocab, p.suppress, parts, per, pv, pi);
        else accept_scan_kernel<unsigned short><<<grid, 256, 0, s>>>(static_cast<const unsigned short*>(p.logits), p.stride, p.vocab, p.suppress, parts, per, pv, pi);
    }
    accept_walk_kernel<<<(unsigned)p.batch, 256, 0, s>>>(p, parts, pv, pi);
}

void launch_paged_compact(const PagedCacheView& c, int layers, long layer_stride, long scale_layer_stride, int dim, const int* table,
                          long table_stride, int max_pages, const int* kept, const int* path, int path_cols, const int* count, int batch,
                          hipStream_t s) {
    const int esize = c.ks ? 1 : 2;
    const int threads = 2 * c.heads * (dim * esize / 16) + (c.ks ? 2 * c.heads : 0);
    paged_compact_kernel<<<dim3((threads + 255) / 256, layers, batch), 256, 0, s>>>(c, layer_stride, scale_layer_stride, esize, dim, table,
                                                                                    table_stride, max_pages, kept, path, path_cols, count);
}

}  // namespace mw
