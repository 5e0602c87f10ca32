// C entry points of the operators over a K/V cache in pages (include/mwhip.h, "drafted tokens over a K/V cache in pages").
// They are stateless: arguments are checked on the host before anything touches the GPU, then the launches are queued on
// the caller's stream.
#include "../../include/mwhip.h"
#include "mw_kernels.h"

#include <math.h>
#include <stdio.h>
#include <stdlib.h>

#include <string>

using namespace mw;

namespace mw { void set_call_error(const std::string& msg); }          // engine.hip: what mw_last_error(NULL) returns

namespace {

int refuse(const char* who, const std::string& what) {
    set_call_error(std::string(who) + ": " + what);
    return MW_ERR_ARG;
}
#define REFUSE_IF(cond, what)                                       \
    do { if (cond) return refuse(who, what); } while (0)

// The device of a call is made current for its launches and the caller's put back, also on errors.
struct OnDevice {
    int before = -1;
    hipError_t err;
    explicit OnDevice(int device) {
        err = hipGetDevice(&before);
        if (err == hipSuccess && before != device) err = hipSetDevice(device);
        else if (err == hipSuccess) before = -1;             // nothing to put back
    }
    ~OnDevice() { if (before >= 0) (void)hipSetDevice(before); }
};
int launched(const char* who, hipError_t e) {
    if (e == hipSuccess) return MW_OK;
    (void)hipGetLastError();                                 // told here, not by the next call that asks
    set_call_error(std::string(who) + ": " + hipGetErrorString(e));
    return MW_ERR_HIP;
}

constexpr int64_t kMaxThreads = (1LL << 32) - 256;           // of a launch along one dimension

bool misaligned(const void* p, uintptr_t n) { return reinterpret_cast<uintptr_t>(p) % n != 0; }

// whether rows of `dim` values, n x m of them at these strides, share memory
bool overlapping(int64_t n, int64_t n_stride, int64_t m, int64_t m_stride, int64_t dim) {
    const int64_t a = llabs(n_stride), b = llabs(m_stride);
    if ((n > 1 && a < dim) || (m > 1 && b < dim)) return true;
    return n > 1 && m > 1 && a < (m - 1) * b + dim && b < (n - 1) * a + dim;
}

int check_cache(const char* who, const mw_paged_cache* c) {
    REFUSE_IF(!c || !c->k || !c->v, "null cache");
    REFUSE_IF(c->dtype != MW_F16 && c->dtype != MW_BF16 && c->dtype != MW_E4M3, "the cache's dtype must be MW_F16, MW_BF16 or MW_E4M3");
    REFUSE_IF(c->head_dim != 64 && c->head_dim != 128, "head_dim must be 64 or 128");
    REFUSE_IF(c->n_heads < 1 || c->n_heads > 1024, "n_heads must be in 1..1024");
    REFUSE_IF(c->page_size < 16 || c->page_size > 4096 || (c->page_size & (c->page_size - 1)), "page_size must be a power of two in 16..4096");
    REFUSE_IF(c->n_pages < 1 || (int64_t)c->n_pages * c->page_size > INT32_MAX, "n_pages must be at least 1 and the cache hold less than 2^31 tokens");
    REFUSE_IF((c->dtype == MW_E4M3) != (c->k_scale != nullptr) || (c->dtype == MW_E4M3) != (c->v_scale != nullptr),
              "row scales belong to an e4m3 cache, and only to one");
    const int64_t unit = c->dtype == MW_E4M3 ? 16 : 8;
    REFUSE_IF(c->page_stride % unit || c->head_stride % unit || c->token_stride % unit || misaligned(c->k, 16) || misaligned(c->v, 16),
              "rows of the cache must start at multiples of 16 bytes");
    REFUSE_IF(c->token_stride < c->head_dim || c->head_stride < c->head_dim || c->page_stride < c->head_dim, "strides of the cache must be at least head_dim");
    REFUSE_IF(c->token_stride > (1 << 26) || c->page_stride > UINT32_MAX, "token_stride must be at most 2^26 and page_stride below 2^32");
    return MW_OK;
}
int log2i(int n) { int s = 0; while ((1 << s) < n) ++s; return s; }
PagedCacheView view_of(const mw_paged_cache& c) {
    return PagedCacheView{c.k, c.v, c.k_scale, c.v_scale, c.page_stride, c.head_stride, c.token_stride, c.n_pages, log2i(c.page_size), c.n_heads};
}

}  // namespace

extern "C" int mw_paged_plan(const mw_plan_args* a, int device, void* stream) {
    const char* who = "mw_paged_plan";
    REFUSE_IF(!a, "null argument");
    REFUSE_IF(a->batch < 1 || a->batch > kPlanMaxBatch, "batch must be in 1.." + std::to_string(kPlanMaxBatch));
    REFUSE_IF(a->rows < 0 || a->rows >= (1 << 30), "rows must be in 0..2^30 - 1");
    REFUSE_IF(a->page_size < 16 || a->page_size > 4096 || (a->page_size & (a->page_size - 1)), "page_size must be a power of two in 16..4096");
    REFUSE_IF(a->max_pages < 1 || (int64_t)a->max_pages * a->page_size > INT32_MAX, "max_pages must be at least 1 and a request hold less than 2^31 tokens");
    REFUSE_IF(a->table_stride < a->max_pages, "table_stride must be at least max_pages");
    REFUSE_IF(a->n_pages < 1 || (int64_t)a->n_pages * a->page_size > INT32_MAX, "n_pages must be at least 1 and the pool hold less than 2^31 tokens");
    REFUSE_IF(!a->kept || !a->fresh || !a->table || !a->pages_in || !a->pages_out || !a->free_list || !a->n_free_in || !a->n_free_out ||
              !a->row_start || !a->admitted, "null array");
    REFUSE_IF(a->pages_in == a->pages_out || a->n_free_in == a->n_free_out, "the counts after the step need arrays of their own");
    REFUSE_IF(a->rows > 0 && (!a->slots || !a->positions), "null slots or positions");
    REFUSE_IF(a->parents && (!a->mask || a->mask_words < 1 || a->mask_words > kPlanMaxWords), "trees need a mask of 1..8 words a row");
    REFUSE_IF((a->units == nullptr) != (a->unit_start == nullptr), "units and unit_start go together");
    REFUSE_IF(a->units && (a->chunk_units < 0 || a->chunk_units > 65536 || a->chunk_min < 1 || misaligned(a->units, 16)),
              "chunk_units must be in 0..65536, chunk_min at least 1 and units 16-byte aligned");
    OnDevice on(device);
    if (on.err != hipSuccess) return launched(who, on.err);
    PlanParams p{};
    p.batch = a->batch; p.rows = a->rows; p.page_shift = log2i(a->page_size); p.max_pages = a->max_pages; p.n_pages = a->n_pages;
    p.kept = a->kept; p.fresh = a->fresh; p.parents = a->parents; p.table = a->table; p.table_stride = a->table_stride;
    p.pages_in = a->pages_in; p.pages_out = a->pages_out; p.free_list = a->free_list; p.n_free_in = a->n_free_in; p.n_free_out = a->n_free_out;
    p.row_start = a->row_start; p.admitted = a->admitted; p.positions = a->positions;
    static_assert(sizeof(long) == sizeof(int64_t), "");
    p.slots = reinterpret_cast<long*>(a->slots); p.mask = a->mask; p.mask_words = a->parents ? a->mask_words : 0;
    p.units = a->units; p.unit_start = a->unit_start; p.chunk_units = a->chunk_units; p.chunk_min = a->chunk_min;
    return launched(who, launch_paged_plan(p, static_cast<hipStream_t>(stream)));
}

extern "C" int mw_paged_write(const mw_paged_cache* cache, const void* k, const void* v, int dtype, int64_t k_row_stride, int64_t k_head_stride,
                              int64_t v_row_stride, int64_t v_head_stride, const int64_t* slots, int64_t rows, int device, void* stream) {
    const char* who = "mw_paged_write";
    int r = check_cache(who, cache);
    if (r) return r;
    REFUSE_IF(dtype != MW_F16 && dtype != MW_BF16, "rows must be MW_F16 or MW_BF16");
    REFUSE_IF(cache->dtype != MW_E4M3 && cache->dtype != dtype, "a 16-bit cache takes rows of its own type");
    REFUSE_IF(rows < 0 || rows > (1 << 30), "rows must be in 0..2^30");
    if (rows == 0) return MW_OK;
    REFUSE_IF(!k || !v || !slots, "null array");
    REFUSE_IF(misaligned(k, 16) || misaligned(v, 16) || k_row_stride % 8 || k_head_stride % 8 || v_row_stride % 8 || v_head_stride % 8,
              "rows must start at multiples of 16 bytes");
    REFUSE_IF(rows * cache->n_heads * (cache->head_dim / 8) > kMaxThreads, "too many rows for one launch");
    OnDevice on(device);
    if (on.err != hipSuccess) return launched(who, on.err);
    return launched(who, launch_paged_write(view_of(*cache), cache->head_dim, dtype == MW_BF16, k, v, k_row_stride, k_head_stride, v_row_stride,
                                            v_head_stride, reinterpret_cast<const long*>(slots), rows, static_cast<hipStream_t>(stream)));
}

static int check_attention(const char* who, const mw_tree_args* a) {
    REFUSE_IF(!a, "null argument");
    int r = check_cache(who, &a->cache);
    if (r) return r;
    REFUSE_IF(a->dtype != MW_F16 && a->dtype != MW_BF16, "q and out must be MW_F16 or MW_BF16");
    REFUSE_IF(a->cache.dtype != MW_E4M3 && a->cache.dtype != a->dtype, "a 16-bit cache is read with queries of its own type");
    REFUSE_IF(a->n_heads < 1 || a->n_heads > 4096 || a->n_heads % a->cache.n_heads, "the query heads must be a multiple of the cache's, at most 4096");
    REFUSE_IF(a->batch < 1 || a->batch > (1 << 20), "batch must be in 1..2^20");
    REFUSE_IF(a->rows < 0 || a->rows > (1 << 30) || a->max_nodes < 0 || a->max_nodes > (1 << 20), "rows must be in 0..2^30 and max_nodes in 0..2^20");
    REFUSE_IF(a->n_units < 0 || a->n_units > (1 << 24), "n_units must be in 0..2^24");
    REFUSE_IF(a->max_pages < 1 || (int64_t)a->max_pages * a->cache.page_size > INT32_MAX - 4096, "max_pages must be at least 1 and a request hold less than 2^31 - 4096 tokens");
    REFUSE_IF(a->table_stride < a->max_pages, "table_stride must be at least max_pages");
    REFUSE_IF(a->mask && (a->mask_words < 1 || a->mask_words > (1 << 15) || a->max_nodes > 32 * a->mask_words), "mask_words must hold a bit for every node");
    REFUSE_IF(!(a->scale > 0.f) || isinf(a->scale), "scale must be positive and finite");
    return MW_OK;
}

extern "C" int64_t mw_tree_attention_workspace(const mw_tree_args* a) {
    int r = check_attention("mw_tree_attention_workspace", a);
    if (r) return r;
    return tree_attn_workspace(a->n_units, a->batch, a->cache.n_heads, a->n_heads / a->cache.n_heads, a->max_nodes, a->cache.head_dim);
}

extern "C" int mw_tree_attention(const mw_tree_args* a, int device, void* stream) {
    const char* who = "mw_tree_attention";
    int r = check_attention(who, a);
    if (r) return r;
    if (a->rows == 0 || a->max_nodes == 0 || a->n_units == 0) return MW_OK;
    REFUSE_IF(!a->q || !a->out || !a->table || !a->kept || !a->row_start || !a->units || !a->unit_start, "null array");
    REFUSE_IF(misaligned(a->q, 16) || a->q_row_stride % 8 || a->q_head_stride % 8, "rows of q must start at multiples of 16 bytes");
    REFUSE_IF(misaligned(a->out, 8) || a->out_row_stride % 4 || a->out_head_stride % 4, "rows of out must start at multiples of 8 bytes");
    REFUSE_IF(overlapping(a->rows, a->out_row_stride, a->n_heads, a->out_head_stride, a->cache.head_dim), "rows of out must not overlap");
    REFUSE_IF(misaligned(a->units, 16), "units must be 16-byte aligned");
    const int group = a->n_heads / a->cache.n_heads;
    const int64_t need = tree_attn_workspace(a->n_units, a->batch, a->cache.n_heads, group, a->max_nodes, a->cache.head_dim);
    REFUSE_IF(need && (!a->workspace || a->workspace_bytes < need || misaligned(a->workspace, 16)),
              "the workspace is smaller than mw_tree_attention_workspace() or not 16-byte aligned");
    REFUSE_IF(((int64_t)a->n_units * a->cache.n_heads + 8) * (((int64_t)a->max_nodes * group + 127) / 128) > kMaxThreads / 256 ||
              (need && (int64_t)a->batch * a->max_nodes * a->n_heads * (a->cache.head_dim / 4) > kMaxThreads), "too many units or rows for one launch");
    OnDevice on(device);
    if (on.err != hipSuccess) return launched(who, on.err);
    TreeAttnParams p{};
    p.c = view_of(a->cache); p.dim = a->cache.head_dim; p.bf16 = a->dtype == MW_BF16; p.heads = a->n_heads; p.rows = a->rows; p.batch = a->batch;
    p.max_nodes = a->max_nodes; p.q = a->q; p.q_row = a->q_row_stride; p.q_head = a->q_head_stride; p.out = a->out;
    p.out_row = a->out_row_stride; p.out_head = a->out_head_stride; p.table = a->table; p.table_stride = a->table_stride; p.max_pages = a->max_pages;
    p.kept = a->kept; p.row_start = a->row_start; p.units = a->units; p.unit_start = a->unit_start; p.n_units = a->n_units;
    p.mask = a->mask; p.mask_words = a->mask ? a->mask_words : 0; p.scale = a->scale; p.workspace = need ? static_cast<float*>(a->workspace) : nullptr;
    return launched(who, launch_tree_attention(p, static_cast<hipStream_t>(stream)));
}

static int check_accept(const char* who, const mw_accept_args* a) {
    REFUSE_IF(!a, "null argument");
    REFUSE_IF(a->dtype != MW_F32 && a->dtype != MW_F16 && a->dtype != MW_BF16, "logits must be MW_F32, MW_F16 or MW_BF16");
    REFUSE_IF(a->rows < 0 || a->rows >= (1 << 24), "rows must be in 0..2^24 - 1");
    REFUSE_IF(a->vocab < 1 || a->vocab > (1 << 24), "vocab must be in 1..2^24");
    REFUSE_IF(a->batch < 1 || a->batch > (1 << 20), "batch must be in 1..2^20");
    REFUSE_IF(a->depth < 1 || a->depth > kAcceptMaxNodes, "depth must be in 1.." + std::to_string(kAcceptMaxNodes));
    return MW_OK;
}

extern "C" int64_t mw_tree_accept_workspace(const mw_accept_args* a) {
    int r = check_accept("mw_tree_accept_workspace", a);
    if (r) return r;
    return (int64_t)a->rows * accept_parts(a->rows, a->vocab) * 8;
}

extern "C" int mw_tree_accept(const mw_accept_args* a, int device, void* stream) {
    const char* who = "mw_tree_accept";
    int r = check_accept(who, a);
    if (r) return r;
    REFUSE_IF(!a->row_start || !a->path || !a->count || !a->out_tokens, "null array");
    REFUSE_IF(a->rows > 0 && (!a->logits || !a->tokens || !a->parents || !a->best || !a->workspace), "null array");
    REFUSE_IF(a->rows > 1 && a->logits_stride < a->vocab, "logits_stride must be at least vocab");
    REFUSE_IF(misaligned(a->logits, a->dtype == MW_F32 ? 4 : 2), "logits must be aligned to their type");
    REFUSE_IF(a->workspace_bytes < (int64_t)a->rows * accept_parts(a->rows, a->vocab) * 8 || misaligned(a->workspace, 4),
              "the workspace is smaller than mw_tree_accept_workspace() or not 4-byte aligned");
    OnDevice on(device);
    if (on.err != hipSuccess) return launched(who, on.err);
    AcceptParams p{};
    p.logits = a->logits; p.stride = a->logits_stride; p.dtype = a->dtype; p.rows = a->rows; p.vocab = a->vocab; p.batch = a->batch; p.depth = a->depth;
    p.suppress = a->suppress; p.tokens = a->tokens; p.parents = a->parents; p.row_start = a->row_start; p.best = a->best; p.path = a->path;
    p.count = a->count; p.out_tokens = a->out_tokens; p.workspace = a->workspace;
    return launched(who, launch_tree_accept(p, static_cast<hipStream_t>(stream)));
}

extern "C" int mw_paged_compact(const mw_paged_cache* cache, int32_t n_layers, int64_t layer_stride, const int32_t* table, int64_t table_stride,
                                int32_t max_pages, const int32_t* kept, const int32_t* path, int32_t path_stride, const int32_t* count,
                                int32_t batch, int device, void* stream) {
    const char* who = "mw_paged_compact";
    int r = check_cache(who, cache);
    if (r) return r;
    REFUSE_IF(n_layers < 1 || n_layers > 65535, "n_layers must be in 1..65535");
    REFUSE_IF(n_layers > 1 && (layer_stride < cache->head_dim || layer_stride % (cache->dtype == MW_E4M3 ? 16 : 8)), "layers must start at multiples of 16 bytes");
    REFUSE_IF(batch < 1 || batch > 65535, "batch must be in 1..65535");
    REFUSE_IF(path_stride < 0 || path_stride > (1 << 20), "path_stride must be in 0..2^20");
    REFUSE_IF(max_pages < 1 || (int64_t)max_pages * cache->page_size > INT32_MAX, "max_pages must be at least 1 and a request hold less than 2^31 tokens");
    REFUSE_IF(table_stride < max_pages, "table_stride must be at least max_pages");
    if (path_stride == 0) return MW_OK;
    REFUSE_IF(!table || !kept || !path || !count, "null array");
    OnDevice on(device);
    if (on.err != hipSuccess) return launched(who, on.err);
    const int64_t scale_stride = (int64_t)cache->n_pages * cache->n_heads * cache->page_size;
    return launched(who, launch_paged_compact(view_of(*cache), n_layers, layer_stride, scale_stride, cache->head_dim, table, table_stride, max_pages,
                                              kept, path, path_stride, count, batch, static_cast<hipStream_t>(stream)));
}
