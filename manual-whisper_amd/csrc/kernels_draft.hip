// Bookkeeping of drafted decoding for gfx950: after every pass, what was accepted is filed and the next trees are grown from
// the caller's drafts; before every pass, the tree rows' embeddings.  Bound by latency, beside a pass of some hundred launches.
#include "mw_kernels.h"

namespace mw {

namespace {

__global__ __launch_bounds__(256) void draft_init_kernel(DraftParams p, int prompt_len) {
    const int tid = threadIdx.x;
    if (blockIdx.x == 0) {
        if (tid == 0) {
            p.st->pos = 0; p.st->prompt_len = prompt_len; p.st->max_new = p.max_new; p.st->eot = p.eot;
            p.st->n_finished = 0; p.st->batch = p.n_audio;
            p.n_free[0] = p.n_pages;
        }
        for (int i = tid; i < p.n_pages; i += 256) p.free_list[i] = p.n_pages - 1 - i;
        for (int i = tid; i < p.n_audio; i += 256) {
            p.kept[i] = 0; p.pages[i] = 0; p.len[i] = 0; p.finished[i] = 0; p.out_len[i] = p.max_new;
            p.fresh_prompt[i] = prompt_len; p.fresh_tree[i] = p.nodes; p.first_rows[i] = i;
        }
        if (tid == 0) p.first_rows[p.n_audio] = p.n_audio;
        for (int i = tid; i < p.n_audio * p.n_drafts; i += 256) p.shift[i] = 0;
    }
    for (long i = (long)blockIdx.x * 256 + tid; i < (long)p.n_audio * p.max_new; i += (long)gridDim.x * 256) p.out_ids[i] = p.eot;
}

// File the accepted tokens of recording b and grow its next tree.  Lane i holds node i of the tree.
//
// A draft proposes what follows the place where it agrees best with the tokens so far: the longest common stretch (up to
// kMatch tokens) that ends in the last token, among equals the one nearest to where the draft was last followed.  Where it
// agrees nowhere (the model just chose another word) the draft is taken up again as far on as its last place was.
// The drafts share the tree: they go in one after another, first with an equal share of its nodes each, then the rest for
// whoever has more; a common beginning is stored once.
// One wave per recording, so that a tree lives in its lanes (a ballot finds a child, a shuffle reads a token) and nothing needs a
// barrier.  16 recordings, two drafts of 100 tokens, trees of 8: 4 us when the drafts have ended, 9 us (the search of both
// drafts, one dependent load a compared token) otherwise.
constexpr int kMatch = 4;
__global__ __launch_bounds__(64) void draft_step_kernel(DraftParams p, int depth, int advance) {
    const int b = blockIdx.x, lane = threadIdx.x;
    // what the plan of the last pass left becomes what the next one starts from
    if (lane == 0) {
        p.pages[b] = p.pages_after[b];
        if (b == 0) p.n_free[0] = p.n_free_after[0];
    }
    int* const tokens = p.tokens + b * p.nodes;
    int* const parents = p.parents + b * p.nodes;
    if (p.finished[b]) {                                     // its rows ride along: nothing is accepted or filed any more
        if (lane < p.nodes) { tokens[lane] = lane ? -1 : p.eot; parents[lane] = lane ? 0 : -1; }
        return;
    }
    // ---- file
    const int m = min(max(p.count[b], 0), depth);
    int len = p.len[b];
    int* const out = p.out_ids + (long)b * p.max_new;
    const int t = lane < m ? p.out_tokens[(long)b * depth + lane] : -1;
    const unsigned long long ends = __ballot(lane < m && t == p.eot);
    const int upto = min(ends ? __ffsll(ends) - 1 : m, p.max_new - len);                // tokens to file
    const bool ended = (ends && upto == __ffsll(ends) - 1 && len + upto < p.max_new) || len + upto >= p.max_new;
    if (lane < upto) out[len + lane] = t;
    len += upto;
    if (ended) {
        if (lane == 0) {
            p.len[b] = len; p.out_len[b] = len; p.finished[b] = 1;
            atomicAdd(&p.st->n_finished, 1);
        }
        if (lane < p.nodes) { tokens[lane] = lane ? -1 : p.eot; parents[lane] = lane ? 0 : -1; }
        return;
    }
    const int kept = advance ? advance : p.kept[b] + m;
    if (lane == 0) { p.len[b] = len; p.kept[b] = kept; }
    __syncthreads();                                         // out[] is read below (one wave: orders its own stores)
    // ---- the next tree: root = the last token
    const int root = __shfl(t, m - 1);
    int tok = lane == 0 ? root : -1, par = lane == 0 ? -1 : 0, n = 1;
    const int longest = min(min(p.nodes - 1, p.max_new - len - 1), p.n_text_ctx - 1 - kept);     // deeper ones could not be filed
    int place[kMaxDrafts];
#pragma unroll 1
    for (int d = 0; d < p.n_drafts; ++d) {
        const int* draft = p.drafts + ((long)b * p.n_drafts + d) * p.max_draft;
        const int dl = p.draft_len[b * p.n_drafts + d];
        const int expect = len + p.shift[b * p.n_drafts + d];
        int best = 0;                                        // (length of the common stretch, nearness, place)
        for (int q = 1 + lane; q <= dl; q += 64) {
            int s = 0;
            while (s < kMatch && s < len && q - 1 - s >= 0 && draft[q - 1 - s] == out[len - 1 - s]) ++s;
            if (s) best = max(best, (s << 20) | ((511 - min(abs(q - expect), 511)) << 10) | (1023 - q));
        }
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) best = max(best, __shfl_xor(best, o));
        const int q = best ? 1023 - (best & 1023) : min(max(expect, 0), dl);
        if (best && lane == 0) p.shift[b * p.n_drafts + d] = q - len;
        place[d & (kMaxDrafts - 1)] = q;
    }
    for (int round = 0; round < 2; ++round) {
        const int share = round == 0 && p.n_drafts > 1 ? (p.nodes - 1 + p.n_drafts - 1) / p.n_drafts : p.nodes;
#pragma unroll 1
        for (int d = 0; d < p.n_drafts; ++d) {
            const int* draft = p.drafts + ((long)b * p.n_drafts + d) * p.max_draft;
            const int q = place[d & (kMaxDrafts - 1)], more = min(min(p.draft_len[b * p.n_drafts + d] - q, longest), share);
            const int ahead = lane < more ? draft[q + lane] : -1;
            int cur = 0;
            for (int j = 0; j < more && n <= p.nodes; ++j) {
                const int want = __shfl(ahead, j);
                const unsigned long long child = __ballot(lane > 0 && lane < n && par == cur && tok == want);
                if (child) cur = __ffsll(child) - 1;
                else if (n < p.nodes) {
                    if (lane == n) { tok = want; par = cur; }
                    cur = n++;
                } else break;
                if (want == p.eot) break;
            }
        }
    }
    if (lane < p.nodes) { tokens[lane] = tok; parents[lane] = par; }
}

// x[row] = token embedding + positional embedding of the row's token and position; rows without a token hold some token's.  A
// workgroup per row; 128 rows of 384: 4.6 us, three dependent loads.
__global__ __launch_bounds__(256) void draft_embed_kernel(const int* __restrict__ tokens, const int* __restrict__ positions, const f16* __restrict__ tok_emb,
                                                          const f16* __restrict__ pos_emb, int D, int n_text_ctx, float* __restrict__ x) {
    const long r = blockIdx.x;
    const int tok = max(tokens[r], 0), pos = min(max(positions[r], 0), n_text_ctx - 1);
    for (int c = threadIdx.x; c < D; c += 256) x[r * D + c] = (float)tok_emb[(long)tok * D + c] + (float)pos_emb[(long)pos * D + c];
}

}  // namespace

void launch_draft_init(const DraftParams& p, int prompt_len, hipStream_t s) {
    const long n = (long)p.n_audio * p.max_new;
    draft_init_kernel<<<(unsigned)((n + 1023) / 1024), 256, 0, s>>>(p, prompt_len);
}
void launch_draft_step(const DraftParams& p, int depth, int advance, hipStream_t s) { draft_step_kernel<<<p.n_audio, 64, 0, s>>>(p, depth, advance); }
void launch_draft_embed(const int* tokens, const int* positions, const f16* tok_emb, const f16* pos_emb, int D, int n_text_ctx, float* x, int rows,
                        hipStream_t s) {
    draft_embed_kernel<<<rows, 256, 0, s>>>(tokens, positions, tok_emb, pos_emb, D, n_text_ctx, x);
}

}  // namespace mw
