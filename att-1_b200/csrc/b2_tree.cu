// b2_tree.cu - the steps around the attention of several new rows per sequence
// (b2_attn_rows.cu): page tables, positions and cache slots from the
// sequences' lengths (b2_kv_plan), RoPE and the K/V store by slot
// (b2_rows_append), greedy verification of drafted trees (b2_tree_accept) and
// the taken rows' K/V moved together (b2_kv_compact).
//
// No kernel here waits for another CTA, keeps a counter between calls or adds
// atomically into a result: what several CTAs need (the prefix sums of
// b2_kv_plan) each computes for itself, so overlapping calls share nothing.
#include "b2_common.cuh"

namespace b2 {

static cudaError_t launch_tree(const void *fn, dim3 grid, dim3 block, size_t smem, int pdl, cudaStream_t st, void **args)
{
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = pdl ? 1 : 0;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelExC(&cfg, fn, args);
}

// ---- b2_kv_plan ---------------------------------------------------------------------

constexpr int kPlanThreads = 512;
constexpr uint32_t kPlanRowsPerCta = 1024;  // rows a CTA expands at a time

// Last index i in [0, n) with start[i] <= at (start ascending, start[0] = 0):
// the sequence a row or a fresh page belongs to; empty ones are skipped.
__device__ __forceinline__ uint32_t plan_find(const uint32_t *start, uint32_t n, uint32_t at)
{
    uint32_t lo = 0, hi = n;
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) >> 1;
        if (start[mid] <= at) lo = mid;
        else hi = mid;
    }
    return lo;
}

// Every CTA forms the exclusive prefix sums of the new rows and of the fresh
// pages over all sequences in shared memory (16 bytes per sequence; reading the
// three length arrays from L2 costs each CTA about a microsecond, less than a
// second launch or a wait between CTAs would), checks the step as a whole, and
// then writes its share of the rows and of the fresh pages. A row's page is
// read from the table below mapped[b] and computed from the free stack above,
// so no CTA depends on another's table writes.
__global__ void __launch_bounds__(kPlanThreads) kv_plan_kernel(const b2_kv_plan_args a)
{
    extern __shared__ uint32_t plan_smem[];
    uint32_t *ctx = plan_smem, *map = ctx + a.batch, *rows0 = map + a.batch, *fresh0 = rows0 + a.batch;
    __shared__ unsigned long long wsum[2][kPlanThreads / 32];
    __shared__ int bad;
    pdl_wait();
    pdl_launch_dependents();
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (tid == 0) bad = 0;
    __syncthreads();
    // consecutive sequences per thread: sums, block scan, then the prefixes
    const uint32_t per = (a.batch + kPlanThreads - 1) / kPlanThreads;
    const uint32_t b0 = min(tid * per, a.batch), b1 = min(b0 + per, a.batch);
    const uint32_t cap = a.pages_per_seq * a.page_tokens;
    unsigned long long nr = 0, nf = 0;
    int wrong = 0;
    for (uint32_t b = b0; b < b1; ++b) {
        const int32_t c = a.ctx_len[b], n = a.new_len[b], mp = a.mapped[b];
        if (c < 0 || n < 0 || (uint32_t)c > cap || (uint32_t)n > cap - (uint32_t)c || mp < 0 ||
            (uint32_t)mp > a.pages_per_seq || (uint64_t)mp * a.page_tokens < (uint64_t)c ||
            (a.tree != nullptr && n > B2_MAX_TREE)) {
            wrong = B2_ERR_POSITION;
            break;
        }
        const uint32_t need = ((uint32_t)c + (uint32_t)n + a.page_tokens - 1) / a.page_tokens;
        const uint32_t fresh = need > (uint32_t)mp ? need - (uint32_t)mp : 0;
        ctx[b] = (uint32_t)c;
        map[b] = (uint32_t)mp;
        rows0[b] = (uint32_t)n;
        fresh0[b] = fresh;
        nr += (uint32_t)n;
        nf += fresh;
    }
    if (wrong) atomicOr(&bad, wrong);
    unsigned long long ir = nr, jf = nf;  // inclusive over the warp
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long r = __shfl_up_sync(0xffffffffu, ir, o), f = __shfl_up_sync(0xffffffffu, jf, o);
        if (lane >= (uint32_t)o) {
            ir += r;
            jf += f;
        }
    }
    if (lane == 31) {
        wsum[0][warp] = ir;
        wsum[1][warp] = jf;
    }
    __syncthreads();
    unsigned long long er = ir - nr, ef = jf - nf, total = 0, fresh_total = 0;
    for (uint32_t w = 0; w < kPlanThreads / 32; ++w) {
        if (w < warp) {
            er += wsum[0][w];
            ef += wsum[1][w];
        }
        total += wsum[0][w];
        fresh_total += wsum[1][w];
    }
    const int32_t have = *a.free_count;
    int status = bad;
    if (status == 0 && (total > a.max_rows || have < 0 || fresh_total > (unsigned long long)have))
        status = B2_ERR_CAPACITY;
    if (status != 0) {  // the step as a whole: no rows, nothing changed
        if (blockIdx.x == 0) {
            for (uint32_t b = tid; b < a.batch; b += kPlanThreads) a.mapped_out[b] = a.mapped[b];
            for (uint32_t b = tid; b <= a.batch; b += kPlanThreads) a.row_start[b] = 0;
            if (tid == 0) {
                *a.free_out = have;
                raise_error(a.err, status);
            }
        }
        return;
    }
    for (uint32_t b = b0; b < b1; ++b) {  // each thread its own entries
        const uint32_t n = rows0[b], f = fresh0[b];
        rows0[b] = (uint32_t)er;
        fresh0[b] = (uint32_t)ef;
        er += n;
        ef += f;
    }
    __syncthreads();
    const uint32_t nrows = (uint32_t)total, nfresh = (uint32_t)fresh_total;
    int fault = 0;
    if (blockIdx.x == 0) {
        for (uint32_t b = tid; b < a.batch; b += kPlanThreads) {
            a.row_start[b] = (int32_t)rows0[b];
            a.mapped_out[b] = (int32_t)(map[b] + (b + 1 < a.batch ? fresh0[b + 1] : nfresh) - fresh0[b]);
        }
        if (tid == 0) {
            a.row_start[a.batch] = (int32_t)nrows;
            *a.free_out = have - (int32_t)nfresh;
        }
    }
    const uint32_t stride = gridDim.x * kPlanThreads;
    for (uint32_t r = blockIdx.x * kPlanThreads + tid; r < nrows; r += stride) {
        const uint32_t b = plan_find(rows0, a.batch, r), i = r - rows0[b], at = ctx[b] + i;
        const uint32_t lp = at / a.page_tokens;
        const int32_t page = lp < map[b] ? a.page_table[(size_t)b * a.pages_per_seq + lp]
                                         : a.free_pages[have - 1 - (int32_t)(fresh0[b] + lp - map[b])];
        const bool ok = page >= 0 && (uint32_t)page < a.pool_pages;
        if (!ok) fault |= B2_ERR_POSITION;
        uint32_t depth = i;
        if (a.tree != nullptr) {
            depth = (uint32_t)__popcll(a.tree[r]);
            if (depth == 0) fault |= B2_ERR_TREE;
            else --depth;
        }
        a.row_item[r] = (int32_t)b;
        a.row_pos[r] = (int32_t)(ctx[b] + depth);
        a.row_slot[r] = ok ? page * (int32_t)a.page_tokens + (int32_t)(at % a.page_tokens) : -1;
    }
    for (uint32_t k = blockIdx.x * kPlanThreads + tid; k < nfresh; k += stride) {
        const uint32_t b = plan_find(fresh0, a.batch, k);
        const int32_t page = a.free_pages[have - 1 - (int32_t)k];
        if (page < 0 || (uint32_t)page >= a.pool_pages) fault |= B2_ERR_POSITION;
        a.page_table[(size_t)b * a.pages_per_seq + map[b] + k - fresh0[b]] = page;
    }
    if (fault) raise_error(a.err, fault);
}

// ---- b2_rows_append -------------------------------------------------------------------

constexpr uint32_t kAppendThreads = 128;  // twice as many for head sizes above 512
constexpr uint32_t kAppendBatch = 4;      // heads a thread loads before it stores them

// grid (head parts, rows): a thread owns four dimensions (two RoPE pairs) of a
// row and takes every hgroups-th head of its part, so the sine and cosine of a
// pair are computed once per thread, not once per head; q | k | v heads in one
// sequence of h + 2 hkv. One float4 in, one out per head. Bound by one load
// round trip for few rows and by HBM for many, which takes enough bytes on
// their way: four heads' loads go out before the row's slot and angles are
// known (2048 rows of the 8B shape: 19.2 us, 5.2 TB/s; one load at a time 25.4;
// six 19.0, with 256 threads 20.8, 512 23.3, whose CTAs leave in coarser steps).
__global__ void __launch_bounds__(2 * kAppendThreads) rows_append_kernel(const b2_rows_append_args a, uint32_t heads_per_part)
{
    pdl_wait();
    pdl_launch_dependents();
    const uint32_t hd = a.kv.head_dim, cols = hd / 4, hgroups = blockDim.x / cols;
    const uint32_t col = threadIdx.x % cols, hg = threadIdx.x / cols;
    const uint32_t qh = a.q_rows / hd, hkv = a.kv.n_kv_heads, heads = qh + 2 * hkv;
    const uint32_t h0 = blockIdx.x * heads_per_part, h1 = min(heads, h0 + heads_per_part);
    // (not a read-only load: the kernel before may write it while this one is resident)
    const uint32_t m = a.n_rows != nullptr ? (uint32_t)min(max(*a.n_rows, 0), (int32_t)min(a.m, 0x7FFFFFFFu)) : a.m;
    const uint32_t slots = a.pool_pages * a.kv.page_tokens;
    if (hg >= hgroups) return;
    for (uint32_t n = blockIdx.y; n < m; n += gridDim.y) {
        const float *y = a.y + (size_t)n * a.y_stride + 4 * col;
        float4 x[kAppendBatch];  // asked for before the row's slot, position and angles are known
        auto load = [&](uint32_t h) {
#pragma unroll
            for (uint32_t k = 0; k < kAppendBatch; ++k)
                if (h + k * hgroups < h1) x[k] = __ldcs(reinterpret_cast<const float4 *>(y + (size_t)(h + k * hgroups) * hd));
        };
        load(h0 + hg);
        const int32_t slot = a.slots[n];
        const int32_t pos = a.rope_freq != nullptr ? a.positions[n] : 0;
        if (pos < 0 || (slot >= 0 && (uint32_t)slot >= slots)) {
            if (threadIdx.x == 0 && blockIdx.x == 0) raise_error(a.err, B2_ERR_POSITION);
            if (pos < 0) continue;
        }
        const bool store = slot >= 0 && (uint32_t)slot < slots;
        const size_t page = store ? (uint32_t)slot / a.kv.page_tokens : 0;
        const uint32_t off = store ? (uint32_t)slot % a.kv.page_tokens : 0;
        float s0 = 0.0f, c0 = 1.0f, s1 = 0.0f, c1 = 1.0f;
        if (a.rope_freq != nullptr) {  // src/rope.c:20-30, the f32 product of position and frequency
            sincosf(__fmul_rn((float)pos, a.rope_freq[2 * col]), &s0, &c0);
            sincosf(__fmul_rn((float)pos, a.rope_freq[2 * col + 1]), &s1, &c1);
        }
        for (uint32_t hb = h0 + hg; hb < h1; hb += kAppendBatch * hgroups) {
            if (hb != h0 + hg) load(hb);
#pragma unroll
            for (uint32_t k = 0; k < kAppendBatch; ++k) {
                const uint32_t h = hb + k * hgroups;
                if (h >= h1) break;
                float4 v = x[k];
                if (h < qh + hkv && a.rope_freq != nullptr) {
                    v = make_float4(__fsub_rn(__fmul_rn(v.x, c0), __fmul_rn(v.y, s0)),
                                    __fadd_rn(__fmul_rn(v.x, s0), __fmul_rn(v.y, c0)),
                                    __fsub_rn(__fmul_rn(v.z, c1), __fmul_rn(v.w, s1)),
                                    __fadd_rn(__fmul_rn(v.z, s1), __fmul_rn(v.w, c1)));
                }
                if (h < qh) {
                    reinterpret_cast<float4 *>(a.q + (size_t)n * a.q_stride + (size_t)h * hd)[col] = v;
                } else if (store) {
                    const uint32_t kh = h < qh + hkv ? h - qh : h - qh - hkv;
                    float *pool = h < qh + hkv ? a.kv.k_pool : a.kv.v_pool;
                    reinterpret_cast<float4 *>(pool + ((page * hkv + kh) * a.kv.page_tokens + off) * hd)[col] = v;
                }
            }
        }
    }
}

// ---- b2_tree_accept -------------------------------------------------------------------

constexpr int kAcceptWarps = 4;

// One warp per item, rows i = lane and lane + 32. A row's parent is the highest
// bit of its mask below itself, and a tree's mask is its parent's and its own
// bit, down to the root's. A row fits when its token is the argmax token of its
// parent and no earlier sibling carries the same token; with M the 64-bit set of
// fitting rows, a row is taken when its mask lies inside M. The taken rows are
// one branch: two taken children of a row would carry the same token. All in
// registers and shared memory; the time is two dependent load round trips.
__global__ void __launch_bounds__(kAcceptWarps * 32) tree_accept_kernel(const b2_tree_accept_args a)
{
    __shared__ uint32_t tok_s[kAcceptWarps][64], next_s[kAcceptWarps][64];
    __shared__ uint64_t mask_s[kAcceptWarps][64];
    __shared__ int8_t par_s[kAcceptWarps][64];
    pdl_wait();
    pdl_launch_dependents();
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t item = blockIdx.x * kAcceptWarps + warp;
    if (item >= a.batch) return;
    const int32_t r0 = a.row_start[item], r1 = a.row_start[item + 1];
    int fault = 0;
    uint32_t n = 0;
    if (r0 < 0 || r1 < r0 || (uint32_t)r1 > a.rows || (uint32_t)(r1 - r0) > a.max_rows) fault = B2_ERR_POSITION;
    else n = (uint32_t)(r1 - r0);
    uint64_t mask[2] = {0, 0};
    int par[2] = {-1, -1};
    bool tree[2] = {false, false};
    uint32_t *tok = tok_s[warp], *nxt = next_s[warp];
    int8_t *pr = par_s[warp];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const uint32_t i = lane + 32 * h;
        if (i < n) {
            mask[h] = a.tree != nullptr ? a.tree[r0 + i] : (2ull << i) - 1;
            mask_s[warp][i] = mask[h];
            tok[i] = a.tokens[r0 + i];
            nxt[i] = 0xFFFFFFFFu - (uint32_t)a.argmax[r0 + i];
        }
    }
    __syncwarp();
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const uint32_t i = lane + 32 * h;
        if (i < n) {
            const uint64_t above = mask[h] & ((1ull << i) - 1);
            const int up = 63 - __clzll(above);  // -1: none
            // itself, nothing after itself, and all that its parent has
            tree[h] = (mask[h] >> i) == 1 && (i == 0 || (up >= 0 && mask_s[warp][up] == above));
            if (!tree[h]) fault |= B2_ERR_TREE;
            par[h] = tree[h] ? up : -1;
            pr[i] = (int8_t)par[h];
        }
    }
    __syncwarp();
    bool fits[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const uint32_t i = lane + 32 * h;
        fits[h] = i < n && tree[h] && (i == 0 || (par[h] >= 0 && tok[i] == nxt[par[h]]));
        if (fits[h] && i > 0)
            for (uint32_t j = 1; j < i; ++j)
                if (pr[j] == par[h] && tok[j] == tok[i]) {
                    fits[h] = false;
                    break;
                }
    }
    const uint32_t mlo = __ballot_sync(0xffffffffu, fits[0]), mhi = __ballot_sync(0xffffffffu, fits[1]);
    const uint64_t M = (uint64_t)mhi << 32 | mlo;
    const bool t0 = fits[0] && (mask[0] & ~M) == 0, t1 = fits[1] && (mask[1] & ~M) == 0;
    const uint32_t alo = __ballot_sync(0xffffffffu, t0), ahi = __ballot_sync(0xffffffffu, t1);
    const uint64_t taken = (uint64_t)ahi << 32 | alo;
    const uint32_t count = (uint32_t)__popcll(taken);
    int32_t *path = a.path + (size_t)item * B2_MAX_TREE;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const uint32_t i = lane + 32 * h;
        if (h == 0 ? t0 : t1) path[__popcll(taken & ((1ull << i) - 1))] = (int32_t)i;
        if (i >= count) path[i] = -1;
    }
    if (lane == 0) {
        a.count[item] = (int32_t)count;
        a.next[item] = count > 0 ? nxt[63 - __clzll(taken)] : 0xFFFFFFFFu;
        a.ctx_out[item] = a.ctx_len[item] + (int32_t)count;
    }
    if (fault) raise_error(a.err, fault);
}

// ---- b2_kv_compact ----------------------------------------------------------------------

constexpr uint32_t kCompactLayers = 64;  // layers of one launch (24 bytes of parameters each)
constexpr int kCompactThreads = 128;
constexpr uint32_t kCompactBatch = 8;  // rows a thread loads before it stores them

struct CompactLayers {
    float *pool[kCompactLayers][2];
    const int32_t *table[kCompactLayers];
};

// CTA (layer, K or V and head group, item). A thread moves one float4 column of
// one head for all rows of the path, in path order: path[i] >= i, so a place
// written for row i is never the source of a later row, and a batch of loads
// may run ahead of its stores. Only one thread ever touches a column, so no
// CTA waits for another. The page lookups of the path's 64 rows happen once per
// CTA. Bound by HBM for large batches, by three load round trips for small.
__global__ void __launch_bounds__(kCompactThreads)
    kv_compact_kernel(const CompactLayers L, b2_kv_layout kv, uint32_t pool_pages, const int32_t *ctx_len,
                      const int32_t *path, const int32_t *count, int32_t *err)
{
    __shared__ uint2 src[B2_MAX_TREE], dst[B2_MAX_TREE];  // page, offset in page
    __shared__ uint32_t moves;
    pdl_wait();
    pdl_launch_dependents();
    const uint32_t layer = blockIdx.x, item = blockIdx.z;
    const uint32_t cols = kv.head_dim / 4, work = 2 * kv.n_kv_heads * cols;  // float4 columns of K and V
    if (threadIdx.x < 32) {
        const uint32_t lane = threadIdx.x;
        const int32_t n = count[item], c = ctx_len[item];
        const uint32_t cap = kv.pages_per_seq * kv.page_tokens;
        const int32_t *row = L.table[layer] + (size_t)item * kv.pages_per_seq;
        const bool fits = n >= 0 && n <= B2_MAX_TREE && c >= 0;
        int fault = fits ? 0 : B2_ERR_POSITION;
        uint32_t kept = 0;
        for (uint32_t i0 = 0; i0 < B2_MAX_TREE; i0 += 32) {
            const uint32_t i = i0 + lane;
            bool move = false;
            uint2 s = make_uint2(0, 0), d = s;
            if (fits && i < (uint32_t)n) {
                const int32_t *at_i = path + (size_t)item * B2_MAX_TREE + i, p = *at_i, before = i > 0 ? at_i[-1] : -1;
                if (p < (int32_t)i || p <= before || p >= B2_MAX_TREE || (uint32_t)c + (uint32_t)p >= cap) {
                    fault = B2_ERR_POSITION;
                } else if (p > (int32_t)i) {
                    const uint32_t at = (uint32_t)c + (uint32_t)p, to = (uint32_t)c + i;
                    const int32_t ps = row[at / kv.page_tokens], pd = row[to / kv.page_tokens];
                    move = ps >= 0 && pd >= 0 && (pool_pages == 0 || ((uint32_t)ps < pool_pages && (uint32_t)pd < pool_pages));
                    if (!move) fault = B2_ERR_POSITION;
                    s = make_uint2((uint32_t)ps, at % kv.page_tokens);
                    d = make_uint2((uint32_t)pd, to % kv.page_tokens);
                }
            }
            const uint32_t who = __ballot_sync(0xffffffffu, move);
            if (move) {
                const uint32_t at = kept + __popc(who & ((1u << lane) - 1));
                src[at] = s;
                dst[at] = d;
            }
            kept += __popc(who);
        }
        if (lane == 0) moves = kept;
        if (fault) raise_error(err, fault);
    }
    __syncthreads();
    const uint32_t n = moves;
    for (uint32_t w = blockIdx.y * kCompactThreads + threadIdx.x; w < work; w += gridDim.y * kCompactThreads) {
        const uint32_t col = w % cols, hh = w / cols, head = hh % kv.n_kv_heads;
        float4 *pool = reinterpret_cast<float4 *>(L.pool[layer][hh / kv.n_kv_heads]) + col;
        for (uint32_t i0 = 0; i0 < n; i0 += kCompactBatch) {
            float4 x[kCompactBatch];
#pragma unroll
            for (uint32_t j = 0; j < kCompactBatch; ++j) {
                if (i0 + j < n) {
                    const uint2 s = src[i0 + j];
                    x[j] = pool[(((size_t)s.x * kv.n_kv_heads + head) * kv.page_tokens + s.y) * cols];
                }
            }
#pragma unroll
            for (uint32_t j = 0; j < kCompactBatch; ++j) {
                if (i0 + j < n) {
                    const uint2 d = dst[i0 + j];
                    pool[(((size_t)d.x * kv.n_kv_heads + head) * kv.page_tokens + d.y) * cols] = x[j];
                }
            }
        }
    }
}

static bool tree_geometry_ok(const b2_kv_layout &kv)
{
    return kv.k_pool != nullptr && kv.v_pool != nullptr && kv.page_tokens != 0 && kv.n_kv_heads != 0 &&
           kv.head_dim != 0 && kv.head_dim % 4 == 0 && kv.head_dim <= 1024 && !((uintptr_t)kv.k_pool & 15) &&
           !((uintptr_t)kv.v_pool & 15);
}

}  // namespace b2

using namespace b2;

extern "C" int b2_kv_plan(const b2_kv_plan_args *a, void *stream)
{
    if (a == nullptr || a->batch == 0 || a->max_rows == 0 || a->max_rows > 0x7FFFFFFFu || a->page_tokens == 0 ||
        a->pages_per_seq == 0 || a->pool_pages == 0)
        return -1;
    if (!a->ctx_len || !a->new_len || !a->mapped || !a->free_pages || !a->free_count || !a->page_table ||
        !a->mapped_out || !a->free_out || !a->row_start || !a->row_item || !a->row_pos || !a->row_slot)
        return -1;
    // the CTAs read the inputs at their own pace, so no output may replace one
    if (a->mapped_out == a->mapped || a->free_out == a->free_count) return -1;
    if ((uint64_t)a->pages_per_seq * a->page_tokens > 0x7FFFFFFFull ||
        (uint64_t)a->pool_pages * a->page_tokens > 0x7FFFFFFFull)
        return -1;  // positions and slots are int32
    if (a->batch > B2_MAX_PLAN_BATCH) return -9;
    const size_t smem = (size_t)a->batch * 4 * sizeof(uint32_t);
    // (the default limit is 48 KB with the kernel's static shared memory, well below 16 KB)
    if (smem > 32 * 1024 && cudaFuncSetAttribute(kv_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                 (int)(B2_MAX_PLAN_BATCH * 4 * sizeof(uint32_t))) != cudaSuccess)
        return -8;
    uint32_t blocks = (a->max_rows + kPlanRowsPerCta - 1) / kPlanRowsPerCta;
    const uint32_t cap = (uint32_t)sm_count();
    if (blocks > cap) blocks = cap;
    b2_kv_plan_args p = *a;
    void *args[] = {&p};
    return launch_tree((const void *)kv_plan_kernel, dim3(blocks), dim3(kPlanThreads), smem, a->pdl,
                       (cudaStream_t)stream, args) == cudaSuccess
               ? 0
               : -8;
}

extern "C" int b2_rows_append(const b2_rows_append_args *a, void *stream)
{
    if (a == nullptr || a->m == 0 || a->m > 0x7FFFFFFFu || a->y == nullptr || a->q == nullptr || a->slots == nullptr ||
        a->pool_pages == 0 || !tree_geometry_ok(a->kv))
        return -1;
    const b2_kv_layout &kv = a->kv;
    if (a->rope_freq != nullptr && a->positions == nullptr) return -1;
    if (a->q_rows == 0 || a->q_rows % kv.head_dim || a->q_stride < a->q_rows || (a->q_stride & 3) || (a->y_stride & 3) ||
        a->y_stride < (uint64_t)a->q_rows + 2ull * kv.n_kv_heads * kv.head_dim || ((uintptr_t)a->y & 15) ||
        ((uintptr_t)a->q & 15))
        return -1;
    if ((uint64_t)a->pool_pages * kv.page_tokens > 0x7FFFFFFFull) return -1;
    const uint32_t heads = a->q_rows / kv.head_dim + 2 * kv.n_kv_heads;
    const uint32_t threads = kv.head_dim / 4 > kAppendThreads ? 2 * kAppendThreads : kAppendThreads;
    const uint32_t hgroups = threads / (kv.head_dim / 4);
    // few rows: a row's heads over several CTAs, at least one pass of the head groups each
    uint32_t parts = ((uint32_t)sm_count() + a->m - 1) / a->m;
    const uint32_t most = (heads + hgroups - 1) / hgroups;
    if (parts > most) parts = most;
    uint32_t per = (heads + parts - 1) / parts;
    per = (per + hgroups - 1) / hgroups * hgroups;
    parts = (heads + per - 1) / per;
    b2_rows_append_args p = *a;
    void *args[] = {&p, &per};
    return launch_tree((const void *)rows_append_kernel, dim3(parts, a->m < 65535u ? a->m : 65535u),
                       dim3(threads), 0, a->pdl, (cudaStream_t)stream, args) == cudaSuccess
               ? 0
               : -8;
}

extern "C" int b2_tree_accept(const b2_tree_accept_args *a, void *stream)
{
    if (a == nullptr || a->batch == 0 || a->batch > 0x7FFFFFFFu || a->max_rows == 0 || a->max_rows > B2_MAX_TREE ||
        a->rows > 0x7FFFFFFFu)
        return -1;
    if (!a->row_start || !a->tokens || !a->argmax || !a->ctx_len || !a->path || !a->count || !a->next || !a->ctx_out)
        return -1;
    b2_tree_accept_args p = *a;
    void *args[] = {&p};
    return launch_tree((const void *)tree_accept_kernel, dim3((a->batch + kAcceptWarps - 1) / kAcceptWarps),
                       dim3(kAcceptWarps * 32), 0, a->pdl, (cudaStream_t)stream, args) == cudaSuccess
               ? 0
               : -8;
}

extern "C" int b2_kv_compact(const b2_kv_compact_args *a, void *stream)
{
    if (a == nullptr || a->n_layers == 0 || a->layers == nullptr || a->batch == 0 || a->batch > 65535u ||
        !a->ctx_len || !a->path || !a->count)
        return -1;
    b2_kv_layout kv = a->layers[0];
    for (uint32_t l = 0; l < a->n_layers; ++l) {
        const b2_kv_layout &k = a->layers[l];
        if (!tree_geometry_ok(k) || k.page_table == nullptr || k.pages_per_seq == 0 || k.page_tokens != kv.page_tokens ||
            k.pages_per_seq != kv.pages_per_seq || k.n_kv_heads != kv.n_kv_heads || k.head_dim != kv.head_dim)
            return -1;
    }
    if ((uint64_t)kv.pages_per_seq * kv.page_tokens > 0x7FFFFFFFull) return -1;
    const uint32_t work = 2 * kv.n_kv_heads * (kv.head_dim / 4);
    uint32_t pool_pages = a->pool_pages;
    const int32_t *ctx_len = a->ctx_len, *path = a->path, *count = a->count;
    int32_t *err = a->err;
    for (uint32_t l0 = 0; l0 < a->n_layers; l0 += kCompactLayers) {
        const uint32_t n = a->n_layers - l0 < kCompactLayers ? a->n_layers - l0 : kCompactLayers;
        CompactLayers L = {};
        for (uint32_t l = 0; l < n; ++l) {
            L.pool[l][0] = a->layers[l0 + l].k_pool;
            L.pool[l][1] = a->layers[l0 + l].v_pool;
            L.table[l] = a->layers[l0 + l].page_table;
        }
        void *args[] = {&L, &kv, &pool_pages, &ctx_len, &path, &count, &err};
        if (launch_tree((const void *)kv_compact_kernel,
                        dim3(n, (work + kCompactThreads - 1) / kCompactThreads, a->batch), dim3(kCompactThreads), 0,
                        a->pdl, (cudaStream_t)stream, args) != cudaSuccess)
            return -8;
    }
    return 0;
}
