// b2_attn_rows.cu - attention of several new rows per sequence (the nodes of a
// drafted tree, or a prompt chunk) over the paged KV cache.
//
//   out[n] = sum_j p_j v_j,  p = softmax over the visible places j of q_n k_j / sqrt(hd)
//
// visible: the ctx_len cached places, and the item's own rows its ancestor mask
// (or the causal chain) names.
//
// One warp per (row, query head), four dimensions per lane: the score of a
// place is a warp sum, and the warp keeps the running maximum and sum of the
// softmax and rescales its weighted value sum when the maximum grows.
#include "b2_common.cuh"

namespace b2 {

constexpr int kRowWarps = 8;

__global__ void __launch_bounds__(kRowWarps * 32) attn_rows_kernel(const b2_attn_rows_args a, float scale)
{
    pdl_wait();
    pdl_launch_dependents();
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint32_t item = blockIdx.z, head = blockIdx.y, i = blockIdx.x * kRowWarps + warp;
    const int32_t r0 = a.row_start[item], r1 = a.row_start[item + 1], ctx = a.ctx_len[item];
    if (r0 < 0 || r1 < r0 || (uint32_t)r1 > a.rows || (uint32_t)(r1 - r0) > a.max_rows || ctx < 0 ||
        (uint32_t)ctx + (uint32_t)(r1 - r0) > a.max_ctx || (a.tree != nullptr && r1 - r0 > B2_MAX_TREE)) {
        if (threadIdx.x == 0 && head == 0 && blockIdx.x == 0) raise_error(a.err, B2_ERR_POSITION);
        return;
    }
    if (i >= (uint32_t)(r1 - r0)) return;
    const uint32_t hd = a.head_dim, n = (uint32_t)(r1 - r0), kvh = head / (a.n_heads / a.n_kv_heads);
    const bool mine = 4 * lane < hd;
    const uint64_t mask = a.tree != nullptr ? a.tree[r0 + i] : 0;
    const size_t qo = (size_t)(r0 + i) * a.q_stride + head * hd;
    float4 q = make_float4(0, 0, 0, 0), o = q;
    if (mine) q = reinterpret_cast<const float4 *>(a.q + qo)[lane];
    float m = -INFINITY, l = 0.0f;
    const uint32_t end = (uint32_t)ctx + (a.tree != nullptr ? n : i + 1);
    int fault = 0;
    for (uint32_t at = 0; at < end; ++at) {
        if (a.tree != nullptr && at >= (uint32_t)ctx && !((mask >> (at - (uint32_t)ctx)) & 1)) continue;
        const int32_t page = a.kv.page_table[(size_t)item * a.kv.pages_per_seq + at / a.kv.page_tokens];
        if (page < 0 || (a.pool_pages != 0 && (uint32_t)page >= a.pool_pages)) {
            fault |= B2_ERR_POSITION;
            continue;
        }
        const size_t row = (((size_t)page * a.n_kv_heads + kvh) * a.kv.page_tokens + at % a.kv.page_tokens) * hd;
        float4 k = make_float4(0, 0, 0, 0), v = k;
        if (mine) {
            k = reinterpret_cast<const float4 *>(a.kv.k_pool + row)[lane];
            v = reinterpret_cast<const float4 *>(a.kv.v_pool + row)[lane];
        }
        bool fine = isfinite(k.x) && isfinite(k.y) && isfinite(k.z) && isfinite(k.w) && isfinite(v.x) &&
                    isfinite(v.y) && isfinite(v.z) && isfinite(v.w);
        fine = __all_sync(0xffffffffu, fine);
        float s = warp_sum(q.x * k.x + q.y * k.y + q.z * k.z + q.w * k.w) * scale;
        if (!fine) s = NAN;
        const float nm = fmaxf(m, s);
        const float f = m == -INFINITY ? 0.0f : expf(m - nm), p = expf(s - nm);
        l = l * f + p;
        o = make_float4(o.x * f + p * v.x, o.y * f + p * v.y, o.z * f + p * v.z, o.w * f + p * v.w);
        m = nm;
    }
    if (l != l) {
        fault |= B2_ERR_NONFINITE;
        o = make_float4(NAN, NAN, NAN, NAN);
        l = 1.0f;
    }
    const float inv = l > 0.0f ? 1.0f / l : 0.0f;
    if (mine)
        reinterpret_cast<float4 *>(a.ctx + (size_t)(r0 + i) * a.ctx_stride + head * hd)[lane] =
            make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
    if (fault && lane == 0) raise_error(a.err, fault);
}

static int attn_rows_check(const b2_attn_rows_args *a)
{
    if (a == nullptr || a->q == nullptr || a->ctx == nullptr || a->row_start == nullptr || a->ctx_len == nullptr)
        return -1;
    if (a->batch == 0 || a->batch > 65535u || a->n_kv_heads == 0 || a->n_heads == 0 || a->n_heads % a->n_kv_heads ||
        a->head_dim == 0 || a->head_dim % 16 || a->head_dim > 128 || a->max_rows == 0 || a->max_rows > 0x7FFFFFFFu ||
        a->rows == 0 || a->rows > 0x7FFFFFFFu || a->max_ctx == 0)
        return -1;
    const uint64_t row = (uint64_t)a->n_heads * a->head_dim;
    if (a->q_stride < row || a->ctx_stride < row || (a->q_stride & 3) || (a->ctx_stride & 3) || ((uintptr_t)a->q & 15) ||
        ((uintptr_t)a->ctx & 15))
        return -1;
    const b2_kv_layout &kv = a->kv;
    if (!kv.k_pool || !kv.v_pool || !kv.page_table || kv.page_tokens == 0 || kv.head_dim != a->head_dim ||
        kv.n_kv_heads != a->n_kv_heads || ((uintptr_t)kv.k_pool & 15) || ((uintptr_t)kv.v_pool & 15))
        return -1;
    if ((uint64_t)kv.page_tokens * kv.pages_per_seq > 0x7FFFFFFFull || a->max_ctx > kv.page_tokens * kv.pages_per_seq)
        return -1;
    return 0;
}

}  // namespace b2

using namespace b2;

extern "C" size_t b2_attn_rows_scratch_bytes(const b2_attn_rows_args *) { return 0; }

extern "C" int b2_attn_rows(const b2_attn_rows_args *a, void *stream)
{
    const int rc = attn_rows_check(a);
    if (rc != 0) return rc;
    if (a->n_heads > 65535u) return -9;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((a->max_rows + kRowWarps - 1) / kRowWarps, a->n_heads, a->batch);
    cfg.blockDim = dim3(kRowWarps * 32);
    cfg.stream = (cudaStream_t)stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = a->pdl ? 1 : 0;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, attn_rows_kernel, *a, 1.0f / sqrtf((float)a->head_dim)) == cudaSuccess ? 0 : -8;
}
