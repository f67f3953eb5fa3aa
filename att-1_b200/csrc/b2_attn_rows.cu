// b2_attn_rows.cu - attention of several new rows per sequence (the nodes of a
// drafted tree, or a prompt chunk) over the paged KV cache.
//
//   out[n] = sum_j p_j v_j,  p = softmax over the visible places j of q_n k_j / sqrt(hd)
//
// visible: the ctx_len cached places, and the item's own rows that its ancestor
// mask (or the causal chain) names.
//
// Work split. The rows of an item times the query heads of one KV head are the
// rows r = token * group + head of a matrix; CTA (split, KV head and block of
// 128 such rows, item) takes a contiguous range of the places in tiles of 64, so
// K and V are read once per 128 rows. 13 warps (at most four per scheduler: 128
// registers a thread):
//   warps 8..11   load K and V (f32) straight into registers, eight keys ahead of
//                 the eight being converted, and store them as matrix operands;
//                 the tiles to come are asked into L2, so that a register load's
//                 round trip is L2's and not HBM's;
//   warp 12       one thread issues the tcgen05 MMAs: S = Q K^T of tile j + 1
//                 before O = P V of tile j, accumulators in tensor memory, two
//                 buffers each;
//   warps 0..7    two per 32 rows: a thread holds one row and 32 of a tile's 64
//                 keys: scores from tensor memory, the row's running maximum
//                 (joined with the other half's through shared memory), P as
//                 matrix operand; then one row and half of the dimensions of O,
//                 summed in registers over the tiles, so a growing maximum
//                 rescales registers, not tensor memory.
// Splits write (maximum, sum, weighted values) per row; a second kernel joins
// them in split order. No counters or atomics: results do not depend on timing.
//
// Precision. Every f32 operand x becomes two f16 numbers of x 2^e (the scale
// exact): hi = f16(x 2^e), lo = f16(x 2^e - hi), and a product is
// hi hi + lo hi + hi lo with f32 accumulation; what is dropped is below 2^-22.
// f16 rather than bf16 pairs (2^-16) because the scale takes care of the range:
// a row of q, eight keys' K and eight keys' V have a power of two each that
// brings their largest magnitude to [2^8, 2^9), so an element 2^-17 of the
// largest still keeps 16 bits. K's scale goes into the scores, V's into P
// relative to the tile's largest, and the tile's into its O when it is summed.
// The softmax statistics and the weighted sums are f32.
//
// Operands are K-major without swizzle as in b2_gemm.cu: 8-row x 16-byte core
// matrices, row groups 128 bytes apart, 8-column chunks R * 16 bytes apart. K's
// hi and lo rows are one operand of 128 rows (one MMA of N = 128 gives
// q_hi k_hi and q_hi k_lo, a second of N = 64 adds q_lo k_hi); V is transposed
// on the way from registers to shared memory (a lane holds eight keys of a
// dimension: one 16-byte store).
#include "b2_common.cuh"
#include "b2_umma.cuh"

#include <cuda_fp16.h>

namespace b2 {

constexpr uint32_t kRowsM = 128;        // (token, query head) rows of a CTA
constexpr uint32_t kRowsKeys = 64;      // places of a tile
constexpr int kRowsSoftWarps = 8;
constexpr int kRowsConvWarps = 4;
constexpr int kRowsThreads = 32 * (kRowsSoftWarps + kRowsConvWarps + 1);
constexpr uint32_t kRowsMeta = 8;       // ring of per-tile K scales: more than the tiles between converting and softmax
constexpr uint32_t kRowsAhead = 3;      // tiles ahead of the conversion whose K and V are asked into L2
constexpr uint32_t kRowsMaxSplits = 64;
constexpr int kRowsTop = 8;             // operands are scaled to [2^kRowsTop, 2^(kRowsTop + 1))
constexpr float kRowsP = 12.0f;         // P is scaled by 2^12

template <int HD>
struct RowsSmem {
    static constexpr uint32_t stages = HD == 128 ? 2 : 4;
    static constexpr uint32_t q_half = kRowsM * HD * 2;            // hi or lo
    static constexpr uint32_t k_stage = 2 * kRowsKeys * HD * 2;    // hi and lo rows of one operand
    static constexpr uint32_t v_half = kRowsKeys * HD * 2;
    static constexpr uint32_t p_half = kRowsM * kRowsKeys * 2;
    static constexpr uint32_t off_q = 0;
    static constexpr uint32_t off_k = off_q + 2 * q_half;
    static constexpr uint32_t off_v = off_k + stages * k_stage;
    static constexpr uint32_t off_p = off_v + stages * 2 * v_half;
    static constexpr uint32_t off_x = off_p + 2 * p_half;          // [2][2][128] f32: the halves' maxima
    static constexpr uint32_t off_ks = off_x + 2 * 2 * kRowsM * 4;  // [kRowsMeta][8] f32: 1 / K scale of eight keys
    static constexpr uint32_t off_km = off_ks + kRowsMeta * 8 * 4;  // [kRowsMeta][8] u32: keys that are NaN | hidden << 8
    static constexpr uint32_t off_ve = off_km + kRowsMeta * 8 * 4;  // [4][8] int: exponent of eight keys' V
    static constexpr uint32_t off_vm = off_ve + 4 * 8 * 4;          // [4][8] u32: keys whose V is NaN
    static constexpr uint32_t off_bar = off_vm + 4 * 8 * 4;
    static constexpr uint32_t bytes = off_bar + 8 * (4 * stages + 4 + 1 + 4 + 2 + 4) + 16;
};
static_assert(RowsSmem<128>::bytes <= 227 * 1024 && RowsSmem<64>::bytes <= 227 * 1024, "shared memory");

struct RowsParams {
    b2_attn_rows_args a;
    uint32_t group, blocks;   // query heads per KV head, 128-row blocks per (item, KV head)
    uint32_t splits;
    float scale;              // log2(e) / sqrt(head_dim)
    float *part;              // splits > 1: [item][KV head][block][split][128][head_dim + 2]
};

// The rows of an item, or false for lengths that do not fit.
__device__ __forceinline__ bool rows_item(const b2_attn_rows_args &a, uint32_t item, uint32_t &r0, uint32_t &n, uint32_t &ctx)
{
    const int32_t s = a.row_start[item], e = a.row_start[item + 1], c = a.ctx_len[item];
    if (s < 0 || e < s || (uint32_t)e > a.rows || (uint32_t)(e - s) > a.max_rows || c < 0 || (uint32_t)c > a.max_ctx ||
        (uint32_t)(e - s) > a.max_ctx - (uint32_t)c || (a.tree != nullptr && e - s > B2_MAX_TREE))
        return false;
    r0 = (uint32_t)s;
    n = (uint32_t)(e - s);
    ctx = (uint32_t)c;
    return true;
}

// Places a block of rows can see, and the tiles [t0, t1) of split s.
__device__ __forceinline__ uint32_t rows_places(const RowsParams &p, uint32_t n, uint32_t ctx, uint32_t blk)
{
    if (p.a.tree != nullptr) return ctx + n;
    return ctx + min(n, (blk * kRowsM + kRowsM - 1) / p.group + 1);
}
__device__ __forceinline__ void rows_range(uint32_t places, uint32_t splits, uint32_t s, uint32_t &t0, uint32_t &t1)
{
    const uint32_t nt = (places + kRowsKeys - 1) / kRowsKeys;
    t0 = (uint32_t)((uint64_t)s * nt / splits);
    t1 = (uint32_t)((uint64_t)(s + 1) * nt / splits);
}

__device__ __forceinline__ float ex2(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ float pow2i(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }  // -126..127

// Unbiased exponent of the largest magnitude (its bits), floored so that the
// scale 2^(kRowsTop - e) and its inverse stay normal.
__device__ __forceinline__ int top_exp(uint32_t amax_bits) { return max((int)(amax_bits >> 23) - 127, -100); }

// f16 hi and lo words of two values.
__device__ __forceinline__ void split_f16(float a, float b, uint32_t &hi, uint32_t &lo)
{
    const __half2 h = __floats2half2_rn(a, b);
    const float2 f = __half22float2(h);
    const __half2 l = __floats2half2_rn(a - f.x, b - f.y);
    hi = *reinterpret_cast<const uint32_t *>(&h);
    lo = *reinterpret_cast<const uint32_t *>(&l);
}

__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7FFFFFFFu; }

__device__ __forceinline__ void tmem_ld16_nowait(uint32_t taddr, uint32_t (&r)[16])
{
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

// All lanes wait; false for the whole warp if any gave up.
__device__ __forceinline__ bool warp_wait(uint64_t *bar, uint32_t phase, int32_t *err)
{
    return __all_sync(0xffffffffu, mbar_wait_bounded(bar, phase & 1u, err));
}

template <int HD>
__global__ void __launch_bounds__(kRowsThreads, 1) attn_rows_kernel(const RowsParams p)
{
    using S = RowsSmem<HD>;
    constexpr uint32_t NST = S::stages;
    extern __shared__ __align__(1024) uint8_t smem[];
    const b2_attn_rows_args &a = p.a;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t split = blockIdx.x, kvh = blockIdx.y / p.blocks, blk = blockIdx.y % p.blocks, item = blockIdx.z;
    const uint32_t hd = a.head_dim;
    float *xmax = reinterpret_cast<float *>(smem + S::off_x);
    float *kscale = reinterpret_cast<float *>(smem + S::off_ks);
    uint32_t *kmark = reinterpret_cast<uint32_t *>(smem + S::off_km);
    int *vexp = reinterpret_cast<int *>(smem + S::off_ve);
    uint32_t *vmark = reinterpret_cast<uint32_t *>(smem + S::off_vm);
    uint64_t *k_full = reinterpret_cast<uint64_t *>(smem + S::off_bar), *k_empty = k_full + NST, *v_full = k_empty + NST,
             *v_empty = v_full + NST, *s_full = v_empty + NST, *s_empty = s_full + 2, *p_full = s_empty + 2,
             *o_full = p_full + 1, *o_empty = o_full + 2, *q_full = o_empty + 2, *done = q_full + 1, *xbar = done + 1;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(xbar + 4);

    pdl_wait();
    pdl_launch_dependents();
    uint32_t r0, n, ctx;
    if (!rows_item(a, item, r0, n, ctx)) {
        if (threadIdx.x == 0 && split == 0 && blockIdx.y == 0) raise_error(a.err, B2_ERR_POSITION);
        return;
    }
    const uint32_t mrows = n * p.group;  // rows of this (item, KV head)
    if (blk * kRowsM >= mrows) return;
    const uint32_t live = min(kRowsM, mrows - blk * kRowsM);
    const uint32_t places = rows_places(p, n, ctx, blk);
    uint32_t t0, t1;
    rows_range(places, p.splits, split, t0, t1);
    if (t0 == t1) return;  // the joining kernel skips the same splits
    const uint32_t nt = t1 - t0;
    const uint32_t nsoft = 2 * ((live + 31) / 32);  // softmax warps with rows: two per quarter of the rows

    if (threadIdx.x == 0) {
        for (uint32_t i = 0; i < NST; ++i) {
            mbar_init(&k_full[i], kRowsConvWarps);
            mbar_init(&k_empty[i], 1);
            mbar_init(&v_full[i], kRowsConvWarps);
            mbar_init(&v_empty[i], 1);
        }
        for (uint32_t i = 0; i < 2; ++i) {
            mbar_init(&s_full[i], 1);
            mbar_init(&s_empty[i], nsoft);
            mbar_init(&o_full[i], 1);
            mbar_init(&o_empty[i], nsoft);
        }
        mbar_init(p_full, nsoft);
        mbar_init(q_full, nsoft);
        mbar_init(done, 1);
        for (uint32_t i = 0; i < 4; ++i) mbar_init(&xbar[i], 2);
        fence_mbar_init();
    }
    if (warp == kRowsSoftWarps + kRowsConvWarps) tmem_alloc(tmem_slot, 512);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;  // S: columns 0..255 (two buffers of hi | lo keys), O: 256 + buffer * HD

    if (warp >= (uint32_t)kRowsSoftWarps && warp < (uint32_t)(kRowsSoftWarps + kRowsConvWarps)) {
        // ---- K and V into operands: keys 16 cw .. 16 cw + 15 of every tile, eight at a time ----
        const uint32_t cw = warp - kRowsSoftWarps, key = lane & 7, ch = lane >> 3;
        const int32_t *table = a.kv.page_table + (size_t)item * a.kv.pages_per_seq;
        const uint32_t pt = a.kv.page_tokens;
        int fault = 0;
        constexpr uint32_t kNoRow = 0xFFFFFFFFu;
        // lane l: the page of the warp's key l % 16 in tile t, and its row in the pools
        auto page_of = [&](uint32_t t) -> int32_t {
            const uint32_t at = t * kRowsKeys + 16 * cw + (lane & 15);
            return t < t1 && at < places ? table[at / pt] : 0;
        };
        auto row_of = [&](uint32_t t, int32_t page, bool &hidden) -> uint32_t {
            const uint32_t at = t * kRowsKeys + 16 * cw + (lane & 15);
            hidden = false;
            if (t >= t1 || at >= places) return kNoRow;
            if (page < 0 || (a.pool_pages != 0 && (uint32_t)page >= a.pool_pages)) {
                fault = B2_ERR_POSITION;
                hidden = true;
                return kNoRow;
            }
            return ((uint32_t)page * a.n_kv_heads + kvh) * pt + at % pt;
        };
        // lanes 0..15 ask for their key's K row, 16..31 for its V row
        auto ask = [&](uint32_t row) {
            if (row == kNoRow) return;
            const float *src = (lane < 16 ? a.kv.k_pool : a.kv.v_pool) + (size_t)row * hd;
            for (uint32_t d = 0; d < hd; d += 32) asm volatile("prefetch.global.L2 [%0];" ::"l"(src + d));
        };
        constexpr int U = HD / 4;  // values a lane holds of eight keys
        // K: eight dimensions each of chunks ch, ch + 4, .. of key `key`
        auto load_k = [&](float (&x)[U], uint32_t rows, uint32_t g) {
            const uint32_t row = __shfl_sync(0xffffffffu, rows, 8 * g + key);
            const float *src = a.kv.k_pool + (size_t)row * hd + 8 * ch;
#pragma unroll
            for (int i = 0; i < HD / 32; ++i) {
                float4 u = make_float4(0, 0, 0, 0), v = u;
                if (row != kNoRow && 32 * i + 8 * ch < hd) {
                    u = *reinterpret_cast<const float4 *>(src + 32 * i);
                    v = *reinterpret_cast<const float4 *>(src + 32 * i + 4);
                }
                x[8 * i] = u.x, x[8 * i + 1] = u.y, x[8 * i + 2] = u.z, x[8 * i + 3] = u.w;
                x[8 * i + 4] = v.x, x[8 * i + 5] = v.y, x[8 * i + 6] = v.z, x[8 * i + 7] = v.w;
            }
        };
        // V: dimensions lane + 32 i of the eight keys
        auto load_v = [&](float (&x)[U], uint32_t rows, uint32_t g) {
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const uint32_t row = __shfl_sync(0xffffffffu, rows, 8 * g + k);
                const float *src = a.kv.v_pool + (size_t)row * hd + lane;
#pragma unroll
                for (int i = 0; i < HD / 32; ++i) x[8 * i + k] = row != kNoRow && lane + 32 * i < hd ? src[32 * i] : 0.0f;
            }
        };
        // largest magnitude of the eight keys (bits)
        auto largest = [&](const float (&x)[U]) -> uint32_t {
            uint32_t top = 0;
#pragma unroll
            for (int i = 0; i < U; ++i) top = max(top, abs_bits(x[i]));
            return __reduce_max_sync(0xffffffffu, top);
        };
        // a NaN or infinity (rare): zero it; bit i of the result: this lane had one among x[8 i' + i]
        auto drop_bad = [&](float (&x)[U]) -> uint32_t {
            uint32_t bad = 0;
#pragma unroll
            for (int i = 0; i < U; ++i) {
                if (abs_bits(x[i]) >= 0x7F800000u) {
                    bad |= 1u << (i & 7);
                    x[i] = 0.0f;
                }
            }
            return bad;
        };
        // eight values in a row (K: dimensions of a key, V: keys of a dimension) are one 16-byte chunk
        auto store = [&](const float (&x)[U], float sc, uint8_t *dst, uint32_t step, uint32_t lo_off, uint32_t first, uint32_t per) {
#pragma unroll
            for (int i = 0; i < HD / 32; ++i) {
                if (first + per * i < hd) {
                    uint4 h, l;
                    split_f16(x[8 * i] * sc, x[8 * i + 1] * sc, h.x, l.x);
                    split_f16(x[8 * i + 2] * sc, x[8 * i + 3] * sc, h.y, l.y);
                    split_f16(x[8 * i + 4] * sc, x[8 * i + 5] * sc, h.z, l.z);
                    split_f16(x[8 * i + 6] * sc, x[8 * i + 7] * sc, h.w, l.w);
                    *reinterpret_cast<uint4 *>(dst + i * step) = h;
                    *reinterpret_cast<uint4 *>(dst + i * step + lo_off) = l;
                }
            }
        };
        auto convert_k = [&](float (&x)[U], uint32_t j, uint32_t g, uint32_t hide) {
            const uint32_t w = 2 * cw + g;
            uint32_t top = largest(x), mark = (hide >> (8 * g) & 0xFFu) << 8;
            if (top >= 0x7F800000u) {
                const uint32_t who = __ballot_sync(0xffffffffu, drop_bad(x) != 0);
                mark |= (who | who >> 8 | who >> 16 | who >> 24) & 0xFFu;
                top = largest(x);
            }
            const int e = top_exp(top);
            // element (key, d): chunk d / 8 of 128 rows (hi rows 0..63, lo rows 64..127)
            store(x, pow2i(kRowsTop - e), smem + S::off_k + (j % NST) * S::k_stage + ch * (2 * kRowsKeys * 16) + w * 128 + key * 16,
                  4 * (2 * kRowsKeys * 16), kRowsKeys * 16, 8 * ch, 32);
            if (lane == 0) {
                kscale[(j % kRowsMeta) * 8 + w] = pow2i(e - kRowsTop);
                kmark[(j % kRowsMeta) * 8 + w] = mark;
            }
        };
        auto convert_v = [&](float (&x)[U], uint32_t j, uint32_t g) {
            const uint32_t w = 2 * cw + g;
            uint32_t top = largest(x), mark = 0;
            if (top >= 0x7F800000u) {
                mark = __reduce_or_sync(0xffffffffu, drop_bad(x));
                top = largest(x);
            }
            const int e = top_exp(top);
            // element (d, key): chunk key / 8 of HD rows
            store(x, pow2i(kRowsTop - e), smem + S::off_v + (j % NST) * 2 * S::v_half + w * (HD * 16) + lane * 16, 512, S::v_half, lane, 32);
            if (lane == 0) {
                vexp[(j % NST) * 8 + w] = e;
                vmark[(j % NST) * 8 + w] = mark;
            }
        };
        auto publish = [&](uint64_t *bar) {
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar);
        };
        bool hidden, unused;
        uint32_t rows = row_of(t0, page_of(t0), hidden);
        ask(rows);
        float xa[U], xb[U];
        load_k(xa, rows, 0);
        for (uint32_t i = 1; i < kRowsAhead; ++i) ask(row_of(t0 + i, page_of(t0 + i), unused));
        int32_t page = page_of(t0 + 1), far = page_of(t0 + kRowsAhead);
        for (uint32_t j = 0; j < nt; ++j) {
            const uint32_t st = j % NST, pass = j / NST, hide = __ballot_sync(0xffffffffu, hidden);
            load_k(xb, rows, 1);
            ask(row_of(t0 + j + kRowsAhead, far, unused));
            far = page_of(t0 + j + 1 + kRowsAhead);
            if (j >= NST && !warp_wait(&k_empty[st], pass - 1, a.err)) break;
            convert_k(xa, j, 0, hide);
            load_v(xa, rows, 0);
            convert_k(xb, j, 1, hide);
            publish(&k_full[st]);
            load_v(xb, rows, 1);
            if (j >= NST && !warp_wait(&v_empty[st], pass - 1, a.err)) break;
            convert_v(xa, j, 0);
            if (j + 1 < nt) {  // K of the next tile on its way while V is converted
                rows = row_of(t0 + j + 1, page, hidden);
                page = page_of(t0 + j + 2);
                load_k(xa, rows, 0);
            }
            convert_v(xb, j, 1);
            publish(&v_full[st]);
        }
        if (fault) raise_error(a.err, fault);
    } else if (warp == kRowsSoftWarps + kRowsConvWarps) {
        // ---- MMA issue ----
        if (lane == 0) {
            const uint32_t id_s2 = umma_idesc_f16(kRowsM, 2 * kRowsKeys), id_s1 = umma_idesc_f16(kRowsM, kRowsKeys);
            const uint32_t id_o = umma_idesc_f16(kRowsM, hd);
            const uint32_t qb = smem_u32(smem + S::off_q), kb = smem_u32(smem + S::off_k), vb = smem_u32(smem + S::off_v),
                           pb = smem_u32(smem + S::off_p);
            bool ok = mbar_wait_bounded(q_full, 0, a.err);
            for (uint32_t j = 0; ok && j <= nt; ++j) {
                if (j < nt) {  // S of tile j
                    const uint32_t st = j % NST, sb = j & 1;
                    ok = mbar_wait_bounded(&k_full[st], (j / NST) & 1, a.err) &&
                         (j < 2 || mbar_wait_bounded(&s_empty[sb], (j / 2 - 1) & 1, a.err));
                    if (!ok) break;
                    tc_fence_after();
                    const uint32_t d = tmem + sb * 2 * kRowsKeys, kt = kb + st * S::k_stage;
                    for (uint32_t kk = 0; kk < hd / 16; ++kk) {
                        const uint64_t b = umma_desc(kt + kk * 2 * (2 * kRowsKeys * 16), 2 * kRowsKeys * 16, 128);
                        umma_16(d, umma_desc(qb + kk * 2 * (kRowsM * 16), kRowsM * 16, 128), b, id_s2, kk > 0);
                        umma_16(d, umma_desc(qb + S::q_half + kk * 2 * (kRowsM * 16), kRowsM * 16, 128), b, id_s1, 1);
                    }
                    umma_commit(&s_full[sb]);
                    umma_commit(&k_empty[st]);
                }
                if (j > 0) {  // O of tile j - 1
                    const uint32_t i = j - 1, st = i % NST, ob = i & 1;
                    ok = mbar_wait_bounded(p_full, i & 1, a.err) && mbar_wait_bounded(&v_full[st], (i / NST) & 1, a.err) &&
                         (i < 2 || mbar_wait_bounded(&o_empty[ob], (i / 2 - 1) & 1, a.err));
                    if (!ok) break;
                    tc_fence_after();
                    const uint32_t d = tmem + 4 * kRowsKeys + ob * HD, vt = vb + st * 2 * S::v_half;
#pragma unroll
                    for (uint32_t kk = 0; kk < kRowsKeys / 16; ++kk) {
                        const uint64_t ph = umma_desc(pb + kk * 2 * (kRowsM * 16), kRowsM * 16, 128);
                        const uint64_t pl = umma_desc(pb + S::p_half + kk * 2 * (kRowsM * 16), kRowsM * 16, 128);
                        const uint64_t vh = umma_desc(vt + kk * 2 * (HD * 16), HD * 16, 128);
                        const uint64_t vl = umma_desc(vt + S::v_half + kk * 2 * (HD * 16), HD * 16, 128);
                        umma_16(d, ph, vh, id_o, kk > 0);
                        umma_16(d, pl, vh, id_o, 1);
                        umma_16(d, ph, vl, id_o, 1);
                    }
                    umma_commit(&o_full[ob]);
                    umma_commit(&v_empty[st]);
                }
            }
            // everything issued has completed before tensor memory is freed
            umma_commit(done);
            mbar_wait_bounded(done, 0, a.err);
        }
        __syncwarp();
    } else {
        const uint32_t qt = warp & 3, half = warp >> 2;
        if (qt < nsoft / 2) {
            // ---- softmax and the sums of O: row r, keys 32 half .. + 31, dimensions of half ----
            const uint32_t r = qt * 32 + lane, m_row = blk * kRowsM + r;
            const bool mine = r < live;
            const uint32_t tok = mine ? m_row / p.group : 0, head = kvh * p.group + (mine ? m_row % p.group : 0);
            const uint32_t lanes = (qt * 32) << 16;
            uint32_t xph = 0;  // exchanges done with the other half's warp
            auto exchange = [&](float mine_v, float &other) -> bool {
                float *x = xmax + (xph & 1) * 2 * kRowsM;
                x[half * kRowsM + r] = mine_v;
                __syncwarp();
                if (lane == 0) mbar_arrive(&xbar[qt]);
                const bool ok = warp_wait(&xbar[qt], xph, a.err);
                other = x[(half ^ 1) * kRowsM + r];
                ++xph;
                return ok;
            };
            float cq;  // score of a row: dot * K scale * cq, in powers of two
            bool ok;
            {
                const float *src = a.q + (size_t)(r0 + tok) * a.q_stride + (size_t)head * hd;
                float x[HD / 2];
                uint32_t top = 0;
#pragma unroll
                for (int c = 0; c < HD / 16; ++c) {
                    const uint32_t d = half * (HD / 2) + 8 * c;
                    float4 u = make_float4(0, 0, 0, 0), v = u;
                    if (mine && d < hd) {
                        u = *reinterpret_cast<const float4 *>(src + d);
                        v = *reinterpret_cast<const float4 *>(src + d + 4);
                    }
                    x[8 * c] = u.x, x[8 * c + 1] = u.y, x[8 * c + 2] = u.z, x[8 * c + 3] = u.w;
                    x[8 * c + 4] = v.x, x[8 * c + 5] = v.y, x[8 * c + 6] = v.z, x[8 * c + 7] = v.w;
                }
#pragma unroll
                for (int i = 0; i < HD / 2; ++i) top = max(top, abs_bits(x[i]));
                float other;
                ok = exchange(__uint_as_float(top), other);
                top = max(top, __float_as_uint(other));
                const bool bad = top >= 0x7F800000u;
                const int e = bad ? 0 : top_exp(top);
                const float sc = bad ? 0.0f : pow2i(kRowsTop - e);
                cq = bad ? NAN : pow2i(e - kRowsTop) * p.scale;
                uint8_t *dst = smem + S::off_q + r * 16;
#pragma unroll
                for (int c = 0; c < HD / 16; ++c) {
                    const uint32_t chunk = half * (HD / 16) + c;
                    uint4 h = make_uint4(0, 0, 0, 0), l = h;
                    if (!bad) {
                        split_f16(x[8 * c] * sc, x[8 * c + 1] * sc, h.x, l.x);
                        split_f16(x[8 * c + 2] * sc, x[8 * c + 3] * sc, h.y, l.y);
                        split_f16(x[8 * c + 4] * sc, x[8 * c + 5] * sc, h.z, l.z);
                        split_f16(x[8 * c + 6] * sc, x[8 * c + 7] * sc, h.w, l.w);
                    }
                    *reinterpret_cast<uint4 *>(dst + chunk * (kRowsM * 16)) = h;
                    *reinterpret_cast<uint4 *>(dst + chunk * (kRowsM * 16) + S::q_half) = l;
                }
                fence_proxy_async();
                __syncwarp();
                if (lane == 0) mbar_arrive(q_full);
            }
            const uint64_t mask = mine && a.tree != nullptr ? a.tree[r0 + tok] : 0;
            float m = -INFINITY, l = 0.0f, corr_prev = 0.0f, osc_prev = 0.0f;
            float acc[HD / 2];
#pragma unroll
            for (int i = 0; i < HD / 2; ++i) acc[i] = 0.0f;
            // O of tile i into the sums: acc = acc * corr + O * osc
            auto take_o = [&](uint32_t i) {
                const uint32_t col = tmem + lanes + 4 * kRowsKeys + (i & 1) * HD + half * (HD / 2);
                tc_fence_after();
#pragma unroll
                for (int c = 0; c < HD / 2; c += 16) {
                    uint32_t v[16];
                    tmem_ld16_nowait(col + c, v);
                    tmem_wait_ld();
#pragma unroll
                    for (int k = 0; k < 16; ++k) acc[c + k] = fmaf(__uint_as_float(v[k]), osc_prev, acc[c + k] * corr_prev);
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&o_empty[i & 1]);
            };
            uint32_t j = 0;
            for (; ok && j < nt; ++j) {
                const uint32_t sb = j & 1, mt = j % kRowsMeta, vt = j % NST;
                ok = warp_wait(&s_full[sb], j / 2, a.err) && warp_wait(&v_full[vt], j / NST, a.err);
                if (!ok) break;
                tc_fence_after();
                float s[32];
                const float4 ks = *reinterpret_cast<const float4 *>(kscale + mt * 8 + half * 4);
                const float ksc[4] = {ks.x, ks.y, ks.z, ks.w};
                const uint4 km = *reinterpret_cast<const uint4 *>(kmark + mt * 8 + half * 4);
                const uint4 vm = *reinterpret_cast<const uint4 *>(vmark + vt * 8 + half * 4);
                const int4 e0 = *reinterpret_cast<const int4 *>(vexp + vt * 8), e1 = *reinterpret_cast<const int4 *>(vexp + vt * 8 + 4);
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    uint32_t u[16], v[16];
                    const uint32_t col = tmem + lanes + sb * 2 * kRowsKeys + half * 32 + c * 16;
                    tmem_ld16_nowait(col, u);
                    tmem_ld16_nowait(col + kRowsKeys, v);
                    tmem_wait_ld();
#pragma unroll
                    for (int k = 0; k < 16; ++k)
                        s[c * 16 + k] = (__uint_as_float(u[k]) + __uint_as_float(v[k])) * ksc[(c * 16 + k) / 8];
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&s_empty[sb]);
                // keys this row does not see, and keys whose K or V is not finite
                const uint32_t key0 = (t0 + j) * kRowsKeys + half * 32;
                uint32_t vis = 0xFFFFFFFFu;
                if (key0 + 32 > ctx) {
                    if (a.tree != nullptr) {
                        if (key0 >= ctx) {
                            const uint32_t sh = key0 - ctx;
                            vis = sh < 64 ? (uint32_t)(mask >> sh) : 0;
                        } else {
                            const uint32_t sh = ctx - key0;  // 1..31
                            vis = (uint32_t)(mask << sh) | ((1u << sh) - 1);
                        }
                    } else {
                        const uint32_t seen = ctx + tok + 1;  // places 0 .. seen - 1
                        vis = seen >= key0 + 32 ? 0xFFFFFFFFu : seen <= key0 ? 0 : (1u << (seen - key0)) - 1;
                    }
                }
                if (key0 + 32 > places) vis &= places <= key0 ? 0 : (1u << (places - key0)) - 1;
                const uint32_t any = km.x | km.y | km.z | km.w | vm.x | vm.y | vm.z | vm.w;
                if (any != 0) {
                    const uint32_t bad = ((km.x | vm.x) & 0xFF) | ((km.y | vm.y) & 0xFF) << 8 | ((km.z | vm.z) & 0xFF) << 16 |
                                         ((km.w | vm.w) & 0xFF) << 24;
                    vis &= ~((km.x >> 8) | (km.y >> 8) << 8 | (km.z >> 8) << 16 | (km.w >> 8) << 24);
#pragma unroll
                    for (int k = 0; k < 32; ++k)
                        if (bad >> k & 1) s[k] = NAN;
                }
                if (vis != 0xFFFFFFFFu) {
#pragma unroll
                    for (int k = 0; k < 32; ++k)
                        if (!(vis >> k & 1)) s[k] = -INFINITY;
                }
                float top = s[0];
#pragma unroll
                for (int k = 1; k < 32; ++k) top = fmaxf(top, s[k]);
                float other;
                ok = exchange(top, other);
                if (!ok) break;
                const float m_new = fmaxf(m, fmaxf(top, other) * cq);
                const float m_use = m_new == -INFINITY ? 0.0f : m_new;
                const float corr = ex2(m - m_use), shift = kRowsP - m_use;
                const int emax = max(max(max(e0.x, e0.y), max(e0.z, e0.w)), max(max(e1.x, e1.y), max(e1.z, e1.w)));
                const int4 eh = half ? e1 : e0;
                const int eg[4] = {eh.x, eh.y, eh.z, eh.w};
                float sum = 0.0f;
                uint32_t hi[16], lo[16];
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const float f = pow2i(max(eg[g] - emax, -126));
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const float p0 = ex2(fmaf(s[8 * g + 2 * k], cq, shift)), p1 = ex2(fmaf(s[8 * g + 2 * k + 1], cq, shift));
                        sum += p0 + p1;
                        split_f16(p0 * f, p1 * f, hi[4 * g + k], lo[4 * g + k]);
                    }
                }
                l = fmaf(l, corr, sum);
                m = m_new;
                if (j > 0) {
                    ok = warp_wait(&o_full[(j - 1) & 1], (j - 1) / 2, a.err);  // P is free, and O of tile j - 1 is there
                    if (!ok) break;
                }
                uint8_t *dst = smem + S::off_p + half * 4 * (kRowsM * 16) + r * 16;
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    *reinterpret_cast<uint4 *>(dst + g * (kRowsM * 16)) = make_uint4(hi[4 * g], hi[4 * g + 1], hi[4 * g + 2], hi[4 * g + 3]);
                    *reinterpret_cast<uint4 *>(dst + g * (kRowsM * 16) + S::p_half) =
                        make_uint4(lo[4 * g], lo[4 * g + 1], lo[4 * g + 2], lo[4 * g + 3]);
                }
                fence_proxy_async();
                __syncwarp();
                if (lane == 0) mbar_arrive(p_full);
                if (j > 0) take_o(j - 1);
                corr_prev = corr;
                osc_prev = pow2i(emax - kRowsTop - (int)kRowsP);
            }
            if (ok) ok = warp_wait(&o_full[(nt - 1) & 1], (nt - 1) / 2, a.err);
            if (ok) {
                take_o(nt - 1);
                float other;
                ok = exchange(l, other);
                l = (half ? other : l) + (half ? l : other);  // the halves in one order
            }
            if (ok && mine) {
                // the weights carry 2^12, the sums of O do not
                const float lw = l * pow2i(-(int)kRowsP);
                if (p.splits > 1) {
                    float *dst = p.part + ((((size_t)item * a.n_kv_heads + kvh) * p.blocks + blk) * p.splits + split) * kRowsM * (hd + 4) +
                                 (size_t)r * (hd + 4);
                    if (half == 0) *reinterpret_cast<float2 *>(dst) = make_float2(m, lw);
                    dst += 4;
#pragma unroll
                    for (int c = 0; c < HD / 2; c += 4)
                        if (half * (HD / 2) + c < hd)
                            *reinterpret_cast<float4 *>(dst + half * (HD / 2) + c) = make_float4(acc[c], acc[c + 1], acc[c + 2], acc[c + 3]);
                } else {
                    const float inv = lw > 0.0f ? 1.0f / lw : lw == 0.0f ? 0.0f : lw;  // NaN stays
                    if (lw != lw && half == 0) raise_error(a.err, B2_ERR_NONFINITE);
                    float *dst = a.ctx + (size_t)(r0 + tok) * a.ctx_stride + (size_t)head * hd;
#pragma unroll
                    for (int c = 0; c < HD / 2; c += 4)
                        if (half * (HD / 2) + c < hd)
                            *reinterpret_cast<float4 *>(dst + half * (HD / 2) + c) =
                                make_float4(acc[c] * inv, acc[c + 1] * inv, acc[c + 2] * inv, acc[c + 3] * inv);
                }
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == kRowsSoftWarps + kRowsConvWarps) {
        tc_fence_after();
        tmem_free(tmem, 512);
    }
}

// Joins the splits of every (item, KV head, row) in split order: one warp per
// row, four dimensions per lane.
constexpr int kJoinWarps = 8;

__global__ void __launch_bounds__(kJoinWarps * 32) attn_rows_join_kernel(const RowsParams p)
{
    pdl_wait();
    pdl_launch_dependents();
    const b2_attn_rows_args &a = p.a;
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint32_t kvh = blockIdx.y, item = blockIdx.z, m_row = blockIdx.x * kJoinWarps + warp, hd = a.head_dim;
    uint32_t r0, n, ctx;
    if (!rows_item(a, item, r0, n, ctx)) return;
    if (m_row >= n * p.group) return;
    const uint32_t blk = m_row / kRowsM, r = m_row % kRowsM;
    const uint32_t places = rows_places(p, n, ctx, blk);
    const size_t stride = (size_t)kRowsM * (hd + 4);
    const float *base = p.part + (((size_t)item * a.n_kv_heads + kvh) * p.blocks + blk) * p.splits * stride + (size_t)r * (hd + 4);
    // the splits' statistics, one per lane and pass
    float ms[kRowsMaxSplits / 32], ls[kRowsMaxSplits / 32], top = -INFINITY;
#pragma unroll
    for (int i = 0; i < (int)kRowsMaxSplits / 32; ++i) {
        const uint32_t s = lane + 32 * i;
        ms[i] = -INFINITY;
        ls[i] = 0.0f;
        if (s < p.splits) {
            uint32_t t0, t1;
            rows_range(places, p.splits, s, t0, t1);
            if (t0 < t1) {
                const float2 x = *reinterpret_cast<const float2 *>(base + s * stride);
                ms[i] = x.x;
                ls[i] = x.y;
            }
        }
        top = fmaxf(top, ms[i]);
    }
    top = warp_max(top);
    if (top == -INFINITY) top = 0.0f;
    float4 o = make_float4(0, 0, 0, 0);
    float l = 0.0f;
#pragma unroll
    for (int i = 0; i < (int)kRowsMaxSplits / 32; ++i) {
        const float f = ex2(ms[i] - top);
        for (uint32_t s = 32 * i; s < min(p.splits, 32u * (i + 1)); ++s) {
            const float fs = __shfl_sync(0xffffffffu, f, s - 32 * i), lsum = __shfl_sync(0xffffffffu, ls[i], s - 32 * i);
            uint32_t t0, t1;
            rows_range(places, p.splits, s, t0, t1);
            if (t0 == t1) continue;
            l = fmaf(lsum, fs, l);
            if (4 * lane < hd) {
                const float4 x = reinterpret_cast<const float4 *>(base + s * stride + 4)[lane];
                o = make_float4(fmaf(x.x, fs, o.x), fmaf(x.y, fs, o.y), fmaf(x.z, fs, o.z), fmaf(x.w, fs, o.w));
            }
        }
    }
    const float inv = l > 0.0f ? 1.0f / l : l == 0.0f ? 0.0f : l;
    if (l != l && lane == 0) raise_error(a.err, B2_ERR_NONFINITE);
    if (4 * lane < hd)
        reinterpret_cast<float4 *>(a.ctx + (size_t)(r0 + m_row / p.group) * a.ctx_stride +
                                   (size_t)(kvh * p.group + m_row % p.group) * hd)[lane] =
            make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
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

// Blocks and splits. A CTA costs about kSetup tiles of time besides its own
// (launch, q, the pipeline's ends), a split launch about kJoin more for the
// joining kernel: the split count with the least waves x (tiles + kSetup).
static void attn_rows_plan(const b2_attn_rows_args *a, uint32_t &blocks, uint32_t &splits)
{
    const uint64_t group = a->n_heads / a->n_kv_heads;
    blocks = (uint32_t)((a->max_rows * group + kRowsM - 1) / kRowsM);
    const uint64_t ctas = (uint64_t)a->batch * a->n_kv_heads * blocks, sms = (uint64_t)sm_count();
    const uint64_t tiles = (a->max_ctx + kRowsKeys - 1) / kRowsKeys;
    constexpr uint64_t kSetup = 4, kJoin = 3;
    uint64_t best = ~0ull;
    splits = 1;
    for (uint64_t s = 1; s <= kRowsMaxSplits && s <= tiles; ++s) {
        const uint64_t waves = (ctas * s + sms - 1) / sms;
        const uint64_t cost = waves * ((tiles + s - 1) / s + kSetup) + (s > 1 ? kJoin : 0);
        if (cost < best) {
            best = cost;
            splits = (uint32_t)s;
        }
    }
}

static size_t attn_rows_scratch(const b2_attn_rows_args *a, uint32_t blocks, uint32_t splits)
{
    if (splits == 1) return 0;
    return (size_t)a->batch * a->n_kv_heads * blocks * splits * kRowsM * (a->head_dim + 4) * sizeof(float);
}

static cudaError_t launch_rows_attn(const void *fn, dim3 grid, int threads, size_t smem, int pdl, cudaStream_t st, const RowsParams &p)
{
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = pdl ? 1 : 0;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    void *args[] = {const_cast<RowsParams *>(&p)};
    return cudaLaunchKernelExC(&cfg, fn, args);
}

}  // namespace b2

using namespace b2;

extern "C" size_t b2_attn_rows_scratch_bytes(const b2_attn_rows_args *a)
{
    if (attn_rows_check(a) != 0) return 0;
    uint32_t blocks, splits;
    attn_rows_plan(a, blocks, splits);
    return attn_rows_scratch(a, blocks, splits);
}

extern "C" int b2_attn_rows(const b2_attn_rows_args *a, void *stream)
{
    const int rc = attn_rows_check(a);
    if (rc != 0) return rc;
    RowsParams p = {};
    p.a = *a;
    p.group = a->n_heads / a->n_kv_heads;
    attn_rows_plan(a, p.blocks, p.splits);
    if ((uint64_t)a->n_kv_heads * p.blocks > 65535u) return -9;
    const size_t need = attn_rows_scratch(a, p.blocks, p.splits);
    if (need > 0 && (a->scratch == nullptr || a->scratch_bytes < need || ((uintptr_t)a->scratch & 15))) return -1;
    p.part = (float *)a->scratch;
    p.scale = (float)(1.4426950408889634 / sqrt((double)a->head_dim));
    const cudaStream_t st = (cudaStream_t)stream;
    const bool wide = a->head_dim > 64;
    const void *fn = wide ? (const void *)attn_rows_kernel<128> : (const void *)attn_rows_kernel<64>;
    const size_t smem = wide ? RowsSmem<128>::bytes : RowsSmem<64>::bytes;
    if (cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess) return -8;
    if (launch_rows_attn(fn, dim3(p.splits, a->n_kv_heads * p.blocks, a->batch), kRowsThreads, smem, a->pdl, st, p) != cudaSuccess)
        return -8;
    if (p.splits > 1) {
        const uint32_t rows = a->max_rows * p.group;
        if (launch_rows_attn((const void *)attn_rows_join_kernel, dim3((rows + kJoinWarps - 1) / kJoinWarps, a->n_kv_heads, a->batch),
                             kJoinWarps * 32, 0, a->pdl, st, p) != cudaSuccess)
            return -8;
    }
    return 0;
}
