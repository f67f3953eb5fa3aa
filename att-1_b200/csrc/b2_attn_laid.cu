// b2_attn_laid.cu - attention of many new rows per sequence (prompt chunks) over the
// paged KV cache: b2_attn_rows where several blocks of 128 rows share an (item, KV
// head)'s K and V. Arithmetic and split are b2_attn_rows.cu's.
//
// There each block converts K and V for itself, which takes as many instruction slots as
// its softmax. Here a first kernel converts every tile once, into scratch (hi and lo are
// as many bytes as the f32), and the attention kernel's tiles arrive as operands, by bulk
// copies. 16 warps, by role:
//   warps 0..3, 4..7    softmax of the even and of the odd tiles, a row per thread, each
//                       group with its own P in tensor memory, running maximum and sum;
//   warps 8..11         32 rows each: every tile's O from tensor memory into f32 sums in
//                       registers, rescaled where a group's maximum passed the sums'
//                       (both groups' P are relative to their own; the maxima come along);
//   warps 12, 13        one thread each issues the MMAs of S, for a pair of tiles as soon as
//                       both groups have read the pair before, and those of O, when P is
//                       there (one thread for both was behind with waits and commits);
//   warps 14, 15        one thread each copies: K and the marks of a pair, two ahead, and V
//                       of a tile, two ahead (head sizes up to 64: four).
// An MMA of 128 rows and K = 16 costs 64 cycles with N = 128 and hardly less with fewer, so
// S is taken of pairs of tiles. S of a pair, two P, q and O fill the 512 columns.
//
// 8B shape: a chunk of 512 at context 2500 77 us with the conversion (8 us), 300 TFLOP/s
// of f32 products (three f16 products each); 2000 rows at context 6000 634 us. Each block
// converting for itself: 110 and 992 us. A tile takes 2500 cycles, its MMAs 1580: O of a tile
// (800), its reading out (600) and the hand-overs between the roles (200 to 300 each) follow
// one another, because tensor memory has no room for a second O.
#include "b2_attn_rows.cuh"

#include <type_traits>

namespace b2 {

constexpr uint32_t kLaidSoftWarps = 4;  // per group
constexpr uint32_t kLaidSumWarp = 2 * kLaidSoftWarps, kLaidMmaWarp = kLaidSumWarp + 4, kLaidCopyWarp = kLaidMmaWarp + 2;
constexpr int kLaidThreads = 512;  // whole warpgroups
// Registers a thread of the softmax warpgroups (two), the summing one and the last; the
// launch gives every thread 128.
constexpr int kLaidSoftRegs = 128, kLaidSumRegs = 224, kLaidLastRegs = 32;
static_assert(256 * kLaidSoftRegs + 128 * kLaidSumRegs + 128 * kLaidLastRegs <= kLaidThreads * 128, "register split");

constexpr uint32_t kLaidMarks = 4;   // ring of marks: more than the pairs between the copy and the end of a softmax

// A tile's marks: [8] u32 of K's units, [8] of V's; [64] s8 places' exponents of K, of V.
struct TileMarks {
    static constexpr uint32_t off_vm = 8 * 4, off_ke = off_vm + 8 * 4, off_ve = off_ke + kRowsKeys, bytes = off_ve + kRowsKeys;
};
// A pair of tiles in memory: K as one operand of 128 places [hi, lo], V per tile [hi, lo], marks per tile.
template <int HD>
struct LaidPair {
    static constexpr uint32_t k_half = kLaidKeys * HD * 2, v_tile = 2 * kRowsKeys * HD * 2;
    static constexpr uint32_t off_v = 2 * k_half, off_m = off_v + 2 * v_tile, bytes = off_m + 2 * TileMarks::bytes;
    static_assert(bytes % 128 == 0, "alignment");
};

template <int HD>
struct LaidSmem {
    using P = LaidPair<HD>;
    static constexpr uint32_t k_stages = 2, v_stages = HD == 128 ? 2 : 4;
    static constexpr uint32_t off_k = 0;
    static constexpr uint32_t off_v = off_k + k_stages * 2 * P::k_half;
    static constexpr uint32_t off_m = off_v + v_stages * P::v_tile;  // [kLaidMarks][2] marks of a tile
    static constexpr uint32_t off_cq = off_m + kLaidMarks * 2 * TileMarks::bytes;  // [128] f32: the rows' score factors
    static constexpr uint32_t off_qt = off_cq + kRowsM * 4;         // [128] u32: bits of their largest |q|
    static constexpr uint32_t off_ri = off_qt + kRowsM * 4;         // [4][128] (f32, f32): a tile's maximum and factor per row
    static constexpr uint32_t off_l = off_ri + 4 * kRowsM * 8;      // [group][128] (f32, f32): maximum and sum at the end
    static constexpr uint32_t off_bar = off_l + 2 * kRowsM * 8;
    static constexpr uint32_t bytes = off_bar + 8 * (2 * k_stages + 2 * v_stages + 2 + 2 * 2 + 4) + 16;
};
static_assert(LaidSmem<128>::bytes <= 227 * 1024 && LaidSmem<64>::bytes <= 227 * 1024, "shared memory");

// Every item's K and V as operands, for the blocks of rows to share: CTA (tile, KV head,
// item), eight warps, 16 places of K or V each. The pair's second tile is written whole,
// zeros past the end.
constexpr int kLayWarps = 8;

template <int HD, bool EXACT>
__global__ void __launch_bounds__(kLayWarps * 32) attn_rows_lay_kernel(const RowsParams p)
{
    extern __shared__ __align__(1024) uint8_t smem[];
    const b2_attn_rows_args &a = p.a;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, tile = blockIdx.x, kvh = blockIdx.y, item = blockIdx.z;
    const uint32_t hd = EXACT ? HD : a.head_dim, pt = a.kv.page_tokens;
    const bool is_v = warp >= kLayWarps / 2;
    pdl_wait();
    pdl_launch_dependents();
    uint32_t r0, n, ctx;
    if (!rows_item(a, item, r0, n, ctx) || n == 0 || tile / 2 * kLaidKeys >= ctx + n) return;
    const uint32_t u = warp % (kLayWarps / 2), at = tile * kRowsKeys + u * kRowsUnit + (lane & 15);
    const bool in = at < ctx + n;
    const int32_t page = in ? a.kv.page_table[(size_t)item * a.kv.pages_per_seq + at / pt] : 0;
    const bool wrong = in && (page < 0 || (a.pool_pages != 0 && (uint32_t)page >= a.pool_pages));
    const uint32_t hidden = __ballot_sync(0xffffffffu, wrong) & 0xFFFFu, live = __ballot_sync(0xffffffffu, in && !wrong) & 0xFFFFu;
    if (wrong) raise_error(a.err, B2_ERR_POSITION);
    const size_t row = in && !wrong ? ((size_t)(uint32_t)page * a.n_kv_heads + kvh) * pt + at % pt : 0;
    float *mine = reinterpret_cast<float *>(smem) + warp * kRowsUnit * HD;
    const float *pool = is_v ? a.kv.v_pool : a.kv.k_pool;
#pragma unroll
    for (uint32_t i = 0; i < kRowsUnit; ++i) {
        const size_t r = __shfl_sync(0xffffffffu, row, i);
        if (4 * lane < hd && (live >> i & 1)) cp_async16(mine + i * hd + 4 * lane, pool + r * hd + 4 * lane, 16);
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncwarp();
    using P = LaidPair<HD>;
    uint8_t *out = p.laid + (((size_t)item * a.n_kv_heads + kvh) * p.pairs + tile / 2) * P::bytes, *marks = out + P::off_m + tile % 2 * TileMarks::bytes;
    // K: the tile's 64 of the pair's 128 rows
    uint8_t *to = is_v ? out + P::off_v + tile % 2 * P::v_tile : out + tile % 2 * kRowsKeys * 16;
#pragma unroll 1
    for (uint32_t h = 0; h < kRowsUnit / 8; ++h) {
        const uint32_t w = u * (kRowsUnit / 8) + h;
        const uint32_t m = lay_unit<HD, EXACT>(mine + 8 * h * hd, hd, is_v, w, ~live >> (8 * h) & 0xFFu, hidden >> (8 * h) & 0xFFu, to, P::k_half,
                                               reinterpret_cast<int8_t *>(marks + (is_v ? TileMarks::off_ve : TileMarks::off_ke)));
        if (lane == 0) reinterpret_cast<uint32_t *>(marks + (is_v ? TileMarks::off_vm : 0))[w] = m;
    }
}

// A block's rows of q as operand A, in two steps of eight warps w with a barrier between:
// whole rows, coalesced, into hi and lo images in shared memory (128 rows of HD f16 each;
// 16-byte pieces of a row are permuted by it, so that a thread per row reads without
// conflicts), with the rows' score factors and largest |q|; then a thread's row into
// tensor memory, the dimensions of one half.
template <int HD>
__device__ __forceinline__ void stage_q(const RowsParams &p, uint32_t w, uint32_t r0, uint32_t kvh, uint32_t first, uint32_t live, uint8_t *hi,
                                        uint8_t *lo, float *cqs, uint32_t *tops)
{
    constexpr uint32_t kAhead = 8;  // rows asked for at a time
    const b2_attn_rows_args &a = p.a;
    const uint32_t lane = threadIdx.x & 31, hd = a.head_dim;
#pragma unroll 1
    for (uint32_t b = w; b < live; b += 8 * kAhead) {
        float4 f[kAhead];
#pragma unroll
        for (uint32_t i = 0; i < kAhead; ++i) {
            const uint32_t r = b + 8 * i, m_row = first + r;
            f[i] = make_float4(0, 0, 0, 0);
            if (r < live && 4 * lane < hd)
                f[i] = __ldcg(reinterpret_cast<const float4 *>(a.q + (size_t)(r0 + m_row / p.group) * a.q_stride + (size_t)(kvh * p.group + m_row % p.group) * hd) + lane);
        }
#pragma unroll
        for (uint32_t i = 0; i < kAhead; ++i) {
            const uint32_t r = b + 8 * i;
            if (r >= live) break;
            uint32_t top = max(max(abs_bits(f[i].x), abs_bits(f[i].y)), max(abs_bits(f[i].z), abs_bits(f[i].w)));
            top = __reduce_max_sync(0xffffffffu, top);
            const bool bad = top >= 0x7F800000u;
            const int e = bad ? 0 : top_exp(top);
            const float sc = pow2i(-e);
            if (bad) f[i] = make_float4(0, 0, 0, 0);
            if (lane == 0) {
                cqs[r] = bad ? NAN : pow2i(e) * p.scale;
                tops[r] = bad ? 0 : top;
            }
            if (4 * lane < HD) {
                uint2 h2, l2;
                split_f16(f[i].x * sc, f[i].y * sc, h2.x, l2.x);
                split_f16(f[i].z * sc, f[i].w * sc, h2.y, l2.y);
                const uint32_t at = r * HD * 2 + (((lane >> 1) ^ (r & (HD / 8 - 1))) * 16 + (lane & 1) * 8);
                *reinterpret_cast<uint2 *>(hi + at) = h2;
                *reinterpret_cast<uint2 *>(lo + at) = l2;
            }
        }
    }
}
template <int HD>
__device__ __forceinline__ void put_q(uint32_t tm_q, uint32_t half, uint32_t r, const uint8_t *hi, const uint8_t *lo)
{
#pragma unroll
    for (uint32_t c = 0; c < HD / 2; c += 32) {  // 32 dimensions: 16 columns of hi, 16 of lo
#pragma unroll
        for (uint32_t k = 0; k < 2; ++k) {
            uint32_t v[16];
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) {
                const uint32_t piece = (half * (HD / 2) + c) / 8 + i;
                const uint4 x = *reinterpret_cast<const uint4 *>((k ? lo : hi) + r * HD * 2 + (piece ^ (r & (HD / 8 - 1))) * 16);
                v[4 * i] = x.x, v[4 * i + 1] = x.y, v[4 * i + 2] = x.z, v[4 * i + 3] = x.w;
            }
            tmem_st16(tm_q + k * (HD / 2) + half * (HD / 4) + c / 2, v);
        }
    }
}

template <int HD>
__global__ void __launch_bounds__(kLaidThreads, 1) attn_laid_kernel(const RowsParams p)
{
    using S = LaidSmem<HD>;
    using P = LaidPair<HD>;
    constexpr uint32_t NK = S::k_stages, NV = S::v_stages;
    extern __shared__ __align__(1024) uint8_t smem[];
    const b2_attn_rows_args &a = p.a;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t split = blockIdx.x, kvh = blockIdx.y / p.blocks, blk = blockIdx.y % p.blocks, item = blockIdx.z;
    const uint32_t hd = a.head_dim;
    float2 *info = reinterpret_cast<float2 *>(smem + S::off_ri), *ends = reinterpret_cast<float2 *>(smem + S::off_l);
    float *cqs = reinterpret_cast<float *>(smem + S::off_cq);
    // by stage: K (with the marks) and V there, read by their products; S there and read; by group: P and O there
    uint64_t *k_full = reinterpret_cast<uint64_t *>(smem + S::off_bar), *k_free = k_full + NK, *v_full = k_free + NK, *v_free = v_full + NV,
             *s_full = v_free + NV, *s_empty = s_full + 1, *p_full = s_empty + 1, *o_full = p_full + 2,
             *o_empty = o_full + 2, *q_full = o_empty + 1, *done = q_full + 1;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(done + 2);

    // Launched while attn_rows_lay_kernel still runs: what came before that has completed, and
    // only the copies read what it writes. The lengths, q and the masks are read without this
    // kernel's own wait, so from L2: nothing says that an SM's L1 no longer holds what the same
    // buffers had in the layer before.
    pdl_launch_dependents();
    uint32_t r0, n, ctx;
    if (!rows_fit(a, __ldcg(a.row_start + item), __ldcg(a.row_start + item + 1), __ldcg(a.ctx_len + item), r0, n, ctx)) {
        if (threadIdx.x == 0 && split == 0 && blockIdx.y == 0) raise_error(a.err, B2_ERR_POSITION);
        pdl_wait();
        return;
    }
    const uint32_t mrows = n * p.group;  // rows of this (item, KV head)
    if (blk * kRowsM >= mrows) {
        pdl_wait();
        return;
    }
    const uint32_t live = min(kRowsM, mrows - blk * kRowsM);
    const uint32_t places = rows_places(p, n, ctx, blk);
    uint32_t t0, t1;
    rows_range(p, places, split, t0, t1);
    if (t0 == t1) {  // the joining kernel skips the same splits
        pdl_wait();
        return;
    }
    const uint32_t np = t1 - t0, nt = 2 * np;  // pairs of tiles, tiles
    const uint32_t nq = (live + 31) / 32;  // quarters of the rows in use

    if (threadIdx.x == 0) {
        for (uint32_t i = 0; i < NK; ++i) {
            mbar_init(&k_full[i], 1);
            mbar_init(&k_free[i], 1);
        }
        for (uint32_t i = 0; i < NV; ++i) {
            mbar_init(&v_full[i], 1);
            mbar_init(&v_free[i], 1);
        }
        for (uint32_t i = 0; i < 2; ++i) {
            mbar_init(&p_full[i], nq);
            mbar_init(&o_full[i], 2);  // the products, and the issuing thread with what it saw of P's
        }
        mbar_init(s_full, 2);  // and of the marks'
        mbar_init(s_empty, 2 * nq);
        mbar_init(o_empty, nq);
        mbar_init(q_full, 2 * nq);
        mbar_init(&done[0], 1);
        mbar_init(&done[1], 1);
        fence_mbar_init();
    }
    if (warp == kLaidMmaWarp) tmem_alloc(tmem_slot, 512);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    // columns: S 64 per tile of the pair | P hi 32, lo 32 per group | Q hi HD / 2, lo HD / 2 | O from 384
    const uint32_t tm_s = tmem, tm_p = tmem + 128, tm_q = tmem + 256, tm_o = tmem + 384;

    if (warp >= kLaidMmaWarp) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kLaidLastRegs));
        if (warp >= kLaidCopyWarp) {
            if (lane == 0) {
                const uint8_t *src = p.laid + (((size_t)item * a.n_kv_heads + kvh) * p.pairs + t0) * P::bytes;
                bool ok = true;
                uint32_t i = 0;
                pdl_wait();
                // (no copy is in flight when the CTA ends, not even after a wait that gave up)
                if (warp == kLaidCopyWarp) {
                    for (; i < np; ++i, src += P::bytes) {
                        const uint32_t st = i % NK;
                        if (i == NK - 1) ok = mbar_wait_bounded(q_full, 0, a.err);  // q came through this stage
                        if (i >= NK) ok = mbar_wait_bounded(&k_free[st], (i / NK - 1) & 1, a.err);
                        if (!ok) break;
                        mbar_arrive_expect_tx(&k_full[st], 2 * P::k_half + 2 * TileMarks::bytes);
                        bulk_g2s(smem + S::off_k + st * 2 * P::k_half, src, 2 * P::k_half, &k_full[st]);
                        bulk_g2s(smem + S::off_m + i % kLaidMarks * 2 * TileMarks::bytes, src + P::off_m, 2 * TileMarks::bytes, &k_full[st]);
                    }
                    for (uint32_t k = i > NK ? i - NK : 0; k < i; ++k) mbar_wait_bounded(&k_full[k % NK], (k / NK) & 1, a.err);
                } else {
                    for (src += P::off_v; i < nt; ++i, src += i & 1 ? P::v_tile : P::bytes - P::v_tile) {
                        const uint32_t st = i % NV;
                        if (i >= NV) ok = mbar_wait_bounded(&v_free[st], (i / NV - 1) & 1, a.err);
                        if (!ok) break;
                        mbar_arrive_expect_tx(&v_full[st], P::v_tile);
                        bulk_g2s(smem + S::off_v + st * P::v_tile, src, P::v_tile, &v_full[st]);
                    }
                    for (uint32_t k = i > NV ? i - NV : 0; k < i; ++k) mbar_wait_bounded(&v_full[k % NV], (k / NV) & 1, a.err);
                }
            }
            __syncwarp();
        } else if (warp == kLaidMmaWarp) {
            if (elect_one()) {
                const uint32_t id_s = umma_idesc_f16(kRowsM, kLaidKeys), kb = smem_u32(smem + S::off_k);
                bool ok = mbar_wait_bounded(q_full, 0, a.err);
                for (uint32_t i = 0; ok && i < np; ++i) {
                    const uint32_t st = i % NK;
                    ok = spin_wait(&k_full[st], (i / NK) & 1, a.err) && (i == 0 || spin_wait(s_empty, (i - 1) & 1, a.err));
                    if (!ok) break;
                    tc_fence_after();
                    // (a descriptor's address field counts 16 bytes)
                    const uint64_t kh = umma_desc(kb + st * 2 * P::k_half, kLaidKeys * 16, 128), kl = umma_desc(kb + st * 2 * P::k_half + P::k_half, kLaidKeys * 16, 128);
#pragma unroll 1
                    for (uint32_t kk = 0; kk < hd / 16; ++kk) {
                        umma_16_ts(tm_s, tm_q + kk * 8, kh + kk * 2 * kLaidKeys, id_s, kk > 0);
                        umma_16_ts(tm_s, tm_q + HD / 2 + kk * 8, kh + kk * 2 * kLaidKeys, id_s, 1);
                        umma_16_ts(tm_s, tm_q + kk * 8, kl + kk * 2 * kLaidKeys, id_s, 1);
                    }
                    umma_commit(s_full);
                    mbar_arrive(s_full);
                    umma_commit(&k_free[st]);
                }
                // everything issued has completed before tensor memory is freed
                umma_commit(&done[0]);
                mbar_wait_bounded(&done[0], 0, a.err);
            }
            __syncwarp();
        } else if (warp == kLaidMmaWarp + 1) {
            if (elect_one()) {
                const uint32_t id_o = umma_idesc_f16(kRowsM, hd), vb = smem_u32(smem + S::off_v);
                bool ok = true;
                for (uint32_t j = 0; ok && j < nt; ++j) {
                    const uint32_t st = j % NV, g = j & 1;
                    const uint64_t vh = umma_desc(vb + st * P::v_tile, HD * 16, 128), vl = umma_desc(vb + st * P::v_tile + P::v_tile / 2, HD * 16, 128);
                    const uint32_t pp = tm_p + g * kRowsKeys;
                    // O's buffer, free once the tile before was summed, is what comes last
                    ok = spin_wait(&v_full[st], (j / NV) & 1, a.err) && spin_wait(&p_full[g], (j / 2) & 1, a.err) &&
                         (j == 0 || spin_wait(o_empty, (j - 1) & 1, a.err));
                    if (!ok) break;
                    tc_fence_after();
#pragma unroll 1
                    for (uint32_t kk = 0; kk < kRowsKeys / 16; ++kk) {
                        umma_16_ts(tm_o, pp + kk * 8, vh + kk * 2 * HD, id_o, kk > 0);
                        umma_16_ts(tm_o, pp + 32 + kk * 8, vh + kk * 2 * HD, id_o, 1);
                        umma_16_ts(tm_o, pp + kk * 8, vl + kk * 2 * HD, id_o, 1);
                    }
                    umma_commit(&o_full[g]);
                    umma_commit(&v_free[st]);
                    mbar_arrive(&o_full[g]);
                }
                umma_commit(&done[1]);
                mbar_wait_bounded(&done[1], 0, a.err);
            }
            __syncwarp();
        }
        tc_fence_before();
        __syncthreads();
        if (warp == kLaidMmaWarp) {
            tc_fence_after();
            tmem_free(tmem, 512);
        }
    } else if (warp >= kLaidSumWarp) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kLaidSumRegs));
        // ---- the sums of O: row r, all dimensions ----
        const uint32_t qt = warp & 3, r = qt * 32 + lane;
        bool ok = true;
        float m = -INFINITY;      // what the sums are relative to
        uint64_t acc[HD / 2];     // pairs of dimensions
#pragma unroll
        for (int i = 0; i < HD / 2; ++i) acc[i] = 0;
        for (uint32_t j = 0; ok && qt < nq && j < nt; ++j) {
            ok = warp_wait(&o_full[j & 1], j / 2, a.err);
            if (!ok) break;
            tc_fence_after();
            uint32_t v[16];
            tmem_ld16_nowait(tm_o + ((qt * 32) << 16), v);
            const float2 f = info[(j & 3) * kRowsM + r];
            const float m_new = fmaxf(m, f.x), m_use = m_new == -INFINITY ? 0.0f : m_new;
            if (__any_sync(0xffffffffu, m_new != m)) {
                const float c = ex2(m - m_use);
                const uint64_t c2 = pair(c, c);
#pragma unroll
                for (int k = 0; k < HD / 2; ++k) acc[k] = mul2(acc[k], c2);
            }
            m = m_new;
            const float o1 = f.y * ex2(f.x - m_use);
            const uint64_t o2 = pair(o1, o1);
#pragma unroll
            for (int c = 0; c < HD; c += 16) {
                tmem_wait_ld();
#pragma unroll
                for (int k = 0; k < 8; ++k)
                    acc[c / 2 + k] = fma2(pair(__uint_as_float(v[2 * k]), __uint_as_float(v[2 * k + 1])), o2, acc[c / 2 + k]);
                if (c + 16 < HD) tmem_ld16_nowait(tm_o + ((qt * 32) << 16) + c + 16, v);
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(o_empty);
        }
        tc_fence_before();
        __syncthreads();
        if (ok && r < live) {
            const float m_use = m == -INFINITY ? 0.0f : m;
            float l = 0.0f;
#pragma unroll
            for (int g = 0; g < 2; ++g) {
                const float2 x = ends[g * kRowsM + r];
                l = fmaf(x.y, ex2(x.x - m_use), l);
            }
            l *= pow2i(-(int)kRowsP);  // the weights carry 2^11, the sums of O do not
            const uint32_t m_row = blk * kRowsM + r;
            float *dst;
            float inv = 1.0f;
            if (p.splits > 1) {
                dst = rows_part(p, item, kvh, blk, split) + (size_t)r * (hd + 4);
                *reinterpret_cast<float2 *>(dst) = make_float2(m, l);
                dst += 4;
            } else {
                inv = l > 0.0f ? 1.0f / l : l == 0.0f ? 0.0f : l;  // NaN stays
                if (l != l) raise_error(a.err, B2_ERR_NONFINITE);
                dst = a.ctx + (size_t)(r0 + m_row / p.group) * a.ctx_stride + (size_t)(kvh * p.group + m_row % p.group) * hd;
            }
#pragma unroll
            for (int c = 0; c < HD; c += 4) {
                if (c < (int)hd) {
                    float4 f;
                    unpair(acc[c / 2], f.x, f.y);
                    unpair(acc[c / 2 + 1], f.z, f.w);
                    *reinterpret_cast<float4 *>(dst + c) = make_float4(f.x * inv, f.y * inv, f.z * inv, f.w * inv);
                }
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kLaidSoftRegs));
        // ---- softmax of every other tile: row r ----
        const uint32_t g = warp / kLaidSoftWarps, qt = warp & 3, r = qt * 32 + lane;
        uint8_t *q_hi = smem + S::off_k + (NK - 1) * 2 * P::k_half, *q_lo = q_hi + P::k_half;
        stage_q<HD>(p, warp, r0, kvh, blk * kRowsM, live, q_hi, q_lo, cqs, reinterpret_cast<uint32_t *>(smem + S::off_qt));
        asm volatile("bar.sync 1, 256;" ::: "memory");
        if (qt < nq) {
            const bool mine = r < live;
            const uint32_t tok = mine ? (blk * kRowsM + r) / p.group : 0;
            const uint32_t lanes = (qt * 32) << 16;
            // score of a row: dot * K scale * cq, in powers of two; the sign says whether the warp's rows
            // are far (a register of its own, held over the loop, cost 1.5 percent)
            const bool far = rows_far(mine ? reinterpret_cast<const uint32_t *>(smem + S::off_qt)[r] : 0, p.reach);
            const float cq = copysignf(mine ? cqs[r] : 0.0f, far ? -1.0f : 1.0f);
            put_q<HD>(tm_q + lanes, g, r, q_hi, q_lo);
            tmem_wait_st();
            fence_proxy_async();  // (a copy writes there next)
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(q_full);
            const uint64_t mask = mine && a.tree != nullptr ? __ldcg(reinterpret_cast<const unsigned long long *>(a.tree) + r0 + tok) : 0;
            float m = -INFINITY, l = 0.0f;
            bool ok = true;
            // One tile; those with units of different scale, marked places or scores past 2^23 have
            // a copy of the code of their own.
            auto tile = [&](uint32_t j, auto rare, const uint8_t *marks) {
                constexpr bool RARE = decltype(rare)::value;
                const uint32_t *ks = reinterpret_cast<const uint32_t *>(marks), *vs = reinterpret_cast<const uint32_t *>(marks + TileMarks::off_vm);
                const int8_t *ke = reinterpret_cast<const int8_t *>(marks + TileMarks::off_ke), *ve = reinterpret_cast<const int8_t *>(marks + TileMarks::off_ve);
                const uint32_t key0 = t0 * kLaidKeys + j * kRowsKeys;
                auto visible = [&](uint32_t c) { return rows_visible(a.tree != nullptr, mask, tok, ctx, places, key0 + c); };
                // a tile that all rows see whole needs no masks
                uint64_t vis = ~0ull;
                if (key0 + kRowsKeys > ctx) vis = (uint64_t)visible(32) << 32 | visible(0);
                if (RARE) vis &= ~((uint64_t)meta_bytes(*reinterpret_cast<const uint4 *>(ks + 4), 8) << 32 | meta_bytes(*reinterpret_cast<const uint4 *>(ks), 8));
                const float cqk = RARE ? 1.0f : score_factor(cq, meta_exp(ks[0]));
                float s[64];
                {
                    uint32_t x[32], y[32];
                    tmem_ld32(tm_s + lanes + g * kRowsKeys, x);
                    tmem_ld32(tm_s + lanes + g * kRowsKeys + 32, y);
                    tmem_wait_ld();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(s_empty);
#pragma unroll
                    for (int k = 0; k < 32; ++k) s[k] = __uint_as_float(x[k]), s[32 + k] = __uint_as_float(y[k]);
                }
                if (RARE) {
#pragma unroll
                    for (int k = 0; k < 64; ++k) {
                        s[k] = place_score(s[k], fabsf(cq), exp_of(ks, ke, k));
                        if (ks[k / 8] >> (k & 7) & 1) s[k] = NAN;
                    }
                }
                if (vis != ~0ull) {
#pragma unroll
                    for (int k = 0; k < 64; ++k)
                        if (!((k < 32 ? (uint32_t)vis : (uint32_t)(vis >> 32)) >> (k & 31) & 1)) s[k] = -INFINITY;
                }
                float top = fmaxf(s[0], s[1]), top2 = fmaxf(s[2], s[3]);
#pragma unroll
                for (int k = 4; k < 64; k += 4) {
                    top = max3(top, s[k], s[k + 1]);
                    top2 = max3(top2, s[k + 2], s[k + 3]);
                }
                top = fmaxf(top, top2) * cqk;
                // (kept while it grows by less than kRowsSlack, so that the sums are seldom rescaled)
                const float m_new = top > m + kRowsSlack ? top : m;
                const float m_use = m_new == -INFINITY ? 0.0f : m_new;
                const float corr = ex2(m - m_use);
                m = m_new;
                const float shift = RARE ? kRowsP : kRowsP - m_use;
                if (RARE) {
#pragma unroll
                    for (int k = 0; k < 64; ++k) s[k] -= m_use;
                }
                const uint64_t cq2 = pair(cqk, cqk), sh2 = pair(shift, shift);
                uint64_t sum = 0;
#pragma unroll
                for (int k = 0; k < 64; k += 2) {
                    float y, z;
                    unpair(fma2(pair(s[k], s[k + 1]), cq2, sh2), y, z);
                    s[k] = ex2(y);
                    s[k + 1] = ex2(z);
                    sum = add2(sum, pair(s[k], s[k + 1]));
                }
                float sy, sz;
                unpair(sum, sy, sz);
                l = fmaf(l, corr, sy + sz);
                int emax = meta_exp(vs[0]);
                if (RARE && !units_plain(vs)) {  // P takes V's scales relative to the row's own largest weighted place
                    emax = -100;
#pragma unroll
                    for (int k = 0; k < 64; ++k) emax = max(emax, weight_exp(s[k], exp_of(vs, ve, k)));
#pragma unroll
                    for (int k = 0; k < 64; ++k) s[k] *= pow2c(exp_of(vs, ve, k) - emax);
                    const uint64_t bad = (uint64_t)meta_bytes(*reinterpret_cast<const uint4 *>(vs + 4), 0) << 32 | meta_bytes(*reinterpret_cast<const uint4 *>(vs), 0);
                    if ((bad & vis) != 0) l = NAN;
                }
                uint32_t hi[2][16], lo[2][16];
#pragma unroll
                for (int k = 0; k < 32; ++k) cut_f16(s[2 * k], s[2 * k + 1], hi[k / 16][k % 16], lo[k / 16][k % 16]);
                if (j >= 2) ok = ok && warp_wait(&o_full[g], j / 2 - 1, a.err);  // P of the group's tile before was read
                info[(j & 3) * kRowsM + r] = make_float2(m, pow2i(emax - (int)kRowsP));
                tc_fence_after();
                const uint32_t to = tm_p + lanes + g * kRowsKeys;
                tmem_st16(to, hi[0]);
                tmem_st16(to + 16, hi[1]);
                tmem_st16(to + 32, lo[0]);
                tmem_st16(to + 48, lo[1]);
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&p_full[g]);
            };
            for (uint32_t j = g; ok && j < nt; j += 2) {
                const uint32_t i = j / 2;
                ok = warp_wait(s_full, i, a.err);
                if (!ok) break;
                tc_fence_after();
                const uint8_t *marks = smem + S::off_m + (i % kLaidMarks * 2 + g) * TileMarks::bytes;
                const uint32_t *ks = reinterpret_cast<const uint32_t *>(marks);
                if (units_plain(ks) && ks[0] <= meta_of_exp(0) && __float_as_int(cq) >= 0 && units_plain(ks + 8)) tile(j, std::false_type(), marks);
                else tile(j, std::true_type(), marks);
            }
            ends[g * kRowsM + r] = make_float2(m, l);
        }
        tc_fence_before();
        __syncthreads();
    }
}

template <int HD, bool EXACT>
static cudaError_t launch_laid(const RowsParams &p, cudaStream_t st)
{
    const b2_attn_rows_args &a = p.a;
    auto launch = [&](void (*kernel)(const RowsParams), dim3 grid, uint32_t threads, uint32_t smem, int pdl) {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) return e;
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
        return cudaLaunchKernelEx(&cfg, kernel, p);
    };
    const cudaError_t e = launch(attn_rows_lay_kernel<HD, EXACT>, dim3(2 * p.pairs, a.n_kv_heads, a.batch), kLayWarps * 32, kRowsKeys * 2 * HD * 4, a.pdl);
    return e != cudaSuccess ? e : launch(attn_laid_kernel<HD>, dim3(p.splits, a.n_kv_heads * p.blocks, a.batch), kLaidThreads, LaidSmem<HD>::bytes, 1);
}

size_t attn_laid_pair(uint32_t head_dim) { return head_dim > 64 ? LaidPair<128>::bytes : LaidPair<64>::bytes; }

cudaError_t attn_laid_launch(const RowsParams &p, cudaStream_t st)
{
    return p.a.head_dim == 128  ? launch_laid<128, true>(p, st)
           : p.a.head_dim > 64  ? launch_laid<128, false>(p, st)
           : p.a.head_dim == 64 ? launch_laid<64, true>(p, st)
                                : launch_laid<64, false>(p, st);
}

}  // namespace b2
