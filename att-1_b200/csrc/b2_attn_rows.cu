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
// K and V are read once per 128 rows. 20 warps (two idle), by role:
//   warp 17       streams K and V (f32) into a ring of tiles with bulk copies, a
//                 run of places on one page each;
//   warps 8..15   convert 16 places each of every tile's K (8..11) or V (12..15) from
//                 the ring into matrix operands;
//   warp 16       one thread issues the tcgen05 MMAs: S = Q K^T of tile j + 1
//                 before O = P V of tile j; Q, P, S and O live in tensor memory,
//                 only K and V are read from shared memory;
//   warps 0..7    two per 32 rows: a thread holds one row and 32 of a tile's 64
//                 places: its scores from tensor memory, the row's running maximum
//                 (over all 64, so the two need not talk), P back into tensor
//                 memory; and half of the dimensions of the row's O, summed in
//                 registers over the tiles: a growing maximum rescales registers,
//                 not tensor memory, and no sum runs through more than 12 MMAs.
// Splits write (maximum, sum, weighted values) per row; a second kernel joins
// them in split order. No counters or atomics: results do not depend on timing.
//
// Precision. Every f32 operand x becomes two f16 numbers of x 2^e (the scale
// exact): hi = f16(x 2^e), lo = f16(x 2^e - hi), and a product is
// hi hi + lo hi + hi lo with f32 accumulation; what is dropped is below 2^-22.
// f16 rather than bf16 pairs (2^-16) because the scale takes care of the range:
// a row of q, eight places' K and eight places' V have a power of two each, 1 for
// largest magnitudes from 2^-4 to 2^12, else what brings the largest to [1, 16). So an
// element keeps 22 bits down to 2^-3, and what a smaller one loses is below 2^-25 (both
// of 1, or of the scaled largest). The scaling exponents are multiples of four, so that
// neighbours mostly share one, and mostly have none to apply. A
// place of 2^12 and more that is far above one of its neighbours gets its own scale,
// as they do: a place that a row does not see, or gives no weight, takes nothing from
// the others, whatever it holds. K's scale goes into the scores; V's into P, relative
// to the row's largest weighted place where they differ, and that into its O when it
// is summed. The softmax statistics and the weighted sums are f32.
//
// Operands in shared memory are K-major without swizzle as in b2_gemm.cu: 8-row
// x 16-byte core matrices, row groups 128 bytes apart, 8-column chunks R * 16
// bytes apart. V is transposed on its way through the registers (a lane holds
// eight places of a dimension: one 16-byte store). Operand A of every MMA comes
// from tensor memory, two f16 to a column: 128 rows of A would cost as many
// shared-memory cycles per MMA as B does, and shared memory is what a tile of 64
// places uses most (copies in 64 KB, conversion 64 + 64 KB, MMAs 96 KB).
#include "b2_attn_rows.cuh"
#include "b2_umma.cuh"

#include <type_traits>

namespace b2 {

constexpr int kRowsSoftWarps = 8;
constexpr int kRowsConvWarps = 8;
constexpr uint32_t kRowsMmaWarp = kRowsSoftWarps + kRowsConvWarps, kRowsCopyWarp = kRowsMmaWarp + 1;
constexpr int kRowsThreads = 32 * (kRowsSoftWarps + kRowsConvWarps + 4);  // whole warpgroups: two warps idle
// Registers a thread of the softmax warpgroups (two), the converting ones (two) and
// the last one; the launch gives every thread 96 (five warps per scheduler).
constexpr int kRowsSoftRegs = 136, kRowsConvRegs = 80, kRowsLastRegs = 40;
static_assert(kRowsThreads == 640 && 256 * kRowsSoftRegs + 256 * kRowsConvRegs + 128 * kRowsLastRegs <= 640 * 96, "register split");
constexpr uint32_t kRowsMeta = 4;       // ring of per-tile scales: more than the tiles between converting and softmax

template <int HD>
struct RowsSmem {
    static constexpr uint32_t stages = 2;                           // operands of two tiles
    static constexpr uint32_t slots = HD == 128 ? 3 : 6;           // ring of f32 tiles, K and V in turn
    // A slot's fill is waited for by parity, so every warp has to see every phase of a barrier it
    // waits on. Where a slot is K's and V's in turn (an odd number of slots), whose warps are not
    // the same, each has a barrier of its own there: that of fill i is i % fills.
    static constexpr uint32_t fills = slots % 2 ? 2 * slots : slots;
    static constexpr uint32_t slot = kRowsKeys * HD * 4;
    static constexpr uint32_t half = kRowsKeys * HD * 2;           // hi or lo of an operand
    static constexpr uint32_t off_k = 0;
    static constexpr uint32_t off_v = off_k + stages * 2 * half;
    static constexpr uint32_t off_r = off_v + stages * 2 * half;
    static constexpr uint32_t off_x = off_r + slots * slot;         // [2][2][128] f32: the halves' maxima, by tile parity
    static constexpr uint32_t off_km = off_x + 4 * kRowsM * 4;      // [kRowsMeta][8] u32: a K unit's exponent and marks
    static constexpr uint32_t off_vm = off_km + kRowsMeta * 8 * 4;  // [2][8] u32: the same of V
    static constexpr uint32_t off_ke = off_vm + 2 * 8 * 4;          // [kRowsMeta][64] s8: the places' exponents of K
    static constexpr uint32_t off_ve = off_ke + kRowsMeta * kRowsKeys;  // [2][64] s8: of V
    static constexpr uint32_t off_rh = off_ve + 2 * kRowsKeys;      // [slots] u64: places whose page is bad
    static constexpr uint32_t off_bar = off_rh + 8 * slots;
    static constexpr uint32_t bytes = off_bar + 8 * (fills + slots + 12) + 48;
};
static_assert(RowsSmem<128>::bytes <= 227 * 1024 && RowsSmem<64>::bytes <= 227 * 1024, "shared memory");

template <int HD, bool EXACT>
__global__ void __launch_bounds__(kRowsThreads, 1) attn_rows_kernel(const RowsParams p)
{
    using S = RowsSmem<HD>;
    constexpr uint32_t NR = S::slots, NF = S::fills;
    extern __shared__ __align__(1024) uint8_t smem[];
    const b2_attn_rows_args &a = p.a;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t split = blockIdx.x, kvh = blockIdx.y / p.blocks, blk = blockIdx.y % p.blocks, item = blockIdx.z;
    const uint32_t hd = EXACT ? HD : a.head_dim;  // EXACT: head_dim == HD
    float *xmax = reinterpret_cast<float *>(smem + S::off_x);
    uint32_t *kmeta = reinterpret_cast<uint32_t *>(smem + S::off_km), *vmeta = reinterpret_cast<uint32_t *>(smem + S::off_vm);
    int8_t *kexp = reinterpret_cast<int8_t *>(smem + S::off_ke), *vexp = reinterpret_cast<int8_t *>(smem + S::off_ve);
    uint64_t *rhide = reinterpret_cast<uint64_t *>(smem + S::off_rh);
    // by parity of the tile: K and V converted, S and O computed (which frees that K and V)
    uint64_t *r_full = reinterpret_cast<uint64_t *>(smem + S::off_bar), *r_empty = r_full + NF, *k_full = r_empty + NR,
             *v_full = k_full + 2, *s_full = v_full + 2, *o_full = s_full + 2, *s_empty = o_full + 2, *p_full = s_empty + 1,
             *q_full = p_full + 1, *done = q_full + 1;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(done + 1), *met = tmem_slot + 2;  // [4][2]: the halves' meetings

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
    rows_range(p, places, split, t0, t1);
    if (t0 == t1) return;  // the joining kernel skips the same splits
    const uint32_t nt = t1 - t0;
    const uint32_t nsoft = 2 * ((live + 31) / 32);  // softmax warps with rows: two per quarter of the rows

    if (threadIdx.x == 0) {
        for (uint32_t i = 0; i < NF; ++i) mbar_init(&r_full[i], 1);
        for (uint32_t i = 0; i < NR; ++i) mbar_init(&r_empty[i], kRowsKeys / kRowsUnit);
        for (uint32_t i = 0; i < 2; ++i) {
            mbar_init(&k_full[i], kRowsKeys / kRowsUnit);
            mbar_init(&v_full[i], kRowsKeys / kRowsUnit);
            mbar_init(&s_full[i], 1);
            mbar_init(&o_full[i], 1);
        }
        mbar_init(s_empty, nsoft);
        mbar_init(p_full, nsoft);
        mbar_init(q_full, nsoft);
        mbar_init(done, 1);
        for (uint32_t i = 0; i < 8; ++i) met[i] = 0;
        fence_mbar_init();
    }
    if (warp == kRowsMmaWarp) tmem_alloc(tmem_slot, 512);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    // columns: S with K's hi 64, with its lo 64 | P hi 32, lo 32 | Q hi HD / 2, lo HD / 2 | O from 320
    const uint32_t tm_s = tmem, tm_p = tmem + 128, tm_q = tmem + 192, tm_o = tmem + 320;

    if (warp >= kRowsMmaWarp) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRowsLastRegs));
        if (warp == kRowsCopyWarp) {
            // ---- K and V tiles into the ring: lane l looks after places l and l + 32 ----
            const int32_t *table = a.kv.page_table + (size_t)item * a.kv.pages_per_seq;
            const uint32_t pt = a.kv.page_tokens, rowb = hd * sizeof(float);
            const uint64_t pol = l2_evict_first_policy();
            int fault = 0;
            auto page_of = [&](uint32_t t, uint32_t h) -> int32_t {
                const uint32_t at = (t0 + t) * kRowsKeys + lane + 32 * h;
                return t < nt && at < places ? table[at / pt] : 0;
            };
            int32_t page[2] = {page_of(0, 0), page_of(0, 1)};
            uint32_t filled = 0;
            bool ok = true;
            for (uint32_t j = 0; ok && j < nt; ++j) {
                size_t row[2];
                uint32_t run[2], bytes = 0, bad[2];
#pragma unroll
                for (uint32_t h = 0; h < 2; ++h) {
                    const uint32_t k = lane + 32 * h, at = (t0 + j) * kRowsKeys + k, off = at % pt;
                    const bool in = at < places;
                    const bool wrong = in && (page[h] < 0 || (a.pool_pages != 0 && (uint32_t)page[h] >= a.pool_pages));
                    bad[h] = __ballot_sync(0xffffffffu, wrong);
                    if (wrong) fault = B2_ERR_POSITION;
                    // a run: the tile's places on one page, copied by its first place's lane
                    const bool first = in && !wrong && (k == 0 || off == 0);
                    run[h] = first ? min(min(kRowsKeys - k, pt - off), places - at) : 0;
                    row[h] = (((size_t)(uint32_t)page[h] * a.n_kv_heads + kvh) * pt + off) * hd;
                    bytes += run[h] * rowb;
                    page[h] = page_of(j + 1, h);
                }
                bytes = __reduce_add_sync(0xffffffffu, bytes);
#pragma unroll
                for (uint32_t op = 0; op < 2 && ok; ++op) {
                    const uint32_t i = 2 * j + op, sl = i % NR;
                    if (i >= NR) ok = warp_wait(&r_empty[sl], i / NR - 1, a.err);
                    if (!ok) break;
                    uint64_t *full = &r_full[i % NF];
                    if (lane == 0) {
                        rhide[sl] = (uint64_t)bad[1] << 32 | bad[0];
                        mbar_arrive_expect_tx(full, bytes);
                    }
                    __syncwarp();
                    const float *pool = op == 0 ? a.kv.k_pool : a.kv.v_pool;
#pragma unroll
                    for (uint32_t h = 0; h < 2; ++h)
                        if (run[h] != 0)
                            bulk_g2s_stream(smem + S::off_r + sl * S::slot + (lane + 32 * h) * rowb, pool + row[h], run[h] * rowb,
                                            full, pol);
                    filled = i + 1;
                }
            }
            // no copy is in flight when the CTA ends, not even after a wait that gave up
            for (uint32_t i = filled > NR ? filled - NR : 0; i < filled; ++i) warp_wait(&r_full[i % NF], i / NF, a.err);
            if (fault) raise_error(a.err, fault);
        } else if (warp == kRowsMmaWarp) {
            // ---- MMA issue ----
            if (elect_one()) {
                const uint32_t id_s2 = umma_idesc_f16(kRowsM, 2 * kRowsKeys), id_s = umma_idesc_f16(kRowsM, kRowsKeys),
                           id_o = umma_idesc_f16(kRowsM, hd);
                const uint32_t kb = smem_u32(smem + S::off_k), vb = smem_u32(smem + S::off_v);
                // S of tile j + 1 before O of tile j: its operands are there first. (Polling for
                // whichever came first cost the scheduler's softmax warps more than it gained.)
                bool ok = mbar_wait_bounded(q_full, 0, a.err);
                for (uint32_t j = 0; ok && j <= nt; ++j) {
                    if (j < nt) {
                        ok = spin_wait(&k_full[j & 1], (j / 2) & 1, a.err) && (j == 0 || spin_wait(s_empty, (j - 1) & 1, a.err));
                        if (!ok) break;
                        tc_fence_after();
                        // 64 rows of hi, 64 of lo (a descriptor's address field counts 16 bytes)
                        uint64_t kd = umma_desc(kb + (j & 1) * 2 * S::half, 2 * kRowsKeys * 16, 128);
#pragma unroll 1
                        for (uint32_t kk = 0; kk < hd / 16; ++kk, kd += 4 * kRowsKeys) {
                            umma_16_ts(tm_s, tm_q + kk * 8, kd, id_s2, kk > 0);
                            umma_16_ts(tm_s, tm_q + HD / 2 + kk * 8, kd, id_s, 1);  // the hi rows
                        }
                        umma_commit(&s_full[j & 1]);
                    }
                    if (j > 0) {
                        // P of a tile is published after its V was converted and the O before it taken
                        const uint32_t i = j - 1, vt = vb + (i & 1) * 2 * S::half;
                        ok = spin_wait(p_full, i & 1, a.err);
                        if (!ok) break;
                        tc_fence_after();
                        uint64_t vh = umma_desc(vt, HD * 16, 128), vl = umma_desc(vt + S::half, HD * 16, 128);
#pragma unroll 1
                        for (uint32_t kk = 0; kk < kRowsKeys / 16; ++kk, vh += 2 * HD, vl += 2 * HD) {
                            umma_16_ts(tm_o, tm_p + kk * 8, vh, id_o, kk > 0);
                            umma_16_ts(tm_o, tm_p + 32 + kk * 8, vh, id_o, 1);
                            umma_16_ts(tm_o, tm_p + kk * 8, vl, id_o, 1);
                        }
                        umma_commit(&o_full[i & 1]);
                    }
                }
                // everything issued has completed before tensor memory is freed
                umma_commit(done);
                mbar_wait_bounded(done, 0, a.err);
            }
            __syncwarp();
        }
    } else if (warp >= (uint32_t)kRowsSoftWarps) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRowsConvRegs));
        // ---- ring tiles into operands ----
        // Every warp takes part in every tile's K, or in every tile's V, so (with r_full apart for
        // the two) none can be two phases of a barrier away from the others. K and V differ in
        // how a lane picks its values; the conversion of its HD / 32 chunks of eight (16 bytes of
        // hi, 16 of lo) is one piece of code for both: the roles of this kernel run different
        // code side by side, and instruction fetch is what they run out of first.
        const bool is_v = warp >= (uint32_t)kRowsSoftWarps + 4;
        for (uint32_t j = 0; j < nt; ++j) {
            const uint32_t i = 2 * j + is_v, sl = i % NR;
            const uint32_t st = j & 1;
            if (!warp_wait(&r_full[i % NF], i / NF, a.err)) break;
            if (j >= 2 && !warp_wait((is_v ? o_full : s_full) + st, j / 2 - 1, a.err)) break;
            const uint64_t hide = rhide[sl];
#pragma unroll 1
            for (uint32_t w = (warp & 3) * (kRowsUnit / 8), we = w + kRowsUnit / 8; w < we; ++w) {
                const uint32_t place = (t0 + j) * kRowsKeys + 8 * w;
                // places past the end (never copied) and on bad pages are zeros, hidden from every row
                const uint32_t hidden = (uint32_t)(hide >> (8 * w)) & 0xFFu;  // (the softmax knows the end itself)
                uint32_t none = hidden;
                if (place + 8 > places) none |= places <= place ? 0xFFu : (0xFFu << (places - place)) & 0xFFu;
                const uint32_t m = lay_unit<HD, EXACT>(reinterpret_cast<float *>(smem + S::off_r + sl * S::slot) + 8 * w * hd, hd, is_v, w, none, hidden,
                                                       smem + (is_v ? S::off_v : S::off_k) + st * 2 * S::half, kRowsKeys * 16,
                                                       is_v ? vexp + st * kRowsKeys : kexp + (j % kRowsMeta) * kRowsKeys);
                if (lane == 0) (is_v ? vmeta + st * 8 : kmeta + (j % kRowsMeta) * 8)[w] = m;
            }
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(&r_empty[sl]);
                mbar_arrive((is_v ? v_full : k_full) + st);
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRowsSoftRegs));
        const uint32_t qt = warp & 3, half = warp >> 2;
        if (qt < nsoft / 2) {
            // ---- softmax and the sums of O: row r, places 32 half .. + 31, dimensions of half ----
            const uint32_t r = qt * 32 + lane, m_row = blk * kRowsM + r;
            const bool mine = r < live;
            const uint32_t tok = mine ? m_row / p.group : 0, head = kvh * p.group + (mine ? m_row % p.group : 0);
            const uint32_t lanes = (qt * 32) << 16;
            float cq;  // score of a row: dot * K scale * cq, in powers of two
            bool far;  // the warp's rows
            {
                const float *src = a.q + (size_t)(r0 + tok) * a.q_stride + (size_t)head * hd;
                uint32_t top = 0;
                for (uint32_t d = 0; mine && d < hd; d += 4) {  // the row's largest magnitude
                    const float4 f = *reinterpret_cast<const float4 *>(src + d);
                    top = max(max(top, max(abs_bits(f.x), abs_bits(f.y))), max(abs_bits(f.z), abs_bits(f.w)));
                }
                const bool bad = top >= 0x7F800000u;
                const int e = bad ? 0 : top_exp(top);
                const float sc = pow2i(-e);
                cq = bad ? NAN : pow2i(e) * p.scale;
                far = rows_far(bad ? 0 : top, p.reach);
#pragma unroll
                for (uint32_t c = 0; c < HD / 2; c += 32) {  // 32 dimensions: 16 columns of hi, 16 of lo
                    uint32_t hi[16], lo[16];
#pragma unroll
                    for (uint32_t k = 0; k < 8; ++k) {
                        const uint32_t d = half * (HD / 2) + c + 4 * k;
                        float4 f = make_float4(0, 0, 0, 0);
                        if (mine && !bad && d < hd) f = *reinterpret_cast<const float4 *>(src + d);
                        split_f16(f.x * sc, f.y * sc, hi[2 * k], lo[2 * k]);
                        split_f16(f.z * sc, f.w * sc, hi[2 * k + 1], lo[2 * k + 1]);
                    }
                    tmem_st16(tm_q + lanes + half * (HD / 4) + c / 2, hi);
                    tmem_st16(tm_q + lanes + HD / 2 + half * (HD / 4) + c / 2, lo);
                }
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(q_full);
            }
            const uint64_t mask = mine && a.tree != nullptr ? a.tree[r0 + tok] : 0;
            float m = -INFINITY, l = 0.0f, corr_prev = 0.0f, osc_prev = 0.0f;
            uint64_t acc[HD / 4];  // pairs of the half's dimensions
#pragma unroll
            for (int i = 0; i < HD / 4; ++i) acc[i] = 0;
            // The two warps of a quarter meet at a named barrier once a tile, so neither may leave
            // the loop alone: after a wait that gave up both run on without waiting.
            bool ok = true;
            auto wait = [&](uint64_t *bar, uint32_t phase) { ok = ok && warp_wait(bar, phase, a.err); };
            auto meet = [&]() { asm volatile("bar.sync %0, 64;" ::"r"(1 + qt) : "memory"); };
            // Where only some tiles meet: want grows from meeting to meeting, and it ends by itself
            // even if one of the two never comes.
            auto meet_again = [&](uint32_t want) {
                volatile uint32_t *at = met + 2 * qt;
                __threadfence_block();
                __syncwarp();
                at[half] = want;
                for (uint32_t i = 0; ok && at[half ^ 1] < want; ++i) ok = i < (1u << 22);
                ok = __all_sync(0xffffffffu, ok);
                __threadfence_block();
            };
            // O of the tile before into the sums: acc = acc * corr + O * osc
            auto take_o = [&]() {
                const uint32_t col = tm_o + lanes + half * (HD / 2);
                if (!__all_sync(0xffffffffu, corr_prev == 1.0f || !mine)) {
                    const uint64_t c2 = pair(corr_prev, corr_prev);
#pragma unroll
                    for (int k = 0; k < HD / 4; ++k) acc[k] = mul2(acc[k], c2);
                }
                const uint64_t o2 = pair(osc_prev, osc_prev);
#pragma unroll
                for (int c = 0; c < HD / 2; c += 32) {
                    uint32_t v[32];
                    tmem_ld32(col + c, v);
                    tmem_wait_ld();
#pragma unroll
                    for (int k = 0; k < 16; ++k)
                        acc[c / 2 + k] = fma2(pair(__uint_as_float(v[2 * k]), __uint_as_float(v[2 * k + 1])), o2, acc[c / 2 + k]);
                }
            };
            auto visible = [&](uint32_t key0) { return rows_visible(a.tree != nullptr, mask, tok, ctx, places, key0); };
            // One tile. Units of K or V of different scale, marked places and scores that may pass
            // 2^23 are rare and cost the others next to nothing: they have a copy of the code of
            // their own (in one, the branches and what they keep in registers slowed every tile by
            // 5 to 9 percent).
            auto tile = [&](uint32_t j, auto rare, const uint4 &km, const uint4 &va, const uint4 &vb) {
                constexpr bool RARE = decltype(rare)::value;
                const uint32_t mt = j % kRowsMeta, vt = j & 1, key0 = (t0 + j) * kRowsKeys + half * 32;
                uint32_t raw[32], low[16];
                tmem_ld32(tm_s + lanes + half * 32, raw);
                tmem_ld16_nowait(tm_s + lanes + kRowsKeys + half * 32, low);
                float s[32];
                tmem_wait_ld();
                auto sum16 = [&](int k0) {
#pragma unroll
                    for (int k = 0; k < 16; k += 2)
                        unpair(add2(pair(__uint_as_float(raw[k0 + k]), __uint_as_float(raw[k0 + k + 1])),
                                    pair(__uint_as_float(low[k]), __uint_as_float(low[k + 1]))),
                               s[k0 + k], s[k0 + k + 1]);
                };
                sum16(0);
                tmem_ld16_nowait(tm_s + lanes + kRowsKeys + half * 32 + 16, low);
                tmem_wait_ld();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(s_empty);
                sum16(16);
                float cqk = score_factor(cq, meta_exp(km.x));
                uint32_t vis = key0 + 32 > ctx ? visible(key0) : 0xFFFFFFFFu;
                if (RARE) {
                    const uint32_t bad = meta_bytes(km, 0);
                    vis &= ~meta_bytes(km, 8);
#pragma unroll
                    for (int k = 0; k < 32; ++k) {
                        s[k] = place_score(s[k], cq, exp_of(kmeta + mt * 8, kexp + mt * kRowsKeys, half * 32 + k));
                        if (bad >> k & 1) s[k] = NAN;
                    }
                    cqk = 1.0f;
                }
                if (vis != 0xFFFFFFFFu) {
#pragma unroll
                    for (int k = 0; k < 32; ++k)
                        if (!(vis >> k & 1)) s[k] = -INFINITY;
                }
                float top = fmaxf(s[0], s[1]), top2 = fmaxf(s[2], s[3]);
#pragma unroll
                for (int k = 4; k < 32; k += 4) {
                    top = max3(top, s[k], s[k + 1]);
                    top2 = max3(top2, s[k + 2], s[k + 3]);
                }
                top = fmaxf(top, top2);
                // the row's maximum over both halves
                float *x = xmax + (j & 1) * 2 * kRowsM;
                x[half * kRowsM + r] = top * cqk;
                meet();
                // (kept while it grows by less than kRowsSlack, so that the sums are seldom rescaled)
                float m_new = fmaxf(top * cqk, x[(half ^ 1) * kRowsM + r]);
                m_new = m_new > m + kRowsSlack ? m_new : m;
                const float m_use = m_new == -INFINITY ? 0.0f : m_new;
                const float corr = ex2(m - m_use);
                m = m_new;
                const float shift = RARE ? kRowsP : kRowsP - m_use;
                if (RARE) {
#pragma unroll
                    for (int k = 0; k < 32; ++k) s[k] -= m_use;
                }
                const uint64_t cq2 = pair(cqk, cqk), sh2 = pair(shift, shift);
                uint64_t sum = 0;
#pragma unroll
                for (int k = 0; k < 32; k += 2) {
                    float y, z;
                    unpair(fma2(pair(s[k], s[k + 1]), cq2, sh2), y, z);
                    s[k] = ex2(y);
                    s[k + 1] = ex2(z);
                    sum = add2(sum, pair(s[k], s[k + 1]));
                }
                float sy, sz;
                unpair(sum, sy, sz);
                l = fmaf(l, corr, sy + sz);
                int emax = meta_exp(va.x);
                if (RARE && !(meta_plain(va) && meta_plain(vb) && va.x == vb.x)) {
                    // P takes V's scales relative to the row's own largest weighted place
                    const uint4 vh = half ? vb : va;
                    const uint32_t *mu = vmeta + vt * 8;
                    const int8_t *pe = vexp + vt * kRowsKeys;
                    emax = -100;
#pragma unroll
                    for (int k = 0; k < 32; ++k) emax = max(emax, weight_exp(s[k], exp_of(mu, pe, half * 32 + k)));
                    meet_again(2 * j + 1);  // both have read the maxima
                    x[half * kRowsM + r] = __int_as_float(emax);
                    meet_again(2 * j + 2);
                    emax = max(emax, __float_as_int(x[(half ^ 1) * kRowsM + r]));
#pragma unroll
                    for (int k = 0; k < 32; ++k) s[k] *= pow2c(exp_of(mu, pe, half * 32 + k) - emax);
                    if ((meta_bytes(vh, 0) & visible(key0)) != 0) l = NAN;
                }
                uint32_t hi[16], lo[16];
#pragma unroll
                for (int k = 0; k < 16; ++k) cut_f16(s[2 * k], s[2 * k + 1], hi[k], lo[k]);
                if (j > 0) wait(&o_full[(j - 1) & 1], (j - 1) / 2);  // P is free, and O of the tile before is there
                tc_fence_after();
                tmem_st16(tm_p + lanes + half * 16, hi);
                tmem_st16(tm_p + lanes + 32 + half * 16, lo);
                if (j > 0) take_o();
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(p_full);
                corr_prev = corr;
                osc_prev = pow2i(emax - (int)kRowsP);
            };
            for (uint32_t j = 0; j < nt; ++j) {
                wait(&s_full[j & 1], j / 2);
                wait(&v_full[j & 1], j / 2);
                tc_fence_after();
                const uint4 km = *reinterpret_cast<const uint4 *>(kmeta + (j % kRowsMeta) * 8 + half * 4),
                            va = *reinterpret_cast<const uint4 *>(vmeta + (j & 1) * 8), vb = *reinterpret_cast<const uint4 *>(vmeta + (j & 1) * 8 + 4);
                if (meta_plain(km) && km.x <= meta_of_exp(0) && !far && meta_plain(va) && meta_plain(vb) && va.x == vb.x) tile(j, std::false_type(), km, va, vb);
                else tile(j, std::true_type(), km, va, vb);
            }
            wait(&o_full[(nt - 1) & 1], (nt - 1) / 2);
            tc_fence_after();
            take_o();
            // the row's sum: both halves', in one order
            float *x = xmax + (nt & 1) * 2 * kRowsM;
            x[half * kRowsM + r] = l;
            meet();
            l = x[r] + x[kRowsM + r];
            auto acc4 = [&](int c) {
                float4 f;
                unpair(acc[c / 2], f.x, f.y);
                unpair(acc[c / 2 + 1], f.z, f.w);
                return f;
            };
            if (!ok && lane == 0) raise_error(a.err, B2_ERR_TIMEOUT);
            if (ok && mine) {
                // the weights carry 2^11, the sums of O do not
                const float lw = l * pow2i(-(int)kRowsP);
                if (p.splits > 1) {
                    float *dst = rows_part(p, item, kvh, blk, split) + (size_t)r * (hd + 4);
                    if (half == 0) *reinterpret_cast<float2 *>(dst) = make_float2(m, lw);
                    dst += 4;
#pragma unroll
                    for (int c = 0; c < HD / 2; c += 4)
                        if (half * (HD / 2) + c < hd)
                            *reinterpret_cast<float4 *>(dst + half * (HD / 2) + c) = acc4(c);
                } else {
                    const float inv = lw > 0.0f ? 1.0f / lw : lw == 0.0f ? 0.0f : lw;  // NaN stays
                    if (lw != lw && half == 0) raise_error(a.err, B2_ERR_NONFINITE);
                    float *dst = a.ctx + (size_t)(r0 + tok) * a.ctx_stride + (size_t)head * hd;
#pragma unroll
                    for (int c = 0; c < HD / 2; c += 4)
                        if (half * (HD / 2) + c < hd)
                            *reinterpret_cast<float4 *>(dst + half * (HD / 2) + c) =
                                make_float4(acc4(c).x * inv, acc4(c).y * inv, acc4(c).z * inv, acc4(c).w * inv);
                }
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == kRowsMmaWarp) {
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
    const uint32_t blk = m_row / p.block, r = m_row % p.block;
    const uint32_t places = rows_places(p, n, ctx, blk);
    const size_t stride = (size_t)p.block * (hd + 4);
    const float *base = rows_part(p, item, kvh, blk, 0) + (size_t)r * (hd + 4);
    // (with fewer units than splits the first ones have one each)
    const uint32_t splits = min(p.splits, (places + p.unit - 1) / p.unit);
    // the splits' statistics, one per lane and pass
    float ms[kRowsMaxSplits / 32], ls[kRowsMaxSplits / 32], top = -INFINITY;
#pragma unroll
    for (int i = 0; i < (int)kRowsMaxSplits / 32; ++i) {
        const uint32_t s = lane + 32 * i;
        const float2 x = s < splits ? *reinterpret_cast<const float2 *>(base + s * stride) : make_float2(-INFINITY, 0.0f);
        ms[i] = x.x;
        ls[i] = x.y;
        top = fmaxf(top, ms[i]);
    }
    top = warp_max(top);
    if (top == -INFINITY) top = 0.0f;
    float4 o = make_float4(0, 0, 0, 0);
    float l = 0.0f;
#pragma unroll
    for (int i = 0; i < (int)kRowsMaxSplits / 32; ++i) {
        const float f = ex2(ms[i] - top);
        const uint32_t n32 = splits > 32u * i ? min(splits - 32 * i, 32u) : 0;
#pragma unroll 4
        for (uint32_t s = 0; s < n32; ++s) {
            const float fs = __shfl_sync(0xffffffffu, f, s), lsum = __shfl_sync(0xffffffffu, ls[i], s);
            l = fmaf(lsum, fs, l);
            if (4 * lane < hd) {
                const float4 x = reinterpret_cast<const float4 *>(base + (32 * i + s) * stride + 4)[lane];
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
    if ((uint64_t)a->max_rows * (a->n_heads / a->n_kv_heads) > 0x7FFFFFFFull) return -1;
    if ((uint64_t)kv.page_tokens * kv.pages_per_seq > 0x7FFFFFFFull || a->max_ctx > kv.page_tokens * kv.pages_per_seq)
        return -1;
    return 0;
}

constexpr uint32_t kFewCtx = 2048;
constexpr uint32_t kLaidBlocks = 4;
constexpr size_t kLaidBytes = (size_t)512 << 20;

// Kernel, blocks and splits. Up to kFewRows rows of an (item, KV head) over up to kFewCtx
// places go to attn_few_kernel, which converts K and V in registers and multiplies with
// mma.sync: no tensor-memory set-up, no roles to synchronise, no 128-row products for a
// handful of rows, no second kernel. Against attn_rows_kernel, one token of the 8B shape
// (4 rows) at context 1000 9.8 us and 14.8, 1900 13.5 and 17.7, 4000 23.9 and 23.0; 8
// sequences of it 25.0 and 25.2, 40.9 and 39.0, 77.6 and 71.1. (A form for 32 rows took 8
// tokens at context 1000 in 15.7, where attn_rows_kernel takes 16.5, but 8 sequences of
// that in 35, against 28.)
//
// From kLaidBlocks blocks of 128 rows on, K and V are laid out as operands once for all of
// them (b2_attn_laid.cu). 2000 cached places, laid out and each block for itself: 8B shape,
// 8 sequences of 128 rows (4 blocks) 123 us and 143, 512 rows (16 blocks) 67 and 97; 8
// sequences of 64 (2 blocks) 79.1 and 80.7; 9 heads of 64, 8 sequences of 64 rows (2 blocks)
// 33.9 and 31.0. That takes scratch of the size of the batch's K and V, and is left out
// where it would be more than kLaidBytes.
//
// The splits take the least modelled time, in quarters of a tile's: what a CTA costs besides
// its tiles (launch, q, the pipeline's ends) and what joining costs, by a kernel also one
// per split. Measured (attn_rows_kernel): 8B shape, 8 tokens at context 1000 8 splits 16.5
// us, 16 splits 17.8, 4 18.6; one KV head of the 70B shape, 8 sequences to 30000 18 splits
// 78 us, 12 97, 24 91. Items of different lengths have the same number of splits: evener
// shares were worth little where a call is long enough for the power cap (8B shape, 16
// trees of 32, contexts 4000 to 8000: 1 to 4 splits 288 to 290 us, at 990 W and 1770 to
// 1687 MHz; 261 to 252 from rest).
static void attn_rows_plan(const b2_attn_rows_args *a, RowsParams &p, bool &few)
{
    p.group = a->n_heads / a->n_kv_heads;
    const uint64_t rows = (uint64_t)a->max_rows * p.group, sms = (uint64_t)sm_count();
    few = rows <= kFewRows && a->max_ctx <= kFewCtx;
    p.block = few ? kFewRows : kRowsM;
    p.blocks = (uint32_t)((rows + p.block - 1) / p.block);
    const uint64_t ctas = (uint64_t)a->batch * a->n_kv_heads * p.blocks, pairs = (a->max_ctx + kLaidKeys - 1) / kLaidKeys;
    const bool laid = !few && p.blocks >= kLaidBlocks && (uint64_t)a->batch * a->n_kv_heads * pairs <= kLaidBytes / attn_laid_pair(a->head_dim);
    p.pairs = laid ? (uint32_t)pairs : 0;
    p.unit = few ? kFewUnit : laid ? kLaidKeys : kRowsKeys;
    // a tile: 64 places of a tcgen05 CTA (128 laid out), or a pass of 16 places per warp
    const uint64_t tile = few ? kFewUnit * kFewWarps : p.unit, tiles = (a->max_ctx + tile - 1) / tile;
    const uint64_t setup = few ? 6 : 16, join = few ? 1 : 8;  // quarters of a tile
    uint64_t best = ~0ull;
    p.splits = 1;
    for (uint64_t s = 1; s <= (few ? kFewCluster : kRowsMaxSplits) && s <= tiles; s = few ? 2 * s : s + 1) {
        const uint64_t waves = (ctas * s + sms - 1) / sms;
        const uint64_t cost = waves * (4 * ((tiles + s - 1) / s) + setup) + (s == 1 ? 0 : few ? join : join + s);
        if (cost < best) {
            best = cost;
            p.splits = (uint32_t)s;
        }
    }
}

static size_t attn_rows_scratch(const b2_attn_rows_args *a, const RowsParams &p, bool few)
{
    const size_t laid = (size_t)a->batch * a->n_kv_heads * p.pairs * attn_laid_pair(a->head_dim);
    if (p.splits == 1 || few) return laid;
    return laid + (size_t)a->batch * a->n_kv_heads * p.blocks * p.splits * p.block * (a->head_dim + 4) * sizeof(float);
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
    RowsParams p = {};
    bool few;
    attn_rows_plan(a, p, few);
    return (uint64_t)a->n_kv_heads * p.blocks > 65535u ? 0 : attn_rows_scratch(a, p, few);
}

extern "C" int b2_attn_rows(const b2_attn_rows_args *a, void *stream)
{
    const int rc = attn_rows_check(a);
    if (rc != 0) return rc;
    RowsParams p = {};
    p.a = *a;
    bool few;
    attn_rows_plan(a, p, few);
    if ((uint64_t)a->n_kv_heads * p.blocks > 65535u) return -9;
    const size_t need = attn_rows_scratch(a, p, few);
    if (need > 0 && (a->scratch == nullptr || a->scratch_bytes < need || ((uintptr_t)a->scratch & 15))) return -1;
    p.laid = (uint8_t *)a->scratch;
    p.part = (float *)((uint8_t *)a->scratch + (size_t)a->batch * a->n_kv_heads * p.pairs * attn_laid_pair(a->head_dim));
    p.scale = (float)(1.4426950408889634 / sqrt((double)a->head_dim));
    p.reach = p.scale * (float)a->head_dim;
    const cudaStream_t st = (cudaStream_t)stream;
    if (few) {
        if (attn_few_launch(p, st) != cudaSuccess) return -8;
    } else if (p.pairs != 0) {
        if (attn_laid_launch(p, st) != cudaSuccess) return -8;
    } else {
        const bool wide = a->head_dim > 64;
        const void *fn = a->head_dim == 128  ? (const void *)attn_rows_kernel<128, true>
                         : wide              ? (const void *)attn_rows_kernel<128, false>
                         : a->head_dim == 64 ? (const void *)attn_rows_kernel<64, true>
                                             : (const void *)attn_rows_kernel<64, false>;
        const size_t smem = wide ? RowsSmem<128>::bytes : RowsSmem<64>::bytes;
        if (cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess) return -8;
        if (launch_rows_attn(fn, dim3(p.splits, a->n_kv_heads * p.blocks, a->batch), kRowsThreads, smem, a->pdl, st, p) != cudaSuccess)
            return -8;
    }
    if (p.splits > 1 && !few) {  // (launched early in any case: it waits for the kernel before)
        const uint32_t rows = a->max_rows * p.group;
        if (launch_rows_attn((const void *)attn_rows_join_kernel, dim3((rows + kJoinWarps - 1) / kJoinWarps, a->n_kv_heads, a->batch),
                             kJoinWarps * 32, 0, 1, st, p) != cudaSuccess)
            return -8;
    }
    return 0;
}
