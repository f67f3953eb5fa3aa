// b2_attn_few.cu - attention of a few new rows per sequence over the paged KV cache:
// b2_attn_rows for up to 16 rows (tokens x query heads of a KV head). Same arithmetic
// as b2_attn_rows.cu: every f32 operand as two f16 numbers of a power-of-two multiple,
// three products, f32 sums.
//
// With few rows the work is the stream of K and V, so the kernel is built around it:
// CTA (split, KV head, item) takes a contiguous range of the places, its eight warps
// 16 places each in turn. A warp owns a ring of shared-memory slots that it fills with
// cp.async (every lane copies its own pieces, of places on any page; a bulk copy per run
// of places would take the thread that issues it some 300 cycles each) and waits for
// nobody: it reads a slot straight into mma.sync fragments (m16n8k16), converting in
// registers, so K and V cross shared memory once and no warp synchronises with another
// before the end.
//   S = Q K^T: the fragment of Q comes from shared memory (prepared once); a lane's four
//   K values of a 16-dimension step are consecutive (both operands take the
//   dimensions of a step in the order 4 t, 4 t + 1 | 4 t + 2, 4 t + 3).
//   O = P V: P's fragment is S's accumulator; V's columns are dealt so that a lane reads
//   four consecutive dimensions of a place. Each product starts from zero and is added
//   to the f32 sums with the 16 places' scale, so no sum runs through more than three
//   MMAs of O, or 3 head_dim / 16 of S.
// A lane holds the softmax statistics of its rows; the warps' sums are joined in shared
// memory in warp order, then the splits' in split order: up to eight, a cluster whose CTAs
// read each other's shared memory.
#include "b2_attn_rows.cuh"

namespace b2 {

static_assert(kFewRows == 16, "one MMA tile of rows");

template <int HD>
struct FewSmem {
    static constexpr uint32_t slots = HD == 128 ? 3 : 6;          // per warp
    static constexpr uint32_t slot = kFewUnit * HD * 4;
    static constexpr uint32_t ring = slots * slot;
    static constexpr uint32_t q_step = 2 * 32 * 16;                // hi and lo fragments of 16 rows x 16 dimensions
    static constexpr uint32_t off_q = kFewWarps * ring;
    static constexpr uint32_t off_cq = off_q + (HD / 16) * q_step;  // [16] f32: a row's score factor
    static constexpr uint32_t off_qt = off_cq + kFewRows * 4;       // [16] u32: bits of its largest |q|
    static constexpr uint32_t off_mask = off_qt + kFewRows * 4;     // [16] u64
    static constexpr uint32_t off_hide = off_mask + kFewRows * 8;   // [warps][4] u32: places on bad pages
    static constexpr uint32_t bytes = off_hide + kFewWarps * 4 * 4;
    // the warps' sums at the end, in the drained ring: values, then (maximum, sum), the CTA's last
    static constexpr uint32_t off_o = 0, off_ml = kFewWarps * kFewRows * HD * 4;
    static_assert(off_ml + (kFewWarps + 1) * kFewRows * 8 <= off_q && bytes <= 227 * 1024, "shared memory");
};

__device__ __forceinline__ void mma_f16(float (&d)[4], const uint4 &a, uint32_t b0, uint32_t b1)
{
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}

// All threads of the cluster; what was written to shared memory before is seen after.
__device__ __forceinline__ void cluster_sync()
{
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Shared memory of CTA `rank` of the cluster, at the place of p in this one's.
__device__ __forceinline__ uint32_t cluster_addr(const void *p, uint32_t rank)
{
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_u32(p)), "r"(rank));
    return r;
}
__device__ __forceinline__ float2 cluster_ld2(const void *p, uint32_t rank)
{
    float2 v;
    asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(cluster_addr(p, rank)) : "memory");
    return v;
}
__device__ __forceinline__ float4 cluster_ld4(const void *p, uint32_t rank)
{
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(cluster_addr(p, rank)) : "memory");
    return v;
}

template <int HD>
__global__ void __launch_bounds__(kFewWarps * 32, 1) attn_few_kernel(const RowsParams p)
{
    using S = FewSmem<HD>;
    constexpr uint32_t NS = S::slots;
    constexpr int KS = HD / 16, QG = HD / 32;  // 16-dimension steps; groups of 32 dimensions
    extern __shared__ __align__(128) uint8_t smem[];
    const b2_attn_rows_args &a = p.a;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g8 = lane >> 2, t4 = lane & 3;
    const uint32_t split = blockIdx.x, kvh = blockIdx.y, item = blockIdx.z, hd = a.head_dim;
    uint8_t *ring = smem + warp * S::ring;
    float *cqs = reinterpret_cast<float *>(smem + S::off_cq);
    uint32_t *tops = reinterpret_cast<uint32_t *>(smem + S::off_qt);
    uint64_t *masks = reinterpret_cast<uint64_t *>(smem + S::off_mask);
    uint32_t *hides = reinterpret_cast<uint32_t *>(smem + S::off_hide) + warp * 4;
    pdl_wait();
    pdl_launch_dependents();
    uint32_t r0, n, ctx;
    if (!rows_item(a, item, r0, n, ctx)) {
        if (threadIdx.x == 0 && split == 0 && kvh == 0) raise_error(a.err, B2_ERR_POSITION);
        return;
    }
    const uint32_t rows = n * p.group;
    if (rows == 0) return;
    const uint32_t places = rows_places(p, n, ctx, 0);
    uint32_t t0, t1;
    rows_range(p, places, split, t0, t1);
    const uint32_t nc = t1 - t0 > warp ? (t1 - t0 - warp + kFewWarps - 1) / kFewWarps : 0;  // this warp's units

    // ---- the ring: unit c of this warp is K in fill 2 c, V in fill 2 c + 1 ----
    const int32_t *table = a.kv.page_table + (size_t)item * a.kv.pages_per_seq;
    const uint32_t pt = a.kv.page_tokens;
    int fault = 0;
    auto first_of = [&](uint32_t c) { return (t0 + warp + c * kFewWarps) * kFewUnit; };
    auto page_of = [&](uint32_t c) -> int32_t {  // lane: the page of place `lane` % 16 of unit c
        const uint32_t at = first_of(c) + (lane & 15);
        return c < nc && at < places ? table[at / pt] : 0;
    };
    uint32_t fills = 0;                       // fills asked for
    int32_t page = page_of(0), page1 = page_of(1);  // of the units of the next fills of K
    uint32_t row = 0, live = 0;               // of the unit being filled: pool row of a lane's place, places with one
    // One cp.async group per fill, empty past the last. Places without a row (past the
    // end, bad pages) are filled with zeros.
    auto fill = [&]() {
        const uint32_t c = fills / 2;
        if (c < nc) {
            if ((fills & 1) == 0) {
                const uint32_t at = first_of(c) + (lane & 15);
                const bool in = at < places, wrong = in && (page < 0 || (a.pool_pages != 0 && (uint32_t)page >= a.pool_pages));
                live = __ballot_sync(0xffffffffu, in && !wrong) & 0xFFFFu;
                const uint32_t hide = __ballot_sync(0xffffffffu, wrong) & 0xFFFFu;
                if (wrong) fault = B2_ERR_POSITION;
                if (lane == 0) hides[c & 3] = hide;
                row = in && !wrong ? ((uint32_t)page * a.n_kv_heads + kvh) * pt + at % pt : 0;
                page = page1;
                page1 = page_of(c + 2);
            }
            constexpr uint32_t C4 = HD / 4, PL = 32 / C4;  // 16-byte columns of a place, places of one instruction
            const uint32_t col = lane % C4;
            const float *pool = (fills & 1 ? a.kv.v_pool : a.kv.k_pool) + 4 * col;
            uint8_t *dst = ring + (fills % NS) * S::slot + (lane / C4) * hd * 4 + 16 * col;
#pragma unroll
            for (uint32_t i = 0; i < kFewUnit / PL; ++i) {
                const uint32_t pl = i * PL + lane / C4;
                const uint32_t r = __shfl_sync(0xffffffffu, row, pl);
                if (4 * col < hd) cp_async16(dst + i * PL * hd * 4, pool + (size_t)r * hd, live >> pl & 1 ? 16 : 0);
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
        ++fills;
    };
    auto landed = [&]() {  // the oldest of the NS latest fills
        asm volatile("cp.async.wait_group %0;" ::"n"(NS - 1) : "memory");
        __syncwarp();
    };
    for (uint32_t i = 0; i < NS; ++i) fill();

    // ---- Q: rows dealt to the warps, fragments of hi and lo, score factors, masks ----
    for (uint32_t r = warp; r < kFewRows; r += kFewWarps) {
        const bool mine = r < rows;
        const uint32_t tok = mine ? r / p.group : 0;
        float4 f = make_float4(0, 0, 0, 0);
        if (mine && 4 * lane < hd)
            f = reinterpret_cast<const float4 *>(a.q + (size_t)(r0 + tok) * a.q_stride + (size_t)(kvh * p.group + r % p.group) * hd)[lane];
        uint32_t top = max(max(abs_bits(f.x), abs_bits(f.y)), max(abs_bits(f.z), abs_bits(f.w)));
        top = __reduce_max_sync(0xffffffffu, top);
        const bool bad = top >= 0x7F800000u;
        const int e = bad ? 0 : top_exp(top);
        const float sc = bad ? 0.0f : pow2i(-e);
        if (bad) f = make_float4(0, 0, 0, 0);
        if (4 * lane < HD) {
            uint32_t h0, h1, l0, l1;
            split_f16(f.x * sc, f.y * sc, h0, l0);
            split_f16(f.z * sc, f.w * sc, h1, l1);
            // dimensions 16 ks + 4 t ..: registers (row half) and 2 + (row half) of lane 4 g + t
            uint32_t *dst = reinterpret_cast<uint32_t *>(smem + S::off_q + lane / 4 * S::q_step) +
                            ((r & 7) * 4 + (lane & 3)) * 4 + ((r >> 3) & 1);
            dst[0] = h0, dst[2] = h1;
            dst[32 * 4] = l0, dst[32 * 4 + 2] = l1;
        }
        if (lane == 0) {
            cqs[r] = bad ? NAN : pow2i(e) * p.scale;
            tops[r] = bad ? 0 : top;
            masks[r] = mine && a.tree != nullptr ? a.tree[r0 + tok] : 0;
        }
    }
    __syncthreads();

    // a lane's rows: g8 (i = 0) and g8 + 8
    float cq[2], m[2], l[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        cq[i] = cqs[g8 + i * 8];
        m[i] = -INFINITY;
        l[i] = 0.0f;
    }
    const bool far = rows_far(tops[lane % kFewRows], p.reach);
    float acc[4 * QG][4];  // column (q, i): dimensions 32 q + 4 col + i, col 2 t4 and 2 t4 + 1
#pragma unroll
    for (int k = 0; k < 4 * QG; ++k)
#pragma unroll
        for (int v = 0; v < 4; ++v) acc[k][v] = 0.0f;
    // places of the 16 from p0 that row r sees
    auto visible = [&](uint32_t r, uint32_t p0) -> uint32_t {
        uint32_t vis = 0xFFFFu;
        if (p0 + kFewUnit > ctx) {
            if (a.tree != nullptr) {
                const uint64_t mask = masks[r];
                if (p0 >= ctx) {
                    vis = p0 - ctx < 64 ? (uint32_t)(mask >> (p0 - ctx)) : 0;
                } else {
                    const uint32_t sh = ctx - p0;  // 1..15
                    vis = (uint32_t)(mask << sh) | ((1u << sh) - 1);
                }
            } else {
                const uint32_t seen = ctx + r / p.group + 1;
                vis = seen >= p0 + kFewUnit ? 0xFFFFu : seen <= p0 ? 0 : (1u << (seen - p0)) - 1;
            }
        }
        if (p0 + kFewUnit > places) vis &= (1u << (places - p0)) - 1;
        return vis & 0xFFFFu;
    };
    for (uint32_t c = 0; c < nc; ++c) {
        const uint32_t p0 = first_of(c), none0 = p0 + kFewUnit > places ? (0xFFFFu << (places - p0)) & 0xFFFFu : 0;
        // ---- S: 16 rows x 16 places (column tiles of 8) ----
        float s[2][4];
#pragma unroll
        for (int nt = 0; nt < 2; ++nt)
#pragma unroll
            for (int v = 0; v < 4; ++v) s[nt][v] = 0.0f;
        uint32_t sl = (2 * c) % NS;
        landed();
        const uint32_t hide = hides[c & 3], none = hide | none0;
        uint32_t kbad = 0;
        int ke, kpe = 0;  // exponent of K; if kwide, of place `lane`
        bool kwide = false;
        {
            float4 x[2][KS];  // the lane's K: place 8 nt + g8, dimensions 16 ks + 4 t4 ..
            float *rows0 = reinterpret_cast<float *>(ring + sl * S::slot);
            auto load = [&]() -> uint32_t {  // bits of the largest magnitude
                const float *src = rows0 + 4 * t4;
#pragma unroll
                for (int nt = 0; nt < 2; ++nt)
#pragma unroll
                    for (int ks = 0; ks < KS; ++ks)
                        x[nt][ks] = 16 * ks < (int)hd ? *reinterpret_cast<const float4 *>(src + (8 * nt + g8) * hd + 16 * ks) : make_float4(0, 0, 0, 0);
                float big = 0.0f;
#pragma unroll
                for (int nt = 0; nt < 2; ++nt)
#pragma unroll
                    for (int ks = 0; ks < KS; ++ks)
                        big = max3_nan(max3_nan(big, fabsf(x[nt][ks].x), fabsf(x[nt][ks].y)), fabsf(x[nt][ks].z), fabsf(x[nt][ks].w));
                return __reduce_max_sync(0xffffffffu, abs_bits(big));
            };
            uint32_t top = load();
            if (__builtin_expect(top >= kRowsWide, 0)) {
                kwide = settle_places(rows0, kFewUnit, hd, 0, kpe, kbad);
                top = load();
            }
            ke = top_exp(top);
            const float sc = pow2i(-ke);
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                uint32_t h[2][2], lo[2][2];
#pragma unroll
                for (int nt = 0; nt < 2; ++nt) {
                    float4 f = x[nt][ks];
                    if (ke != 0) f = make_float4(f.x * sc, f.y * sc, f.z * sc, f.w * sc);
                    split_f16(f.x, f.y, h[nt][0], lo[nt][0]);
                    split_f16(f.z, f.w, h[nt][1], lo[nt][1]);
                }
                const uint4 *qf = reinterpret_cast<const uint4 *>(smem + S::off_q + ks * S::q_step) + lane;
                const uint4 qh = qf[0], ql = qf[32];
#pragma unroll
                for (int nt = 0; nt < 2; ++nt) {
                    mma_f16(s[nt], qh, h[nt][0], h[nt][1]);
                    mma_f16(s[nt], ql, h[nt][0], h[nt][1]);
                    mma_f16(s[nt], qh, lo[nt][0], lo[nt][1]);
                }
            }
        }
        __syncwarp();
        fill();  // into the slot just read
        // ---- softmax: a lane holds columns 8 nt + 2 t4, + 1 of its rows ----
        const bool masked = p0 + kFewUnit > ctx || none != 0 || kbad != 0;
        const bool apart = kwide || ke > 0 || far;  // scores rounded before the maximum is subtracted
        if (__builtin_expect(apart, 0)) {
#pragma unroll
            for (int nt = 0; nt < 2; ++nt)
#pragma unroll
                for (int v = 0; v < 2; ++v) {
                    const int own = __shfl_sync(0xffffffffu, kpe, 8 * nt + 2 * t4 + v), e = kwide ? own : ke;
#pragma unroll
                    for (int i = 0; i < 2; ++i) s[nt][2 * i + v] = place_score(s[nt][2 * i + v], cq[i], e);
                }
        }
        float corr[2];
        bool rescale = false;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            float *s0 = &s[0][2 * i], *s1 = &s[1][2 * i];
            const float cqk = apart ? 1.0f : score_factor(cq[i], ke);
            if (masked) {
                const uint32_t vis = visible(g8 + i * 8, p0) & ~none;
#pragma unroll
                for (int v = 0; v < 2; ++v) {
                    if (kbad >> (2 * t4 + v) & 1) s0[v] = NAN;
                    if (kbad >> (8 + 2 * t4 + v) & 1) s1[v] = NAN;
                    if (!(vis >> (2 * t4 + v) & 1)) s0[v] = -INFINITY;
                    if (!(vis >> (8 + 2 * t4 + v) & 1)) s1[v] = -INFINITY;
                }
            }
            float top = fmaxf(max3(s0[0], s0[1], s1[0]), s1[1]) * cqk;
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            // kept while it grows by less than kRowsSlack, so that the sums are seldom rescaled
            const float m_new = top > m[i] + kRowsSlack ? top : m[i];
            const float m_use = m_new == -INFINITY ? 0.0f : m_new, shift = apart ? kRowsP : kRowsP - m_use;
            if (__builtin_expect(apart, 0)) s0[0] -= m_use, s0[1] -= m_use, s1[0] -= m_use, s1[1] -= m_use;
            corr[i] = ex2(m[i] - m_use);
            rescale |= m_new != m[i];
            m[i] = m_new;
            s0[0] = ex2(fmaf(s0[0], cqk, shift)), s0[1] = ex2(fmaf(s0[1], cqk, shift));
            s1[0] = ex2(fmaf(s1[0], cqk, shift)), s1[1] = ex2(fmaf(s1[1], cqk, shift));
            l[i] = fmaf(l[i], corr[i], (s0[0] + s0[1]) + (s1[0] + s1[1]));
        }
        if (__any_sync(0xffffffffu, rescale)) {
#pragma unroll
            for (int k = 0; k < 4 * QG; ++k)
#pragma unroll
                for (int v = 0; v < 4; ++v) acc[k][v] *= corr[v / 2];
        }
        uint4 ph, pl;  // P's fragments: rows g8, g8 + 8 of columns 2 t4, then of 8 + 2 t4
        auto split_p = [&]() {
            cut_f16(s[0][0], s[0][1], ph.x, pl.x);
            cut_f16(s[0][2], s[0][3], ph.y, pl.y);
            cut_f16(s[1][0], s[1][1], ph.z, pl.z);
            cut_f16(s[1][2], s[1][3], ph.w, pl.w);
        };
        split_p();
        // ---- O: the lane's V: places 2 t4, 2 t4 + 1, 8 + 2 t4, 9 + 2 t4, dimensions 32 q + 4 g8 .. ----
        sl = (2 * c + 1) % NS;
        landed();
        {
            float4 x[4][QG];
            float *rows0 = reinterpret_cast<float *>(ring + sl * S::slot);
            uint32_t vbad = 0;
            int vpe = 0;
            bool vwide = false;
            auto load = [&]() -> uint32_t {  // bits of the largest magnitude
                const float *src = rows0 + 4 * g8;
#pragma unroll
                for (int k = 0; k < 4; ++k)
#pragma unroll
                    for (int q = 0; q < QG; ++q)
                        x[k][q] = 32 * q + 4 * g8 < hd ? *reinterpret_cast<const float4 *>(src + (2 * t4 + (k & 1) + (k >> 1) * 8) * hd + 32 * q)
                                                       : make_float4(0, 0, 0, 0);
                float big = 0.0f;
#pragma unroll
                for (int k = 0; k < 4; ++k)
#pragma unroll
                    for (int q = 0; q < QG; ++q)
                        big = max3_nan(max3_nan(big, fabsf(x[k][q].x), fabsf(x[k][q].y)), fabsf(x[k][q].z), fabsf(x[k][q].w));
                return __reduce_max_sync(0xffffffffu, abs_bits(big));
            };
            uint32_t top = load();
            if (__builtin_expect(top >= kRowsWide, 0)) {
                vwide = settle_places(rows0, kFewUnit, hd, 0, vpe, vbad);
                top = load();
            }
            const int ve = top_exp(top);
            const float sc = pow2i(-ve);
            if (__builtin_expect(vbad != 0, 0)) {  // the rows that see a place with a NaN or infinity become NaN
#pragma unroll
                for (int i = 0; i < 2; ++i)
                    if ((vbad & ~none & visible(g8 + i * 8, p0)) != 0) l[i] = NAN;
            }
            auto values = [&](auto &&osc) {  // osc(i): what row i's products are added with
#pragma unroll
                for (int q = 0; q < QG; ++q) {
                    const float *f0 = reinterpret_cast<const float *>(&x[0][q]), *f1 = reinterpret_cast<const float *>(&x[1][q]),
                                *f2 = reinterpret_cast<const float *>(&x[2][q]), *f3 = reinterpret_cast<const float *>(&x[3][q]);
#pragma unroll
                    for (int v = 0; v < 4; ++v) {
                        float y[4] = {f0[v], f1[v], f2[v], f3[v]};
                        if (ve != 0) y[0] *= sc, y[1] *= sc, y[2] *= sc, y[3] *= sc;
                        uint32_t h0, h1, l0, l1;
                        split_f16(y[0], y[1], h0, l0);
                        split_f16(y[2], y[3], h1, l1);
                        float o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                        mma_f16(o, ph, h0, h1);
                        mma_f16(o, pl, h0, h1);
                        mma_f16(o, ph, l0, l1);
#pragma unroll
                        for (int k = 0; k < 4; ++k) acc[4 * q + v][k] = fmaf(o[k], osc(k / 2), acc[4 * q + v][k]);
                    }
                }
            };
            if (__builtin_expect(!vwide, 1)) {
                const float vsc = pow2i(ve - (int)kRowsP);
                values([=](int) { return vsc; });
            } else {  // P gets the places' scales relative to the row's largest weighted place
                float rsc[2];
                int pe[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) pe[k] = __shfl_sync(0xffffffffu, vpe, 2 * t4 + (k & 1) + (k >> 1) * 8);
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    int em = -100;
#pragma unroll
                    for (int k = 0; k < 4; ++k) em = max(em, weight_exp(s[k >> 1][2 * i + (k & 1)], pe[k]));
                    em = max(em, __shfl_xor_sync(0xffffffffu, em, 1));
                    em = max(em, __shfl_xor_sync(0xffffffffu, em, 2));
#pragma unroll
                    for (int k = 0; k < 4; ++k) s[k >> 1][2 * i + (k & 1)] *= pow2c(pe[k] - em);
                    rsc[i] = pow2i(em - (int)kRowsP);
                }
                split_p();
                values([&](int i) { return rsc[i]; });
            }
        }
        __syncwarp();
        fill();
    }
    if (fault) raise_error(a.err, fault);
    // ---- the warps' sums, joined in warp order, where the rings were ----
    __syncthreads();
    float *O = reinterpret_cast<float *>(smem + S::off_o) + (size_t)warp * kFewRows * HD;
    float2 *ML = reinterpret_cast<float2 *>(smem + S::off_ml);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
        l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
        const uint32_t r = g8 + i * 8;
        if (t4 == 0) ML[warp * kFewRows + r] = make_float2(m[i], l[i] * pow2i(-(int)kRowsP));
#pragma unroll
        for (int q = 0; q < QG; ++q)
#pragma unroll
            for (int col = 0; col < 2; ++col)
                *reinterpret_cast<float4 *>(O + r * HD + 32 * q + 4 * (2 * t4 + col)) =
                    make_float4(acc[4 * q][2 * i + col], acc[4 * q + 1][2 * i + col], acc[4 * q + 2][2 * i + col], acc[4 * q + 3][2 * i + col]);
    }
    __syncthreads();
    // A thread joins the warps' four dimensions of a row. In a cluster it leaves the result
    // in place of warp 0's (which no other thread reads), and the CTAs share out the rows.
    auto finish = [&](uint32_t r, uint32_t d, float L, const float4 &o) {
        const float inv = L > 0.0f ? 1.0f / L : L == 0.0f ? 0.0f : L;  // NaN stays
        if (L != L && d == 0) raise_error(a.err, B2_ERR_NONFINITE);
        *reinterpret_cast<float4 *>(a.ctx + (size_t)(r0 + r / p.group) * a.ctx_stride + (size_t)(kvh * p.group + r % p.group) * hd + d) =
            make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
    };
    float *O0 = reinterpret_cast<float *>(smem + S::off_o);
    for (uint32_t i = threadIdx.x; i < rows * (HD / 4); i += kFewWarps * 32) {
        const uint32_t r = i / (HD / 4), d = i % (HD / 4) * 4;
        if (d >= hd) continue;
        float M = -INFINITY;
#pragma unroll
        for (int w = 0; w < kFewWarps; ++w) M = fmaxf(M, ML[w * kFewRows + r].x);
        const float ref = M == -INFINITY ? 0.0f : M;
        float4 o = make_float4(0, 0, 0, 0);
        float L = 0.0f;
#pragma unroll
        for (int w = 0; w < kFewWarps; ++w) {
            const float2 ml = ML[w * kFewRows + r];
            const float f = ex2(ml.x - ref);
            const float4 x = *reinterpret_cast<const float4 *>(O0 + ((size_t)w * kFewRows + r) * HD + d);
            L = fmaf(ml.y, f, L);
            o = make_float4(fmaf(x.x, f, o.x), fmaf(x.y, f, o.y), fmaf(x.z, f, o.z), fmaf(x.w, f, o.w));
        }
        if (p.splits > 1) {
            *reinterpret_cast<float4 *>(O0 + (size_t)r * HD + d) = o;
            if (d == 0) ML[kFewWarps * kFewRows + r] = make_float2(M, L);
        } else {
            finish(r, d, L, o);
        }
    }
    if (p.splits == 1) return;
    cluster_sync();
    for (uint32_t i = split * kFewWarps * 32 + threadIdx.x; i < rows * (HD / 4); i += p.splits * kFewWarps * 32) {
        const uint32_t r = i / (HD / 4), d = i % (HD / 4) * 4;
        if (d >= hd) continue;
        float2 ml[kFewCluster];
        float4 x[kFewCluster];
        float M = -INFINITY;
#pragma unroll
        for (uint32_t s = 0; s < kFewCluster; ++s) {
            ml[s] = make_float2(-INFINITY, 0.0f);
            x[s] = make_float4(0, 0, 0, 0);
            if (s < p.splits) {
                ml[s] = cluster_ld2(&ML[kFewWarps * kFewRows + r], s);
                x[s] = cluster_ld4(O0 + (size_t)r * HD + d, s);
                M = fmaxf(M, ml[s].x);
            }
        }
        const float ref = M == -INFINITY ? 0.0f : M;
        float4 o = make_float4(0, 0, 0, 0);
        float L = 0.0f;
#pragma unroll
        for (uint32_t s = 0; s < kFewCluster; ++s) {
            const float f = ex2(ml[s].x - ref);
            L = fmaf(ml[s].y, f, L);
            o = make_float4(fmaf(x[s].x, f, o.x), fmaf(x[s].y, f, o.y), fmaf(x[s].z, f, o.z), fmaf(x[s].w, f, o.w));
        }
        finish(r, d, L, o);
    }
    cluster_sync();  // no CTA ends while another reads its sums
}

template <int HD>
static cudaError_t launch_few(const RowsParams &p, cudaStream_t st)
{
    const cudaError_t e = cudaFuncSetAttribute(attn_few_kernel<HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)FewSmem<HD>::bytes);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(p.splits, p.a.n_kv_heads, p.a.batch);
    cfg.blockDim = dim3(kFewWarps * 32);
    cfg.dynamicSmemBytes = FewSmem<HD>::bytes;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = p.a.pdl ? 1 : 0;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = p.splits;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = p.splits > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, attn_few_kernel<HD>, p);
}

cudaError_t attn_few_launch(const RowsParams &p, cudaStream_t st)
{
    return p.a.head_dim > 64 ? launch_few<128>(p, st) : launch_few<64>(p, st);
}

}  // namespace b2
