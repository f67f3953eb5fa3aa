// b2_attn_rows.cuh - what the kernels of attention of several new rows per
// sequence share: the items' lengths and the split of their places, power-of-two
// scales, f16 pairs and packed f32 arithmetic.
#pragma once

#include "b2_umma.cuh"

#include <cuda_fp16.h>

namespace b2 {

constexpr float kRowsP = 11.0f;         // P is scaled by 2^11,
constexpr float kRowsSlack = 4.0f;      // and may pass that by 2^4 (f16 ends at 2^16) before the maximum is raised
constexpr uint32_t kRowsMaxSplits = 64;

struct RowsParams {
    b2_attn_rows_args a;
    uint32_t group;           // query heads per KV head
    uint32_t block, unit;     // (token, query head) rows of a block; places of a unit of the split
    uint32_t blocks, splits;  // blocks per (item, KV head), splits of their places
    uint32_t pairs;           // K and V are laid out as operands first: pairs of tiles of an (item, KV head), else 0
    uint8_t *laid;            // [item][KV head][pair]
    float scale, reach;       // log2(e) / sqrt(head_dim), and head_dim times that
    float *part;              // splits to be joined by a kernel: [item][KV head][block][split][rows of a block][head_dim + 4]:
                              // maximum (log2), sum, -, -, weighted values
};

// The rows of an item, or false for lengths that do not fit.
__device__ __forceinline__ bool rows_fit(const b2_attn_rows_args &a, int32_t s, int32_t e, int32_t c, uint32_t &r0, uint32_t &n, uint32_t &ctx)
{
    if (s < 0 || e < s || (uint32_t)e > a.rows || (uint32_t)(e - s) > a.max_rows || c < 0 || (uint32_t)c > a.max_ctx ||
        (uint32_t)(e - s) > a.max_ctx - (uint32_t)c || (a.tree != nullptr && e - s > B2_MAX_TREE))
        return false;
    r0 = (uint32_t)s;
    n = (uint32_t)(e - s);
    ctx = (uint32_t)c;
    return true;
}
__device__ __forceinline__ bool rows_item(const b2_attn_rows_args &a, uint32_t item, uint32_t &r0, uint32_t &n, uint32_t &ctx)
{
    return rows_fit(a, a.row_start[item], a.row_start[item + 1], a.ctx_len[item], r0, n, ctx);
}

// Places a block of rows can see, and the units [t0, t1) of split s.
__device__ __forceinline__ uint32_t rows_places(const RowsParams &p, uint32_t n, uint32_t ctx, uint32_t blk)
{
    if (p.a.tree != nullptr) return ctx + n;
    return ctx + min(n, ((blk + 1) * p.block - 1) / p.group + 1);
}
__device__ __forceinline__ void rows_range(const RowsParams &p, uint32_t places, uint32_t s, uint32_t &t0, uint32_t &t1)
{
    const uint32_t nt = (places + p.unit - 1) / p.unit, per = nt / p.splits, more = nt - per * p.splits;
    t0 = s * per + min(s, more);
    t1 = t0 + per + (s < more);
}
// The rows of a partial result.
__device__ __forceinline__ float *rows_part(const RowsParams &p, uint32_t item, uint32_t kvh, uint32_t blk, uint32_t split)
{
    return p.part + ((((size_t)item * p.a.n_kv_heads + kvh) * p.blocks + blk) * p.splits + split) * p.block * (p.a.head_dim + 4);
}

__device__ __forceinline__ float ex2(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7FFFFFFFu; }

__device__ __forceinline__ float pow2i(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }  // -126..127

// The exponent e that operands of this largest magnitude (its bits) are scaled by, as
// x 2^-e: 0 from 2^-4 up to 2^12 and for zeros, else what brings it to [1, 16), floored so
// that 2^-e stays normal.
__device__ __forceinline__ int top_exp(uint32_t amax_bits)
{
    const int e = (int)(amax_bits >> 23) - 127;
    return (uint32_t)(e + 4) < 16u || amax_bits == 0 ? 0 : max(e & ~3, -100);
}
constexpr uint32_t kRowsWide = 139u << 23;  // bits of 2^12

// Two f32 in one register pair.
__device__ __forceinline__ uint64_t pair(float a, float b)
{
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void unpair(uint64_t v, float &a, float &b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c)
{
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b)
{
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b)
{
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

// f16 hi and lo words of two values.
__device__ __forceinline__ void split_f16(float a, float b, uint32_t &hi, uint32_t &lo)
{
    const __half2 h = __floats2half2_rn(a, b);
    const float2 f = __half22float2(h);
    float x, y;
    unpair(fma2(pair(f.x, f.y), pair(-1.0f, -1.0f), pair(a, b)), x, y);  // exact
    const __half2 l = __floats2half2_rn(x, y);
    hi = *reinterpret_cast<const uint32_t *>(&h);
    lo = *reinterpret_cast<const uint32_t *>(&l);
}

// The same with hi cut off instead of rounded (a mask instead of a conversion
// back): 21 bits together, for the weights, whose lo is then never negative.
__device__ __forceinline__ void cut_f16(float a, float b, uint32_t &hi, uint32_t &lo)
{
    const float ha = __uint_as_float(__float_as_uint(a) & 0xFFFFE000u), hb = __uint_as_float(__float_as_uint(b) & 0xFFFFE000u);
    float x, y;
    unpair(fma2(pair(ha, hb), pair(-1.0f, -1.0f), pair(a, b)), x, y);  // exact
    const __half2 h = __floats2half2_rn(ha, hb), l = __floats2half2_rn(x, y);
    hi = *reinterpret_cast<const uint32_t *>(&h);
    lo = *reinterpret_cast<const uint32_t *>(&l);
}

// What the softmax needs to know of a unit: exponent, whether its places have their
// own, places hidden from every row, places with a NaN or infinity.
__device__ __forceinline__ uint32_t unit_meta(int e, bool wide, uint32_t hidden, uint32_t bad)
{
    return (uint32_t)wide << 24 | (uint32_t)(e + 128) << 16 | hidden << 8 | bad;
}
__host__ __device__ constexpr uint32_t meta_of_exp(int e) { return (uint32_t)(e + 128) << 16; }  // nothing marked
__device__ __forceinline__ int meta_exp(uint32_t m) { return (int)(m >> 16 & 0xFF) - 128; }
// byte i of the result: (m_i >> shift) & 0xFF
__device__ __forceinline__ uint32_t meta_bytes(const uint4 &m, uint32_t shift)
{
    return (m.x >> shift & 0xFF) | (m.y >> shift & 0xFF) << 8 | (m.z >> shift & 0xFF) << 16 | (m.w >> shift & 0xFF) << 24;
}
// Four units that share an exponent and have nothing marked.
__device__ __forceinline__ bool meta_plain(const uint4 &m) { return m.x == m.y && m.x == m.z && m.x == m.w && (m.x & 0x100FFFF) == 0; }

// Places that share an exponent e lose what is below 2^-25 of the largest (of 1, if that
// is between 1 and 2^12). A larger place that few rows see, or that has next to no weight,
// must not take that from its neighbours: among places of 2^12 and more, each has its own
// exponent if one is kRowsSpread or more below another.
// rows: `places` rows of hd values in shared memory, all a warp's; bits of none: rows that
// are not there. Zeroes NaNs and infinities (bits of bad), and if it returns true has scaled
// row i by 2^-pe of lane i.
constexpr int kRowsSpread = 8;
__device__ __forceinline__ bool settle_places(float *rows, uint32_t places, uint32_t hd, uint32_t none, int &pe, uint32_t &bad)
{
    const uint32_t lane = threadIdx.x & 31;
    uint32_t mine = 0;
#pragma unroll 1
    for (uint32_t c = 0; c < places; ++c) {
        uint32_t top = 0;
        bool b = false;
#pragma unroll 1
        for (uint32_t d = none >> c & 1 ? hd : lane; d < hd; d += 32) {
            const uint32_t v = abs_bits(rows[c * hd + d]);
            if (v < 0x7F800000u) {
                top = max(top, v);
            } else {
                b = true;
                rows[c * hd + d] = 0.0f;
            }
        }
        top = __reduce_max_sync(0xffffffffu, top);
        if (__any_sync(0xffffffffu, b)) bad |= 1u << c;
        if (lane == c) mine = top;
    }
    const int e = top_exp(__reduce_max_sync(0xffffffffu, mine));
    pe = mine == 0 ? e : top_exp(mine);
    const bool wide = __any_sync(0xffffffffu, pe <= e - kRowsSpread) && e > 0;
#pragma unroll 1
    for (uint32_t c = 0; wide && c < places; ++c) {
        const float sc = pow2i(-__shfl_sync(0xffffffffu, pe, c));
#pragma unroll 1
        for (uint32_t d = none >> c & 1 ? hd : lane; d < hd; d += 32) rows[c * hd + d] *= sc;
    }
    __syncwarp();
    return wide;
}
// Exponent of a weighted place, p 2^e, with p (times 2^kRowsP) at most 1.
__device__ __forceinline__ int weight_exp(float p, int e) { return p > 0.0f ? e + ((int)(__float_as_uint(p) >> 23) - 127) - (int)kRowsP : -100; }
__device__ __forceinline__ float pow2c(int e) { return pow2i(min(max(e, -126), 127)); }


__device__ __forceinline__ float max3(float a, float b, float c)
{
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
// Largest of three, NaN if one is.
__device__ __forceinline__ float max3_nan(float a, float b, float c)
{
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// 16 bytes global to shared, or zeros (from 0).
__device__ __forceinline__ void cp_async16(void *dst, const void *src, uint32_t from)
{
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(from) : "memory");
}

// What a row's dot products are multiplied by: its own factor and K's scale, never 0
// (which would make a NaN of a hidden place's -infinity).
__device__ __forceinline__ float score_factor(float cq, int e)
{
    const float f = cq * pow2i(e);
    return f == 0.0f ? 1e-38f : f;
}

// Scores and their distance to the maximum come from one fused multiply-add, of which the
// maximum is a rounding: below 2^23 they differ by less than 1/2, and a weight does not pass
// f16's range. Beyond, scores are rounded first (place_score), and the maximum subtracted
// from that: for K of exponents above 0 (2^12 and more), and where a warp's rows are far,
// their largest |q_i| (its bits) times head_dim times 2^12, scaled like a score, at 2^23.
__device__ __forceinline__ bool rows_far(uint32_t top, float reach)
{
    return __uint_as_float(__reduce_max_sync(0xffffffffu, top)) * reach >= 2048.0f;
}
// The rounded score of a place of exponent e, in two steps of e: the row's factor and e may
// both be far from 1, and s * cq or cq * 2^e out of range where the score is not.
__device__ __forceinline__ float place_score(float s, float cq, int e) { return s * (cq * pow2i(e / 2)) * pow2i(e - e / 2); }

// All lanes wait; false for the whole warp if any gave up.
__device__ __forceinline__ bool warp_wait(uint64_t *bar, uint32_t phase, int32_t *err)
{
    return __all_sync(0xffffffffu, mbar_wait_bounded(bar, phase & 1u, err));
}

// ---- the tcgen05 kernels (b2_attn_rows.cu, b2_attn_laid.cu) -----------------------------

constexpr uint32_t kRowsM = 128;        // (token, query head) rows of a CTA
constexpr uint32_t kRowsKeys = 64;      // places of a tile
constexpr uint32_t kRowsUnit = 16;      // places a converting warp takes of a tile
constexpr uint32_t kLaidKeys = 128;     // places of a pair of tiles (b2_attn_laid.cu)

// Places of the 32 from key0 that a row sees: the first ctx, and of the item's own those
// in `mask` (tree) or up to its own.
__device__ __forceinline__ uint32_t rows_visible(bool tree, uint64_t mask, uint32_t tok, uint32_t ctx, uint32_t places, uint32_t key0)
{
    uint32_t vis = 0xFFFFFFFFu;
    if (key0 + 32 > ctx) {
        if (tree) {
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
    return vis;
}

// What the marks of a tile say: units of V that share an exponent and have nothing
// marked; the exponent of a place.
__device__ __forceinline__ bool units_plain(const uint32_t *m)
{
    const uint4 x = *reinterpret_cast<const uint4 *>(m), y = *reinterpret_cast<const uint4 *>(m + 4);
    return meta_plain(x) && meta_plain(y) && x.x == y.x;
}
__device__ __forceinline__ int exp_of(const uint32_t *unit, const int8_t *place, uint32_t k)
{
    return unit[k / 8] >> 24 ? (int)place[k] : meta_exp(unit[k / 8]);
}

// 32 lanes x 32 columns: thread i gets lane (base + i), columns col..col+31. The
// registers hold after tmem_wait_ld.
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&r)[32])
{
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
                 : "r"(taddr)
                 : "memory");
}
__device__ __forceinline__ void tmem_ld16_nowait(uint32_t taddr, uint32_t (&r)[16])
{
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16])
{
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

// mbar_wait_bounded of one thread without the suspension of mbar_try_wait.
__device__ __forceinline__ bool spin_wait(uint64_t *bar, uint32_t parity, int32_t *err)
{
    for (uint32_t i = 0; i < (1u << 26); ++i) {
        uint32_t ok;
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(ok)
            : "r"(smem_u32(bar)), "r"(parity)
            : "memory");
        if (ok) return true;
    }
    raise_error(err, B2_ERR_TIMEOUT);
    return false;
}

// Eight places (unit w of a tile) from f32 rows in shared memory into the tile's
// operand of K or V at `to`; one warp. Bits of none: places to take as zeros. Returns
// the unit's marks, and sets the places' exponents where it has its own. K's operand has
// 128 rows, lo k_lo bytes behind hi; V's HD, lo behind the tile's hi.
template <int HD, bool EXACT>
__device__ __forceinline__ uint32_t lay_unit(float *src, uint32_t hd, bool is_v, uint32_t w, uint32_t none, uint32_t hidden, uint8_t *to, uint32_t k_lo,
                                             int8_t *exps)
{
    constexpr int U = HD / 4;  // values a lane holds of eight places
    const uint32_t lane = threadIdx.x & 31, key = lane & 7, c0 = ((lane >> 3) + key) & 3, swap = key & 4;
    uint32_t bad = 0;
    float x[U];
    const uint32_t first = is_v ? lane : 8 * c0;  // dimension of the lane's first chunk (V: of its first column)
    bool wide = false;
    auto load = [&]() -> uint32_t {  // bits of the largest magnitude
        if (!is_v) {
            // the lane's key is `key`, its chunks of eight dimensions c0, c0 + 4, ..; the rotation by
            // the key and the swapped halves keep the reads of eight rows and the writes of one
            // 16-byte column each free of bank conflicts
            const float *from = src + key * hd + 8 * c0;
#pragma unroll
            for (int k = 0; k < HD / 32; ++k) {
                const float *at = EXACT || 32 * k + 8 * c0 < hd ? from + 32 * k : from - 8 * c0;
                const float4 f = *reinterpret_cast<const float4 *>(at + swap), g = *reinterpret_cast<const float4 *>(at + (swap ^ 4));
                x[8 * k] = swap ? g.x : f.x, x[8 * k + 1] = swap ? g.y : f.y, x[8 * k + 2] = swap ? g.z : f.z,
                x[8 * k + 3] = swap ? g.w : f.w, x[8 * k + 4] = swap ? f.x : g.x, x[8 * k + 5] = swap ? f.y : g.y,
                x[8 * k + 6] = swap ? f.z : g.z, x[8 * k + 7] = swap ? f.w : g.w;
            }
        } else {
            // dimensions lane + 32 k of the eight places
#pragma unroll
            for (int c = 0; c < 8; ++c)
#pragma unroll
                for (int k = 0; k < HD / 32; ++k)
                    x[8 * k + c] = src[c * hd + (EXACT || lane + 32 * k < hd ? lane + 32 * k : 0)];
        }
        if (none != 0) {
#pragma unroll
            for (int k = 0; k < U; ++k)
                if (none >> (is_v ? k & 7 : key) & 1) x[k] = 0.0f;
        }
        float big = 0.0f;
#pragma unroll
        for (int k = 0; k < U; k += 2) big = max3_nan(big, fabsf(x[k]), fabsf(x[k + 1]));
        return __reduce_max_sync(0xffffffffu, abs_bits(big));  // a NaN's bits are above infinity's
    };
    uint32_t top = load();
    if (__builtin_expect(top >= kRowsWide, 0)) {
        int pe;
        wide = settle_places(src, 8, hd, none, pe, bad);
        if (wide && lane < 8) exps[8 * w + lane] = (int8_t)pe;
        top = load();
    }
    const int e = top_exp(top);
    if (e != 0) {
        const float sc = pow2i(-e);
        const uint64_t sc2 = pair(sc, sc);
#pragma unroll
        for (int k = 0; k < U; k += 2) unpair(mul2(pair(x[k], x[k + 1]), sc2), x[k], x[k + 1]);
    }
    // element (key, d) of K: chunk d / 8 of 128 rows; (d, place) of V: chunk place / 8 of HD rows
    uint8_t *dst = to + (is_v ? w * (HD * 16) + lane * 16 : c0 * (2 * kRowsKeys * 16) + w * 128 + key * 16);
    const uint32_t step = is_v ? 32 * 16 : 4 * (2 * kRowsKeys * 16), to_lo = is_v ? kRowsKeys * HD * 2 : k_lo;
#pragma unroll
    for (uint32_t k = 0; k < HD / 32; ++k) {
        if (EXACT || first + 32 * k < hd) {
            uint4 h, l;
            split_f16(x[8 * k], x[8 * k + 1], h.x, l.x);
            split_f16(x[8 * k + 2], x[8 * k + 3], h.y, l.y);
            split_f16(x[8 * k + 4], x[8 * k + 5], h.z, l.z);
            split_f16(x[8 * k + 6], x[8 * k + 7], h.w, l.w);
            *reinterpret_cast<uint4 *>(dst + k * step) = h;
            *reinterpret_cast<uint4 *>(dst + k * step + to_lo) = l;
        }
    }
    return unit_meta(e, wide, hidden, bad);
}

// K and V laid out as operands first (b2_attn_laid.cu): bytes of a pair of tiles, and its launches.
size_t attn_laid_pair(uint32_t head_dim);
cudaError_t attn_laid_launch(const RowsParams &p, cudaStream_t st);

// ---- b2_attn_few.cu ----------------------------------------------------------------------

constexpr uint32_t kFewRows = 16;        // most rows of an (item, KV head)
constexpr uint32_t kFewUnit = 16;        // places a warp takes at a time
constexpr int kFewWarps = 8;
constexpr uint32_t kFewCluster = 8;      // most splits
cudaError_t attn_few_launch(const RowsParams &p, cudaStream_t st);

}  // namespace b2
