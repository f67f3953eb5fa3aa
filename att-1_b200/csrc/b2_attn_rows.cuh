// b2_attn_rows.cuh - what the kernels of attention of several new rows per
// sequence share: the items' lengths and the split of their places, power-of-two
// scales, f16 pairs and packed f32 arithmetic.
#pragma once

#include "b2_common.cuh"

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
    uint32_t cluster;         // the splits are a cluster that joins them itself
    float scale;              // log2(e) / sqrt(head_dim)
    float *part;              // splits > 1: [item][KV head][block][split][rows of a block][head_dim + 4]:
                              // maximum (log2), sum, -, -, weighted values
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

// All lanes wait; false for the whole warp if any gave up.
__device__ __forceinline__ bool warp_wait(uint64_t *bar, uint32_t phase, int32_t *err)
{
    return __all_sync(0xffffffffu, mbar_wait_bounded(bar, phase & 1u, err));
}

// The kernel for few rows (b2_attn_few.cu): p.block (16 or 32), p.unit and the splits
// as planned.
constexpr uint32_t kFewRows = 32;        // most rows of an (item, KV head) it takes
constexpr uint32_t kFewUnit = 16;        // places a warp takes at a time
constexpr int kFewWarps = 8;
constexpr uint32_t kFewCluster = 8;      // most splits of a cluster
cudaError_t attn_few_launch(const RowsParams &p, cudaStream_t st);

}  // namespace b2
