// b2_attn_rows.cuh - what the kernels of attention of several new rows per
// sequence share: the items' lengths and the split of their places, power-of-two
// scales, f16 pairs and packed f32 arithmetic.
#pragma once

#include "b2_common.cuh"

#include <cuda_fp16.h>

namespace b2 {

constexpr int kRowsTop = 0;             // operands are scaled to [2^kRowsTop, 2^(kRowsTop + 4))
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

__device__ __forceinline__ float pow2i(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }  // -126..127

// Exponent of the largest magnitude (its bits), down to a multiple of four and
// floored so that the scale 2^(kRowsTop - e) and its inverse stay normal.
__device__ __forceinline__ int top_exp(uint32_t amax_bits) { return max(((int)(amax_bits >> 23) - 127) & ~3, -100); }

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

// What the softmax needs to know of a unit: exponent, places hidden from every
// row, places with a NaN or infinity.
__device__ __forceinline__ uint32_t unit_meta(int e, uint32_t hidden, uint32_t bad) { return (uint32_t)(e + 128) << 16 | hidden << 8 | bad; }
__device__ __forceinline__ int meta_exp(uint32_t m) { return (int)(m >> 16) - 128; }
// byte i of the result: (m_i >> shift) & 0xFF
__device__ __forceinline__ uint32_t meta_bytes(const uint4 &m, uint32_t shift)
{
    return (m.x >> shift & 0xFF) | (m.y >> shift & 0xFF) << 8 | (m.z >> shift & 0xFF) << 16 | (m.w >> shift & 0xFF) << 24;
}
// Four units that share an exponent and have nothing marked.
__device__ __forceinline__ bool meta_plain(const uint4 &m) { return m.x == m.y && m.x == m.z && m.x == m.w && (m.x & 0xFFFF) == 0; }

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

__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7FFFFFFFu; }

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
