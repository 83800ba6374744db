// What the attention kernels over packed documents share.
#pragma once

#include <cuda.h>
#include <cuda_fp16.h>

#include "device_common.cuh"
#include "kernels.hpp"

namespace ltx {

constexpr int BQ = 128, BKV = 128;
constexpr float kRescaleLog2 = 8.0f;
constexpr float kLog2e = 1.4426950408889634f;

struct PackedParams {
    __nv_bfloat16 *out;
    int64_t ldo;
    const int *qo, *ko, *prefix;
    const float *slopes;
    int docs, rows_q, rows_k, kv_heads, group, tile_tokens, causal, pairs, splits, head_group, item_tiles;
    float scale, softcap;
    int *flag;
};

// A document's rows, the first query tile and the key head a CTA works on there;
// how many K and V tiles the CTA loaded before it.
struct Item {
    int qs, lq, ks, lk, tile0, doc, kvh;
    uint32_t load0;
};

// Document i's rows [s, e) of an offsets array, kept inside [0, rows] whatever
// the array holds; an entry that descends or lies outside raises the flag.
__device__ __forceinline__ void doc_span(const int *off, int i, int rows, int *flag, int &s, int &e) {
    const int a = off[i], b = off[i + 1];
    if (a < 0 || b < a || b > rows) report_index(flag, kErrBadOffsets);
    s = min(max(a, 0), rows);
    e = min(max(b, s), rows);
}

// Keys that token `t` of the document sees: the first of them.
__device__ __forceinline__ int limit_of(const PackedParams &p, const Item &it, int t, int prefix) {
    if (!p.causal) return it.lk;
    const int64_t upto = (int64_t)t + it.lk - it.lq + 1;
    return max(prefix, (int)min((int64_t)it.lk, max((int64_t)0, upto)));
}

// The key from which token `t`'s distances count.  A token that stands before the
// first key takes that one: all its distances are then less by the same number, which
// the softmax does not see and f32 scores would lose bits to.
__device__ __forceinline__ int key_beside(int lq, int lk, int t) { return max(t + lk - lq, 0); }

// 2^x on the FMA pipe, two at a time, as exp2_fma2 of attention.cu: x = n + f with
// n = rint(x), 2^f by a cubic (7.7e-5 relative, under f16's half step), 2^n added
// to the exponent; below 2^-120 it stays there.  Not for a NaN (whose exponent the
// addition would change): the caller's other values have to carry it.
__device__ __forceinline__ float2 exp2_poly2(float2 x) {
    constexpr float kRound = 12582912.0f;   // 1.5 * 2^23
    constexpr float c0 = 0x1.fff682p-1f, c1 = 0x1.62f1e0p-1f, c2 = 0x1.f0e03ap-3f, c3 = 0x1.c46242p-5f;
    x = make_float2(fmaxf(x.x, -120.f), fmaxf(x.y, -120.f));
    const float2 t = __fadd2_rn(x, make_float2(kRound, kRound));
    const float2 n = __fadd2_rn(t, make_float2(-kRound, -kRound));
    const float2 f = __ffma2_rn(n, make_float2(-1.f, -1.f), x);
    float2 q = __ffma2_rn(make_float2(c3, c3), f, make_float2(c2, c2));
    q = __ffma2_rn(q, f, make_float2(c1, c1));
    q = __ffma2_rn(q, f, make_float2(c0, c0));
    return make_float2(__uint_as_float(__float_as_uint(q.x) + (__float_as_uint(t.x) << 23)),
                       __uint_as_float(__float_as_uint(q.y) + (__float_as_uint(t.y) << 23)));
}

// tanh(u), two at a time: u q(u^2), q fitted here to the least absolute error of
// tanh: for |u| <= 1 of degree 5 (3.0e-7), for |u| <= 1/2 of degree 3 (1.5e-7).
__device__ __forceinline__ float2 tanh_poly2(float2 u) {
    constexpr float t0 = 0x1.ffff96p-1f, t1 = -0x1.553ce0p-2f, t2 = 0x1.0f6ea4p-3f, t3 = -0x1.a191d8p-5f,
                    t4 = 0x1.0803c6p-6f, t5 = -0x1.742ca4p-9f;
    const float2 z = __fmul2_rn(u, u);
    float2 q = __ffma2_rn(make_float2(t5, t5), z, make_float2(t4, t4));
    q = __ffma2_rn(q, z, make_float2(t3, t3));
    q = __ffma2_rn(q, z, make_float2(t2, t2));
    q = __ffma2_rn(q, z, make_float2(t1, t1));
    q = __ffma2_rn(q, z, make_float2(t0, t0));
    return __fmul2_rn(q, u);
}
__device__ __forceinline__ float2 tanh_small2(float2 u) {
    constexpr float h0 = 0x1.ffffb2p-1f, h1 = -0x1.55341ap-2f, h2 = 0x1.0d366cp-3f, h3 = -0x1.634eb0p-5f;
    const float2 z = __fmul2_rn(u, u);
    float2 q = __ffma2_rn(make_float2(h3, h3), z, make_float2(h2, h2));
    q = __ffma2_rn(q, z, make_float2(h1, h1));
    q = __ffma2_rn(q, z, make_float2(h0, h0));
    return __fmul2_rn(q, u);
}

// tanh(u) = 1 - 2 / (2^(2u log2e) + 1): right at both ends, absolute error at most 4e-7
__device__ __forceinline__ float tanh_exp(float u) { return 1.f - __fdividef(2.f, ex2(u * (2.f * kLog2e)) + 1.f); }
// With the polynomial where that would be many times a small u's last bits, which a
// large cap turns into a score's: relative error 3e-6 of any u.
__device__ __forceinline__ float2 tanh_any2(float2 u) {
    const float2 s = tanh_small2(u);
    return make_float2(fabsf(u.x) <= 0.5f ? s.x : tanh_exp(u.x), fabsf(u.y) <= 0.5f ? s.y : tanh_exp(u.y));
}

// How two raw scores of a key, of neighbouring rows, become scores in the log2
// domain when they are capped or biased.
struct ScoreMod {
    float2 scale;      // scale / cap, or scale log2e without a cap
    float cap2;        // cap log2e, 0 without
    __device__ __forceinline__ float2 operator()(float2 s, float2 slope2, float2 away) const {   // slope log2e, distance
        s = __fmul2_rn(s, scale);
        if (cap2 > 0.f) s = __fmul2_rn(tanh_any2(s), make_float2(cap2, cap2));
        return make_float2(s.x - slope2.x * fabsf(away.x), s.y - slope2.y * fabsf(away.y));
    }
};

// Two f32 to a pair of f16 or bf16, the first in the low half.
template <bool F16>
__device__ __forceinline__ uint32_t pack16(float2 v) {
    uint32_t r;
    if constexpr (F16) asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(v.y), "f"(v.x));
    else asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(v.y), "f"(v.x));
    return r;
}

__device__ __forceinline__ float2 unpack_bf16(uint32_t v) {
    return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
}

// attention_packed_few.cu: few query rows per document, as rows_per_doc counts
// them (heads of a group included).  Enqueues the attention and the join of
// what several CTAs share.
int attention_packed_few(ltx_ctx *ctx, const CUtensorMap &tk, const CUtensorMap &tv, const void *q, int64_t ldq,
                         const PackedParams &p, int heads, int head_dim, bool v_f16, int rows_per_doc);
constexpr int kMaxFewRows = 64;
// [rows, heads, D] of 16-bit values with row stride ld (elements), box {64, box_heads, box_rows}.
bool packed_map(CUtensorMap *m, const void *ptr, int64_t rows, int heads, int d, int64_t ld, bool f16, int box_heads,
                int box_rows);

}  // namespace ltx
