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
    int docs, rows_q, rows_k, kv_heads, group, tile_tokens, causal, pairs, splits;
    float scale, softcap;
    int *flag;
};

// A document's rows, and the first query tile a CTA works on there.
struct Item {
    int qs, lq, ks, lk, tile0, doc;
};

// Document i's rows [s, e) of an offsets array, kept inside [0, rows] whatever
// the array holds; an entry that descends or lies outside raises the flag.
__device__ __forceinline__ void doc_span(const int *off, int i, int rows, int *flag, int &s, int &e) {
    const int a = off[i], b = off[i + 1];
    if (a < 0 || b < a || b > rows) atomicExch(flag, kErrBadOffsets);
    s = min(max(a, 0), rows);
    e = min(max(b, s), rows);
}

// Keys that token `t` of the document sees: the first of them.
__device__ __forceinline__ int limit_of(const PackedParams &p, const Item &it, int t, int prefix) {
    if (!p.causal) return it.lk;
    const int64_t upto = (int64_t)t + it.lk - it.lq + 1;
    return max(prefix, (int)min((int64_t)it.lk, max((int64_t)0, upto)));
}

// How a raw score becomes one in the log2 domain when it is capped or biased.
struct ScoreMod {
    float scale, twice_over_cap, cap2;   // scale; 2 log2e / cap (0 = no cap); cap log2e
    float slope2, place;                 // slope log2e (0 = no bias), the row's key less the tile's first
    __device__ __forceinline__ float operator()(float s, int e) const {
        s *= scale;
        // tanh(u) = 1 - 2 / (2^(2u log2e) + 1): absolute error of some 1e-7, right at both ends
        s = twice_over_cap > 0.f ? cap2 * (1.f - __fdividef(2.f, ex2(s * twice_over_cap) + 1.f)) : s * kLog2e;
        return s - slope2 * fabsf(place - (float)e);
    }
};

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
