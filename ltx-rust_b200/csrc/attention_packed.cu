// Attention over packed documents: softmax over the keys of the row's own
// document only, with optional causal and prefix masks, scores capped by a
// tanh, and a bias that falls with distance.
//
// The simplest form: one warp per (query row, head) walks its visible keys
// once with the running maximum and sum of the softmax.
#include <cuda_fp16.h>

#include <cmath>

#include "device_common.cuh"
#include "internal.hpp"
#include "kernels.hpp"

namespace ltx {

namespace {

struct PackedParams {
    const __nv_bfloat16 *q, *k;
    const void *v;
    __nv_bfloat16 *out;
    int64_t ldq, ldk, ldv, ldo;
    const int *qo, *ko, *prefix;
    const float *slopes;
    int docs, rows_q, rows_k, heads, kv_heads, causal, v_f16;
    float scale, softcap;
    int *flag;
};

// Document i's rows [s, e) of an offsets array, kept inside [0, rows] whatever
// the array holds; an entry that descends or lies outside raises the flag.
__device__ __forceinline__ void doc_span(const int *off, int i, int rows, int *flag, int &s, int &e) {
    const int a = off[i], b = off[i + 1];
    if (a < 0 || b < a || b > rows) atomicExch(flag, kErrBadOffsets);
    s = min(max(a, 0), rows);
    e = min(max(b, s), rows);
}

template <int D>
__global__ void __launch_bounds__(256) packed_rows_kernel(PackedParams p) {
    const int lane = threadIdx.x & 31;
    const int64_t item = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) >> 5;
    if (item >= (int64_t)p.rows_q * p.heads) return;
    const int row = (int)(item / p.heads), h = (int)(item % p.heads), kv = h / (p.heads / p.kv_heads);
    int qs = 0, qe = 0, doc = 0;
    for (; doc < p.docs; ++doc) {
        doc_span(p.qo, doc, p.rows_q, p.flag, qs, qe);
        if (row >= qs && row < qe) break;
    }
    if (doc == p.docs) return;   // in no document: the row of out stays as it was
    int ks, ke;
    doc_span(p.ko, doc, p.rows_k, p.flag, ks, ke);
    const int lk = ke - ks, place = (row - qs) + lk - (qe - qs);
    int lim = lk;
    if (p.causal) {
        lim = min(lk, max(0, place + 1));
        if (p.prefix) lim = max(lim, min(max(p.prefix[doc], 0), lk));
    }
    constexpr int V = D / 32;
    float qv[V], acc[V];
    for (int i = 0; i < V; ++i) {
        qv[i] = __bfloat162float(p.q[(int64_t)row * p.ldq + h * D + i * 32 + lane]);
        acc[i] = 0.f;
    }
    float m = -INFINITY, l = 0.f;
    for (int j = 0; j < lim; ++j) {
        const int64_t kr = (int64_t)(ks + j);
        float s = 0.f;
        for (int i = 0; i < V; ++i) s += qv[i] * __bfloat162float(p.k[kr * p.ldk + kv * D + i * 32 + lane]);
#pragma unroll
        for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        s *= p.scale;
        if (p.softcap > 0.f) s = p.softcap * tanhf(s / p.softcap);
        if (p.slopes) s -= p.slopes[h] * fabsf((float)(place - j));
        const float mn = fmaxf(m, s), a = __expf(m - mn), w = __expf(s - mn);
        l = l * a + w;
        for (int i = 0; i < V; ++i) {
            const int64_t at = kr * p.ldv + kv * D + i * 32 + lane;
            const float vv = p.v_f16 ? __half2float(static_cast<const __half *>(p.v)[at])
                                     : __bfloat162float(static_cast<const __nv_bfloat16 *>(p.v)[at]);
            acc[i] = acc[i] * a + w * vv;
        }
        m = mn;
    }
    for (int i = 0; i < V; ++i)
        p.out[(int64_t)row * p.ldo + h * D + i * 32 + lane] = __float2bfloat16_rn(lim > 0 ? acc[i] / l : 0.f);
}

}  // namespace

}  // namespace ltx

extern "C" int ltx_attention_packed_fwd(ltx_ctx *ctx, const void *q_dev, int64_t ldq, const void *k_dev, int64_t ldk,
                                        const void *v_dev, int64_t ldv, int32_t v_dtype, const int32_t *q_offsets_dev,
                                        const int32_t *k_offsets_dev, int32_t docs, int32_t rows_q, int32_t rows_k,
                                        int32_t heads, int32_t kv_heads, int32_t head_dim, float scale, float softcap,
                                        const float *slopes_dev, int32_t causal, const int32_t *prefix_dev,
                                        void *out_dev, int64_t ldo) {
    using namespace ltx;
    if (!ctx) return LTX_ERR_INVALID_ARG;
    const char *w = "attention_packed";
    if (v_dtype != LTX_BF16 && v_dtype != LTX_F16) return fail(ctx, LTX_ERR_DTYPE, "%s: V must be BF16 or F16", w);
    if (head_dim != 64 && head_dim != 128)
        return fail(ctx, LTX_ERR_UNSUPPORTED, "%s: head_dim %d (64 or 128)", w, head_dim);
    if (docs < 0 || rows_q < 0 || rows_k < 0 || heads < 1 || kv_heads < 1 || heads % kv_heads)
        return fail(ctx, LTX_ERR_SHAPE, "%s: %d documents, %d x %d rows, %d heads over %d key heads", w, docs, rows_q,
                    rows_k, heads, kv_heads);
    if (heads / kv_heads > 128) return fail(ctx, LTX_ERR_UNSUPPORTED, "%s: more than 128 heads per key head", w);
    if (!(scale > 0.f) || !std::isfinite(scale) || !(softcap >= 0.f) || !std::isfinite(softcap))
        return fail(ctx, LTX_ERR_INVALID_ARG, "%s: scale must be finite and > 0, softcap finite and >= 0", w);
    if (prefix_dev && !causal) return fail(ctx, LTX_ERR_INVALID_ARG, "%s: a prefix needs the causal mask", w);
    if (docs == 0 || rows_q == 0) return LTX_OK;
    if (!q_dev || !out_dev || !q_offsets_dev || !k_offsets_dev || (rows_k && (!k_dev || !v_dev)))
        return fail(ctx, LTX_ERR_INVALID_ARG, "%s: null pointer", w);
    const int64_t qc = (int64_t)heads * head_dim, kc = (int64_t)kv_heads * head_dim;
    if (ldq % 8 || ldk % 8 || ldv % 8 || ldo % 8 || ldq < qc || ldo < qc || ldk < kc || ldv < kc ||
        (((uintptr_t)q_dev | (uintptr_t)k_dev | (uintptr_t)v_dev | (uintptr_t)out_dev) & 15))
        return fail(ctx, LTX_ERR_SHAPE, "%s: rows must be 16-byte aligned and as long as the heads", w);
    DeviceGuard guard(ctx);
    PackedParams p{static_cast<const __nv_bfloat16 *>(q_dev), static_cast<const __nv_bfloat16 *>(k_dev), v_dev,
                   static_cast<__nv_bfloat16 *>(out_dev), ldq, ldk, ldv, ldo, q_offsets_dev, k_offsets_dev, prefix_dev,
                   slopes_dev, docs, rows_q, rows_k, heads, kv_heads, causal, v_dtype == LTX_F16, scale, softcap,
                   ctx->timeout_flag};
    const unsigned grid = (unsigned)(((int64_t)rows_q * heads + 7) / 8);
    if (head_dim == 64) packed_rows_kernel<64><<<grid, 256, 0, ctx->stream>>>(p);
    else packed_rows_kernel<128><<<grid, 256, 0, ctx->stream>>>(p);
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? LTX_OK : cuda_fail(ctx, e, w);
}
