// Projection with one low-rank adapter per row:
//   out[m] = epilogue(x[m] W^T + c_a (x[m] A_a^T) B_a^T),  a = idx[m].
//
// The simplest form: one kernel for the low-rank products low[m] = c_a x[m]
// A_a^T in f32 (a warp per value), one tiled f32 kernel for everything else.
#include <cmath>

#include "device_common.cuh"
#include "internal.hpp"
#include "kernels.hpp"

namespace ltx {

namespace {

struct AdapterParams {
    const __nv_bfloat16 *x, *w, *a, *b;
    int64_t ldx, ldw, ldo, ld_gate;
    int m, n, k, rank, adapters, epilogue;
    const int *idx, *gate_idx;
    const float *coeff, *bias, *gate;
    float *low;   // [m, rank]
    void *out;
    int *flag;
};

// The adapter of row m, -1 for none; an index beyond the pool counts as none
// and raises the flag.
__device__ __forceinline__ int adapter_of(const AdapterParams &p, int m) {
    const int a = p.idx[m];
    if (a >= p.adapters) {
        atomicExch(p.flag, kErrBadAdapter);
        return -1;
    }
    return a < 0 ? -1 : a;
}

__global__ void low_kernel(AdapterParams p) {
    const int lane = threadIdx.x & 31;
    const int64_t item = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) >> 5;
    if (item >= (int64_t)p.m * p.rank) return;
    const int m = (int)(item / p.rank), r = (int)(item % p.rank), a = adapter_of(p, m);
    float s = 0.f;
    if (a >= 0) {
        const __nv_bfloat16 *ar = p.a + ((int64_t)a * p.rank + r) * p.k, *xr = p.x + m * p.ldx;
        for (int e = lane; e < p.k; e += 32) s += __bfloat162float(ar[e]) * __bfloat162float(xr[e]);
#pragma unroll
        for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        s *= p.coeff[a];
    }
    if (lane == 0) p.low[item] = s;
}

__global__ void __launch_bounds__(256) adapter_tile_kernel(AdapterParams p) {
    __shared__ float xs[64][33], ws[64][33];
    const int m0 = blockIdx.y * 64, n0 = blockIdx.x * 64, tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    float acc[4][4] = {};
    for (int k0 = 0; k0 < p.k; k0 += 32) {
        __syncthreads();
        for (int e = threadIdx.x; e < 64 * 32; e += 256) {
            const int r = e >> 5, c = e & 31;
            xs[r][c] = m0 + r < p.m && k0 + c < p.k ? __bfloat162float(p.x[(int64_t)(m0 + r) * p.ldx + k0 + c]) : 0.f;
            ws[r][c] = n0 + r < p.n && k0 + c < p.k ? __bfloat162float(p.w[(int64_t)(n0 + r) * p.ldw + k0 + c]) : 0.f;
        }
        __syncthreads();
        for (int c = 0; c < 32; ++c)
            for (int i = 0; i < 4; ++i)
                for (int j = 0; j < 4; ++j) acc[i][j] += xs[ty * 4 + i][c] * ws[tx + 16 * j][c];
    }
    for (int i = 0; i < 4; ++i) {
        const int m = m0 + ty * 4 + i;
        if (m >= p.m) continue;
        const int a = adapter_of(p, m);
        for (int j = 0; j < 4; ++j) {
            const int n = n0 + tx + 16 * j;
            if (n >= p.n) continue;
            float y = acc[i][j];
            if (a >= 0)
                for (int r = 0; r < p.rank; ++r)
                    y += p.low[(int64_t)m * p.rank + r] * __bfloat162float(p.b[((int64_t)a * p.n + n) * p.rank + r]);
            if (p.bias) y += p.bias[n];
            if (p.epilogue == LTX_EPI_GELU_BF16)
                y = 0.5f * y * (1.f + tanhf(0.7978845608028654f * (y + 0.044715f * y * y * y)));
            const int64_t at = (int64_t)m * p.ldo + n;
            if (p.epilogue == LTX_EPI_F32) static_cast<float *>(p.out)[at] = y;
            else if (p.epilogue == LTX_EPI_RESID)
                static_cast<float *>(p.out)[at] +=
                    p.gate ? y * p.gate[(int64_t)(p.gate_idx ? p.gate_idx[m] : 0) * p.ld_gate + n] : y;
            else static_cast<__nv_bfloat16 *>(p.out)[at] = __float2bfloat16_rn(y);
        }
    }
}

}  // namespace

}  // namespace ltx

extern "C" int ltx_gemm_adapters(ltx_ctx *ctx, const void *x_dev, int64_t ldx, const void *w_dev, int64_t ldw, int32_t m,
                                 int32_t n, int32_t k, int32_t epilogue, const float *bias_dev, void *out_dev,
                                 int64_t ldo, const float *gate_dev, const int32_t *gate_idx_dev, int64_t ld_gate,
                                 const int32_t *adapter_idx_dev, const void *lora_a_dev, const void *lora_b_dev,
                                 const float *coeff_dev, int32_t adapters, int32_t rank) {
    using namespace ltx;
    if (!ctx) return LTX_ERR_INVALID_ARG;
    const char *w = "gemm_adapters";
    if (epilogue < LTX_EPI_BF16 || epilogue > LTX_EPI_RESID)
        return fail(ctx, LTX_ERR_INVALID_ARG, "%s: bad epilogue %d", w, epilogue);
    if (m < 0 || n < 1 || k < 1) return fail(ctx, LTX_ERR_SHAPE, "%s: %d x %d x %d", w, m, n, k);
    if (adapters < 0 || adapters > LTX_MAX_ADAPTERS || rank < 8 || rank > LTX_MAX_ADAPTER_RANK || rank % 8)
        return fail(ctx, LTX_ERR_UNSUPPORTED, "%s: %d adapters of rank %d (at most %d, rank a multiple of 8 up to %d)", w,
                    adapters, rank, LTX_MAX_ADAPTERS, LTX_MAX_ADAPTER_RANK);
    if (m == 0) return LTX_OK;
    if (!x_dev || !w_dev || !out_dev || !adapter_idx_dev || (adapters && (!lora_a_dev || !lora_b_dev || !coeff_dev)))
        return fail(ctx, LTX_ERR_INVALID_ARG, "%s: null pointer", w);
    if (k % 8 || ldx % 8 || ldw % 8 || ldx < k || ldw < k || ldo < n ||
        (((uintptr_t)x_dev | (uintptr_t)w_dev | (uintptr_t)lora_a_dev | (uintptr_t)lora_b_dev) & 15))
        return fail(ctx, LTX_ERR_SHAPE, "%s: operand rows must be 16-byte aligned (k %d, ldx %lld, ldw %lld)", w, k,
                    (long long)ldx, (long long)ldw);
    if (epilogue == LTX_EPI_RESID && gate_dev && ld_gate < n)
        return fail(ctx, LTX_ERR_SHAPE, "%s: gate rows shorter than n", w);
    DeviceGuard guard(ctx);
    void *low = nullptr;
    int rc = work_alloc(ctx, (size_t)m * rank * sizeof(float), &low);
    if (rc != LTX_OK) return rc;
    AdapterParams p{static_cast<const __nv_bfloat16 *>(x_dev), static_cast<const __nv_bfloat16 *>(w_dev),
                    static_cast<const __nv_bfloat16 *>(lora_a_dev), static_cast<const __nv_bfloat16 *>(lora_b_dev), ldx,
                    ldw, ldo, ld_gate, m, n, k, rank, adapters, epilogue, adapter_idx_dev, gate_idx_dev, coeff_dev,
                    bias_dev, gate_dev, static_cast<float *>(low), out_dev, ctx->timeout_flag};
    low_kernel<<<(unsigned)(((int64_t)m * rank + 7) / 8), 256, 0, ctx->stream>>>(p);
    adapter_tile_kernel<<<dim3((n + 63) / 64, (m + 63) / 64), 256, 0, ctx->stream>>>(p);
    const cudaError_t e = cudaGetLastError();
    rc = work_free(ctx, low);
    return e == cudaSuccess ? rc : cuda_fail(ctx, e, w);
}
