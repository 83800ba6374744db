// ltx_ctx: device, stream, last-error text, device timeout flag, scratch.
#include <algorithm>
#include <cstring>
#include <new>
#include <set>
#include <utility>

#include "internal.hpp"
#include "kernels.hpp"

namespace ltx {

int ensure_scratch(ltx_ctx *ctx, size_t bytes) {
    if (ctx->scratch_bytes >= bytes) return LTX_OK;
    if (ctx->scratch) {
        cudaStreamSynchronize(ctx->stream);
        cudaFree(ctx->scratch);
        ctx->scratch = nullptr;
        ctx->scratch_bytes = 0;
    }
    cudaError_t e = cudaMalloc(&ctx->scratch, bytes);
    if (e != cudaSuccess) return fail(ctx, LTX_ERR_OOM, "scratch allocation of %zu bytes: %s", bytes, cudaGetErrorString(e));
    ctx->scratch_bytes = bytes;
    return LTX_OK;
}

// Workspaces up to this size stay with the context between eager calls.
constexpr size_t kKeptWorkBytes = 64u << 20;

int work_alloc(ltx_ctx *ctx, size_t bytes, void **out) {
    *out = nullptr;
    cudaStreamCaptureStatus capturing = cudaStreamCaptureStatusNone;
    LTX_CUDA_TRY(ctx, cudaStreamIsCapturing(ctx->stream, &capturing));
    const bool keep = capturing == cudaStreamCaptureStatusNone && bytes <= kKeptWorkBytes;
    if (keep && ctx->kept_bytes >= bytes) {
        *out = ctx->kept;
        return LTX_OK;
    }
    if (!ctx->pool) {
        cudaMemPoolProps props{};
        props.allocType = cudaMemAllocationTypePinned;
        props.location.type = cudaMemLocationTypeDevice;
        props.location.id = ctx->device;
        LTX_CUDA_TRY(ctx, cudaMemPoolCreate(&ctx->pool, &props));
        uint64_t hold = kKeptWorkBytes;   // what lies free beyond that goes back to the device at the next synchronisation
        LTX_CUDA_TRY(ctx, cudaMemPoolSetAttribute(ctx->pool, cudaMemPoolAttrReleaseThreshold, &hold));
    }
    if (keep && ctx->kept) {   // behind the calls that use it
        void *old = ctx->kept;
        ctx->kept = nullptr;
        ctx->kept_bytes = 0;
        LTX_CUDA_TRY(ctx, cudaFreeAsync(old, ctx->stream));
    }
    const cudaError_t e = cudaMallocFromPoolAsync(out, bytes, ctx->pool, ctx->stream);
    if (e == cudaErrorMemoryAllocation) {
        cudaGetLastError();   // reported here, not by the next launch check
        return fail(ctx, LTX_ERR_OOM, "workspace of %zu bytes: %s", bytes, cudaGetErrorString(e));
    }
    if (e != cudaSuccess) return cuda_fail(ctx, e, "workspace");
    if (keep) {
        ctx->kept = *out;
        ctx->kept_bytes = bytes;
    }
    return LTX_OK;
}

int work_free(ltx_ctx *ctx, void *p) {
    if (p && p != ctx->kept) LTX_CUDA_TRY(ctx, cudaFreeAsync(p, ctx->stream));
    return LTX_OK;
}

cudaError_t allow_smem(const ltx_ctx *ctx, const void *kernel, int bytes) {
    static std::mutex lock;
    static std::set<std::pair<const void *, int>> done;
    const std::lock_guard<std::mutex> hold(lock);
    if (done.count({kernel, ctx->device})) return cudaSuccess;
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != cudaSuccess) return e;
    try {
        done.insert({kernel, ctx->device});
    } catch (const std::bad_alloc &) {   // asked again next time
    }
    return e;
}

int upload(ltx_ctx *ctx, void *dst_dev, const void *src_host, size_t bytes) {
    if (bytes == 0) return LTX_OK;
    // The staging buffer is reused: the previous upload must have left it.
    LTX_CUDA_TRY(ctx, cudaEventSynchronize(ctx->upload_done));
    if (ctx->pinned_bytes < bytes) {
        if (ctx->pinned) cudaFreeHost(ctx->pinned);
        ctx->pinned = nullptr;
        ctx->pinned_bytes = 0;
        const size_t want = std::max<size_t>(bytes, 1 << 20);
        if (cudaHostAlloc(&ctx->pinned, want, cudaHostAllocDefault) != cudaSuccess)
            return fail(ctx, LTX_ERR_OOM, "pinned staging of %zu bytes", want);
        ctx->pinned_bytes = want;
    }
    memcpy(ctx->pinned, src_host, bytes);
    LTX_CUDA_TRY(ctx, cudaMemcpyAsync(dst_dev, ctx->pinned, bytes, cudaMemcpyHostToDevice, ctx->stream));
    LTX_CUDA_TRY(ctx, cudaEventRecord(ctx->upload_done, ctx->stream));
    return LTX_OK;
}

}  // namespace ltx

extern "C" int ltx_ctx_create(int device, void *stream, ltx_ctx **out) {
    if (!out) return LTX_ERR_INVALID_ARG;
    *out = nullptr;
    int n = 0;
    if (cudaGetDeviceCount(&n) != cudaSuccess || device < 0 || device >= n) return LTX_ERR_CUDA;
    ltx_ctx *ctx = new (std::nothrow) ltx_ctx();
    if (!ctx) return LTX_ERR_OOM;
    ctx->device = device;
    if (cudaSetDevice(device) != cudaSuccess) {
        delete ctx;
        return LTX_ERR_CUDA;
    }
    cudaDeviceGetAttribute(&ctx->sm_count, cudaDevAttrMultiProcessorCount, device);
    // The caller's stream; NULL is the CUDA default (legacy) stream, which is
    // also what PyTorch and most hosts enqueue on by default.
    ctx->stream = static_cast<cudaStream_t>(stream);
    if (cudaEventCreateWithFlags(&ctx->upload_done, cudaEventDisableTiming) != cudaSuccess ||
        cudaMalloc(&ctx->timeout_flag, sizeof(int)) != cudaSuccess ||
        cudaMemsetAsync(ctx->timeout_flag, 0, sizeof(int), ctx->stream) != cudaSuccess) {
        if (ctx->own_stream) cudaStreamDestroy(ctx->stream);
        delete ctx;
        return LTX_ERR_CUDA;
    }
    *out = ctx;
    return LTX_OK;
}

extern "C" void ltx_ctx_destroy(ltx_ctx *ctx) {
    if (!ctx) return;
    cudaSetDevice(ctx->device);
    cudaStreamSynchronize(ctx->stream);
    ltx::comm_release(ctx, false);
    if (ctx->kept) cudaFreeAsync(ctx->kept, ctx->stream);
    if (ctx->pool) {
        cudaStreamSynchronize(ctx->stream);
        cudaMemPoolDestroy(ctx->pool);
    }
    if (ctx->scratch) cudaFree(ctx->scratch);
    if (ctx->work) cudaFree(ctx->work);
    if (ctx->pinned) cudaFreeHost(ctx->pinned);
    if (ctx->upload_done) cudaEventDestroy(ctx->upload_done);
    if (ctx->timeout_flag) cudaFree(ctx->timeout_flag);
    if (ctx->own_stream) cudaStreamDestroy(ctx->stream);
    delete ctx;
}

extern "C" const char *ltx_last_error(const ltx_ctx *ctx) { return ctx ? ctx->last_error.c_str() : "null context"; }

extern "C" const char *ltx_host_last_error(void) { return ltx::host_error().c_str(); }

extern "C" void *ltx_ctx_stream(const ltx_ctx *ctx) { return ctx ? static_cast<void *>(ctx->stream) : nullptr; }

extern "C" int ltx_ctx_synchronize(ltx_ctx *ctx) {
    if (!ctx) return LTX_ERR_INVALID_ARG;
    cudaError_t e = cudaStreamSynchronize(ctx->stream);
    if (e != cudaSuccess) return ltx::cuda_fail(ctx, e, "cudaStreamSynchronize");
    int flag = 0;
    e = cudaMemcpy(&flag, ctx->timeout_flag, sizeof(int), cudaMemcpyDeviceToHost);
    if (e != cudaSuccess) return ltx::cuda_fail(ctx, e, "reading the timeout flag");
    if (flag) {
        cudaMemset(ctx->timeout_flag, 0, sizeof(int));
        if (flag == ltx::kErrTooManyTimesteps)
            return ltx::fail(ctx, LTX_ERR_UNSUPPORTED,
                             "a forward had more than %d distinct timesteps on the device (pass them from the host: "
                             "ltx_denoise_step's mask_host)", ltx::kMaxDistinctTs);
        if (flag == ltx::kErrBadPosition)
            return ltx::fail(ctx, LTX_ERR_INVALID_ARG, "qk_norm_rope: a position lies outside the cos/sin tables");
        if (flag == ltx::kErrBadAdapter)
            return ltx::fail(ctx, LTX_ERR_INVALID_ARG, "gemm_adapters: an adapter index lies beyond the pool");
        if (flag == ltx::kErrBadGate)
            return ltx::fail(ctx, LTX_ERR_INVALID_ARG, "gemm_adapters: a gate index lies outside the gate's rows");
        if (flag == ltx::kErrBadOffsets)
            return ltx::fail(ctx, LTX_ERR_INVALID_ARG,
                             "attention_packed: document offsets descend or lie outside the rows");
        return ltx::fail(ctx, LTX_ERR_TIMEOUT, "a device-side wait gave up (code %d)", flag);
    }
    return LTX_OK;
}
