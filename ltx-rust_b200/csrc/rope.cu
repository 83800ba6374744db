// Rotary positions for packed batches: the cos/sin tables of 1-D positions
// (stretched for long contexts) and the per-head RMSNorm of queries and keys
// with the rotation in the same pass.
//
// Both are bound by the bytes they move.  The table writes rot_dim * 4 bytes
// per position: 14.4 us for 131072 x 128, 4.7 TB/s, where a fill of the same bytes
// takes 12.4.  The norm reads and writes every query and key value once and adds
// one table row per token: 80 us for 12288 x (32 + 32) heads x 128 in bf16, 5.1 TB/s
// (a copy of that size runs at 6.3).
#include <cuda_fp16.h>

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "device_common.cuh"
#include "internal.hpp"
#include "kernels.hpp"

namespace ltx {

namespace {

constexpr int kMaxRot = 512, kMaxHeadDim = 512;

// ── tables ───────────────────────────────────────────────────────────────────

struct TableParams {
    const int *pos;
    int rows, half;
    double powers[8];                // theta^(-2 2^b / rot_dim): a frequency is their product over the bits of its index
    double inv_factor, orig_turns;   // orig_turns = original_len / 2pi, 0 = stretch every frequency
    double turns_low, inv_span;
    float amplitude;
    float *cos_out, *sin_out;
};

// The angle is kept as a 64-bit fraction of a turn: a frequency's turns per
// position times 2^64, rounded from f64, times the position, modulo 2^64: whole
// turns (2.7 million at position 2^24) fall off the top exactly, by two integer
// multiplications.  The upper 32 bits are the angle to 2^-32 turns: two bits of
// quarter and the rest r, |r| <= 1/2 quarter.  sin(pi r/2) = r S(r^2) and
// cos(pi r/2) = C(r^2) with S of degree 3 and C of degree 4, fitted here to the
// least absolute error: with the f32 roundings 9.4e-8 at most, 2e-8 root mean
// square.  (A value took 16 f64 and conversion cycles more with the reduction in
// f64: 18.4 us for 131072 x 128 instead of 14.4.)
struct SinCos {
    float s[4], c[5];   // the polynomials, the amplitude multiplied in
    __device__ __forceinline__ explicit SinCos(float a)
        : s{a * 0x1.921fb4p+0f, a * -0x1.4abba8p-1f, a * 0x1.465a3ep-4f, a * -0x1.2cf5d4p-8f},
          c{a, a * -0x1.3bd3ccp+0f, a * 0x1.03c1dcp-2f, a * -0x1.55c57cp-6f, a * 0x1.d9c364p-11f} {}
    // pos: the position's absolute value; sign: its sign bit
    __device__ __forceinline__ void operator()(unsigned pos, unsigned sign, uint2 turns, float &sn, float &cs) const {
        const unsigned angle = __umulhi(pos, turns.x) + pos * turns.y;   // bits 32..63 of the product
        const unsigned q = (angle + 0x20000000u) >> 30;
        const float r = (float)(int)(angle << 2) * 0x1p-32f, z = r * r;
        const float a = r * fmaf(fmaf(fmaf(s[3], z, s[2]), z, s[1]), z, s[0]);
        const float b = fmaf(fmaf(fmaf(fmaf(c[4], z, c[3]), z, c[2]), z, c[1]), z, c[0]);
        sn = __uint_as_float(__float_as_uint(q & 1 ? b : a) ^ (((q & 2) << 30) ^ sign));
        cs = __uint_as_float(__float_as_uint(q & 1 ? a : b) ^ (((q + 1) & 2) << 30));
    }
};

// A thread keeps VEC neighbouring frequencies of its own and walks down the
// rows: no division per value, 16-byte stores (VEC 4; 1 where rot_dim / 2 is
// no multiple of 4).
template <int VEC>
__global__ void __launch_bounds__(256) rope_table_1d_kernel(TableParams p) {
    __shared__ uint2 s_turns[kMaxRot / 2];   // per position, lower and upper word
    for (int i = threadIdx.x; i < p.half; i += blockDim.x) {
        double f = 1.0;   // theta^(-2i/rot)
#pragma unroll
        for (int b = 0; b < 8; ++b) f *= i >> b & 1 ? p.powers[b] : 1.0;
        const double w = p.orig_turns > 0 ? fmin(fmax((p.orig_turns * f - p.turns_low) * p.inv_span, 0.0), 1.0) : 0.0;
        double t = f * (w + (1.0 - w) * p.inv_factor) * 0.15915494309189533577;   // 1/2pi
        t -= floor(t);
        const unsigned long long u = t < 1.0 ? __double2ull_rn(t * 18446744073709551616.0) : 0ull;
        s_turns[i] = make_uint2((unsigned)u, (unsigned)(u >> 32));
    }
    __syncthreads();
    const int per_row = p.half / VEC, rows_at_once = 256 / per_row;   // per_row <= 256: rot_dim <= 512
    const int i = threadIdx.x % per_row * VEC;
    if (threadIdx.x / per_row >= rows_at_once) return;
    uint2 turns[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) turns[v] = s_turns[i + v];
    const SinCos sincos(p.amplitude);
    // the next row's position is fetched under this one's values
    const int step = (int)gridDim.x * rows_at_once;
    int64_t r = (int64_t)blockIdx.x * rows_at_once + threadIdx.x / per_row;
    int next = p.pos && r < p.rows ? p.pos[r] : (int)r;
    for (; r < p.rows; r += step) {
        const int at_pos = next;
        next = !p.pos ? (int)(r + step) : r + step < p.rows ? p.pos[r + step] : 0;
        const unsigned pos = at_pos < 0 ? 0u - (unsigned)at_pos : (unsigned)at_pos, sign = (unsigned)at_pos & 0x80000000u;
        float c[VEC], s[VEC];
#pragma unroll
        for (int v = 0; v < VEC; ++v) sincos(pos, sign, turns[v], s[v], c[v]);
        const int64_t at = r * p.half + i;
        if constexpr (VEC == 4) {
            __stcs(reinterpret_cast<float4 *>(p.cos_out + at), make_float4(c[0], c[1], c[2], c[3]));
            __stcs(reinterpret_cast<float4 *>(p.sin_out + at), make_float4(s[0], s[1], s[2], s[3]));
        } else {
            p.cos_out[at] = c[0];
            p.sin_out[at] = s[0];
        }
    }
}

// ── per-head norm + rotation ─────────────────────────────────────────────────

struct NormRopeParams {
    const void *q, *k;
    void *qo, *ko;
    int64_t ldq, ldk, ldqo, ldko;
    int rows, heads, kv_heads, d, norm;
    float eps;
    const float *gq, *gk, *cos_t, *sin_t;
    int table_rows, half, interleaved;
    const int *pos;
    int *flag;
};

template <typename T>
__device__ __forceinline__ float to_f32(T v) {
    if constexpr (sizeof(T) == 4) return v;
    else if constexpr (std::is_same_v<T, __half>) return __half2float(v);
    else return __bfloat162float(v);
}
template <typename T>
__device__ __forceinline__ T from_f32(float v) {
    if constexpr (sizeof(T) == 4) return v;
    else if constexpr (std::is_same_v<T, __half>) return __float2half_rn(v);
    else return __float2bfloat16_rn(v);
}

// The table row of token `row`: its position, or the row itself modulo the
// table.  A position outside the table takes the nearest row and raises the flag.
__device__ __forceinline__ int64_t table_row(const NormRopeParams &p, int row) {
    if (!p.pos) return row % p.table_rows;
    const int r = p.pos[row];
    if ((unsigned)r >= (unsigned)p.table_rows) {
        report_index(p.flag, kErrBadPosition);
        return r < 0 ? 0 : p.table_rows - 1;
    }
    return r;
}

// Any head_dim, rot_dim, layout and alignment (what the kernel below does not
// take): one warp per (row, head), the
// head in shared memory as f32 between the norm and the rotation.
template <typename T>
__global__ void __launch_bounds__(256) qk_norm_rope_any_kernel(NormRopeParams p) {
    __shared__ float xs[8][kMaxHeadDim];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int all = p.heads + p.kv_heads;
    const int64_t item = (int64_t)blockIdx.x * 8 + warp;
    if (item >= (int64_t)p.rows * all) return;
    const int row = (int)(item / all), h = (int)(item % all);
    const bool is_q = h < p.heads;
    const int hh = is_q ? h : h - p.heads;
    const T *x = static_cast<const T *>(is_q ? p.q : p.k) + (int64_t)row * (is_q ? p.ldq : p.ldk) + (int64_t)hh * p.d;
    T *y = static_cast<T *>(is_q ? p.qo : p.ko) + (int64_t)row * (is_q ? p.ldqo : p.ldko) + (int64_t)hh * p.d;
    const float *g = is_q ? p.gq : p.gk;
    float *s = xs[warp];
    float ss = 0.f;
    for (int e = lane; e < p.d; e += 32) {
        const float v = to_f32(x[e]);
        s[e] = v;
        ss += v * v;
    }
    float inv = 1.f;
    if (p.norm) {
#pragma unroll
        for (int o = 16; o; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        inv = 1.f / sqrtf(ss / (float)p.d + p.eps);
        for (int e = lane; e < p.d; e += 32) s[e] *= g ? inv * g[e] : inv;
    }
    __syncwarp();
    if (p.half) {
        const int64_t tr = table_row(p, row) * p.half;
        for (int j = lane; j < p.half; j += 32) {
            const int a = p.interleaved ? 2 * j : j, b = p.interleaved ? 2 * j + 1 : j + p.half;
            const float c = p.cos_t[tr + j], sn = p.sin_t[tr + j], u = s[a], v = s[b];
            y[a] = from_f32<T>(c * u - sn * v);
            y[b] = from_f32<T>(sn * u + c * v);
        }
    }
    for (int e = 2 * p.half + lane; e < p.d; e += 32) y[e] = from_f32<T>(s[e]);
}

// The same with 16-byte accesses: a lane holds 8 neighbouring values, LANES
// lanes a head (the power of two that covers head_dim / 8), and a warp works on
// 32 / LANES heads of one row at a time, kHeadsDeep times, all of queries or all
// of keys, with every load issued before the first sum.  gamma is folded into the
// rotation once per warp: out = (x c gamma + partner s gamma') / rms, so a
// value costs a conversion, its square, two products and its share of the
// partner's fetch (packed: a pair of the half layout lies rot_dim/16 lanes apart,
// one of the interleaved layout in the same word).  Four heads deep at 63 registers:
// two 6 to 35% slower, eight 2 to 45%, more blocks to an SM (spills) 3 to 80%.
constexpr int kHeadsDeep = 4;

template <typename T>
struct Vec8 {
    static constexpr int kWords = 2 * sizeof(T);
    uint32_t w[kWords];
    __device__ __forceinline__ void load(const T *p) {
#pragma unroll
        for (int i = 0; i < kWords; i += 4) *reinterpret_cast<uint4 *>(w + i) = *reinterpret_cast<const uint4 *>(reinterpret_cast<const uint32_t *>(p) + i);
    }
    __device__ __forceinline__ void get(float (&v)[8]) const {
#pragma unroll
        for (int i = 0; i < kWords; ++i) {
            if constexpr (sizeof(T) == 4) v[i] = __uint_as_float(w[i]);
            else if constexpr (std::is_same_v<T, __half>) {
                const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
                v[2 * i] = f.x;
                v[2 * i + 1] = f.y;
            } else {
                v[2 * i] = __uint_as_float(w[i] << 16);
                v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
            }
        }
    }
    __device__ __forceinline__ void put(const float (&v)[8], T *p) {
#pragma unroll
        for (int i = 0; i < kWords; ++i) {
            if constexpr (sizeof(T) == 4) w[i] = __float_as_uint(v[i]);
            else if constexpr (std::is_same_v<T, __half>) {
                const __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
                w[i] = *reinterpret_cast<const uint32_t *>(&h);
            } else {
                const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
                w[i] = *reinterpret_cast<const uint32_t *>(&h);
            }
        }
#pragma unroll
        for (int i = 0; i < kWords; i += 4) *reinterpret_cast<uint4 *>(reinterpret_cast<uint32_t *>(p) + i) = *reinterpret_cast<uint4 *>(w + i);
    }
    // the values of the lane `from`, or (interleaved) the neighbours in the pairs
    __device__ __forceinline__ Vec8 partner(bool interleaved, int from) const {
        Vec8 o;
        if (!interleaved) {
#pragma unroll
            for (int i = 0; i < kWords; ++i) o.w[i] = __shfl_sync(0xffffffffu, w[i], from);
        } else {
#pragma unroll
            for (int i = 0; i < kWords; ++i) {
                if constexpr (sizeof(T) == 4) o.w[i] = w[i ^ 1];
                else o.w[i] = (w[i] << 16) | (w[i] >> 16);
            }
        }
        return o;
    }
};

__device__ __forceinline__ void load8(const float *p, float (&v)[8]) {
    const float4 a = __ldg(reinterpret_cast<const float4 *>(p)), b = __ldg(reinterpret_cast<const float4 *>(p) + 1);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}

template <typename T, int LANES, bool INTERLEAVED>
__global__ void __launch_bounds__(256) qk_norm_rope_vec_kernel(NormRopeParams p) {
    constexpr int kSide = 32 / LANES;   // heads side by side in a warp
    const int lane = threadIdx.x & 31, sub = lane / LANES, e0 = lane % LANES * 8;
    const int64_t row64 = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (row64 >= p.rows) return;
    const int row = (int)row64;
    const int q_chunks = (p.heads + kSide * kHeadsDeep - 1) / (kSide * kHeadsDeep);
    const bool is_q = (int)blockIdx.y < q_chunks;
    const int heads = is_q ? p.heads : p.kv_heads;
    const int h0 = ((int)blockIdx.y - (is_q ? 0 : q_chunks)) * kSide * kHeadsDeep + sub;
    const T *in = static_cast<const T *>(is_q ? p.q : p.k) + (int64_t)row * (is_q ? p.ldq : p.ldk) + h0 * p.d + e0;
    T *out = static_cast<T *>(is_q ? p.qo : p.ko) + (int64_t)row * (is_q ? p.ldqo : p.ldko) + h0 * p.d + e0;
    const int step = kSide * p.d;
    const bool in_head = e0 < p.d;

    Vec8<T> x[kHeadsDeep];
#pragma unroll
    for (int u = 0; u < kHeadsDeep; ++u) {
        x[u] = Vec8<T>{};
        if (in_head && h0 + u * kSide < heads) x[u].load(in + u * step);
    }
    // this lane's 8 values: out = x * a + partner * b, gamma included
    const int rot = 2 * p.half, apart = p.half / 8;   // half layout: lanes between a pair
    const bool turns = e0 < rot, second = !INTERLEAVED && turns && e0 >= p.half;
    const int from = (second ? lane - apart : lane + apart) & 31;
    float a[8], b[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) a[i] = 1.f;
    const float *g = p.norm ? (is_q ? p.gq : p.gk) : nullptr;
    if (g && in_head) load8(g + e0, a);
    if (turns) {
        float c[8];
        const int64_t at = table_row(p, row) * p.half;
        if constexpr (!INTERLEAVED) {
            const int j = second ? e0 - p.half : e0;
            load8(p.cos_t + at + j, c);
            load8(p.sin_t + at + j, b);
        } else {
            const float4 c4 = __ldg(reinterpret_cast<const float4 *>(p.cos_t + at + e0 / 2));
            const float4 s4 = __ldg(reinterpret_cast<const float4 *>(p.sin_t + at + e0 / 2));
            const float cc[4] = {c4.x, c4.y, c4.z, c4.w}, sv[4] = {s4.x, s4.y, s4.z, s4.w};
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                c[i] = cc[i / 2];
                b[i] = sv[i / 2];
            }
        }
        float gp[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) gp[i] = INTERLEAVED ? a[i ^ 1] : 1.f;
        if (!INTERLEAVED && g) load8(g + (second ? e0 - p.half : e0 + p.half), gp);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            b[i] *= (INTERLEAVED ? !(i & 1) : !second) ? -gp[i] : gp[i];
            a[i] *= c[i];
        }
    }
    const float inv_d = 1.f / (float)p.d;
#pragma unroll
    for (int u = 0; u < kHeadsDeep; ++u) {
        float v[8], w[8], inv = 1.f;
        x[u].get(v);
        if (rot) x[u].partner(INTERLEAVED, from).get(w);
        if (p.norm) {
            float ss = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) ss = fmaf(v[i], v[i], ss);
#pragma unroll
            for (int o = LANES / 2; o; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
            inv = rsqrtf(fmaf(ss, inv_d, p.eps));
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = (turns ? fmaf(w[i], b[i], v[i] * a[i]) : v[i] * a[i]) * inv;
        if (in_head && h0 + u * kSide < heads) x[u].put(v, out + u * step);
    }
}

template <typename T, int LANES>
void launch_vec(const NormRopeParams &p, cudaStream_t st) {
    constexpr int kHeads = 32 / LANES * kHeadsDeep;
    const dim3 grid((unsigned)(((int64_t)p.rows + 7) / 8), (unsigned)((p.heads + kHeads - 1) / kHeads + (p.kv_heads + kHeads - 1) / kHeads));
    if (p.interleaved) qk_norm_rope_vec_kernel<T, LANES, true><<<grid, 256, 0, st>>>(p);
    else qk_norm_rope_vec_kernel<T, LANES, false><<<grid, 256, 0, st>>>(p);
}

template <typename T>
void launch_norm_rope(const NormRopeParams &p, cudaStream_t st) {
    // 16-byte accesses need whole groups of 8 values everywhere: the head, each
    // half of the rotated part (interleaved: the part), rows and bases.
    constexpr int kAlign = 16 / sizeof(T);
    const uintptr_t bases = (uintptr_t)p.q | (uintptr_t)p.qo | (uintptr_t)p.k | (uintptr_t)p.ko | (uintptr_t)p.gq |
                            (uintptr_t)p.gk | (uintptr_t)p.cos_t | (uintptr_t)p.sin_t;
    const int64_t lds = p.ldq | p.ldqo | p.ldk | p.ldko;
    if (p.d % 8 == 0 && p.d <= 256 && p.half % (p.interleaved ? 4 : 8) == 0 && !(bases & 15) && lds % kAlign == 0 &&
        p.heads + (int64_t)p.kv_heads <= 65535) {   // the grid's second dimension
        if (p.d <= 32) launch_vec<T, 4>(p, st);
        else if (p.d <= 64) launch_vec<T, 8>(p, st);
        else if (p.d <= 128) launch_vec<T, 16>(p, st);
        else launch_vec<T, 32>(p, st);
        return;
    }
    const int64_t items = (int64_t)p.rows * (p.heads + p.kv_heads);
    qk_norm_rope_any_kernel<T><<<(unsigned)((items + 7) / 8), 256, 0, st>>>(p);
}

}  // namespace

}  // namespace ltx

extern "C" int ltx_rope_table(ltx_ctx *ctx, const int32_t *pos_dev, int32_t rows, int32_t rot_dim, double theta,
                              double factor, int64_t original_len, double turns_low, double turns_high,
                              double amplitude, float *cos_dev, float *sin_dev) {
    using namespace ltx;
    if (!ctx) return LTX_ERR_INVALID_ARG;
    if (rows < 0 || rot_dim < 2 || rot_dim > kMaxRot || rot_dim % 2)
        return fail(ctx, LTX_ERR_SHAPE, "rope_table: %d rows, rot_dim %d (even, 2..%d)", rows, rot_dim, kMaxRot);
    if (!(theta > 0) || !std::isfinite(theta) || !(factor > 0) || !std::isfinite(factor) || !std::isfinite((float)amplitude) ||
        original_len < 0)
        return fail(ctx, LTX_ERR_INVALID_ARG, "rope_table: theta and factor must be finite and > 0, original_len >= 0");
    if (original_len > 0 && !(turns_high > turns_low && std::isfinite(turns_high) && std::isfinite(turns_low)))
        return fail(ctx, LTX_ERR_INVALID_ARG, "rope_table: turns_high must exceed turns_low");
    if (rows == 0) return LTX_OK;
    if (!cos_dev || !sin_dev) return fail(ctx, LTX_ERR_INVALID_ARG, "rope_table: null output");
    DeviceGuard guard(ctx);
    TableParams p{pos_dev, rows, rot_dim / 2, {}, 1.0 / factor, (double)original_len * 0.15915494309189533577, turns_low,
                  original_len > 0 ? 1.0 / (turns_high - turns_low) : 0.0, (float)amplitude, cos_dev, sin_dev};
    for (int b = 0; b < 8; ++b) p.powers[b] = std::pow(theta, -(double)(1 << b) / p.half);
    const bool vec = p.half % 4 == 0 && !(((uintptr_t)cos_dev | (uintptr_t)sin_dev) & 15);
    const int at_once = 256 / (vec ? p.half / 4 : p.half);
    const int grid = (int)std::min<int64_t>(((int64_t)rows + at_once - 1) / at_once, ctx->sm_count * 6);   // all at once
    if (vec) rope_table_1d_kernel<4><<<grid, 256, 0, ctx->stream>>>(p);
    else rope_table_1d_kernel<1><<<grid, 256, 0, ctx->stream>>>(p);
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? LTX_OK : cuda_fail(ctx, e, "rope_table launch");
}

extern "C" int ltx_qk_norm_rope(ltx_ctx *ctx, const ltx_norm_rope *args) {
    using namespace ltx;
    if (!ctx) return LTX_ERR_INVALID_ARG;
    if (!args) return fail(ctx, LTX_ERR_INVALID_ARG, "qk_norm_rope: null arguments");
    const auto &[q_dev, k_dev, q_out_dev, k_out_dev, gamma_q_dev, gamma_k_dev, cos_dev, sin_dev, pos_dev, ldq, ldk, ldqo, ldko,
                 dtype, rows, heads, kv_heads, head_dim, norm, table_rows, rot_dim, layout, eps] = *args;
    if (dtype != LTX_BF16 && dtype != LTX_F16 && dtype != LTX_F32)
        return fail(ctx, LTX_ERR_DTYPE, "qk_norm_rope: dtype %d (BF16, F16 or F32)", dtype);
    if (rows < 0 || heads < 0 || kv_heads < 0 || head_dim < 1 || head_dim > kMaxHeadDim)
        return fail(ctx, LTX_ERR_SHAPE, "qk_norm_rope: %d rows, %d + %d heads of %d (1..%d)", rows, heads, kv_heads,
                    head_dim, kMaxHeadDim);
    if (rot_dim < 0 || rot_dim > head_dim || rot_dim % 2)
        return fail(ctx, LTX_ERR_SHAPE, "qk_norm_rope: rot_dim %d must be even and at most head_dim %d", rot_dim, head_dim);
    if (layout != LTX_ROPE_HALF && layout != LTX_ROPE_INTERLEAVED)
        return fail(ctx, LTX_ERR_INVALID_ARG, "qk_norm_rope: bad layout %d", layout);
    if (norm && !(eps >= 0.f && std::isfinite(eps)))
        return fail(ctx, LTX_ERR_INVALID_ARG, "qk_norm_rope: eps must be finite and >= 0");
    if (rot_dim > 0 && (!cos_dev || !sin_dev || table_rows < 1))
        return fail(ctx, LTX_ERR_INVALID_ARG, "qk_norm_rope: a rotation needs cos/sin tables with at least one row");
    const int64_t qc = (int64_t)heads * head_dim, kc = (int64_t)kv_heads * head_dim;
    if (rows == 0 || qc + kc == 0) return LTX_OK;
    if ((heads && (!q_dev || !q_out_dev)) || (kv_heads && (!k_dev || !k_out_dev)))
        return fail(ctx, LTX_ERR_INVALID_ARG, "qk_norm_rope: null q or k");
    if ((heads && (ldq < qc || ldqo < qc)) || (kv_heads && (ldk < kc || ldko < kc)))
        return fail(ctx, LTX_ERR_SHAPE, "qk_norm_rope: leading dimensions shorter than the heads");
    if ((int64_t)rows * (heads + (int64_t)kv_heads) > (int64_t)1 << 33)
        return fail(ctx, LTX_ERR_UNSUPPORTED, "qk_norm_rope: more than 2^33 heads in one call");
    DeviceGuard guard(ctx);
    NormRopeParams p{q_dev, k_dev, q_out_dev, k_out_dev, ldq, ldk, ldqo, ldko, rows, heads, kv_heads, head_dim, norm,
                     eps, gamma_q_dev, gamma_k_dev, cos_dev, sin_dev, table_rows, rot_dim / 2,
                     layout == LTX_ROPE_INTERLEAVED, pos_dev, ctx->timeout_flag};
    if (dtype == LTX_F32) launch_norm_rope<float>(p, ctx->stream);
    else if (dtype == LTX_F16) launch_norm_rope<__half>(p, ctx->stream);
    else launch_norm_rope<__nv_bfloat16>(p, ctx->stream);
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? LTX_OK : cuda_fail(ctx, e, "qk_norm_rope launch");
}
