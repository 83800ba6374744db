// Attention over packed documents: softmax over the keys of the row's own
// document only, with optional causal and prefix masks, scores capped by a
// tanh, and a bias that falls with distance.
//
// Every mask here leaves a row the first `lim` keys of its document (the
// document mask: all of them; causal: up to the key beside it; a prefix: at
// least that many), so a row needs one number and a tile of keys is either
// whole for all rows of a warp or compared against it.
//
// One CTA per (document, key head, up to 256 query rows).  A query row is a
// (token, head of the key head's group): a 128-row tile holds 128 / group
// tokens times the group's heads, so the heads that share a key head read
// each K/V tile once, and a single new token still brings `group` rows.
// Both 128-row tiles A and B of the CTA share every K/V tile.
// TMEM (512 columns): S_A, S_B (128 f32 columns each), O_A, O_B; P goes back
// into the upper half of its S as packed 16-bit pairs and is the A operand of
// P.V from there.
// 10 warps:
//   warp 0     TMA: the Q tiles, then K_j, V_j through a ring.  Afterwards it
//              zeroes the V rows behind the document's end in the last tile:
//              P is 0 there, but 0 times another document's NaN is not.
//   warp 1     one thread issues QK_A QK_B | PV_A(j) QK_A(j+1) PV_B(j) QK_B(j+1).
//   warps 2-5  softmax of tile A, 6-9 of tile B, one row per thread: running
//              maximum and sum in f32, O rescaled in TMEM only when a row's
//              maximum grew by more than 2^kRescaleLog2.
// With few CTAs (few rows over long keys) a cluster of S CTAs shares the
// keys of one item and joins its partial O, maximum and sum through
// distributed shared memory, in the order of the ranks.
// All waits are bounded (2 s) and report LTX_ERR_TIMEOUT through the flag.
#include <cuda.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <cmath>

#include "attention_packed.cuh"
#include "device_common.cuh"
#include "internal.hpp"
#include "kernels.hpp"

namespace ltx {

namespace {

constexpr int kThreads = 320;

// D 128: 16-bit K and V tiles of 32 KB (two 64-column swizzle blocks), D 64: 16 KB.
template <int D>
struct Smem {
    static constexpr int TILE = 128 * D * 2, HALF = 128 * 64 * 2;
    static constexpr int RING_SLOTS = D == 128 ? 5 : 8;
    static constexpr int Q = 0, RING = 2 * TILE, BAR = RING + RING_SLOTS * TILE;
    // float2 [2][128], a row's maximum and sum (splits > 1): where Q was, which no product reads any more
    static constexpr int ML = Q;
    static constexpr int BYTES = BAR + 256 + 1024;
    static_assert((8 + 2 * RING_SLOTS) * 8 + 8 + 32 <= 256, "barriers and document words exceed their block");
    static_assert(2 * 128 * D * 4 <= RING_SLOTS * TILE, "the f32 partials of both tiles fit the ring");
    static_assert(BYTES <= 232448, "shared memory exceeds the per-CTA limit");
};

// The pair-th pair of query tiles over all documents, found by one warp; false
// when there are fewer.  A causal document's last tiles have the most keys and
// go first.
__device__ __forceinline__ bool find_item(const PackedParams &p, int pair, int lane, Item &it) {
    const int per = 2 * p.tile_tokens;
    int before = 0;
    for (int base = 0; base < p.docs; base += 32) {
        int s = 0, e = 0;
        if (base + lane < p.docs) doc_span(p.qo, base + lane, p.rows_q, p.flag, s, e);
        const int n = (e - s + per - 1) / per;
        int incl = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += v;
        }
        const unsigned hit = __ballot_sync(0xffffffffu, before + incl > pair);
        if (hit) {
            const int src = __ffs(hit) - 1;
            const int local = pair - before - __shfl_sync(0xffffffffu, incl - n, src);
            const int nn = __shfl_sync(0xffffffffu, n, src);
            it.qs = __shfl_sync(0xffffffffu, s, src);
            it.lq = __shfl_sync(0xffffffffu, e, src) - it.qs;
            it.tile0 = 2 * (p.causal ? nn - 1 - local : local);
            it.doc = base + src;
            int ke;
            doc_span(p.ko, it.doc, p.rows_k, p.flag, it.ks, ke);
            it.lk = ke - it.ks;
            return true;
        }
        before += __shfl_sync(0xffffffffu, incl, 31);
    }
    return false;
}

__device__ __forceinline__ void cluster_sync() {
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t peer_addr(const void *smem, uint32_t rank) {
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(smem)), "r"(rank));
    return a;
}
__device__ __forceinline__ float4 ld_peer4(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                 : "r"(addr)
                 : "memory");
    return v;
}
__device__ __forceinline__ float2 ld_peer2(uint32_t addr) {
    float2 v;
    asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
    return v;
}

// VF16: V (and so P) are f16, otherwise bf16; Q and K are bf16.  MOD: scores
// are capped or biased.
template <int D, bool VF16, bool MOD>
__global__ void __launch_bounds__(kThreads, 1)
    packed_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                  const __grid_constant__ CUtensorMap tmV, PackedParams p) {
    using L = Smem<D>;
    constexpr int kRing = L::RING_SLOTS;
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    unsigned char *smem = reinterpret_cast<unsigned char *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    unsigned char *sQ = smem + L::Q, *sRing = smem + L::RING;
    uint64_t *bars = reinterpret_cast<uint64_t *>(smem + L::BAR);
    uint64_t *q_full = bars, *v_clean = bars + 1;
    uint64_t *s_full = bars + 2, *p_full = bars + 4, *pv_done = bars + 6;   // [2] each
    uint64_t *slot_full = bars + 8, *slot_empty = slot_full + kRing;        // [kRing] each
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(slot_empty + kRing);
    Item *s_item = reinterpret_cast<Item *>(tmem_slot + 2);
    int *s_found = reinterpret_cast<int *>(s_item + 1);
    float2 *s_ml = reinterpret_cast<float2 *>(smem + L::ML);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int item = blockIdx.x / p.splits, split = blockIdx.x % p.splits;
    const int kvh = item / p.pairs;

    if (warp == 1) {
        Item it{};
        const bool found = find_item(p, item % p.pairs, lane, it);
        if (lane == 0) {
            *s_item = it;
            *s_found = found;
        }
    }
    if (threadIdx.x == 0) {
        mbar_init(q_full, 1);
        mbar_init(v_clean, 32);
        for (int s = 0; s < kRing; ++s) {
            mbar_init(&slot_full[s], 1);
            mbar_init(&slot_empty[s], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&s_full[i], 1);
            mbar_init(&p_full[i], 4);
            mbar_init(&pv_done[i], 1);
        }
        fence_barrier_init();
    }
    __syncthreads();
    if (!*s_found) return;   // the whole cluster: its CTAs have one item
    if (warp == 0) {
        tmem_alloc(tmem_slot, 512);
        tmem_relinquish();
    }
    const Item it = *s_item;
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    bool aborted = false;

    const int tt = p.tile_tokens;
    const int prefix = p.causal && p.prefix ? min(max(p.prefix[it.doc], 0), it.lk) : 0;
    const int nt = it.lq > (it.tile0 + 1) * tt ? 2 : 1;   // query tiles of this CTA
    // K/V tiles [j0, j0 + cnt[t]) of query tile t: what its last token sees, and this CTA's share of it
    int cnt[2], j0, all;
    {
        int n[2];
#pragma unroll
        for (int t = 0; t < 2; ++t)
            n[t] = t < nt ? (limit_of(p, it, min((it.tile0 + t + 1) * tt, it.lq) - 1, prefix) + BKV - 1) / BKV : 0;
        const int most = max(n[0], n[1]);
        const int per = (most + p.splits - 1) / p.splits;
        j0 = split * per;
        const int j1 = min(most, j0 + per);
#pragma unroll
        for (int t = 0; t < 2; ++t) cnt[t] = max(0, min(j1, n[t]) - j0);
        all = max(cnt[0], cnt[1]);
    }
    // the document ends inside the last tile loaded here
    const int tail = it.lk - (j0 + all - 1) * BKV;
    const bool cleans = all > 0 && tail < BKV;

    if (warp == 0) {
        if (all > 0 && elect_one()) {
            tma_prefetch_desc(&tmQ);
            tma_prefetch_desc(&tmK);
            tma_prefetch_desc(&tmV);
            mbar_arrive_expect_tx(q_full, nt * (D / 64) * tt * p.group * 128);
            for (int t = 0; t < nt; ++t)
                for (int x = 0; x < D; x += 64)
                    tma_load_3d(sQ + t * L::TILE + (x / 64) * L::HALF, &tmQ, q_full, x, kvh * p.group,
                                it.qs + (it.tile0 + t) * tt);
            // load sequence: s = 2j -> K_j, s = 2j + 1 -> V_j, slot s % kRing
            int issued = 0;
            for (int s = 0; s < 2 * all; ++s, ++issued) {
                const int slot = s % kRing;
                if (!mbar_wait(&slot_empty[slot], ((s / kRing) & 1) ^ 1, p.flag, 301, &aborted)) break;
                mbar_arrive_expect_tx(&slot_full[slot], L::TILE);
                for (int x = 0; x < D; x += 64)
                    tma_load_3d(sRing + slot * L::TILE + (x / 64) * L::HALF, (s & 1) ? &tmV : &tmK, &slot_full[slot], x,
                                kvh, it.ks + (j0 + (s >> 1)) * BKV);
            }
            // Wait for every copy this thread started before the CTA can exit.
            bool a2 = false;
            mbar_wait(q_full, 0, nullptr, 0, &a2);
            for (int s = issued > kRing ? issued - kRing : 0; s < issued; ++s)
                mbar_wait(&slot_full[s % kRing], (s / kRing) & 1, nullptr, 0, &a2);
        }
        aborted = __any_sync(0xffffffffu, aborted);
        if (cleans && !aborted) {
            const int s = 2 * all - 1;
            mbar_wait(&slot_full[s % kRing], (s / kRing) & 1, p.flag, 302, &aborted);
            unsigned char *v = sRing + (s % kRing) * L::TILE;
            constexpr int kChunks = D / 64 * 8;   // 16-byte pieces of a row
            for (int i = tail * kChunks + lane; i < BKV * kChunks; i += 32)
                *reinterpret_cast<uint4 *>(v + (i % kChunks) / 8 * L::HALF + i / kChunks * 128 + (i % 8) * 16) =
                    make_uint4(0, 0, 0, 0);
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            mbar_arrive(v_clean);
        }
    } else if (warp == 1) {
        if (all > 0 && elect_one()) {
            constexpr uint32_t idesc_qk = idesc_f16(BQ, BKV, true, false);
            constexpr uint32_t idesc_pv = idesc_f16(BQ, D, !VF16, true);   // A = P (TMEM), B = V, MN-major
            const uint32_t q_addr = smem_u32(sQ);
            auto wait_slot = [&](int s, int code) {
                return mbar_wait(&slot_full[s % kRing], (s / kRing) & 1, p.flag, code, &aborted);
            };
            auto issue_qk = [&](int t, int j) {   // S_t = Q_t K_j^T
                const uint32_t k_addr = smem_u32(sRing + (2 * j) % kRing * L::TILE);
#pragma unroll
                for (int kk = 0; kk < D / 16; ++kk) {
                    const uint32_t off = (kk >> 2) * L::HALF + (kk & 3) * 32;
                    umma_f16_ss(tmem + t * 128, sdesc_sw128(q_addr + t * L::TILE + off, 16, 1024),
                                sdesc_sw128(k_addr + off, 16, 1024), idesc_qk, kk ? 1u : 0u);
                }
                umma_commit(&s_full[t]);
            };
            auto issue_pv = [&](int t, int j) {   // O_t (+)= P_t V_j; P_t: TMEM columns 64..127 of S_t
                const uint32_t v_addr = smem_u32(sRing + (2 * j + 1) % kRing * L::TILE);
#pragma unroll
                for (int kk = 0; kk < BKV / 16; ++kk) {   // 16 keys = 8 packed columns per MMA
                    const uint64_t bd = sdesc_sw128(v_addr + kk * 2048, L::HALF, 1024);
                    umma_f16_ts(tmem + 256 + t * 128, tmem + t * 128 + 64 + kk * 8, bd, idesc_pv,
                                (j > 0 || kk > 0) ? 1u : 0u);
                }
            };
            bool ok = mbar_wait(q_full, 0, p.flag, 305, &aborted) && wait_slot(0, 306);
            if (ok) {
                tc_fence_after();
                for (int t = 0; t < 2; ++t)
                    if (cnt[t] > 0) issue_qk(t, 0);
                umma_commit(&slot_empty[0]);   // K_0 read by both
            }
            for (int j = 0; ok && j < all; ++j) {
                // Per tile: PV_t(j) once the softmax has stored P_t(j) (p_full),
                // then QK_t(j+1) into the same columns: MMAs of one thread run
                // in issue order, so P_t(j) is read before S_t(j+1) lands.
                if (!wait_slot(2 * j + 1, 307)) break;
                const bool next = j + 1 < all;
                if (next && !wait_slot(2 * j + 2, 308)) break;
                if (!next && cleans && !mbar_wait(v_clean, 0, p.flag, 303, &aborted)) break;
                for (int t = 0; t < 2; ++t) {
                    if (j >= cnt[t]) continue;
                    if (!mbar_wait(&p_full[t], j & 1, p.flag, 309 + t, &aborted)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    issue_pv(t, j);
                    if (j + 1 < cnt[t])
                        issue_qk(t, j + 1);
                    else
                        umma_commit(&pv_done[t]);
                }
                if (!ok) break;
                umma_commit(&slot_empty[(2 * j + 1) % kRing]);             // V_j read
                if (next) umma_commit(&slot_empty[(2 * j + 2) % kRing]);   // K_{j+1} read
            }
        }
    }

    // Softmax warps: tile t = 0 (warps 2-5) or 1 (warps 6-9), row quad*32 + lane.
    const int t = (warp - 2) >> 2;
    const int quad = warp & 3;
    const int r_in = quad * 32 + lane;
    const int token = (it.tile0 + t) * tt + r_in / p.group;   // in the document
    const bool row_ok = warp >= 2 && t < nt && r_in < tt * p.group && token < it.lq;
    const int head = kvh * p.group + r_in % p.group;
    const uint32_t lane_base = (uint32_t)(quad * 32) << 16;
    const uint32_t o_tmem = tmem + lane_base + 256 + t * 128;
    float m_ref = -INFINITY;   // the max P is taken against (log2 domain)
    float l = 0.f;
    if (warp >= 2) {
        const int n_mine = t ? cnt[1] : cnt[0];
        const uint32_t s_tmem = tmem + lane_base + t * 128;
        const int lim = row_ok ? limit_of(p, it, token, prefix) : 0x7fffffff;
        const int lim_min = __reduce_min_sync(0xffffffffu, lim);
        const bool active = lim_min != 0x7fffffff;   // the warp holds rows
        ScoreMod mod{};
        float sc = p.scale * kLog2e;
        if constexpr (MOD) {
            mod.scale = p.scale;
            mod.twice_over_cap = p.softcap > 0.f ? 2.f * kLog2e / p.softcap : 0.f;
            mod.cap2 = p.softcap * kLog2e;
            mod.slope2 = p.slopes && row_ok ? p.slopes[head] * kLog2e : 0.f;
            sc = 1.f;
        }
        const float2 sl2 = make_float2(sc, sc);
        for (int j = 0; j < n_mine && !aborted; ++j) {
            // warp-uniform outcome: the tcgen05.ld/st below are warp-collective
            if (!warp_wait(&s_full[t], j & 1, p.flag, 311, &aborted)) break;
            if (!active) {   // no row here: P may hold anything, its O is not read
                if (lane == 0) mbar_arrive(&p_full[t]);
                continue;
            }
            tc_fence_after();
            const int kv0 = (j0 + j) * BKV;
            const int left = lim - kv0;                       // keys of this tile the row sees
            const bool masked = lim_min < kv0 + BKV;          // not all of them for every row of the warp
            if constexpr (MOD) mod.place = (float)((int64_t)token + it.lk - it.lq - kv0);
            // pass 1: the row max over the 128 scores.  Keys 64..127 stay in
            // registers (rh) for pass 2; keys 0..63 are read again (MOD: they
            // are put back changed).
            uint32_t rh[2][32];
            float mx;
            {
                uint32_t r01[2][32];
                tmem_ld_32x32b_x32(s_tmem + 0, r01[0]);
                tmem_ld_32x32b_x32(s_tmem + 32, r01[1]);
                tmem_ld_32x32b_x32(s_tmem + 64, rh[0]);
                tmem_ld_32x32b_x32(s_tmem + 96, rh[1]);
                tmem_ld_wait_regs(r01[0]);
                tmem_ld_wait_regs(r01[1]);
                tmem_ld_wait_regs(rh[0]);
                tmem_ld_wait_regs(rh[1]);
                if constexpr (MOD) {
#pragma unroll
                    for (int e = 0; e < 64; ++e) {
                        r01[e >> 5][e & 31] = __float_as_uint(mod(__uint_as_float(r01[e >> 5][e & 31]), e));
                        rh[e >> 5][e & 31] = __float_as_uint(mod(__uint_as_float(rh[e >> 5][e & 31]), 64 + e));
                    }
                }
                if (masked) {
#pragma unroll
                    for (int e = 0; e < 64; ++e) {
                        if (e >= left) r01[e >> 5][e & 31] = __float_as_uint(-INFINITY);
                        if (64 + e >= left) rh[e >> 5][e & 31] = __float_as_uint(-INFINITY);
                    }
                }
                if constexpr (MOD) {
                    tmem_st_32x32b_x32(s_tmem + 0, r01[0]);
                    tmem_st_32x32b_x32(s_tmem + 32, r01[1]);
                }
                float m8[8];
#pragma unroll
                for (int u = 0; u < 8; ++u) m8[u] = -INFINITY;
#pragma unroll
                for (int e = 0; e < 64; ++e) {
                    m8[e & 7] = fmaxf(m8[e & 7], __uint_as_float(r01[e >> 5][e & 31]));
                    m8[(e + 4) & 7] = fmaxf(m8[(e + 4) & 7], __uint_as_float(rh[e >> 5][e & 31]));
                }
                mx = fmaxf(fmaxf(fmaxf(m8[0], m8[1]), fmaxf(m8[2], m8[3])), fmaxf(fmaxf(m8[4], m8[5]), fmaxf(m8[6], m8[7])));
            }
            mx *= sc;   // scale > 0: max(s * scale) = scale * max(s)
            // The rows of one warp decide together: tcgen05.ld/st are
            // warp-collective (.sync.aligned), so the O rescale runs for the
            // whole warp when any of its rows needs it; a row that does not
            // keeps its reference (alpha = 1).
            const bool grow = mx > m_ref + kRescaleLog2;
            if (__any_sync(0xffffffffu, grow)) {
                // O_t and l are relative to m_ref; move them to mx (PV_t(j-1)
                // was issued before QK_t(j), whose completion was waited for).
                const float alpha = grow ? ex2(m_ref - mx) : 1.0f;   // 0 when m_ref = -inf
                if (j > 0) {
                    const float2 a2 = make_float2(alpha, alpha);
#pragma unroll
                    for (int c = 0; c < D / 32; ++c) {
                        uint32_t o[32];
                        tmem_ld_32x32b_x32(o_tmem + c * 32, o);
                        tmem_ld_wait_regs(o);
#pragma unroll
                        for (int e = 0; e < 16; ++e) {
                            const float2 v = __fmul2_rn(make_float2(__uint_as_float(o[2 * e]), __uint_as_float(o[2 * e + 1])), a2);
                            o[2 * e] = __float_as_uint(v.x);
                            o[2 * e + 1] = __float_as_uint(v.y);
                        }
                        tmem_st_32x32b_x32(o_tmem + c * 32, o);
                    }
                    tmem_st_wait();
                }
                l *= alpha;
                if (grow) m_ref = mx;
            }
            if constexpr (MOD) tmem_st_wait();
            // pass 2: P = 2^(s - m_ref), at most 2^kRescaleLog2, in f32, stored as
            // packed 16-bit pairs (key 2c in the low half of column c) into
            // columns 64..127 of S_t, which pass 1 has read.  A row that has seen
            // no key yet has m_ref = -inf and P = 2^-inf = 0.
            const float base = m_ref == -INFINITY ? 0.f : -m_ref;
            const float2 nm2 = make_float2(base, base);
            float2 sum2 = make_float2(0.f, 0.f);
            auto p_store = [&](const uint32_t (&r)[32], uint32_t col) {   // 32 keys -> 16 columns
                uint32_t pk[16];
#pragma unroll
                for (int u = 0; u < 16; ++u) {
                    const float2 x = __ffma2_rn(make_float2(__uint_as_float(r[2 * u]), __uint_as_float(r[2 * u + 1])),
                                                sl2, nm2);
                    const float2 pf = make_float2(ex2(x.x), ex2(x.y));
                    sum2 = __fadd2_rn(sum2, pf);
                    if constexpr (VF16) {
                        uint32_t out;
                        asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(out) : "f"(pf.y), "f"(pf.x));
                        pk[u] = out;
                    } else {
                        __nv_bfloat162 hv = __floats2bfloat162_rn(pf.x, pf.y);
                        pk[u] = *reinterpret_cast<uint32_t *>(&hv);
                    }
                }
                tmem_st_32x32b_x16(s_tmem + col, pk);
            };
            {
                uint32_t r0[2][32];
                tmem_ld_32x32b_x32(s_tmem + 0, r0[0]);
                tmem_ld_32x32b_x32(s_tmem + 32, r0[1]);
                p_store(rh[0], 96);
                p_store(rh[1], 112);
                tmem_ld_wait_regs(r0[0]);
                tmem_ld_wait_regs(r0[1]);
                if (!MOD && masked) {
#pragma unroll
                    for (int e = 0; e < 64; ++e)
                        if (e >= left) r0[e >> 5][e & 31] = __float_as_uint(-INFINITY);
                }
                p_store(r0[0], 64);
                p_store(r0[1], 80);
            }
            l += sum2.x + sum2.y;
            tmem_st_wait();             // P_t(j) in TMEM ...
            tc_fence_before();          // ... and ordered before the arrive for the MMA thread
            __syncwarp();
            if (lane == 0) mbar_arrive(&p_full[t]);
        }
        // O_t is final once the last P.V has completed; the ring is free once both tiles' have.
        for (int u = 0; u < 2; ++u)
            if (cnt[u] > 0) warp_wait(&pv_done[u], 0, p.flag, 312, &aborted);
        tc_fence_after();
    }

    __nv_bfloat16 *dst = p.out + (int64_t)(it.qs + token) * p.ldo + head * D;
    const bool any_o = warp >= 2 && (t ? cnt[1] : cnt[0]) > 0;   // warp-uniform
    if (p.splits == 1) {
        if (warp >= 2 && !aborted) {
            const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);   // a row that saw no key is 0, NaN stays
#pragma unroll
            for (int c = 0; c < D / 32; ++c) {
                uint32_t r[32];
                if (any_o) {
                    tmem_ld_32x32b_x32(o_tmem + c * 32, r);
                    tmem_ld_wait_regs(r);
                }
                if (!row_ok) continue;
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    uint32_t w[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        __nv_bfloat162 hv = __floats2bfloat162_rn(__uint_as_float(r[g * 8 + 2 * e]) * inv,
                                                                  __uint_as_float(r[g * 8 + 2 * e + 1]) * inv);
                        w[e] = any_o ? *reinterpret_cast<uint32_t *>(&hv) : 0u;
                    }
                    *reinterpret_cast<uint4 *>(dst + c * 32 + g * 8) = make_uint4(w[0], w[1], w[2], w[3]);
                }
            }
        }
    } else {
        // Join the cluster's partial results.  Every CTA publishes its rows'
        // (maximum, sum) and, weighted by them, its O in the ring's place; then
        // rank s sums columns [s D/S, (s+1) D/S) over the ranks, in their order.
        if (warp >= 2) s_ml[t * 128 + r_in] = make_float2(m_ref, l);
        cluster_sync();
        float w_own = 0.f;
        if (row_ok) {
            float top = -INFINITY;
            for (int s = 0; s < p.splits; ++s) top = fmaxf(top, ld_peer2(peer_addr(&s_ml[t * 128 + r_in], s)).x);
            float total = 0.f;
            for (int s = 0; s < p.splits; ++s) {
                const float2 ml = ld_peer2(peer_addr(&s_ml[t * 128 + r_in], s));
                total += ml.y * (ml.x == -INFINITY ? 0.f : ex2(ml.x - top));
            }
            // no key seen anywhere: all weights 0; a NaN sum stays NaN
            if (m_ref != -INFINITY) w_own = ex2(m_ref - top) / total;
            else if (l != l) w_own = l;
        }
        float4 *part = reinterpret_cast<float4 *>(sRing) + (t * 128 + r_in) * (D / 4);
        if (warp >= 2) {
#pragma unroll
            for (int c = 0; c < D / 32; ++c) {
                uint32_t r[32];
                if (any_o) {
                    tmem_ld_32x32b_x32(o_tmem + c * 32, r);
                    tmem_ld_wait_regs(r);
                }
                if (!row_ok) continue;
#pragma unroll
                for (int q = 0; q < 8; ++q) {   // 16-byte piece i of a row sits at i ^ (row % 8)
                    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
                    if (any_o && w_own != 0.f)
                        v = make_float4(__uint_as_float(r[4 * q]) * w_own, __uint_as_float(r[4 * q + 1]) * w_own,
                                        __uint_as_float(r[4 * q + 2]) * w_own, __uint_as_float(r[4 * q + 3]) * w_own);
                    part[(c * 8 + q) ^ (r_in & 7)] = v;
                }
            }
        }
        cluster_sync();
        if (row_ok && !aborted) {
            const int per = D / 4 / p.splits;   // 16-byte pieces of a row for each rank
            for (int i = split * per; i < (split + 1) * per; ++i) {
                float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
                for (int s = 0; s < p.splits; ++s) {
                    const float4 v = ld_peer4(peer_addr(&part[i ^ (r_in & 7)], s));
                    a.x += v.x;
                    a.y += v.y;
                    a.z += v.z;
                    a.w += v.w;
                }
                __nv_bfloat162 h0 = __floats2bfloat162_rn(a.x, a.y), h1 = __floats2bfloat162_rn(a.z, a.w);
                *reinterpret_cast<uint2 *>(dst + i * 4) =
                    make_uint2(*reinterpret_cast<uint32_t *>(&h0), *reinterpret_cast<uint32_t *>(&h1));
            }
        }
        cluster_sync();   // the peers have read this CTA's shared memory
    }

    tc_fence_before();
    __syncthreads();
    if (warp == 0) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

template <int D>
cudaError_t launch_packed(bool f16, bool mod, const CUtensorMap &tq, const CUtensorMap &tk, const CUtensorMap &tv,
                          const PackedParams &p, cudaStream_t st) {
    auto kern = f16 ? (mod ? packed_kernel<D, true, true> : packed_kernel<D, true, false>)
                    : (mod ? packed_kernel<D, false, true> : packed_kernel<D, false, false>);
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Smem<D>::BYTES);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)((int64_t)p.pairs * p.kv_heads * p.splits));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = Smem<D>::BYTES;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = p.splits;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kern, tq, tk, tv, p);
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                                  const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn encode_tiled() {
    static EncodeTiledFn fn = nullptr;
    static std::once_flag once;
    std::call_once(once, [] {
        void *f = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<EncodeTiledFn>(f);
    });
    return fn;
}

}  // namespace

bool packed_map(CUtensorMap *m, const void *ptr, int64_t rows, int heads, int d, int64_t ld, bool f16, int box_heads,
              int box_rows) {
    EncodeTiledFn fn = encode_tiled();
    if (!fn) return false;
    cuuint64_t dims[3] = {(cuuint64_t)d, (cuuint64_t)heads, (cuuint64_t)rows};
    cuuint64_t strides[2] = {(cuuint64_t)d * 2, (cuuint64_t)ld * 2};
    cuuint32_t box[3] = {64, (cuuint32_t)box_heads, (cuuint32_t)box_rows};
    cuuint32_t estr[3] = {1, 1, 1};
    return fn(m, f16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void *>(ptr),
              dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

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
    if (rows_q > 1 << 30 || rows_k > 1 << 30) return fail(ctx, LTX_ERR_UNSUPPORTED, "%s: more than 2^30 rows", w);
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
    const int group = heads / kv_heads, tokens = 128 / group;
    CUtensorMap tq, tk, tv;
    bool ok = packed_map(&tq, q_dev, rows_q, heads, head_dim, ldq, false, group, tokens);
    tk = tv = tq;   // never read without keys
    if (rows_k)
        ok = ok && packed_map(&tk, k_dev, rows_k, kv_heads, head_dim, ldk, false, 1, BKV) &&
             packed_map(&tv, v_dev, rows_k, kv_heads, head_dim, ldv, v_dtype == LTX_F16, 1, BKV);
    if (!ok) return fail(ctx, LTX_ERR_CUDA, "%s: cuTensorMapEncodeTiled failed", w);
    PackedParams p{static_cast<__nv_bfloat16 *>(out_dev), ldo, q_offsets_dev, k_offsets_dev, prefix_dev, slopes_dev,
                   docs, rows_q, rows_k, kv_heads, group, tokens, causal, 0, 1, scale, softcap, ctx->timeout_flag};
    // Few rows per document over many keys, by their averages (the host does
    // not see the offsets): the kernel whose tiles have keys as rows and whose
    // CTAs share every document.  Under some 512 keys its join and its start
    // cost more than it saves.
    const int some = std::min(docs, rows_q);
    const int64_t rows_per_doc = (int64_t)((rows_q + some - 1) / some) * group;
    if (rows_per_doc <= kMaxFewRows && rows_k / docs >= 512)
        return attention_packed_few(ctx, tk, tv, q_dev, ldq, p, heads, head_dim, v_dtype == LTX_F16, (int)rows_per_doc);
    // Pairs of query tiles over all documents: sum ceil(lq / per) <= (rows + docs (per - 1)) / per.
    const int64_t per = 2 * tokens;
    const int64_t pairs = (rows_q + (int64_t)some * (per - 1)) / per, items = pairs * kv_heads;
    if (items > 0x7fffffff / 8) return fail(ctx, LTX_ERR_UNSUPPORTED, "%s: more than 2^28 tiles", w);
    // Too few CTAs for the SMs: split the keys over a cluster, at least two K/V
    // tiles each if one document had them all.
    while (p.splits < 8 && items * p.splits * 2 <= ctx->sm_count && (int64_t)p.splits * 4 * BKV <= rows_k) p.splits *= 2;
    p.pairs = (int)pairs;
    const bool mod = softcap > 0.f || slopes_dev;
    const cudaError_t e = head_dim == 64 ? launch_packed<64>(v_dtype == LTX_F16, mod, tq, tk, tv, p, ctx->stream)
                                         : launch_packed<128>(v_dtype == LTX_F16, mod, tq, tk, tv, p, ctx->stream);
    return e == cudaSuccess ? LTX_OK : cuda_fail(ctx, e, w);
}
