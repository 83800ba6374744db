// Projection with one low-rank adapter per row:
//   out[m] = epilogue(x[m] W^T + c_a (x[m] A_a^T) B_a^T),  a = idx[m].
//
// Two kernels.  low_kernel forms low[m] = c_a x[m] A_a^T, a tenth of a percent
// to a few percent of the work, and keeps it as bf16 (f32 epilogues: two bf16
// parts).  project_kernel is the shared projection with low as more of its K
// loop: for every adapter a in a tile of tokens, one more block multiplies
// B_a's rows by low with the rows of other adapters set to 0, into the same
// f32 accumulator.  So an adapter costs rank / 64 blocks beside the K / 64
// that every tile has, whatever the order of the rows.
//
// Few tokens are bound by latency (8 x 4096 x 4096 with 8 adapters of rank 16: 16.8 us,
// 5.4 to read the weights), many by the tensor cores; f32 outputs carry the tensor
// cores' own rounding: each of k / 16 additions cuts what lies below the sum's last
// bit, 3.7e-6 relative at k 4096.
// Both work on D[128 weight rows, TN tokens]: weight rows are the MMA's M, so
// few tokens (TN 16) cost no wasted rows and the weights stream at HBM's rate,
// and many (TN 256) give the widest tile.
#include <cuda.h>

#include <algorithm>
#include <cmath>

#include "device_common.cuh"
#include "internal.hpp"
#include "kernels.hpp"

namespace ltx {

namespace {

constexpr int BM = 128;             // weight rows of a tile
constexpr int kMaxWords = LTX_MAX_ADAPTERS / 32;

struct AdapterParams {
    int m, n, k, rank, adapters, rank_blocks, parts, splits, m_tiles, n_tiles, group_m;
    int gate_rows;
    int early;                          // the projection starts while low is formed
    int tile_lanes, unit, low_stages;   // low_kernel: clusters per tile, adapters in one product, depth of its ring
    const int *idx, *gate_idx;
    const float *coeff, *bias, *gate;
    int64_t ldo, ld_gate;
    __nv_bfloat16 *low;   // [parts][m][rank_blocks * 64]
    void *out;
    int *flag;
};

// The threads of a list builder: one warp, or four on named barrier 1.
template <int NT>
__device__ __forceinline__ void builder_sync() {
    if constexpr (NT == 32) __syncwarp();
    else asm volatile("bar.sync 1, %0;" ::"n"(NT) : "memory");
}
__device__ __forceinline__ void cluster_sync() {
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// The address of this CTA's shared memory word `smem` in the CTA `rank` of the
// cluster, and a store there.
__device__ __forceinline__ uint32_t peer_addr(const void *smem, uint32_t rank) {
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(smem)), "r"(rank));
    return a;
}
__device__ __forceinline__ void st_peer(uint32_t addr, uint32_t v) {
    asm volatile("st.shared::cluster.b32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}

// Joins the partial sums of a cluster's `splits` CTAs: rank d receives tokens
// [d per, (d + 1) per), per = TN / splits, as part[source][per][128].  Each of
// four warps sends the 32 rows of TMEM that are its own, straight to the owners'
// shared memory (stores: nothing waits for a peer's answer); the first `count`
// tokens are wanted.
template <int TN>
__device__ __forceinline__ void send_partials(uint32_t acc, int row, const float *part, int splits, int rank, int count) {
    const int per = TN / splits, shift = __ffs(per) - 1;   // both powers of two
    uint32_t to = 0;
#pragma unroll 1
    for (int c = 0; c < count; c += 16) {
        uint32_t r[16];
        tmem_ld_32x32b_x16(acc + c, r);
        tmem_ld_wait_regs(r);
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            if (j == 0 || ((c + j) & (per - 1)) == 0)   // the next owner
                to = peer_addr(part + (rank * per + ((c + j) & (per - 1))) * BM + row, min(c + j, TN - 1) >> shift);
            if (c + j < TN) st_peer(to, r[j]);
            to += BM * 4;
        }
    }
}
// 8 tokens from j0 of this rank's share, summed over the sources in their order.
__device__ __forceinline__ void sum_partials(const float *part, int per, int splits, int j0, int row, float (&v)[8]) {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = 0.f;
    const float *at = part + j0 * BM + row;
    for (int s = 0; s < splits; ++s, at += per * BM)
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (j0 + j < per) v[j] += at[j * BM];
}

// The adapters of a tile of tokens.
template <int TN>
struct alignas(8) TileList {
    int count;
    uint16_t ids[TN];   // ascending
};
template <int TN>
struct ListScratch {
    uint32_t bits[kMaxWords];
    int sums[4];
    alignas(8) int16_t tok[TN + 8];   // each token's adapter, -1 for none (8 more: read in eights)
};

// Fills `l` and `s.tok` for tokens [m0, m0 + TN), by NT threads (tid of them).  An index beyond the pool counts as none and raises the
// flag.
template <int TN, int NT>
__device__ __forceinline__ void build_list(const AdapterParams &p, int m0, int tid, TileList<TN> &l,
                                           ListScratch<TN> &s) {
    constexpr int W = (kMaxWords + NT - 1) / NT;   // words of the bit set for each thread
    for (int i = tid; i < kMaxWords; i += NT) s.bits[i] = 0;
    builder_sync<NT>();
    for (int i = tid; i < TN; i += NT) {
        int a = m0 + i < p.m ? p.idx[m0 + i] : -1;
        if (a >= p.adapters) {
            report_index(p.flag, kErrBadAdapter);
            a = -1;
        }
        s.tok[i] = (int16_t)max(a, -1);
        if (a >= 0) atomicOr(&s.bits[a >> 5], 1u << (a & 31));
    }
    builder_sync<NT>();
    uint32_t w[W];
    int n = 0;
#pragma unroll
    for (int i = 0; i < W; ++i) n += __popc(w[i] = tid * W + i < kMaxWords ? s.bits[tid * W + i] : 0u);
    int incl = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, incl, o);
        if ((tid & 31) >= o) incl += v;
    }
    if ((tid & 31) == 31) s.sums[tid >> 5] = incl;
    builder_sync<NT>();
    int at = incl - n;
    for (int i = 0; i < (tid >> 5); ++i) at += s.sums[i];
    if (tid == NT - 1) l.count = at + n;
#pragma unroll
    for (int i = 0; i < W; ++i)
        for (uint32_t b = w[i]; b; b &= b - 1) l.ids[at++] = (uint16_t)((tid * W + i) * 32 + __ffs(b) - 1);
    builder_sync<NT>();
}

// Splits v into bf16 parts hi + lo: together 16 significant bits.
__device__ __forceinline__ void split_bf16(float v, __nv_bfloat16 &hi, __nv_bfloat16 &lo) {
    hi = __float2bfloat16_rn(v);
    lo = __float2bfloat16_rn(v - __bfloat162float(hi));
}

// ── low[m] = c_a x[m] A_a^T ──────────────────────────────────────────────────
//
// One cluster of `splits` CTAs per (tile of TN tokens, lane of its adapters):
// D[ranks, TN] = A . x^T over the cluster's shares of K, joined in the order of
// the ranks of the cluster.  One product takes `unit` adapters at once, their
// ranks behind one another in its 128 rows, so a mixed tile reads x once; with
// few tiles, lanes of CTAs share a tile's adapters instead.  Bound by latency for few
// tokens (some 7 us from launch to end), by reading x for many: 12288 x 4096, rank
// 64, takes 30 us, 3.4 TB/s.

// A stage is x's tile and the ranks in hand (a_bytes of them).  The product reads
// 128 rows from there whatever is behind (rows that nothing reads), so a pad ends
// the ring where they are fewer.  As many stages as the SM holds for the CTAs it
// gets: what bounds this kernel is the latency of x.
template <int TN>
struct LowCfg {
    static constexpr int X_BYTES = TN * 128, MAX_STAGES = 8;
    static constexpr int REST = 256 + (int)sizeof(TileList<TN>) + (int)sizeof(ListScratch<TN>);
    static constexpr int COLS = TN < 32 ? 32 : TN;
    __host__ __device__ static int ring(int a_bytes, int stages) {
        const int bytes = stages * (X_BYTES + a_bytes) + (BM * 128 - a_bytes), partials = TN * BM * 4;
        return bytes > partials ? bytes : partials;
    }
    static int bytes(int a_bytes, int stages) { return 1024 + ring(a_bytes, stages) + REST; }
};
constexpr int kLowThreads = 192;

template <int TN>
__global__ void __launch_bounds__(kLowThreads)
    low_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmX, AdapterParams p) {
    using C = LowCfg<TN>;
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    unsigned char *smem = reinterpret_cast<unsigned char *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const int box = min(p.rank, BM), a_bytes = p.unit * box * 128, stage = C::X_BYTES + a_bytes;   // rank % 8 == 0: whole swizzle blocks
    const int stages = p.low_stages;
    unsigned char *behind = smem + C::ring(a_bytes, stages);
    uint64_t *full = reinterpret_cast<uint64_t *>(behind), *empty = full + C::MAX_STAGES, *done = empty + C::MAX_STAGES;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(done + 1);
    TileList<TN> &list = *reinterpret_cast<TileList<TN> *>(behind + 256);
    ListScratch<TN> &scratch = *reinterpret_cast<ListScratch<TN> *>(behind + 256 + sizeof(TileList<TN>));
    float *part = reinterpret_cast<float *>(smem);   // partial sums in the ring's place

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int split = blockIdx.x % p.splits, job = blockIdx.x / p.splits;
    const int m0 = job / p.tile_lanes * TN;
    grid_dep_launch();
    if (threadIdx.x == 0) {
        tma_prefetch_desc(&tmA);
        tma_prefetch_desc(&tmX);
        for (int s = 0; s < stages; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        mbar_init(done, 1);
        fence_barrier_init();
    }
    if (warp == 0) {
        tmem_alloc(tmem_slot, C::COLS);
        tmem_relinquish();
    }
    if (warp >= 2) build_list<TN, 128>(p, m0, threadIdx.x - 64, list, scratch);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    bool aborted = false;

    const int kb = (p.k + 63) / 64;
    const int k0 = kb * split / p.splits, k1 = kb * (split + 1) / p.splits;
    const int m_blocks = (p.rank + BM - 1) / BM;   // unit is 1 where m_blocks is not
    const int units = (list.count + p.unit - 1) / p.unit * m_blocks;
    uint32_t it = 0, turn = 0;
    for (int u = job % p.tile_lanes; u < units; u += p.tile_lanes, ++turn) {
        const int first = u / m_blocks * p.unit, n_here = min(p.unit, list.count - first), r0 = u % m_blocks * BM;
        // an epilogue thread's row: rank r0 + row % box of adapter `mine`
        const int row = (warp & 3) * 32 + lane, slot = row / box, mine = slot < n_here ? list.ids[first + slot] : -2;
        const float c = warp >= 2 && mine >= 0 ? __ldg(p.coeff + mine) : 0.f;
        const uint32_t acc = tmem + ((uint32_t)((warp & 3) * 32) << 16);
        if (warp == 0) {
            if (elect_one())
                for (int kk = k0; kk < k1; ++kk, ++it) {
                    const int s = it % stages;
                    if (!mbar_wait(&empty[s], ((it / stages) & 1) ^ 1, p.flag, 401, &aborted)) break;
                    mbar_arrive_expect_tx(&full[s], n_here * box * 128 + TN * 128);
                    for (int i = 0; i < n_here; ++i)
                        tma_load_2d(smem + s * stage + C::X_BYTES + i * box * 128, &tmA, &full[s], kk * 64,
                                    list.ids[first + i] * p.rank + r0);
                    tma_load_2d(smem + s * stage, &tmX, &full[s], kk * 64, m0);
                }
        } else if (warp == 1) {
            if (elect_one()) {
                constexpr uint32_t idesc = idesc_f16(BM, TN, true);
                for (int kk = k0; kk < k1; ++kk, ++it) {
                    const int s = it % stages;
                    if (!mbar_wait(&full[s], (it / stages) & 1, p.flag, 402, &aborted)) break;
                    tc_fence_after();
                    const uint32_t bd = smem_u32(smem + s * stage), ad = bd + C::X_BYTES;
#pragma unroll
                    for (int q = 0; q < 4; ++q)
                        umma_f16_ss(tmem, sdesc_sw128(ad + q * 32, 16, 1024), sdesc_sw128(bd + q * 32, 16, 1024), idesc,
                                    kk > k0 || q ? 1u : 0u);
                    umma_commit(&empty[s]);
                }
                if (!aborted) umma_commit(done);
            }
        } else {
            warp_wait(done, turn & 1, p.flag, 403, &aborted);   // every load has been read
            tc_fence_after();
        }
        if (p.splits > 1) {   // the partials take the ring's place, in every CTA of the cluster
            cluster_sync();
            if (warp >= 2 && !aborted && (warp & 3) * 32 < n_here * box)
                send_partials<TN>(acc, row, part, p.splits, split, min(TN, p.m - m0));
            tc_fence_before();
            cluster_sync();
        }
        if (warp >= 2 && !aborted) {   // lanes run along the ranks
            const int ld = p.rank_blocks * 64, r = r0 + row - slot * box, tokens = TN / p.splits;
            const bool used = r < p.rank;
            __nv_bfloat16 *low = p.low + (int64_t)(m0 + split * tokens) * ld + r;
#pragma unroll 1
            for (int j0 = 0; j0 < tokens; j0 += 8) {
                float v[8];
                if (p.splits > 1) {
                    sum_partials(part, tokens, p.splits, j0, row, v);
                } else {
                    uint32_t u[8];
                    tmem_ld_32x32b_x8(acc + j0, u);
                    tmem_ld_wait_regs(u);
#pragma unroll
                    for (int j = 0; j < 8; ++j) v[j] = __uint_as_float(u[j]);
                }
                // adapters of the 8 tokens: 16 bits each
                int16_t of[8];
                *reinterpret_cast<uint2 *>(of) = reinterpret_cast<const uint2 *>(scratch.tok)[(split * tokens + j0) / 4];
                *reinterpret_cast<uint2 *>(of + 4) = reinterpret_cast<const uint2 *>(scratch.tok)[(split * tokens + j0) / 4 + 1];
                if (tokens < 4) of[0] = scratch.tok[split * tokens], of[1] = scratch.tok[split * tokens + 1];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    if (!used || j0 + j >= tokens || of[j] != mine) continue;
                    __nv_bfloat16 hi, lo;
                    split_bf16(v[j] * c, hi, lo);
                    low[(j0 + j) * ld] = hi;
                    if (p.parts == 2) low[(int64_t)p.m * ld + (j0 + j) * ld] = lo;
                }
            }
            tc_fence_before();
        }
        // the ring may be filled again, by TMA, once this CTA has read it; the
        // peers send into it only after the next unit's first cluster_sync
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncthreads();
        tc_fence_after();
    }
    if (aborted && warp == 0) {   // let the copies already issued land before the CTA exits
        bool a2 = false;
        for (uint32_t j = it > (uint32_t)stages ? it - stages : 0; j < it; ++j)
            mbar_wait(&full[j % stages], (j / stages) & 1, nullptr, 0, &a2);
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 0) {
        tc_fence_after();
        tmem_dealloc(tmem, C::COLS);
    }
}

// ── the projection ───────────────────────────────────────────────────────────
//
// 12 to 14 warps: 0 TMA, 1 MMA, 2-9 epilogue (two accumulators: the epilogue of one
// tile runs under the next one's products), from 10 on the builders: they list each
// tile's adapters and copy its rows of low, zeros for other adapters' tokens, into
// buffers beside the ring while the main blocks are multiplied.
// Few tiles: a cluster of `splits` CTAs shares a tile's blocks and joins its
// f32 sums through distributed shared memory in the order of the ranks.

template <int TN>
struct ProjCfg {
    static constexpr int A_BYTES = BM * 128, B_BYTES = TN * 128, STAGE = A_BYTES + B_BYTES;
    // up to 128 tokens: as deep as HBM's latency asks (96 KB and more), and no
    // deeper, so that low_kernel's CTAs run beside these
    static constexpr int STAGES = TN >= 128 ? 3 : TN == 64 ? 4 : TN == 32 ? 6 : 7;
    static constexpr int BUFS = TN <= 32 ? 4 : TN == 256 ? 2 : 3, BUILDERS = TN == 256 ? 2 : 3;   // for rows of low, and who copies them
    static constexpr int THREADS = (10 + BUILDERS) * 32;
    static constexpr int RING = STAGES * STAGE, BUF = RING, BAR = BUF + BUFS * B_BYTES;
    static constexpr int LIST = BAR + ((2 * STAGES + 9 + 2 * BUFS) * 8 + 8 + 15) / 16 * 16;
    static constexpr int BYTES = 1024 + LIST + 2 * (int)sizeof(TileList<TN>) + (int)sizeof(ListScratch<TN>);
    static constexpr int ACC = TN < 32 ? 32 : TN, COLS = 2 * ACC;
    static_assert(TN * BM * 4 <= RING, "the f32 partials fit the ring");
    static_assert(BYTES <= 232448, "shared memory exceeds the per-CTA limit");
};

// Tile -> (token tile, weight tile): groups of group_m token tiles, token tiles
// fastest inside a group.
__device__ __forceinline__ void tile_at(const AdapterParams &p, int t, int &mt, int &nt) {
    const int per = p.group_m * p.n_tiles, g = t / per, first = g * p.group_m, gm = min(p.group_m, p.m_tiles - first);
    const int r = t - g * per;
    mt = first + r % gm;
    nt = r / gm;
}

// One tile's blocks in order: `nk` of the main product with `na` of the adapters'
// spread evenly among them, so that the builder has time for each.
template <typename F, typename G>
__device__ __forceinline__ void blocks_in_order(int nk, int na, F main_block, G adapter_block) {
    int i = 0, next = na > 0 ? nk / (na + 1) : nk + 1;   // adapter block i comes before main block `next`
    for (int k = 0; k <= nk; ++k) {
        while (next == k) {
            if (!adapter_block(i)) return;
            next = ++i < na ? (i + 1) * nk / (na + 1) : nk + 1;
        }
        if (k < nk && !main_block(k)) return;
    }
}

// What the residual epilogue reads for 16 tokens from m on (count of them
// inside), weight row n: fetched ahead of its use.
struct Ahead {
    float x[16], g[16];
    // Called by whole warps; gidx: in lanes `at` to `at` + 15 the tokens' gate rows.
    __device__ __forceinline__ void fetch(const AdapterParams &p, int m, int count, int n, int gidx, int at) {
        const int64_t o = (int64_t)m * p.ldo + n;
        const bool in = n < p.n;
#pragma unroll
        for (int j = 0; j < 16; ++j) x[j] = in && j < count ? static_cast<const float *>(p.out)[o + j * p.ldo] : 0.f;
        if (!p.gate) return;
        const int g0 = __shfl_sync(0xffffffffu, gidx, at), l = threadIdx.x & 31;
        if (__all_sync(0xffffffffu, l < at || l >= at + 16 || gidx == g0)) {   // one row for all, as tokens of one request have
            const float one = in ? __ldg(p.gate + g0 * p.ld_gate + n) : 0.f;
#pragma unroll
            for (int j = 0; j < 16; ++j) g[j] = one;
            return;
        }
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            const int64_t row = __shfl_sync(0xffffffffu, gidx, at + j) * p.ld_gate;
            g[j] = in && j < count ? __ldg(p.gate + row + n) : 0.f;
        }
    }
};
// The gate rows of tokens m + lane.  One outside the gate takes its nearest and raises the flag.
__device__ __forceinline__ int gate_row(const AdapterParams &p, int m, int lane) {
    int g = p.gate && p.gate_idx && m + lane < p.m ? __ldg(p.gate_idx + m + lane) : 0;
    if ((unsigned)g >= (unsigned)p.gate_rows && p.gate) {
        report_index(p.flag, kErrBadGate);
        g = g < 0 ? 0 : p.gate_rows - 1;
    }
    return g;
}

// 16 tokens from m on (count of them inside), weight row n of this thread; a
// warp's threads hold 32 weight rows side by side.
template <int EPI>
__device__ __forceinline__ void finish16(const AdapterParams &p, int m, int count, int n, float bias, const float (&v)[16],
                                         const Ahead &h) {
    if (n >= p.n) return;
    if constexpr (EPI == LTX_EPI_BF16 || EPI == LTX_EPI_GELU_BF16) {
        __nv_bfloat16 *o = static_cast<__nv_bfloat16 *>(p.out) + (int64_t)m * p.ldo + n;
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            float y = v[j] + bias;
            // gelu_tanh(y) = y / (1 + e^(-2u)), u = sqrt(2/pi) (y + 0.044715 y^3)
            if constexpr (EPI == LTX_EPI_GELU_BF16)
                y = __fdividef(y, 1.f + ex2(-2.302208198f * y * (1.f + 0.044715f * y * y)));
            if (j < count) o[j * p.ldo] = __float2bfloat16_rn(y);
        }
    } else {
        float *o = static_cast<float *>(p.out) + (int64_t)m * p.ldo + n;
#pragma unroll
        for (int j = 0; j < 16; ++j)
            if (j < count) o[j * p.ldo] = EPI == LTX_EPI_RESID ? h.x[j] + (v[j] + bias) * (p.gate ? h.g[j] : 1.f) : v[j] + bias;
    }
}

// A tile's epilogue, every other 32 tokens of it from `side` on, by a warp whose
// lanes hold 32 weight rows.
template <int EPI>
struct TileEpilogue {
    Ahead cur, next;
    int gidx = 0;
    __device__ __forceinline__ void begin(const AdapterParams &p, int m0, int tokens, int n, int side, int lane) {
        if (EPI == LTX_EPI_RESID && side < tokens) {
            gidx = gate_row(p, m0 + side, lane);
            next.fetch(p, m0 + side, tokens - side, n, gidx, 0);
        }
    }
    __device__ __forceinline__ void run(const AdapterParams &p, uint32_t acc, int m0, int tokens, int n, int side, int lane,
                                        float bias) {
#pragma unroll 1
        for (int c = side; c < tokens; c += 64) {
            uint32_t r[32];
            tmem_ld_32x32b_x32(acc + c, r);
            int gnext = 0;
            if (EPI == LTX_EPI_RESID && c + 64 < tokens) gnext = gate_row(p, m0 + c + 64, lane);
            tmem_ld_wait_regs(r);
#pragma unroll
            for (int h = 0; h < 32; h += 16) {
                if (c + h >= tokens) break;
                if constexpr (EPI == LTX_EPI_RESID) {
                    cur = next;
                    const int to = h ? c + 64 : c + 16;
                    if (to < tokens) next.fetch(p, m0 + to, tokens - to, n, h ? gnext : gidx, h ? 0 : 16);
                }
                float v[16];
#pragma unroll
                for (int j = 0; j < 16; ++j) v[j] = __uint_as_float(r[h + j]);
                finish16<EPI>(p, m0 + c + h, tokens - c - h, n, bias, v, cur);
            }
            gidx = gnext;
        }
    }
};

// K steps (16 ranks each) of a rank block.
__device__ __forceinline__ int rank_steps(const AdapterParams &p, int rb) { return (min(p.rank - rb * 64, 64) + 15) >> 4; }

// One block of `low` for the product with adapter a's columns of B, by a warp:
// rows of ROWS tokens from m0 on, zeros for tokens of other adapters and behind
// the rank.  `which`: 64 ranks and the bf16 part.  Asynchronous (one commit group).
template <int ROWS>
__device__ __forceinline__ void copy_low(const AdapterParams &p, int a, int which, int m0, const int16_t *tok, int lane,
                                         unsigned char *to) {
    const int ld = p.rank_blocks * 64, rb = which / p.parts, c = lane & 7;   // a lane's 16-byte piece of each row
    const __nv_bfloat16 *src = p.low + (which % p.parts ? (int64_t)p.m * ld : 0) + (int64_t)m0 * ld + rb * 64 + c * 8;
    const bool in_rank = rb * 64 + c * 8 < p.rank;
    if (c < 2 * rank_steps(p, rb)) {   // what the product reads
        const uint32_t dst = smem_u32(to);
#pragma unroll 8
        for (int j = lane >> 3; j < ROWS; j += 4) {   // piece c of token j sits at c ^ (j % 8)
            const bool mine = in_rank && tok[j] == a;
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst + j * 128 + ((c ^ (j & 7)) << 4)),
                         "l"(mine ? src + (int64_t)j * ld : p.low), "r"(mine ? 16 : 0)
                         : "memory");
        }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
}

// Whether a barrier's phase has ended, without waiting for it.
__device__ __forceinline__ bool mbar_ready(uint64_t *bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity)
        : "memory");
    return ok;
}

// The builder warps, BUILDERS from warp 10 on: the first lists a tile's adapters,
// then they take its blocks of `low` in turn.  What a block costs is the latency
// of its copy and the way to the MMA thread and back, so several are on their way.
// tile(i): the i-th tile's first token, -1 behind the last; copy(a, which, m0, buffer);
// hand_over(buffer).
// BUFS >= BUILDERS: a builder is then never two rounds of a buffer ahead of the
// products, which the parity of a barrier could not tell from none.
template <int TN, int BUFS, int BUILDERS, typename Tile, typename Share, typename Copy, typename HandOver>
__device__ __forceinline__ void build_blocks(const AdapterParams &p, int who, int lane, TileList<TN> *lists, ListScratch<TN> &scratch,
                                             uint64_t *lfull, uint64_t *lempty, uint64_t *tfree, uint64_t *bempty, int code,
                                             bool &aborted, Tile tile, Share share, Copy copy, HandOver hand_over) {
    static_assert(BUFS >= BUILDERS);
    const int per_adapter = p.rank_blocks * p.parts;
    bool waited = false;
    uint32_t built = 0;   // blocks of the tiles before
    for (uint32_t i = 0; !aborted; ++i) {
        const int m0 = tile(i);
        if (m0 < 0) break;
        TileList<TN> &list = lists[i & 1];
        if (who == 0) {
            if (!warp_wait(&lempty[i & 1], ((i >> 1) & 1) ^ 1, p.flag, code, &aborted)) break;
            if (!warp_wait(tfree, (i & 1) ^ 1, p.flag, code, &aborted)) break;   // the others still read the last tile's tokens
            if (p.adapters) build_list<TN, 32>(p, m0, lane, list, scratch);
            else if (lane == 0) list.count = 0;
            mbar_arrive(&lfull[i & 1]);
            __syncwarp();
        } else if (!warp_wait(&lfull[i & 1], (i >> 1) & 1, p.flag, code, &aborted)) {
            break;
        }
        int a0, na;
        share(list.count, a0, na);
        if (na > 0 && !waited) {
            grid_dep_wait();
            waited = true;
        }
        int pending = -1;   // a block that is on its way
        for (int b = (who + BUILDERS - built % BUILDERS) % BUILDERS; b < na; b += BUILDERS) {
            const uint32_t at = built + b;
            const int buf = at % BUFS;
            uint64_t *bar = &bempty[buf];
            const uint32_t parity = ((at / BUFS) & 1) ^ 1;
            if (pending >= 0 && !__all_sync(0xffffffffu, mbar_ready(bar, parity))) {
                asm volatile("cp.async.wait_group 0;" ::: "memory");
                hand_over(pending);
                pending = -1;
            }
            if (!warp_wait(bar, parity, p.flag, code + 1, &aborted)) break;
            const int e = a0 + b;
            copy(list.ids[e / per_adapter], e % per_adapter, m0, buf);
            if (pending >= 0) {
                asm volatile("cp.async.wait_group 1;" ::: "memory");
                hand_over(pending);
            }
            pending = buf;
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        if (pending >= 0 && !aborted) hand_over(pending);
        built += na;
        __syncwarp();
        if (who != 0 && lane == 0) mbar_arrive(tfree);
    }
    grid_dep_wait();   // low_kernel has ended before this kernel does: the workspace is free behind it
}

template <int TN, int EPI>
__global__ void __launch_bounds__(ProjCfg<TN>::THREADS, 1)
    project_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmX,
                   const __grid_constant__ CUtensorMap tmB, AdapterParams p) {
    using C = ProjCfg<TN>;
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    unsigned char *smem = reinterpret_cast<unsigned char *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t *full = reinterpret_cast<uint64_t *>(smem + C::BAR), *empty = full + C::STAGES, *tfull = empty + C::STAGES;
    uint64_t *tempty = tfull + 2, *lfull = tempty + 2, *lempty = lfull + 2, *bfull = lempty + 2, *bempty = bfull + C::BUFS;
    uint64_t *tfree = bempty + C::BUFS;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(tfree + 1);
    TileList<TN> *lists = reinterpret_cast<TileList<TN> *>(smem + C::LIST);
    ListScratch<TN> &scratch = *reinterpret_cast<ListScratch<TN> *>(smem + C::LIST + 2 * sizeof(TileList<TN>));
    float *part = reinterpret_cast<float *>(smem);   // partial sums in the ring's place (splits > 1)

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int split = blockIdx.x % p.splits;
    const int first = blockIdx.x / p.splits, stride = gridDim.x / p.splits, tiles = p.m_tiles * p.n_tiles;
    const int kb = (p.k + 63) / 64;
    const int k0 = kb * split / p.splits, nk = kb * (split + 1) / p.splits - k0;
    const int per_adapter = p.rank_blocks * p.parts;
    // this rank's share of a tile's adapter blocks
    auto share = [&](int count, int &a0, int &na) {
        const int all = count * per_adapter;
        a0 = all * split / p.splits;
        na = all * (split + 1) / p.splits - a0;
    };
    // A cluster's one tile: the weights start to stream before anything else, and
    // the adapters' blocks follow them.
    const bool behind = p.splits > 1;
    int mt0, nt0;
    tile_at(p, first, mt0, nt0);
    uint32_t it = 0;   // ring uses of the producer or the MMA thread
    auto load_main = [&](int k, int mt, int nt, int s) {
        tma_load_2d(smem + s * C::STAGE, &tmW, &full[s], (k0 + k) * 64, nt * BM);
        tma_load_2d(smem + s * C::STAGE + C::A_BYTES, &tmX, &full[s], (k0 + k) * 64, mt * TN);
    };

    if (threadIdx.x == 0) {
        tma_prefetch_desc(&tmW);
        tma_prefetch_desc(&tmX);
        for (int s = 0; s < C::STAGES; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&tfull[i], 1);
            mbar_init(&tempty[i], 8);
            mbar_init(&lfull[i], 32);
            mbar_init(&lempty[i], 2);
        }
        for (int i = 0; i < C::BUFS; ++i) {
            mbar_init(&bfull[i], 32);
            mbar_init(&bempty[i], 1);
        }
        mbar_init(tfree, C::BUILDERS - 1);
        fence_barrier_init();
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");   // for the loads of this very thread
        if (behind)
            for (; it < (uint32_t)min(nk, C::STAGES); ++it) {
                mbar_arrive_expect_tx(&full[it], C::STAGE);
                load_main(it, mt0, nt0, it);
            }
    }
    float bias0 = 0.f;   // the cluster's epilogue: fetched now
    if (behind && warp >= 2 && warp < 6 && p.bias && nt0 * BM + (warp & 3) * 32 + lane < p.n)
        bias0 = __ldg(p.bias + nt0 * BM + (warp & 3) * 32 + lane);
    if (warp == 1) {
        tmem_alloc(tmem_slot, C::COLS);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    bool aborted = false;

    if (warp == 0) {
        if (lane == 0) {
            if (p.adapters) tma_prefetch_desc(&tmB);
            uint32_t i = 0;
            for (int t = first; t < tiles && !aborted; t += stride, ++i) {
                int mt, nt;
                tile_at(p, t, mt, nt);
                const TileList<TN> &list = lists[i & 1];
                auto take = [&](uint32_t bytes) {
                    const int s = it % C::STAGES;
                    if (!mbar_wait(&empty[s], ((it / C::STAGES) & 1) ^ 1, p.flag, 412, &aborted)) return -1;
                    mbar_arrive_expect_tx(&full[s], bytes);
                    ++it;
                    return s;
                };
                auto main_block = [&](int k) {
                    const int s = take(C::STAGE);
                    if (s < 0) return false;
                    load_main(k, mt, nt, s);
                    return true;
                };
                int a0, na;
                auto adapter_block = [&](int b) {
                    const int s = take(C::A_BYTES);
                    if (s < 0) return false;
                    const int e = a0 + b, rb = e % per_adapter / p.parts;
                    tma_load_2d(smem + s * C::STAGE, &tmB, &full[s], rb * 64, list.ids[e / per_adapter] * p.n + nt * BM);
                    return true;
                };
                if (behind)
                    for (int k = it; k < nk; ++k)
                        if (!main_block(k)) break;
                if (aborted || !mbar_wait(&lfull[i & 1], (i >> 1) & 1, p.flag, 411, &aborted)) break;
                share(list.count, a0, na);
                blocks_in_order(behind ? 0 : nk, na, main_block, adapter_block);
                mbar_arrive(&lempty[i & 1]);
            }
            if (aborted) {   // let the copies already issued land before the CTA exits
                bool a2 = false;
                for (uint32_t j = it > (uint32_t)C::STAGES ? it - C::STAGES : 0; j < it; ++j)
                    mbar_wait(&full[j % C::STAGES], (j / C::STAGES) & 1, nullptr, 0, &a2);
            }
        }
    } else if (warp == 1) {
        if (elect_one()) {
            constexpr uint32_t idesc = idesc_f16(BM, TN, true);
            uint32_t i = 0, built = 0;
            for (int t = first; t < tiles && !aborted; t += stride, ++i) {
                const uint32_t acc = i & 1;
                if (!mbar_wait(&tempty[acc], ((i >> 1) & 1) ^ 1, p.flag, 414, &aborted)) break;
                tc_fence_after();
                const uint32_t d = tmem + acc * C::ACC;
                uint32_t more = 0;
                auto multiply = [&](uint32_t b_addr, int steps) {
                    const int s = it % C::STAGES;
                    const uint32_t a_addr = smem_u32(smem + s * C::STAGE);
                    if (!b_addr) b_addr = a_addr + C::A_BYTES;
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        if (q >= steps) break;
                        umma_f16_ss(d, sdesc_sw128(a_addr + q * 32, 16, 1024), sdesc_sw128(b_addr + q * 32, 16, 1024), idesc,
                                    more);
                        more = 1;
                    }
                    umma_commit(&empty[s]);
                    ++it;
                };
                auto main_block = [&](int) {
                    if (!mbar_wait(&full[it % C::STAGES], (it / C::STAGES) & 1, p.flag, 415, &aborted)) return false;
                    tc_fence_after();
                    multiply(0, 4);
                    return true;
                };
                int a0, na;
                auto adapter_block = [&](int e) {
                    const int b = built % C::BUFS;
                    if (!mbar_wait(&full[it % C::STAGES], (it / C::STAGES) & 1, p.flag, 416, &aborted) ||
                        !mbar_wait(&bfull[b], (built / C::BUFS) & 1, p.flag, 417, &aborted))
                        return false;
                    tc_fence_after();
                    multiply(smem_u32(smem + C::BUF + b * C::B_BYTES), rank_steps(p, (a0 + e) % per_adapter / p.parts));
                    umma_commit(&bempty[b]);
                    ++built;
                    return true;
                };
                if (behind)
                    for (int k = 0; k < nk; ++k)
                        if (!main_block(k)) break;
                if (aborted || !mbar_wait(&lfull[acc], (i >> 1) & 1, p.flag, 413, &aborted)) break;
                share(lists[acc].count, a0, na);
                blocks_in_order(behind ? 0 : nk, na, main_block, adapter_block);
                if (aborted) break;
                mbar_arrive(&lempty[acc]);
                umma_commit(&tfull[acc]);
            }
        }
    } else if (warp >= 10) {
        build_blocks<TN, C::BUFS, C::BUILDERS>(
            p, warp - 10, lane, lists, scratch, lfull, lempty, tfree, bempty, 418, aborted,
            [&](uint32_t i) {
                const int t = first + (int)i * stride;
                if (t >= tiles) return -1;
                int mt, nt;
                tile_at(p, t, mt, nt);
                return mt * TN;
            },
            share,
            [&](int a, int which, int m0, int buf) {
                copy_low<TN>(p, a, which, m0, scratch.tok, lane, smem + C::BUF + buf * C::B_BYTES);
            },
            [&](int buf) {
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                mbar_arrive(&bfull[buf]);
            });
    } else {
        // warps 2-5 and 6-9 take every other 32 tokens of a tile
        const int quad = warp & 3, side = warp >= 6 ? 32 : 0;
        uint32_t i = 0;
        for (int t = first; t < tiles && !aborted; t += stride, ++i) {
            int mt, nt;
            tile_at(p, t, mt, nt);
            const uint32_t acc = i & 1;
            const int n = nt * BM + quad * 32 + lane, m0 = mt * TN;
            const float bias = p.bias && n < p.n ? p.bias[n] : 0.f;
            const int tokens = min(TN, p.m - m0);
            TileEpilogue<EPI> out;
            if (p.splits == 1) out.begin(p, m0, tokens, n, side, lane);   // under the products
            if (!warp_wait(&tfull[acc], (i >> 1) & 1, p.flag, 420, &aborted)) break;
            tc_fence_after();
            if (p.splits == 1)
                out.run(p, tmem + ((uint32_t)(quad * 32) << 16) + acc * C::ACC, m0, tokens, n, side, lane, bias);
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&tempty[acc]);
        }
    }

    if (p.splits > 1) {   // one tile per cluster; all its loads have been read
        const int row = (warp & 3) * 32 + lane, per = TN / p.splits, mt = mt0, nt = nt0;
        cluster_sync();   // the partials take the ring's place in every CTA
        if (warp >= 2 && warp < 6 && !aborted)
            send_partials<TN>(tmem + ((uint32_t)((warp & 3) * 32) << 16), row, part, p.splits, split,
                              min(TN, p.m - mt * TN));
        cluster_sync();
        if (warp >= 2 && warp < 6 && !aborted) {
            const int n = nt * BM + row;
            for (int j0 = 0; j0 < per; j0 += 16) {
                const int m = mt * TN + split * per + j0, count = min(per - j0, p.m - m);
                if (count <= 0) break;
                Ahead h;
                if (EPI == LTX_EPI_RESID) h.fetch(p, m, count, n, gate_row(p, m, lane), 0);
                float v[16], half[8];
#pragma unroll
                for (int q = 0; q < 16; q += 8) {
                    sum_partials(part, per, p.splits, j0 + q, row, half);
#pragma unroll
                    for (int j = 0; j < 8; ++j) v[q + j] = half[j];
                }
                finish16<EPI>(p, m, count, n, bias0, v, h);
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, C::COLS);
    }
}

// ── the projection, many tokens ──────────────────────────────────────────────
//
// The same with two SMs on one tile of 256 weight rows x 256 tokens, 1250 TFLOP/s for
// 4096 x 16384 x 4096 with low_kernel and rank 128 included, 1560 without adapters
// (cta_group::2): each CTA of a cluster of two loads its 128 weight rows and half
// of the tokens, so a block of 64 K costs an SM 32 KB of loads instead of 48 for
// the same products (one-SM tiles are held up by L2).  The even CTA's thread issues
// the products for both; both CTAs' loads count on its barriers.  Accumulators,
// epilogue and builder are each CTA's own: it holds its 128 weight rows for all 256
// tokens.
struct PairCfg {
    static constexpr int TOKENS = 256, HALF = 128;
    static constexpr int A_BYTES = BM * 128, B_BYTES = HALF * 128, STAGE = A_BYTES + B_BYTES;
    // Four builders and a shorter ring instead of two and six stages: a mixed tile's
    // blocks cost up to a third less (642 x 11552 x 960 with 12 adapters of rank 128:
    // 142 -> 100 us), tiles of one adapter a hundredth more.
    static constexpr int STAGES = 5, BUFS = 4, BUILDERS = 4, THREADS = (10 + BUILDERS) * 32;
    static constexpr int RING = STAGES * STAGE, BUF = RING, BAR = BUF + BUFS * B_BYTES;
    static constexpr int LIST = BAR + ((2 * STAGES + 9 + 2 * BUFS) * 8 + 8 + 15) / 16 * 16;
    static constexpr int BYTES = 1024 + LIST + 2 * (int)sizeof(TileList<TOKENS>) + (int)sizeof(ListScratch<TOKENS>);
    static_assert(BYTES <= 232448, "shared memory exceeds the per-CTA limit");
};

__device__ __forceinline__ void mbar_arrive_at(uint64_t *bar, uint32_t rank) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(peer_addr(bar, rank)) : "memory");
}
// mbar_wait for a barrier on which another CTA of the cluster arrives.
__device__ __forceinline__ bool mbar_wait_cluster(uint64_t *bar, uint32_t parity, int *flag, int code, bool *aborted) {
    if (*aborted) return false;
    uint64_t t0 = 0;
    for (;;) {
        uint32_t ok;
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(ok)
            : "r"(smem_u32(bar)), "r"(parity)
            : "memory");
        if (ok) return true;
        if (!t0) t0 = global_ns();
        else if (global_ns() - t0 > kWaitLimitNs) {
            atomicExch(flag, code);
            *aborted = true;
            return false;
        }
    }
}
// A load into this CTA's shared memory that counts on the barrier at `bar`, an
// address in the pair's even CTA.
__device__ __forceinline__ void pair_load(void *dst, const void *tmap, uint32_t bar, int x, int y) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(
            smem_u32(dst)),
        "l"(tmap), "r"(bar), "r"(x), "r"(y)
        : "memory");
}
__device__ __forceinline__ void pair_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate));
}
// Arrives on `bar` of both CTAs when the products issued so far are done.
__device__ __forceinline__ void pair_commit(uint64_t *bar) {
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(smem_u32(bar)),
        "h"((uint16_t)3)
        : "memory");
}

template <int EPI>
__global__ void __launch_bounds__(PairCfg::THREADS, 1)
    project_pair_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmX,
                        const __grid_constant__ CUtensorMap tmB, AdapterParams p) {
    using C = PairCfg;
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    unsigned char *smem = reinterpret_cast<unsigned char *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t *full = reinterpret_cast<uint64_t *>(smem + C::BAR), *empty = full + C::STAGES;
    uint64_t *tfull = empty + C::STAGES, *tempty = tfull + 2, *lfull = tempty + 2, *lempty = lfull + 2;
    uint64_t *bfull = lempty + 2, *bempty = bfull + C::BUFS;
    uint64_t *tfree = bempty + C::BUFS;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(tfree + 1);
    TileList<C::TOKENS> *lists = reinterpret_cast<TileList<C::TOKENS> *>(smem + C::LIST);
    ListScratch<C::TOKENS> &scratch = *reinterpret_cast<ListScratch<C::TOKENS> *>(smem + C::LIST + 2 * sizeof(TileList<C::TOKENS>));

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = blockIdx.x & 1;
    const int first = blockIdx.x / 2, stride = gridDim.x / 2, tiles = p.m_tiles * p.n_tiles;
    const int nk = (p.k + 63) / 64, per_adapter = p.rank_blocks * p.parts;
    if (threadIdx.x == 0) {
        tma_prefetch_desc(&tmW);
        tma_prefetch_desc(&tmX);
        if (p.adapters) tma_prefetch_desc(&tmB);
        for (int s = 0; s < C::STAGES; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&tfull[i], 1);
            mbar_init(&tempty[i], 16);
            mbar_init(&lfull[i], 32);
            mbar_init(&lempty[i], rank == 0 ? 2 : 1);
        }
        for (int i = 0; i < C::BUFS; ++i) {
            mbar_init(&bfull[i], 2);
            mbar_init(&bempty[i], 1);
        }
        mbar_init(tfree, C::BUILDERS - 1);
        fence_barrier_init();
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::);
    }
    tc_fence_before();
    cluster_sync();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    bool aborted = false;

    if (warp == 0) {
        if (lane == 0) {
            uint32_t it = 0, i = 0;
            for (int t = first; t < tiles && !aborted; t += stride, ++i) {
                int mt, nt;
                tile_at(p, t, mt, nt);
                const TileList<C::TOKENS> &list = lists[i & 1];
                if (!mbar_wait(&lfull[i & 1], (i >> 1) & 1, p.flag, 431, &aborted)) break;
                const int na = list.count * per_adapter, n0 = nt * 2 * BM + rank * BM;
                auto take = [&](uint32_t bytes) {   // bytes that both CTAs load
                    const int s = it % C::STAGES;
                    if (!mbar_wait(&empty[s], ((it / C::STAGES) & 1) ^ 1, p.flag, 432, &aborted)) return -1;
                    if (rank == 0) mbar_arrive_expect_tx(&full[s], bytes);
                    ++it;
                    return s;
                };
                blocks_in_order(
                    nk, na,
                    [&](int k) {
                        const int s = take(2 * C::STAGE);
                        if (s < 0) return false;
                        const uint32_t bar = peer_addr(&full[s], 0);
                        pair_load(smem + s * C::STAGE, &tmW, bar, k * 64, n0);
                        pair_load(smem + s * C::STAGE + C::A_BYTES, &tmX, bar, k * 64, mt * C::TOKENS + rank * C::HALF);
                        return true;
                    },
                    [&](int e) {
                        const int s = take(2 * C::A_BYTES);
                        if (s < 0) return false;
                        pair_load(smem + s * C::STAGE, &tmB, peer_addr(&full[s], 0), e % per_adapter / p.parts * 64,
                                  list.ids[e / per_adapter] * p.n + n0);
                        return true;
                    });
                mbar_arrive(&lempty[i & 1]);
            }
            if (aborted && rank == 0) {   // let the copies already issued land before the CTA exits
                bool a2 = false;
                for (uint32_t j = it > (uint32_t)C::STAGES ? it - C::STAGES : 0; j < it; ++j)
                    mbar_wait(&full[j % C::STAGES], (j / C::STAGES) & 1, nullptr, 0, &a2);
            }
        }
    } else if (warp == 1) {
        if (rank == 0 && elect_one()) {
            constexpr uint32_t idesc = idesc_f16(2 * BM, C::TOKENS, true);
            uint32_t it = 0, i = 0, built = 0;
            for (int t = first; t < tiles && !aborted; t += stride, ++i) {
                const uint32_t acc = i & 1;
                if (!mbar_wait(&lfull[acc], (i >> 1) & 1, p.flag, 433, &aborted)) break;
                const int na = lists[acc].count * per_adapter;
                if (!mbar_wait_cluster(&tempty[acc], ((i >> 1) & 1) ^ 1, p.flag, 435, &aborted)) break;
                tc_fence_after();
                const uint32_t d = tmem + acc * C::TOKENS;
                uint32_t more = 0;
                auto multiply = [&](uint32_t b_addr, int steps) {
                    const int s = it % C::STAGES;
                    if (!mbar_wait_cluster(&full[s], (it / C::STAGES) & 1, p.flag, 436, &aborted)) return false;
                    tc_fence_after();
                    const uint32_t a_addr = smem_u32(smem + s * C::STAGE);
                    if (!b_addr) b_addr = a_addr + C::A_BYTES;
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        if (q >= steps) break;
                        pair_mma(d, sdesc_sw128(a_addr + q * 32, 16, 1024), sdesc_sw128(b_addr + q * 32, 16, 1024), idesc, more);
                        more = 1;
                    }
                    pair_commit(&empty[s]);
                    ++it;
                    return true;
                };
                blocks_in_order(
                    nk, na, [&](int) { return multiply(0, 4); },
                    [&](int e) {
                        const int b = built % C::BUFS;
                        if (!mbar_wait_cluster(&bfull[b], (built / C::BUFS) & 1, p.flag, 437, &aborted) ||
                            !multiply(smem_u32(smem + C::BUF + b * C::B_BYTES), rank_steps(p, e % per_adapter / p.parts)))
                            return false;
                        pair_commit(&bempty[b]);
                        ++built;
                        return true;
                    });
                if (aborted) break;
                pair_commit(&tfull[acc]);
                mbar_arrive(&lempty[acc]);
            }
        }
    } else if (warp >= 10) {
        build_blocks<C::TOKENS, C::BUFS, C::BUILDERS>(
            p, warp - 10, lane, lists, scratch, lfull, lempty, tfree, bempty, 438, aborted,
            [&](uint32_t i) {
                const int t = first + (int)i * stride;
                if (t >= tiles) return -1;
                int mt, nt;
                tile_at(p, t, mt, nt);
                return mt * C::TOKENS;
            },
            [&](int count, int &a0, int &na) {
                a0 = 0;
                na = count * per_adapter;
            },
            [&](int a, int which, int m0, int buf) {
                copy_low<C::HALF>(p, a, which, m0 + rank * C::HALF, scratch.tok + rank * C::HALF, lane, smem + C::BUF + buf * C::B_BYTES);
            },
            [&](int buf) {
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive_at(&bfull[buf], 0);
            });
    } else {
        // warps 2-5 and 6-9 take every other 32 tokens of a tile
        const int quad = warp & 3, side = warp >= 6 ? 32 : 0;
        uint32_t i = 0;
        for (int t = first; t < tiles && !aborted; t += stride, ++i) {
            int mt, nt;
            tile_at(p, t, mt, nt);
            const uint32_t acc = i & 1;
            const int n = nt * 2 * BM + rank * BM + quad * 32 + lane, m0 = mt * C::TOKENS, tokens = min(C::TOKENS, p.m - m0);
            const float bias = p.bias && n < p.n ? p.bias[n] : 0.f;
            TileEpilogue<EPI> out;
            out.begin(p, m0, tokens, n, side, lane);   // under the products
            if (!warp_wait(&tfull[acc], (i >> 1) & 1, p.flag, 440, &aborted)) break;
            tc_fence_after();
            out.run(p, tmem + ((uint32_t)(quad * 32) << 16) + acc * C::TOKENS, m0, tokens, n, side, lane, bias);
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_at(&tempty[acc], 0);
        }
    }

    tc_fence_before();
    cluster_sync();   // neither CTA exits, or frees its TMEM, while the other still uses it
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
    }
}

// ── host side ────────────────────────────────────────────────────────────────

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

// bf16 [rows, cols] with row stride ld (elements), boxes of 64 x box_rows.
bool make_map(CUtensorMap *m, const void *ptr, int64_t rows, int64_t cols, int64_t ld, int box_rows) {
    EncodeTiledFn fn = encode_tiled();
    if (!fn) return false;
    cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
    cuuint64_t strides[1] = {(cuuint64_t)ld * 2};
    cuuint32_t box[2] = {64, (cuuint32_t)box_rows};
    cuuint32_t estr[2] = {1, 1};
    return fn(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void *>(ptr), dims, strides, box, estr,
              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// `most`: the largest dynamic shared memory any call of the kernel asks for.
template <typename K, typename... Args>
cudaError_t launch(const ltx_ctx *ctx, K kern, int grid, int threads, int smem, int most, int cluster, bool dependent,
                   const Args &...args) {
    cudaError_t e = allow_smem(ctx, reinterpret_cast<const void *>(kern), most);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = ctx->stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cluster;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = dependent ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kern, args...);
}

// Shares of K over a cluster: doubled while the CTAs stay within `room` and
// each keeps at least four blocks of K.
int splits_for(int64_t jobs, int room, int kb) {
    int s = 1;
    while (s < 8 && jobs * s * 2 <= room && kb >= s * 2 * 4) s *= 2;
    return s;
}

template <int TN>
cudaError_t run_low(const ltx_ctx *ctx, AdapterParams p, const CUtensorMap &ta, const CUtensorMap &tx) {
    const int tiles = (p.m + TN - 1) / TN, room = (p.rank <= 64 ? 3 : 2) * ctx->sm_count;   // CTAs at once, as their shared memory allows
    p.splits = splits_for(tiles, room, (p.k + 63) / 64);
    // the SMs left over share the adapters of a tile; what one takes goes together
    const int blocks = (p.rank + BM - 1) / BM, most = std::min({p.adapters, TN, p.m});
    p.tile_lanes = std::max(1, std::min(room / (tiles * p.splits), most * blocks));
    p.unit = blocks > 1 ? 1 : std::min(BM / p.rank, (most + p.tile_lanes - 1) / p.tile_lanes);
    using C = LowCfg<TN>;
    const int grid = tiles * p.tile_lanes * p.splits, a_bytes = p.unit * std::min(p.rank, BM) * 128;
    // beside project_kernel's CTA (up to 128 tokens), or by themselves
    const int here = std::max(1, std::min(3, (grid + ctx->sm_count - 1) / ctx->sm_count));
    const int budget = p.m <= 128 ? 72 << 10 : ((227 << 10) / here - 2048);
    p.low_stages = C::MAX_STAGES;
    while (p.low_stages > 2 && C::bytes(a_bytes, p.low_stages) > budget) --p.low_stages;
    return launch(ctx, low_kernel<TN>, grid, kLowThreads, C::bytes(a_bytes, p.low_stages), C::bytes(BM * 128, C::MAX_STAGES), p.splits,
                  false, ta, tx, p);
}

// A weight within 48 MB stays in L2: then the weight tiles of one token tile run
// back to back.  Otherwise as many token tiles go together as keep their rows of x
// within 48 MB, and the weights stream once per group.
int group_of(const AdapterParams &p, int tokens) {
    constexpr int64_t kPanel = 48 << 20;
    return (int64_t)p.n * p.k * 2 <= kPanel ? 1
                                            : (int)std::max<int64_t>(1, std::min<int64_t>(p.m_tiles, kPanel / ((int64_t)tokens * p.k * 2)));
}

template <int TN>
cudaError_t run_project(const ltx_ctx *ctx, AdapterParams p, int epilogue, const CUtensorMap &tw, const CUtensorMap &tx,
                        const CUtensorMap &tb) {
    const int sms = ctx->sm_count;
    p.m_tiles = (p.m + TN - 1) / TN;
    p.n_tiles = (p.n + BM - 1) / BM;
    const int64_t tiles = (int64_t)p.m_tiles * p.n_tiles;
    p.splits = splits_for(tiles, sms, (p.k + 63) / 64);
    p.group_m = group_of(p, TN);
    const int grid = p.splits > 1 ? (int)tiles * p.splits : (int)std::min<int64_t>(tiles, sms);
    auto go = [&](auto kern) {
        return launch(ctx, kern, grid, ProjCfg<TN>::THREADS, ProjCfg<TN>::BYTES, ProjCfg<TN>::BYTES, p.splits, p.early, tw, tx, tb, p);
    };
    switch (epilogue) {
    case LTX_EPI_BF16: return go(project_kernel<TN, LTX_EPI_BF16>);
    case LTX_EPI_GELU_BF16: return go(project_kernel<TN, LTX_EPI_GELU_BF16>);
    case LTX_EPI_F32: return go(project_kernel<TN, LTX_EPI_F32>);
    default: return go(project_kernel<TN, LTX_EPI_RESID>);
    }
}

cudaError_t run_pair(const ltx_ctx *ctx, AdapterParams p, int epilogue, const CUtensorMap &tw, const CUtensorMap &tx,
                     const CUtensorMap &tb) {
    p.m_tiles = (p.m + PairCfg::TOKENS - 1) / PairCfg::TOKENS;
    p.n_tiles = (p.n + 2 * BM - 1) / (2 * BM);
    p.splits = 1;
    p.group_m = group_of(p, PairCfg::TOKENS);
    const int grid = 2 * (int)std::min<int64_t>((int64_t)p.m_tiles * p.n_tiles, ctx->sm_count / 2);
    auto go = [&](auto kern) {
        return launch(ctx, kern, grid, PairCfg::THREADS, PairCfg::BYTES, PairCfg::BYTES, 2, p.early, tw, tx, tb, p);
    };
    switch (epilogue) {
    case LTX_EPI_BF16: return go(project_pair_kernel<LTX_EPI_BF16>);
    case LTX_EPI_GELU_BF16: return go(project_pair_kernel<LTX_EPI_GELU_BF16>);
    case LTX_EPI_F32: return go(project_pair_kernel<LTX_EPI_F32>);
    default: return go(project_pair_kernel<LTX_EPI_RESID>);
    }
}

// Tokens of a tile.  Up to 64: the least that holds them all, so that the weights
// stream once.  More: the widest tile (the fewest bytes per product) that still
// makes work for two SMs in five; a cluster's joined sums and a builder's wider
// copies cost more than they save below that.  Measured, us at 256 / 128 / 64 / 32 /
// 16 tokens: 153 x 600 x 448 - / 25 / 18 / 16 / 14; 512 x 1024 x 2048 41 / 22 / 19 /
// 24 / 32; 200 x 4096 x 4096 29 / 27 / 32 / 44 / 65; 512 x 4096 x 4096 35 / 40 / 50 / 80.
int tokens_for(int m, int n, int sms) {
    if (m <= 64) return m <= 16 ? 16 : m <= 32 ? 32 : 64;
    for (int t = m <= 128 ? 128 : 256; t > 16; t /= 2)
        if ((int64_t)((m + t - 1) / t) * ((n + BM - 1) / BM) * 5 >= sms * 2) return t;
    return 16;
}

}  // namespace

}  // namespace ltx

extern "C" int ltx_gemm_adapters(ltx_ctx *ctx, const ltx_adapter_gemm *args) {
    using namespace ltx;
    if (!ctx) return LTX_ERR_INVALID_ARG;
    const char *w = "gemm_adapters";
    if (!args) return fail(ctx, LTX_ERR_INVALID_ARG, "%s: null arguments", w);
    const auto &[x_dev, w_dev, out_dev, bias_dev, gate_dev, gate_idx_dev, adapter_idx_dev, lora_a_dev, lora_b_dev, coeff_dev,
                 ldx, ldw, ldo, ld_gate, m, n, k, epilogue, adapters, rank, gate_rows] = *args;
    if (epilogue < LTX_EPI_BF16 || epilogue > LTX_EPI_RESID)
        return fail(ctx, LTX_ERR_INVALID_ARG, "%s: bad epilogue %d", w, epilogue);
    if (m < 0 || n < 1 || k < 1 || k > 1 << 24 || m > 1 << 30 || n > 1 << 30)
        return fail(ctx, LTX_ERR_SHAPE, "%s: %d x %d x %d", w, m, n, k);
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
    if (epilogue == LTX_EPI_RESID && gate_dev && (ld_gate < n || gate_rows < 1))
        return fail(ctx, LTX_ERR_SHAPE, "%s: %d gate rows of %lld, shorter than n or none", w, gate_rows, (long long)ld_gate);
    DeviceGuard guard(ctx);
    if ((int64_t)adapters * n > 0x7fffffff || (int64_t)((m + 15) / 16) * ((n + BM - 1) / BM) > 0x7fffffff / 8)
        return fail(ctx, LTX_ERR_UNSUPPORTED, "%s: %d x %d with %d adapters is too large", w, m, n, adapters);
    AdapterParams p{};
    p.m = m;
    p.n = n;
    p.k = k;
    p.rank = rank;
    p.adapters = adapters;
    p.rank_blocks = (rank + 63) / 64;
    p.parts = epilogue == LTX_EPI_F32 || epilogue == LTX_EPI_RESID ? 2 : 1;
    p.idx = adapter_idx_dev;
    p.gate_idx = gate_idx_dev;
    p.coeff = coeff_dev;
    p.bias = bias_dev;
    p.gate = gate_dev;
    p.gate_rows = gate_rows;
    p.ldo = ldo;
    p.ld_gate = ld_gate;
    p.out = out_dev;
    p.flag = ctx->timeout_flag;
    int tn = tokens_for(m, n, ctx->sm_count);
    // enough 256 x 256 tiles for every pair of SMs
    const bool pair = tn == 256 && (int64_t)((m + 255) / 256) * ((n + 255) / 256) * 2 > ctx->sm_count;
    // One SM's tile of 256 tokens has smem for two builders only: where a mixed tile
    // may have more than a quarter of a block for the adapters per block of K, 128
    // tokens.  us at 256 / 128: 136 x 15432 x 256 with 9 of rank 64, gated residual
    // 59 / 42; 160 x 12000 x 640, 8 of 8 34 / 32; 256 x 16384 x 4096, 4 of 64 56 / 70.
    if (tn == 256 && !pair && (int64_t)std::min(adapters, 256) * p.rank_blocks * p.parts * 4 > (k + 63) / 64) tn = 128;
    const int tl = std::min(tn, 64);
    // The waits of a projection that starts early count low_kernel's time in their 2 s.
    // That takes 6e-13 s per value of x and product (tiles of all different adapters of
    // rank 256, A from HBM), so beyond a tenth of the limit the projection comes after it.
    p.early = adapters && (int64_t)m * k * std::min(adapters, tl) * ((rank + BM - 1) / BM) <= (int64_t)1 << 38;
    CUtensorMap tw, tx, txl, ta, tb;
    bool ok = make_map(&tw, w_dev, n, k, ldw, BM) && make_map(&tx, x_dev, m, k, ldx, pair ? 128 : tn);
    ta = tb = txl = tx;
    if (adapters)
        ok = ok && make_map(&txl, x_dev, m, k, ldx, tl) &&
             make_map(&ta, lora_a_dev, (int64_t)adapters * rank, k, k, std::min(rank, BM)) &&
             make_map(&tb, lora_b_dev, (int64_t)adapters * n, rank, rank, BM);
    if (!ok) return fail(ctx, LTX_ERR_CUDA, "%s: cuTensorMapEncodeTiled failed", w);
    void *low = nullptr;
    cudaError_t e = cudaSuccess;
    if (adapters) {
        const int rc = work_alloc(ctx, (size_t)p.parts * m * p.rank_blocks * 128, &low);
        if (rc != LTX_OK) return rc;
        p.low = static_cast<__nv_bfloat16 *>(low);
        e = tl == 16   ? run_low<16>(ctx, p, ta, txl)
            : tl == 32 ? run_low<32>(ctx, p, ta, txl)
                       : run_low<64>(ctx, p, ta, txl);
    }
    if (e == cudaSuccess)
        e = pair        ? run_pair(ctx, p, epilogue, tw, tx, tb)
            : tn == 16  ? run_project<16>(ctx, p, epilogue, tw, tx, tb)
            : tn == 32  ? run_project<32>(ctx, p, epilogue, tw, tx, tb)
            : tn == 64  ? run_project<64>(ctx, p, epilogue, tw, tx, tb)
            : tn == 128 ? run_project<128>(ctx, p, epilogue, tw, tx, tb)
                        : run_project<256>(ctx, p, epilogue, tw, tx, tb);
    const int rc = work_free(ctx, low);
    return e == cudaSuccess ? rc : cuda_fail(ctx, e, w);
}
