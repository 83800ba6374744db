// Attention over packed documents for few query rows per document (new tokens
// over a long cache): bound by reading K and V once.
//
// With N = 16, 32 or 64 rows (tokens x the heads of a key head's group) the
// products are turned round so that the keys fill the MMA's 128 rows:
//   S^T[128 keys, N] = K_tile . Q^T        (A = K, K-major; B = Q)
//   O^T[D, N]      += V_tile^T . P^T       (A = V read M-major; B = P)
// A softmax thread holds one key and the N scores of the rows for it, so a tile
// costs 128 N exponentials, not 128 x 128.  A row's maximum lies across threads;
// it is looked at only when some score exceeds the reference by 2^8 (one vote
// per tile), and sums stay per thread until the document's end.
//
// The work is the line of all K/V tiles of all (document, key head, row tile)
// items, cut into equal lengths, one per CTA, whatever the documents' lengths.
// An item inside one length is finished there; what a cut divides leaves f32
// partials (O, maximum, sum) that a second kernel joins in the order of the CTAs.
//
// Tiles go from a document's last keys to its first: with a bias by distance the
// largest scores come first and the reference hardly moves (upwards, a steep
// slope moved it in every tile, 1500 of a tile's 3400 cycles).
//
// Warps: 0 TMA, 1 MMA (the next tile's S^T is issued before this tile's O^T),
// 2-5 softmax.  All waits are bounded (2 s).
//
// 16 requests of one token x 32/8 heads x 128 over 70001 keys, with slopes: 59 us,
// 4.9 TB/s with the join (a copy runs at 6.5); the first loads wait for the cut of
// the line, the join for the last CTA.
#include <algorithm>

#include "attention_packed.cuh"
#include "internal.hpp"

namespace ltx {

namespace {

constexpr int kFewThreads = 192;
constexpr int kScores = 2;      // S^T buffers in TMEM, P buffers in shared memory
constexpr int kMinTiles = 2;    // a CTA's least length

template <int D, int N>
struct FewSmem {
    static constexpr int TILE = 128 * D * 2, HALF = 128 * 64 * 2;
    static constexpr int Q_BYTES = N * D * 2, P_BYTES = N * 256;
    static constexpr int SLOTS = D == 64 ? (N == 64 ? 9 : 10) : N == 64 ? 4 : 6;
    // D 64: the 128-row O^T product reads 64 columns past a V tile (rows of O^T
    // that nothing reads); behind the last slot lie Q, P and a pad.
    static constexpr int RING = 0, Q = SLOTS * TILE, P = Q + 2 * Q_BYTES;
    static constexpr int PAD = D == 64 ? HALF : 0;
    static constexpr int BAR = P + kScores * P_BYTES + PAD;
    static constexpr int ROWS = BAR + 512;                     // per-row words below
    static constexpr int BYTES = ROWS + N * 4 * (4 + 4 + 4) + 1024;
    static_assert(BYTES <= 232448, "shared memory exceeds the per-CTA limit");
};

// Work of document i: K/V tiles over its row tiles and key heads.  A document
// without keys still has one per row tile, for its zeros.
struct DocWork {
    int qs, lq, ks, lk, tiles, row_tiles;
    __device__ __forceinline__ void load(const PackedParams &p, int i) {
        int e;
        doc_span(p.qo, i, p.rows_q, p.flag, qs, e);
        lq = e - qs;
        doc_span(p.ko, i, p.rows_k, p.flag, ks, e);
        lk = e - ks;
        tiles = max(1, (lk + BKV - 1) / BKV);
        row_tiles = (lq + p.tile_tokens - 1) / p.tile_tokens;
    }
    __device__ __forceinline__ int64_t all(const PackedParams &p) const { return (int64_t)row_tiles * p.kv_heads * tiles; }
};

// A place on the line of tiles: document, item (key head, row tile) and tile.
struct Place {
    DocWork d;
    int doc, tile;
    int64_t item;
};

// A cut of the line, by one warp: finds the length every CTA gets (`per`), the
// tiles of the line from the cut before CTA `c` on (0: none) and the place there.
__device__ __forceinline__ void cut_line(const PackedParams &p, int c, int ctas, int lane, int64_t &per, int64_t &left,
                                         Place &at) {
    int64_t whole = 0, n = 0, incl = 0;
    DocWork d{};
    auto scan = [&](int base) {   // 32 documents from base: work n of this lane's, and up to it
        d = DocWork{};
        n = 0;
        if (base + lane < p.docs) {
            d.load(p, base + lane);
            n = d.all(p);
        }
        incl = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t v = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += v;
        }
    };
    for (int base = 0; base < p.docs; base += 32) {
        scan(base);
        whole += __shfl_sync(0xffffffffu, incl, 31);
    }
    per = max((int64_t)kMinTiles, (whole + ctas - 1) / ctas);
    const int64_t from = per * c;
    left = max((int64_t)0, whole - from);
    if (left == 0) return;
    int64_t before = 0;
    for (int base = 0; base < p.docs; base += 32) {
        if (p.docs > 32) scan(base);
        const unsigned hit = __ballot_sync(0xffffffffu, before + incl > from);
        if (hit) {
            const int src = __ffs(hit) - 1;
            if (lane == src) {
                const int64_t in = from - before - (incl - n);
                at.d = d;
                at.doc = base + lane;
                at.item = in / d.tiles;
                at.tile = (int)(in - at.item * d.tiles);
            }
            at.d.qs = __shfl_sync(0xffffffffu, at.d.qs, src);
            at.d.lq = __shfl_sync(0xffffffffu, at.d.lq, src);
            at.d.ks = __shfl_sync(0xffffffffu, at.d.ks, src);
            at.d.lk = __shfl_sync(0xffffffffu, at.d.lk, src);
            at.d.tiles = __shfl_sync(0xffffffffu, at.d.tiles, src);
            at.d.row_tiles = __shfl_sync(0xffffffffu, at.d.row_tiles, src);
            at.doc = base + src;
            at.item = __shfl_sync(0xffffffffu, at.item, src);
            at.tile = __shfl_sync(0xffffffffu, at.tile, src);
            return;
        }
        before += __shfl_sync(0xffffffffu, incl, 31);
    }
}

// A CTA's stretch of one item.
struct Piece {
    int kvh, token0, t0, t1;   // first token of the row tile; K/V tiles [t0, t1)
};
// Runs body(document, piece) over a CTA's length, by whole warps.
template <typename F>
__device__ __forceinline__ void for_pieces(const PackedParams &p, Place at, int64_t length, F body) {
    DocWork d = at.d;
    while (length > 0) {
        const int take = (int)min((int64_t)(d.tiles - at.tile), length);
        const int kvh = (int)(at.item / d.row_tiles);
        body(d, at.doc, Piece{kvh, (int)(at.item - (int64_t)kvh * d.row_tiles) * p.tile_tokens, at.tile, at.tile + take});
        length -= take;
        at.tile = 0;
        if (length > 0 && ++at.item == (int64_t)d.row_tiles * p.kv_heads) {
            at.item = 0;
            do d.load(p, ++at.doc);
            while (d.row_tiles == 0);
        }
    }
}

__device__ __forceinline__ void softmax_sync() { asm volatile("bar.sync 1, 128;" ::: "memory"); }
// Whether any of the 128 softmax threads says so.
__device__ __forceinline__ bool softmax_any(bool v) {
    uint32_t r;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\t"
        "barrier.cta.red.or.pred q, 1, 128, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
        : "=r"(r)
        : "r"((uint32_t)v)
        : "memory");
    return r != 0;
}

template <int N>
__device__ __forceinline__ void load_columns(uint32_t taddr, float (&v)[N]) {
    uint32_t r[N / 16][16];
#pragma unroll
    for (int c = 0; c < N / 16; ++c) tmem_ld_32x32b_x16(taddr + c * 16, r[c]);
#pragma unroll
    for (int c = 0; c < N / 16; ++c) tmem_ld_wait_regs(r[c]);
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = __uint_as_float(r[i / 16][i % 16]);
}

// A row's value over the 32 lanes of a warp, for N rows that every lane holds: each
// step halves the rows a lane goes on with, so N - 1 exchanges do for all of them.
// A lane ends with first_row in v[0] (N 64: and the row behind it in v[1]).
template <int N>
__device__ __forceinline__ int first_row(int lane) { return N == 16 ? lane >> 1 : N / 32 * lane; }
template <int N, typename F>
__device__ __forceinline__ void over_lanes(float (&v)[N], int lane, F join) {
    int n = N;
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        const bool up = lane & o;
        if (n == 1) {
            v[0] = join(v[0], __shfl_xor_sync(0xffffffffu, v[0], o));
        } else {
            n /= 2;
#pragma unroll
            for (int i = 0; i < N / 2; ++i)
                if (i < n) {
                    const float keep = up ? v[i + n] : v[i], give = up ? v[i] : v[i + n];
                    v[i] = join(keep, __shfl_xor_sync(0xffffffffu, give, o));
                }
        }
    }
}
// The same into a warp's N words of shared memory.
template <int N, typename F>
__device__ __forceinline__ void over_lanes_to(float (&v)[N], int lane, float *to, F join) {
    over_lanes<N>(v, lane, join);
#pragma unroll
    for (int i = 0; i < (N == 64 ? 2 : 1); ++i) to[first_row<N>(lane) + i] = v[i];
}

// Partials: slot 0 of a CTA for the item it goes on with, slot 1 for the one it begins.
struct Partials {
    float *o;     // [ctas * 2][N][D]
    float2 *ml;   // [ctas * 2][N]
};

template <int D, bool VF16, int N>
__global__ void __launch_bounds__(kFewThreads, 1)
    few_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
               const __grid_constant__ CUtensorMap tmV, PackedParams p, Partials part) {
    using L = FewSmem<D, N>;
    constexpr int kSlots = L::SLOTS;
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    unsigned char *smem = reinterpret_cast<unsigned char *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t *bars = reinterpret_cast<uint64_t *>(smem + L::BAR);
    uint64_t *slot_full = bars, *slot_empty = slot_full + kSlots;
    uint64_t *q_full = slot_empty + kSlots, *q_empty = q_full + 2, *o_full = q_empty + 2, *o_empty = o_full + 2;
    uint64_t *s_full = o_empty + 2, *s_empty = s_full + kScores, *p_full = s_empty + kScores, *p_empty = p_full + kScores;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(p_empty + kScores);
    Place *s_place = reinterpret_cast<Place *>(tmem_slot + 2);
    static_assert((2 * kSlots + 8 + 4 * kScores) * 8 + 8 + sizeof(Place) + 8 <= 512, "barriers and place exceed their block");
    int64_t *s_len = reinterpret_cast<int64_t *>(s_place + 1);
    // per row: first keys it sees, key it stands beside, slope log2e, reference maximum, what it moves by or 1 / sum;
    // [4][N] warps' maxima or sums
    int *r_lim = reinterpret_cast<int *>(smem + L::ROWS), *r_place = r_lim + N;
    float *r_slope = reinterpret_cast<float *>(r_place + N), *r_ref = r_slope + N, *r_alpha = r_ref + N, *r_warp = r_alpha + N;
    int64_t *r_out = reinterpret_cast<int64_t *>(r_warp + 4 * N);   // where the row goes, -1 for none

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    grid_dep_launch();
    if (warp == 1) {
        int64_t per, left;
        Place at{};
        cut_line(p, blockIdx.x, gridDim.x, lane, per, left, at);
        if (lane == 0) {
            *s_place = at;
            *s_len = min(per, left);
        }
    }
    if (threadIdx.x == 0) {
        tma_prefetch_desc(&tmQ);
        tma_prefetch_desc(&tmK);
        tma_prefetch_desc(&tmV);
        for (int s = 0; s < kSlots; ++s) {
            mbar_init(&slot_full[s], 1);
            mbar_init(&slot_empty[s], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&q_full[i], 1);
            mbar_init(&q_empty[i], 1);
            mbar_init(&o_full[i], 1);
            mbar_init(&o_empty[i], 4);
        }
        for (int i = 0; i < kScores; ++i) {
            mbar_init(&s_full[i], 1);
            mbar_init(&s_empty[i], 4);
            mbar_init(&p_full[i], 128);
            mbar_init(&p_empty[i], 1);
        }
        fence_barrier_init();
    }
    constexpr int kCols = N == 16 ? 64 : N == 32 ? 128 : 256;   // 2 S^T + 2 O^T buffers of N columns
    if (warp == 0) {
        tmem_alloc(tmem_slot, kCols);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;   // S^T 0, 1, then O^T 0, 1
    const Place start = *s_place;
    const int64_t length = *s_len;
    const int per_tile = p.tile_tokens;
    bool aborted = false;

    if (warp == 0) {
        uint32_t issued = 0, piece = 0;
        for_pieces(p, start, length, [&](const DocWork &d, int, const Piece &w) {
            if (d.lk == 0) return;
            if (!aborted && elect_one()) {
                const int qb = piece & 1;
                if (mbar_wait(&q_empty[qb], ((piece >> 1) & 1) ^ 1, p.flag, 321, &aborted)) {
                    mbar_arrive_expect_tx(&q_full[qb], D / 64 * per_tile * p.group * 128);
                    for (int x = 0; x < D; x += 64)
                        tma_load_3d(smem + L::Q + qb * L::Q_BYTES + x / 64 * N * 128, &tmQ, &q_full[qb], x, w.kvh * p.group,
                                    d.qs + w.token0);
                    for (int s = 0; s < 2 * (w.t1 - w.t0); ++s, ++issued) {   // K_j, V_j, the last tile first
                        const int slot = issued % kSlots;
                        if (!mbar_wait(&slot_empty[slot], ((issued / kSlots) & 1) ^ 1, p.flag, 322, &aborted)) break;
                        mbar_arrive_expect_tx(&slot_full[slot], L::TILE);
                        for (int x = 0; x < D; x += 64)
                            tma_load_3d(smem + L::RING + slot * L::TILE + x / 64 * L::HALF, (s & 1) ? &tmV : &tmK,
                                        &slot_full[slot], x, w.kvh, d.ks + (w.t1 - 1 - (s >> 1)) * BKV);
                    }
                }
                if (aborted) {   // let the copies already issued land before the CTA exits
                    bool a2 = false;
                    mbar_wait(&q_full[qb], (piece >> 1) & 1, nullptr, 0, &a2);
                    a2 = false;
                    for (uint32_t s = issued > (uint32_t)kSlots ? issued - kSlots : 0; s < issued; ++s)
                        mbar_wait(&slot_full[s % kSlots], (s / kSlots) & 1, nullptr, 0, &a2);
                }
            }
            // every lane goes on from the elected one's count
            issued = __reduce_max_sync(0xffffffffu, issued);
            aborted = __any_sync(0xffffffffu, aborted);
            ++piece;
        });
    } else if (warp == 1) {
        uint32_t used = 0, tile = 0, piece = 0;
        constexpr uint32_t idesc_s = idesc_f16(128, N, true);
        constexpr uint32_t idesc_o = idesc_f16(128, N, !VF16) | (1u << 15);   // A = V, M-major
        for_pieces(p, start, length, [&](const DocWork &d, int, const Piece &w) {
            if (d.lk == 0) return;
            const int n = w.t1 - w.t0;
            if (!aborted && elect_one()) {
                const int qb = piece & 1;
                const uint32_t q_addr = smem_u32(smem + L::Q + qb * L::Q_BYTES);
                const uint32_t o_tmem = tmem + (kScores + qb) * N;
                auto scores = [&](int j) {   // S^T of tile j of the piece
                    const uint32_t i = tile + j, sb = i % kScores, slot = (used + 2 * j) % kSlots;
                    if (!mbar_wait(&slot_full[slot], ((used + 2 * j) / kSlots) & 1, p.flag, 323, &aborted) ||
                        !mbar_wait(&s_empty[sb], ((i / kScores) & 1) ^ 1, p.flag, 324, &aborted))
                        return false;
                    tc_fence_after();
                    const uint32_t k_addr = smem_u32(smem + L::RING + slot * L::TILE);
#pragma unroll
                    for (int kk = 0; kk < D / 16; ++kk)
                        umma_f16_ss(tmem + sb * N, sdesc_sw128(k_addr + (kk >> 2) * L::HALF + (kk & 3) * 32, 16, 1024),
                                    sdesc_sw128(q_addr + (kk >> 2) * N * 128 + (kk & 3) * 32, 16, 1024), idesc_s, kk ? 1u : 0u);
                    umma_commit(&slot_empty[slot]);
                    umma_commit(&s_full[sb]);
                    return true;
                };
                bool ok = mbar_wait(&q_full[qb], (piece >> 1) & 1, p.flag, 325, &aborted) &&
                          mbar_wait(&o_empty[qb], ((piece >> 1) & 1) ^ 1, p.flag, 326, &aborted) && scores(0);
                for (int j = 0; ok && j < n; ++j) {
                    if (j + 1 < n) {
                        if (!scores(j + 1)) break;
                    }
                    if (j + 2 >= n && j + 1 >= n) umma_commit(&q_empty[qb]);   // Q's last use is issued
                    const uint32_t i = tile + j, pb = i % kScores, slot = (used + 2 * j + 1) % kSlots;
                    if (!mbar_wait(&p_full[pb], (i / kScores) & 1, p.flag, 327, &aborted) ||
                        !mbar_wait(&slot_full[slot], ((used + 2 * j + 1) / kSlots) & 1, p.flag, 328, &aborted))
                        break;
                    tc_fence_after();
                    const uint32_t v_addr = smem_u32(smem + L::RING + slot * L::TILE);
                    const uint32_t p_addr = smem_u32(smem + L::P + pb * L::P_BYTES);
#pragma unroll
                    for (int kk = 0; kk < BKV / 16; ++kk)   // 16 keys
                        umma_f16_ss(o_tmem, sdesc_sw128(v_addr + kk * 2048, L::HALF, 1024),
                                    sdesc_sw128(p_addr + (kk >> 2) * N * 128 + (kk & 3) * 32, 16, 1024), idesc_o,
                                    j > 0 || kk > 0 ? 1u : 0u);
                    umma_commit(&slot_empty[slot]);
                    umma_commit(&p_empty[pb]);
                    if (j + 1 == n) umma_commit(&o_full[qb]);
                }
            }
            aborted = __any_sync(0xffffffffu, aborted);
            used += 2 * n;
            tile += n;
            ++piece;
        });
    } else {
        // The barriers among these warps are met by all of them in every tile,
        // whatever became of a wait.
        const int quad = warp & 3, key = quad * 32 + lane;
        const uint32_t lanes = (uint32_t)(quad * 32) << 16;
        const bool modified = p.softcap > 0.f || p.slopes;
        ScoreMod mod{};
        const float sl2 = p.scale * kLog2e, over = p.softcap > 0.f ? p.scale / p.softcap : sl2;
        mod.scale = make_float2(over, over);
        mod.cap2 = p.softcap * kLog2e;
        uint32_t used = 0, tile = 0, piece = 0;
        for_pieces(p, start, length, [&](const DocWork &d, int doc, const Piece &w) {
            softmax_sync();   // the row words of the piece before have been read
            if (key < N) {
                const int token = w.token0 + key / p.group;
                const bool ok = key < per_tile * p.group && token < d.lq;
                const int prefix = p.causal && p.prefix ? min(max(p.prefix[doc], 0), d.lk) : 0;
                const Item it{d.qs, d.lq, d.ks, d.lk, 0, doc, w.kvh, 0};
                r_lim[key] = ok ? limit_of(p, it, token, prefix) : 0;
                r_place[key] = key_beside(d.lq, d.lk, token);
                r_slope[key] = ok && p.slopes ? p.slopes[w.kvh * p.group + key % p.group] * kLog2e : 0.f;
                r_ref[key] = -INFINITY;
                r_out[key] = ok ? (int64_t)(d.qs + token) * p.ldo + (w.kvh * p.group + key % p.group) * D : -1;
            }
            softmax_sync();
            const int n = d.lk == 0 ? 0 : w.t1 - w.t0;
            const int qb = piece & 1;
            const uint32_t o_tmem = tmem + lanes + (kScores + qb) * N;
            float l[N];
#pragma unroll
            for (int r = 0; r < N; ++r) l[r] = 0.f;
            for (int j = 0; j < n; ++j) {
                const uint32_t i = tile + j, b = i % kScores, ph = (i / kScores) & 1;
                const int kv = (w.t1 - 1 - j) * BKV + key;   // this thread's key in the document
                float y[N];
                if (warp_wait(&s_full[b], ph, p.flag, 331, &aborted)) {
                    tc_fence_after();
                    load_columns<N>(tmem + lanes + b * N, y);
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&s_empty[b]);
                } else {
#pragma unroll
                    for (int r = 0; r < N; ++r) y[r] = 0.f;
                }
                bool over = false;
#pragma unroll
                for (int r4 = 0; r4 < N; r4 += 4) {
                    const int4 lim = *reinterpret_cast<const int4 *>(r_lim + r4);
                    const float4 ref = *reinterpret_cast<const float4 *>(r_ref + r4);
                    const float4 slope = *reinterpret_cast<const float4 *>(r_slope + r4);
                    const int4 place = *reinterpret_cast<const int4 *>(r_place + r4);
                    const float slopes[4] = {slope.x, slope.y, slope.z, slope.w};
                    const int places[4] = {place.x, place.y, place.z, place.w};
                    const int lims[4] = {lim.x, lim.y, lim.z, lim.w};
                    const float refs[4] = {ref.x, ref.y, ref.z, ref.w};
                    if (modified) {
#pragma unroll
                        for (int e = 0; e < 4; e += 2) {
                            const float2 v = mod(make_float2(y[r4 + e], y[r4 + e + 1]), make_float2(slopes[e], slopes[e + 1]),
                                                 make_float2((float)(places[e] - kv), (float)(places[e + 1] - kv)));
                            y[r4 + e] = v.x;
                            y[r4 + e + 1] = v.y;
                        }
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        float &v = y[r4 + e];
                        if (!modified) v *= sl2;
                        if (kv >= lims[e]) v = -INFINITY;
                        over |= v > refs[e] + kRescaleLog2;
                    }
                }
                if (softmax_any(over)) {
                    // Some row's maximum outgrew its reference: each row's over the
                    // tile, by warps and then all; rows that grew move to it.
                    float m[N];
#pragma unroll
                    for (int r = 0; r < N; ++r) m[r] = y[r];
                    over_lanes_to<N>(m, lane, r_warp + quad * N, [](float a, float b) { return fmaxf(a, b); });
                    softmax_sync();
                    if (key < N) {
                        const float top = fmaxf(fmaxf(r_warp[key], r_warp[N + key]), fmaxf(r_warp[2 * N + key], r_warp[3 * N + key]));
                        const float ref = r_ref[key];
                        const bool grew = top > ref + kRescaleLog2;
                        r_alpha[key] = grew ? ex2(ref - top) : 1.f;
                        if (grew) r_ref[key] = top;
                    }
                    // O^T is stable once the tile before has been added to it
                    if (j > 0) warp_wait(&p_empty[(i - 1) % kScores], ((i - 1) / kScores) & 1, p.flag, 332, &aborted);
                    softmax_sync();
                    if (j > 0) {
                        tc_fence_after();
                        float o[N];
                        load_columns<N>(o_tmem, o);
#pragma unroll
                        for (int r4 = 0; r4 < N; r4 += 4) {
                            const float4 a = *reinterpret_cast<const float4 *>(r_alpha + r4);
                            const float as[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                l[r4 + e] *= as[e];
                                o[r4 + e] *= as[e];
                            }
                        }
#pragma unroll
                        for (int c = 0; c < N; c += 16) {
                            uint32_t u[16];
#pragma unroll
                            for (int r = 0; r < 16; ++r) u[r] = __float_as_uint(o[c + r]);
                            tmem_st_32x32b_x16(o_tmem + c, u);
                        }
                        tmem_st_wait();
                        tc_fence_before();
                    }
                }
                // P (row r, key): 16 bytes of 8 keys at their place ^ (r % 8), 64 keys to a block of N rows
                warp_wait(&p_empty[b], ph ^ 1, p.flag, 333, &aborted);
                unsigned char *pw = smem + L::P + b * L::P_BYTES + (key >> 6) * N * 128 + (key & 7) * 2;
                const int chunk = (key & 63) >> 3;
#pragma unroll
                for (int r4 = 0; r4 < N; r4 += 4) {
                    const float4 ref = *reinterpret_cast<const float4 *>(r_ref + r4);
                    const float refs[4] = {ref.x, ref.y, ref.z, ref.w};
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int r = r4 + e;
                        // a row that has seen no key has reference -inf and all of its scores too
                        const float v = ex2(y[r] - (refs[e] == -INFINITY ? 0.f : refs[e]));
                        unsigned char *to = pw + r * 128 + ((chunk ^ (r & 7)) << 4);
                        // bf16: the sum takes what the product takes, so a row that one key rules is exact;
                        // f16's half step is an eighth of the output's
                        if constexpr (VF16) {
                            l[r] += v;
                            *reinterpret_cast<__half *>(to) = __float2half_rn(v);
                        } else {
                            const __nv_bfloat16 h = __float2bfloat16_rn(v);
                            l[r] += __bfloat162float(h);
                            *reinterpret_cast<__nv_bfloat16 *>(to) = h;
                        }
                    }
                }
                // V rows behind the document's end: P is 0 there, but 0 times another document's NaN is not
                if (kv >= d.lk) {
                    const uint32_t s = used + 2 * j + 1;
                    mbar_wait(&slot_full[s % kSlots], (s / kSlots) & 1, p.flag, 334, &aborted);
                    unsigned char *v = smem + L::RING + (s % kSlots) * L::TILE + key * 128;
#pragma unroll
                    for (int x = 0; x < D / 64; ++x)
#pragma unroll
                        for (int c = 0; c < 8; ++c) *reinterpret_cast<uint4 *>(v + x * L::HALF + c * 16) = make_uint4(0, 0, 0, 0);
                }
                __syncwarp();
                aborted = __any_sync(0xffffffffu, aborted);
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                mbar_arrive(&p_full[b]);
            }
            // the rows' sums over all keys, and O^T: lane = column d of the head
            over_lanes_to<N>(l, lane, r_warp + quad * N, [](float a, float b) { return a + b; });
            softmax_sync();
            const bool whole = w.t0 == 0 && w.t1 == d.tiles;
            const int64_t slot = 2 * blockIdx.x + (w.t0 == 0);
            if (key < N) {
                const float total = r_warp[key] + r_warp[N + key] + r_warp[2 * N + key] + r_warp[3 * N + key];
                r_alpha[key] = total == 0.f ? 0.f : 1.f / total;   // no key seen: 0; a NaN sum stays NaN
                if (!whole) part.ml[slot * N + key] = make_float2(r_ref[key], total);
            }
            if (n > 0) {
                if (warp_wait(&o_full[qb], (piece >> 1) & 1, p.flag, 335, &aborted)) {
                    tc_fence_after();
                    load_columns<N>(o_tmem, l);
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&o_empty[qb]);
                }
            } else {
#pragma unroll
                for (int r = 0; r < N; ++r) l[r] = 0.f;
            }
            softmax_sync();
            if (key < D && !aborted) {
                if (whole) {
#pragma unroll
                    for (int r4 = 0; r4 < N; r4 += 4) {
                        const float4 inv = *reinterpret_cast<const float4 *>(r_alpha + r4);
                        const float is[4] = {inv.x, inv.y, inv.z, inv.w};
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const int64_t to = r_out[r4 + e];
                            if (to >= 0) p.out[to + key] = __float2bfloat16_rn(is[e] == 0.f ? 0.f : l[r4 + e] * is[e]);
                        }
                    }
                } else {
                    float *o = part.o + slot * N * D + key;   // rows that nothing reads included
#pragma unroll
                    for (int r = 0; r < N; ++r) o[r * D] = l[r];
                }
            }
            if (n > 0) {
                used += 2 * n;
                tile += n;
                ++piece;
            }
        });
    }

    tc_fence_before();
    __syncthreads();
    if (warp == 0) {
        tc_fence_after();
        tmem_dealloc(tmem, kCols);
    }
}

// Joins the items that a cut of the line divides.  Block (c - 1, y) looks at the
// cut before CTA c: if it is the first inside its item, the partials of CTA c - 1
// (slot 1) and of the CTAs from c on that reach into the item (slot 0) are one
// result, and the block joins rows 4y to 4y + 3 of it: a warp weighs a row's
// partials, then each warp adds up every fourth of them for all four rows, with
// the loads of a step in flight together, and the four sums become one.
constexpr int kJoinRows = 4, kMaxCtas = 256;
template <int D, int N>
__global__ void __launch_bounds__(128) few_join_kernel(PackedParams p, Partials part, int ctas) {
    __shared__ Place s_place;
    __shared__ int64_t s_per;
    __shared__ int s_go;
    __shared__ float s_weight[kMaxCtas][kJoinRows], s_total[kJoinRows], s_acc[4][kJoinRows][D];
    const int c = blockIdx.x + 1, row0 = blockIdx.y * kJoinRows, warp = threadIdx.x / 32, lane = threadIdx.x & 31;
    if (warp == 0) {
        int64_t per, left;
        Place at{};
        cut_line(p, c, ctas, lane, per, left, at);
        if (lane == 0) {
            s_place = at;
            s_per = per;
            s_go = left > 0 && at.tile > 0 && at.tile <= per;
        }
    }
    __syncthreads();
    grid_dep_wait();   // also where there is nothing to do: this kernel's end stands for the attention's too
    if (!s_go) return;
    const DocWork d = s_place.d;
    const int kvh = (int)(s_place.item / d.row_tiles);
    const int token0 = (int)(s_place.item - (int64_t)kvh * d.row_tiles) * p.tile_tokens;
    // the item goes on for tiles - tile more tiles from this cut
    const int more = (int)((d.tiles - s_place.tile + s_per - 1) / s_per);
    const int rows = min(p.tile_tokens, d.lq - token0) * p.group;
    if (row0 >= rows) return;
    auto slot = [&](int i) { return (int64_t)(i == 0 ? 2 * (c - 1) + 1 : 2 * (c - 1 + i)) * N + row0; };
    float top = -INFINITY, total = 0.f;
    const bool row_ok = row0 + warp < rows;   // a row behind the last has no partials
    for (int i = lane; row_ok && i <= more; i += 32) top = fmaxf(top, part.ml[slot(i) + warp].x);
#pragma unroll
    for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    for (int i = lane; i <= more; i += 32) {
        const float2 ml = row_ok ? part.ml[slot(i) + warp] : make_float2(-INFINITY, 0.f);
        const float f = ml.x == -INFINITY ? 0.f : ex2(ml.x - top);
        s_weight[i][warp] = f;
        total += ml.y * f;
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
    if (lane == 0) s_total[warp] = total;
    __syncthreads();
    float acc[kJoinRows][D / 32] = {};
#pragma unroll 2
    for (int i = warp; i <= more; i += 4) {
        const float *o = part.o + slot(i) * D + lane;
#pragma unroll
        for (int r = 0; r < kJoinRows; ++r) {
            const float f = s_weight[i][r];
#pragma unroll
            for (int x = 0; x < D / 32; ++x)
                if (f != 0.f) acc[r][x] += o[r * D + x * 32] * f;
        }
    }
#pragma unroll
    for (int r = 0; r < kJoinRows; ++r)
#pragma unroll
        for (int x = 0; x < D / 32; ++x) s_acc[warp][r][x * 32 + lane] = acc[r][x];
    __syncthreads();
    if (!row_ok) return;
    const int r = row0 + warp;
    __nv_bfloat16 *out = p.out + (int64_t)(d.qs + token0 + r / p.group) * p.ldo + (kvh * p.group + r % p.group) * D + lane;
#pragma unroll
    for (int x = 0; x < D / 32; ++x) {
        const int at = x * 32 + lane;
        const float v = s_acc[0][warp][at] + s_acc[1][warp][at] + s_acc[2][warp][at] + s_acc[3][warp][at];
        out[x * 32] = __float2bfloat16_rn(s_total[warp] == 0.f ? 0.f : v / s_total[warp]);
    }
}

template <int D, int N>
int run_few(ltx_ctx *ctx, const CUtensorMap &tq, const CUtensorMap &tk, const CUtensorMap &tv, const PackedParams &p,
            bool v_f16) {
    const int ctas = std::min(ctx->sm_count, kMaxCtas);
    void *work = nullptr;
    const size_t o_bytes = (size_t)ctas * 2 * N * D * 4;
    int rc = work_alloc(ctx, o_bytes + (size_t)ctas * 2 * N * 8, &work);
    if (rc != LTX_OK) return rc;
    const Partials part{static_cast<float *>(work), reinterpret_cast<float2 *>(static_cast<char *>(work) + o_bytes)};
    auto kern = v_f16 ? few_kernel<D, true, N> : few_kernel<D, false, N>;
    cudaError_t e = allow_smem(ctx, reinterpret_cast<const void *>(kern), FewSmem<D, N>::BYTES);
    if (e == cudaSuccess) {
        kern<<<ctas, kFewThreads, FewSmem<D, N>::BYTES, ctx->stream>>>(tq, tk, tv, p, part);
        e = cudaGetLastError();
    }
    if (e == cudaSuccess && ctas > 1) {
        cudaLaunchConfig_t cfg{};
        cfg.gridDim = dim3(ctas - 1, N / kJoinRows);
        cfg.blockDim = dim3(128);
        cfg.stream = ctx->stream;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[0].val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        e = cudaLaunchKernelEx(&cfg, few_join_kernel<D, N>, p, part, ctas);
    }
    rc = work_free(ctx, work);
    return e == cudaSuccess ? rc : cuda_fail(ctx, e, "attention_packed");
}

}  // namespace

int attention_packed_few(ltx_ctx *ctx, const CUtensorMap &tk, const CUtensorMap &tv, const void *q, int64_t ldq,
                         const PackedParams &params, int heads, int head_dim, bool v_f16, int rows_per_doc) {
    const int n = rows_per_doc <= 16 ? 16 : rows_per_doc <= 32 ? 32 : 64;
    PackedParams p = params;
    p.tile_tokens = n / p.group;
    CUtensorMap tq;
    if (!packed_map(&tq, q, p.rows_q, heads, head_dim, ldq, false, p.group, p.tile_tokens))
        return fail(ctx, LTX_ERR_CUDA, "attention_packed: cuTensorMapEncodeTiled failed");
    if (head_dim == 64)
        return n == 16   ? run_few<64, 16>(ctx, tq, tk, tv, p, v_f16)
               : n == 32 ? run_few<64, 32>(ctx, tq, tk, tv, p, v_f16)
                         : run_few<64, 64>(ctx, tq, tk, tv, p, v_f16);
    return n == 16   ? run_few<128, 16>(ctx, tq, tk, tv, p, v_f16)
           : n == 32 ? run_few<128, 32>(ctx, tq, tk, tv, p, v_f16)
                     : run_few<128, 64>(ctx, tq, tk, tv, p, v_f16);
}

}  // namespace ltx
