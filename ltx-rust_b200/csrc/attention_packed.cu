// Attention over packed documents: softmax over the keys of the row's own
// document only, with optional causal and prefix masks, scores capped by a
// tanh, and a bias that falls with distance.
//
// Every mask here leaves a row the first `lim` keys of its document (the
// document mask: all of them; causal: up to the key beside it; a prefix: at
// least that many), so a row needs one number and a tile of keys is either
// whole for all rows of a warp or compared against it.
//
// Items are (key head, document, up to 256 query rows; 128 where there are few), one
// per CTA of the grid; a CTA that has told its roles about one takes over the next
// CTA not yet launched (cluster launch control), so its loads and products run on
// under the epilogue and unequal items still spread evenly.  A query row is a
// (token, head of the key head's group): a 128-row tile holds 128 / group tokens times the group's heads, so the heads
// that share a key head read each K/V tile once.  Both 128-row tiles A and B of
// an item share every K/V tile, and tiles go from the last keys to the first
// (with a bias by distance the largest scores come first, and the running
// maximum hardly moves).
// TMEM (512 columns): S_A, S_B (128 f32 columns each), O_A, O_B; P goes back
// into the upper half of its S as packed 16-bit pairs and is the A operand of
// P.V from there.
// 10 warps:
//   warp 0     finds the items and tells the others; TMA: the Q tiles, then K_j,
//              V_j through a ring that runs on into the next item.
//   warp 1     one thread issues QK_A QK_B | PV_A(j) QK_A(j+1) PV_B(j) QK_B(j+1);
//              the next item's QK follows under this one's epilogue.
//   warps 2-5  softmax of tile A, 6-9 of tile B, one row per thread: running
//              maximum and sum in f32, O rescaled in TMEM only when a row's
//              maximum grew by more than 2^kRescaleLog2.
// V rows behind a document's end are zeroed by a softmax warp's threads before
// they hand P over: P is 0 there, but 0 times another document's NaN is not.
// With few items (few rows over long keys) a cluster of S CTAs shares the keys
// of one item and joins its partial O, maximum and sum through distributed
// shared memory, in the order of the ranks.
// Bound by the exponentials and their way from S to P: a row's tile passes max,
// exponential and conversion in one thread while the other tile's products run (three
// clips: tensor pipe 51% busy, special functions 41%).  One document of 8192 rows x 32
// heads x 128: 900 us, 1220 TFLOP/s; with slopes 1430; capped, bf16 V 1280, f16 1775;
// x 64: 792.  Three clips of 8192 rows together: 411, 907 TFLOP/s (1.9 us a K/V tile
// and 8 for each of 1056 items, seven to an SM and twenty more).  4099 capped causal
// rows of 5 documents x 16/4 heads: 47.
// All waits are bounded (2 s) and report LTX_ERR_TIMEOUT through the flag.
#include <cuda.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "attention_packed.cuh"
#include "device_common.cuh"
#include "internal.hpp"
#include "kernels.hpp"

namespace ltx {

namespace {

constexpr int kThreads = 320;
constexpr int kMaxSplits = 8;   // CTAs that share an item, a power of two
// The same value, unknown to the compiler: what is computed from it inside a
// loop is not kept in registers around the loop.
__device__ __forceinline__ int fresh(int v) {
    asm volatile("" : "+r"(v));
    return v;
}
constexpr int kNoRow = 1 << 30;   // keys left of a thread without a row (no document has as many)

// D 128: 16-bit K and V tiles of 32 KB (two 64-column swizzle blocks), D 64: 16 KB.
template <int D>
struct Smem {
    static constexpr int TILE = 128 * D * 2, HALF = 128 * 64 * 2;
    static constexpr int RING_SLOTS = D == 128 ? 5 : 8;
    static constexpr int Q = 0, RING = 2 * TILE, BAR = RING + RING_SLOTS * TILE;
    // float2 [2][128], a row's maximum and sum (splits > 1): where Q was, which no product reads any more
    static constexpr int ML = Q;
    static constexpr int BYTES = BAR + 384 + 1024;
    static_assert((14 + 2 * RING_SLOTS) * 8 + 16 + 2 * sizeof(Item) <= 384, "barriers and items exceed their block");
    static_assert(2 * 128 * D * 4 <= RING_SLOTS * TILE, "the f32 partials of both tiles fit the ring");
    static_assert(BYTES <= 232448, "shared memory exceeds the per-CTA limit");
};

// The pair-th pair of query tiles over all documents, found by one warp; false
// when there are fewer.  32 documents at a time, and among those the pairs with
// the most keys first, whatever documents they are of, so that the CTAs end
// together.  `base`, `before`: where the last search ended (32 documents from
// base, `before` pairs ahead of them); one for a later pair goes on from there.
__device__ __forceinline__ bool find_item(const PackedParams &p, int pair, int lane, int &base, int &before, Item &it) {
    const int per = p.item_tiles * p.tile_tokens;
    if (pair < before) base = before = 0;
    for (; base < p.docs; base += 32) {
        int s = 0, e = 0, ks = 0, ke = 0;
        if (base + lane < p.docs) {
            doc_span(p.qo, base + lane, p.rows_q, p.flag, s, e);
            doc_span(p.ko, base + lane, p.rows_k, p.flag, ks, ke);
        }
        const int n = (e - s + per - 1) / per, all = __reduce_add_sync(0xffffffffu, n);
        if (before + all <= pair) {
            before += all;
            continue;
        }
        // A pair's level is what it sees, in `per` keys: a document's last pair has
        // the highest, causal ones before it one less each.
        const int top = (ke - ks + per - 1) / per, local = pair - before;
        auto above = [&](int level) { return p.causal ? min(max(top - level + 1, 0), n) : level <= top ? n : 0; };   // pairs from level on
        int lo = __reduce_min_sync(0xffffffffu, n ? (p.causal ? top - n + 1 : top) : 1 << 30);
        int hi = __reduce_max_sync(0xffffffffu, n ? top : -(1 << 30)) + 1, higher = 0;   // pairs from hi on
        while (hi - lo > 1) {   // the level of the pair sought: `higher` lie above it, so many or more not
            const int mid = lo + (hi - lo) / 2, count = __reduce_add_sync(0xffffffffu, above(mid));
            if (count > local) lo = mid;
            else hi = mid, higher = count;
        }
        const int here = above(lo) - above(lo + 1);
        int incl = here;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += v;
        }
        const int src = __ffs(__ballot_sync(0xffffffffu, higher + incl > local)) - 1;
        const int which = p.causal ? lo - (top - n + 1) : local - higher - (incl - here);   // of the document's pairs
        it.qs = __shfl_sync(0xffffffffu, s, src);
        it.lq = __shfl_sync(0xffffffffu, e, src) - it.qs;
        it.ks = __shfl_sync(0xffffffffu, ks, src);
        it.lk = __shfl_sync(0xffffffffu, ke, src) - it.ks;
        it.tile0 = p.item_tiles * __shfl_sync(0xffffffffu, which, src);
        it.doc = base + src;
        return true;
    }
    return false;
}

// Cluster launch control: asks for a CTA of the grid that has not been launched
// yet; the 16-byte answer lands in shared memory and counts on the mbarrier.
__device__ __forceinline__ void ask_next_cta(void *answer, uint64_t *bar) {
    asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(
                     smem_u32(answer)),
                 "r"(smem_u32(bar))
                 : "memory");
}
// The index of the CTA taken over, -1 when none was left.
__device__ __forceinline__ int next_cta(const void *answer) {
    uint32_t got, x;
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b128 a;\n\t"
        "ld.shared.b128 a, [%2];\n\t"
        "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, a;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t"
        "mov.u32 %1, 0;\n\t"
        "@p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %1, a;\n\t}"
        : "=r"(got), "=r"(x)
        : "r"(smem_u32(answer))
        : "memory");
    return got ? (int)x : -1;
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
__device__ __forceinline__ void st_peer4(uint32_t addr, float4 v) {
    asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w)
                 : "memory");
}
__device__ __forceinline__ float2 ld_peer2(uint32_t addr) {
    float2 v;
    asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
    return v;
}

// A CTA's share of an item: K/V tiles [j0, j0 + cnt[t]) for query tile t (what
// its last token sees, cut to this rank of the cluster), `all` of them loaded.
struct Share {
    int cnt[2], j0, all, nt, prefix;
    __device__ __forceinline__ Share(const PackedParams &p, const Item &it, int split) {
        prefix = p.causal && p.prefix ? min(max(p.prefix[it.doc], 0), it.lk) : 0;
        nt = p.item_tiles == 2 && it.lq > (it.tile0 + 1) * p.tile_tokens ? 2 : 1;   // query tiles that hold tokens
        int n[2];
#pragma unroll
        for (int t = 0; t < 2; ++t)
            n[t] = t < nt ? (limit_of(p, it, min((it.tile0 + t + 1) * p.tile_tokens, it.lq) - 1, prefix) + BKV - 1) / BKV : 0;
        const int most = max(n[0], n[1]);
        const int per = p.splits == 1 ? most : (most + p.splits - 1) / p.splits;
        j0 = split * per;
        const int j1 = min(most, j0 + per);
#pragma unroll
        for (int t = 0; t < 2; ++t) cnt[t] = max(0, min(j1, n[t]) - j0);
        all = max(cnt[0], cnt[1]);
    }
};

// What changes a row's scores: nothing but the scale, a bias by distance, or a cap
// (and perhaps a bias).  kCapFixed: a cap alone, of at most kFixedCap in the log2
// domain, with bf16 V: 2^score fits f32 and bf16 as it is, so no maximum is kept
// and the scores are gone through once.  kCapFar: a cap above kExpCap (log2 domain),
// where tanh_exp would move small scores by more than half a step of f16's P (2e-4 at
// kExpCap); tanh_any2 for every cap took 1920 us instead of 1775 (8192 x 32 x 128, f16).
enum Mode { kPlain = 0, kBias = 1, kCap = 2, kCapFixed = 3, kCapFar = 4 };
constexpr float kExpCap = 512.f;
constexpr float kFixedCap = 75.f;   // 2^75 by 2^29 keys by values of 2^23 stay within f32

// Scores of one row in the log2 domain.  The scale goes with the log2e, and the
// bias is linear on either side of the key the row stands beside, so a tile that
// lies on one side for every row of the warp needs one multiply-add more.
template <int MODE>
struct RowScores {
    static constexpr bool kCapped = MODE == kCap || MODE == kCapFixed || MODE == kCapFar;
    static constexpr bool kCappedOnline = MODE == kCap || MODE == kCapFar;
    float2 sc;              // kPlain, kBias: scale log2e; capped: scale / cap, 0 in a thread without a row
    float cap2;             // capped: cap log2e
    float slope;            // slope log2e, 0 without
    float place;            // the row's key less the tile's first
    int ends;               // capped: the document's keys in the tile, BKV where it goes on
    int side;               // 1: the tile's keys lie before it for every row, -1: behind, 0: both
    __device__ __forceinline__ void set_tile(int pl) {
        if constexpr (MODE == kBias || kCappedOnline) {
            place = (float)pl;
            side = __all_sync(0xffffffffu, pl >= BKV - 1) ? 1 : __all_sync(0xffffffffu, pl <= 0) ? -1 : 0;
        }
    }
    // 32 scores, keys e0 + 0..31: raw products to the log2 domain (kPlain: as they are).
    // The warp's rows agree on the form of tanh, which moves bits.  What lies outside
    // the document has no say in it: threads without a row have scores of 0, and the
    // keys around the document's end take the form that is right at every size.
    __device__ __forceinline__ void apply(uint32_t (&r)[32], int e0) const {
        if constexpr (MODE == kPlain) return;
        float2 v[16];
#pragma unroll
        for (int u = 0; u < 16; ++u)
            v[u] = __fmul2_rn(make_float2(__uint_as_float(r[2 * u]), __uint_as_float(r[2 * u + 1])), sc);
        if constexpr (MODE == kCapFar) {
#pragma unroll
            for (int u = 0; u < 16; ++u) v[u] = __fmul2_rn(tanh_any2(v[u]), make_float2(cap2, cap2));
        } else if constexpr (kCapped) {
            float big = 0.f;
#pragma unroll
            for (int u = 0; u < 16; ++u) big = fmaxf(big, fmaxf(fabsf(v[u].x), fabsf(v[u].y)));
            if (e0 + 32 > ends) big = 2.f;
            if (!__any_sync(0xffffffffu, big > 0.5f)) {
#pragma unroll
                for (int u = 0; u < 16; ++u) v[u] = __fmul2_rn(tanh_small2(v[u]), make_float2(cap2, cap2));
            } else if (!__any_sync(0xffffffffu, big > 1.f)) {
#pragma unroll
                for (int u = 0; u < 16; ++u) v[u] = __fmul2_rn(tanh_poly2(v[u]), make_float2(cap2, cap2));
            } else {
#pragma unroll
                for (int u = 0; u < 16; ++u) v[u] = make_float2(cap2 * tanh_exp(v[u].x), cap2 * tanh_exp(v[u].y));
            }
        }
        if (MODE == kBias || (kCappedOnline && slope != 0.f)) {
            if (side != 0) {
                const float s = side > 0 ? slope : -slope, base = s * ((float)e0 - place);
#pragma unroll
                for (int u = 0; u < 16; ++u)
                    v[u] = __fadd2_rn(v[u], __ffma2_rn(make_float2(s, s), make_float2(2.f * u, 2.f * u + 1.f), make_float2(base, base)));
            } else {
#pragma unroll
                for (int u = 0; u < 16; ++u) {
                    v[u].x -= slope * fabsf(place - (float)(e0 + 2 * u));
                    v[u].y -= slope * fabsf(place - (float)(e0 + 2 * u + 1));
                }
            }
        }
#pragma unroll
        for (int u = 0; u < 16; ++u) {
            r[2 * u] = __float_as_uint(v[u].x);
            r[2 * u + 1] = __float_as_uint(v[u].y);
        }
    }
};

// Of a row's 16 pairs of exponentials per 32 keys, those computed on the FMA pipe
// (exp2_poly2): the special-function unit alone, at 6 cycles a warp, is as busy as
// the tensor cores at head_dim 128 and busier at 64.  A quarter of them: 768 us at
// 8192 x 32 x 64, 817 with half, 887 with none (head_dim 128 differs by less than
// its runs do).
constexpr uint32_t kPolyPairs = 0x1111u;

// The larger of two, NaN if either is.  For the scores whose exponential is the
// polynomial, which does not keep a NaN (for all of them: 1460 us with slopes
// instead of 1430 at 8192 x 32 x 128).
static_assert(kPolyPairs == (kPolyPairs & 15u) * 0x1111u, "the row maximum's eight chains each hold polynomial scores only or none");
__device__ __forceinline__ float max_nan(float a, float b) {
    float m;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(a), "f"(b));
    return m;
}

// One row's 128 scores of a K/V tile: S from TMEM, the row's maximum, P back
// into TMEM, the row's sum.  `left` keys are the row's to see (`masked`: some row
// of the warp does not see all); O is moved along when the reference grows.
template <int D, bool VF16, int MODE>
__device__ __forceinline__ void softmax_tile(uint32_t s_tmem, uint32_t o_tmem, const RowScores<MODE> &rs, int left,
                                             bool masked, float &m_ref, float &l) {
    auto mask = [&](uint32_t (&r)[32], int e0) {
        if (masked) {
#pragma unroll
            for (int e = 0; e < 32; ++e)
                if (e0 + e >= left) r[e] = __float_as_uint(-INFINITY);
        }
    };
    // pass 1: the row max over the 128 scores.  Keys 64..127 stay in registers
    // (rh) for pass 2; keys 0..63 are read again (kCap, kCapFar: they are put back changed).
    uint32_t rh[2][32];
    float m8[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) m8[u] = -INFINITY;
    auto look = [&](const uint32_t (&r)[32]) {
#pragma unroll
        for (int e = 0; e < 32; ++e)
            m8[e & 7] = (kPolyPairs >> (e & 7) / 2) & 1u ? max_nan(m8[e & 7], __uint_as_float(r[e])) : fmaxf(m8[e & 7], __uint_as_float(r[e]));
    };
    if constexpr (MODE != kPlain) {
        tmem_ld_32x32b_x32(s_tmem + 64, rh[0]);
        tmem_ld_32x32b_x32(s_tmem + 96, rh[1]);
        tmem_ld_wait_regs(rh[0]);
        tmem_ld_wait_regs(rh[1]);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            rs.apply(rh[h], 64 + 32 * h);
            mask(rh[h], 64 + 32 * h);
            look(rh[h]);
        }
#pragma unroll
        for (int c = 0; c < 64; c += 32) {
            uint32_t r[32];
            tmem_ld_32x32b_x32(s_tmem + c, r);
            tmem_ld_wait_regs(r);
            rs.apply(r, c);
            mask(r, c);
            look(r);
            if constexpr (rs.kCappedOnline) tmem_st_32x32b_x32(s_tmem + c, r);
        }
    } else {
        uint32_t r01[2][32];
        tmem_ld_32x32b_x32(s_tmem + 0, r01[0]);
        tmem_ld_32x32b_x32(s_tmem + 32, r01[1]);
        tmem_ld_32x32b_x32(s_tmem + 64, rh[0]);
        tmem_ld_32x32b_x32(s_tmem + 96, rh[1]);
        tmem_ld_wait_regs(r01[0]);
        tmem_ld_wait_regs(r01[1]);
        tmem_ld_wait_regs(rh[0]);
        tmem_ld_wait_regs(rh[1]);
        mask(r01[0], 0);
        mask(r01[1], 32);
        mask(rh[0], 64);
        mask(rh[1], 96);
        look(r01[0]);
        look(r01[1]);
        look(rh[0]);
        look(rh[1]);
    }
    float mx = max_nan(max_nan(max_nan(m8[0], m8[1]), max_nan(m8[2], m8[3])),
                       max_nan(max_nan(m8[4], m8[5]), max_nan(m8[6], m8[7])));
    if constexpr (MODE == kPlain) mx *= rs.sc.x;   // scale > 0: max(s * scale) = scale * max(s)
    // The rows of one warp decide together: tcgen05.ld/st are
    // warp-collective (.sync.aligned), so the O rescale runs for the
    // whole warp when any of its rows needs it; a row that does not
    // keeps its reference (alpha = 1).
    const bool grow = !(mx <= m_ref + kRescaleLog2);   // a NaN becomes the reference, and with it all of the row
    if (__any_sync(0xffffffffu, grow)) {
        // O_t and l are relative to m_ref; move them to mx (the P.V before
        // was issued before this tile's QK, whose completion was waited for).
        const float alpha = grow ? ex2(m_ref - mx) : 1.0f;   // 0 when m_ref = -inf
        // (in an item's first tile O holds the item before's and is about to be overwritten)
        if (__any_sync(0xffffffffu, l != 0.f)) {
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
    if constexpr (rs.kCappedOnline) tmem_st_wait();
    // pass 2: P = 2^(s - m_ref), at most 2^kRescaleLog2, in f32, stored as
    // packed 16-bit pairs (key 2c in the low half of column c) into columns
    // 64..127 of S_t, which pass 1 has read.  A row that has seen no key yet has
    // m_ref = -inf and P = 2^-inf = 0.  Masked tiles take no polynomial: it
    // does not go to 0.  The sum takes P before its rounding to 16 bits, at most half
    // a step of V's type for each key: taking the rounded P costs 3 to 5%.
    const float base = m_ref == -INFINITY ? 0.f : -m_ref;
    const float2 nm2 = make_float2(base, base);
    float2 sum2 = make_float2(0.f, 0.f);
    auto p_store = [&](const uint32_t (&r)[32], uint32_t col, auto with_poly) {   // 32 keys -> 16 columns
        uint32_t pk[16];
#pragma unroll
        for (int u = 0; u < 16; ++u) {
            const float2 s = make_float2(__uint_as_float(r[2 * u]), __uint_as_float(r[2 * u + 1]));
            const float2 x = MODE == kPlain ? __ffma2_rn(s, rs.sc, nm2) : __fadd2_rn(s, nm2);
            const float2 pf = decltype(with_poly)::value && ((kPolyPairs >> u) & 1u) ? exp2_poly2(x) : make_float2(ex2(x.x), ex2(x.y));
            sum2 = __fadd2_rn(sum2, pf);
            pk[u] = pack16<VF16>(pf);
        }
        tmem_st_32x32b_x16(s_tmem + col, pk);
    };
    auto pass2 = [&](auto with_poly) {
        uint32_t r0[2][32];
        tmem_ld_32x32b_x32(s_tmem + 0, r0[0]);
        tmem_ld_32x32b_x32(s_tmem + 32, r0[1]);
        p_store(rh[0], 96, with_poly);
        p_store(rh[1], 112, with_poly);
        tmem_ld_wait_regs(r0[0]);
        tmem_ld_wait_regs(r0[1]);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            if constexpr (MODE == kBias) rs.apply(r0[h], 32 * h);
            if constexpr (!rs.kCappedOnline) mask(r0[h], 32 * h);
            p_store(r0[h], 64 + 16 * h, with_poly);
        }
    };
    if (masked) pass2(std::false_type{});
    else pass2(std::true_type{});
    l += sum2.x + sum2.y;
    tmem_st_wait();             // P_t in TMEM ...
    tc_fence_before();          // ... and ordered before the arrive for the MMA thread
}

// The same for kCapFixed: P = 2^score, 32 keys at a time.  The sum takes P as the
// product takes it, rounded: here a row's largest P is no power of two, and one
// that a single key rules would otherwise carry that rounding into its output.
__device__ __forceinline__ void softmax_tile_fixed(uint32_t s_tmem, const RowScores<kCapFixed> &rs, int left, bool masked,
                                                   float &m_ref, float &l) {
    float2 sum2 = make_float2(0.f, 0.f);
    auto keys32 = [&](uint32_t (&r)[32], int e0, uint32_t col) {
        rs.apply(r, e0);
        if (masked) {
#pragma unroll
            for (int e = 0; e < 32; ++e)
                if (e0 + e >= left) r[e] = __float_as_uint(-INFINITY);
        }
        uint32_t pk[16];
#pragma unroll
        for (int u = 0; u < 16; ++u) {
            const float2 pf = make_float2(ex2(__uint_as_float(r[2 * u])), ex2(__uint_as_float(r[2 * u + 1])));
            pk[u] = pack16<false>(pf);
            sum2 = __fadd2_rn(sum2, unpack_bf16(pk[u]));
        }
        tmem_st_32x32b_x16(s_tmem + col, pk);
    };
    // P's columns 64..127 take the place of the scores of keys 64..127: those first
    uint32_t a[32], b[32], c[32];
    tmem_ld_32x32b_x32(s_tmem + 64, a);
    tmem_ld_32x32b_x32(s_tmem + 96, b);
    tmem_ld_wait_regs(a);
    tmem_ld_wait_regs(b);
    tmem_ld_32x32b_x32(s_tmem + 0, c);
    keys32(a, 64, 96);
    keys32(b, 96, 112);
    tmem_ld_wait_regs(c);
    tmem_ld_32x32b_x32(s_tmem + 32, a);
    keys32(c, 0, 64);
    tmem_ld_wait_regs(a);
    keys32(a, 32, 80);
    l += sum2.x + sum2.y;
    if (left > 0) m_ref = 0.f;
    tmem_st_wait();
    tc_fence_before();
}

// VF16: V (and so P) are f16, otherwise bf16; Q and K are bf16.
template <int D, bool VF16, int MODE>
__global__ void __launch_bounds__(kThreads, 1)
    packed_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                  const __grid_constant__ CUtensorMap tmV, PackedParams p) {
    using L = Smem<D>;
    constexpr int kRing = L::RING_SLOTS;
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    unsigned char *smem = reinterpret_cast<unsigned char *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    unsigned char *sQ = smem + L::Q, *sRing = smem + L::RING;
    uint64_t *bars = reinterpret_cast<uint64_t *>(smem + L::BAR);
    uint64_t *q_full = bars, *q_empty = bars + 1;
    uint64_t *s_full = bars + 2, *p_full = bars + 4, *pv_done = bars + 6;   // [2] each
    uint64_t *i_full = bars + 8, *i_empty = bars + 10;                      // [2] each: items told
    uint64_t *slot_full = bars + 12, *slot_empty = slot_full + kRing;       // [kRing] each
    uint64_t *a_full = slot_empty + kRing;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(a_full + 1);
    uint64_t *answer = a_full + 2;                                          // 16 bytes: 14 + 2 kRing is even
    Item *s_item = reinterpret_cast<Item *>(answer + 2);                    // [2]
    float2 *s_ml = reinterpret_cast<float2 *>(smem + L::ML);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int split = blockIdx.x % p.splits;
    const int tt = p.tile_tokens;
    if (threadIdx.x == 0) {
        tma_prefetch_desc(&tmQ);
        tma_prefetch_desc(&tmK);
        tma_prefetch_desc(&tmV);
        mbar_init(q_full, 1);
        mbar_init(q_empty, 1);
        mbar_init(a_full, 1);
        for (int s = 0; s < kRing; ++s) {
            mbar_init(&slot_full[s], 1);
            mbar_init(&slot_empty[s], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&s_full[i], 1);
            mbar_init(&p_full[i], 4);
            mbar_init(&pv_done[i], 1);
            mbar_init(&i_full[i], 1);
            mbar_init(&i_empty[i], 9);
        }
        fence_barrier_init();
    }
    if (warp == 1) {
        tmem_alloc(tmem_slot, 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    bool aborted = false;

    if (warp == 0) {
        uint32_t issued = 0, n_items = 0, n_q = 0, n_asked = 0;
        int base = 0, before = 0;
        int i = blockIdx.x / p.splits;
        // The next item, asked for when the loads of the one at hand are issued
        // (the ring holds a few microseconds of products then): earlier, a CTA
        // with a long item would sit on a second one.  A cluster has one item.
        auto next = [&]() {
            if (p.splits > 1) return -1;
            if (lane == 0) {
                mbar_arrive_expect_tx(a_full, 16);
                ask_next_cta(answer, a_full);
            }
            if (!warp_wait(a_full, n_asked++ & 1, p.flag, 315, &aborted)) return -1;
            const int x = next_cta(answer);
            __syncwarp();
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");   // read before the next answer lands
            return x;
        };
        for (;;) {
            Item it{};
            bool more = false;
            while (i >= 0) {
                const int g = i / (p.pairs * p.head_group), first = g * p.head_group, in = i - g * p.pairs * p.head_group;
                const int heads = min(p.head_group, p.kv_heads - first);
                it.kvh = first + in % heads;
                if ((more = find_item(p, in / heads, lane, base, before, it))) break;
                i = next();
            }
            if (!more) it.kvh = -1;
            it.load0 = issued;
            const uint32_t b = n_items & 1;
            if (!warp_wait(&i_empty[b], ((n_items >> 1) & 1) ^ 1, p.flag, 300, &aborted)) break;
            if (lane == 0) {
                s_item[b] = it;
                mbar_arrive(&i_full[b]);
            }
            __syncwarp();
            ++n_items;
            if (!more) break;
            const Share sh(p, it, split);
            if (sh.all > 0) {
                if (elect_one() && mbar_wait(q_empty, (n_q & 1) ^ 1, p.flag, 304, &aborted)) {
                    mbar_arrive_expect_tx(q_full, sh.nt * (D / 64) * tt * p.group * 128);
                    for (int t = 0; t < sh.nt; ++t)
                        for (int x = 0; x < D; x += 64)
                            tma_load_3d(sQ + t * L::TILE + (x / 64) * L::HALF, &tmQ, q_full, x, it.kvh * p.group,
                                        it.qs + (it.tile0 + t) * tt);
                    for (int s = 0; s < 2 * sh.all; ++s, ++issued) {   // K_j, V_j, the last tile first
                        const int slot = issued % kRing;
                        if (!mbar_wait(&slot_empty[slot], ((issued / kRing) & 1) ^ 1, p.flag, 301, &aborted)) break;
                        mbar_arrive_expect_tx(&slot_full[slot], L::TILE);
                        for (int x = 0; x < D; x += 64)
                            tma_load_3d(sRing + slot * L::TILE + (x / 64) * L::HALF, (s & 1) ? &tmV : &tmK,
                                        &slot_full[slot], x, it.kvh, it.ks + (sh.j0 + sh.all - 1 - (s >> 1)) * BKV);
                    }
                    if (aborted) {   // let the copies already issued land before the CTA exits
                        bool a2 = false;
                        mbar_wait(q_full, n_q & 1, nullptr, 0, &a2);
                        a2 = false;
                        for (uint32_t s = issued > (uint32_t)kRing ? issued - kRing : 0; s < issued; ++s)
                            mbar_wait(&slot_full[s % kRing], (s / kRing) & 1, nullptr, 0, &a2);
                    }
                }
                ++n_q;
            }
            // every lane goes on from the elected one's count
            issued = __reduce_max_sync(0xffffffffu, issued);
            aborted = __any_sync(0xffffffffu, aborted);
            if (aborted) break;
            i = next();
        }
    } else if (warp == 1) {
        if (elect_one()) {
            constexpr uint32_t idesc_qk = idesc_f16(BQ, BKV, true, false);
            constexpr uint32_t idesc_pv = idesc_f16(BQ, D, !VF16, true);   // A = P (TMEM), B = V, MN-major
            const uint32_t q_addr = smem_u32(sQ);
            uint32_t n_items = 0, n_q = 0, n_p[2] = {0, 0};
            while (!aborted) {
                const uint32_t b = n_items & 1;
                if (!mbar_wait(&i_full[b], (n_items >> 1) & 1, p.flag, 302, &aborted)) break;
                const Item it = s_item[b];
                mbar_arrive(&i_empty[b]);
                ++n_items;
                if (it.kvh < 0) break;
                const Share sh(p, it, split);
                const uint32_t used = it.load0;
                if (sh.all == 0) continue;   // nothing to see, and nobody waits
                auto wait_load = [&](uint32_t s, int code) {
                    return mbar_wait(&slot_full[s % kRing], (s / kRing) & 1, p.flag, code, &aborted);
                };
                auto issue_qk = [&](int t, int j) {   // S_t = Q_t K_j^T
                    const uint32_t k_addr = smem_u32(sRing + (used + 2 * j) % kRing * L::TILE);
#pragma unroll
                    for (int kk = 0; kk < D / 16; ++kk) {
                        const uint32_t off = (kk >> 2) * L::HALF + (kk & 3) * 32;
                        umma_f16_ss(tmem + t * 128, sdesc_sw128(q_addr + t * L::TILE + off, 16, 1024),
                                    sdesc_sw128(k_addr + off, 16, 1024), idesc_qk, kk ? 1u : 0u);
                    }
                    umma_commit(&s_full[t]);
                };
                // tile t works on loads j >= skip(t): its tokens do not see the last keys
                auto skip = [&](int t) { return sh.all - sh.cnt[t]; };
                bool ok = mbar_wait(q_full, n_q & 1, p.flag, 305, &aborted) && wait_load(used, 306);
                ++n_q;
                if (ok) {
                    tc_fence_after();
#pragma unroll
                    for (int t = 0; t < 2; ++t)
                        if (skip(t) == 0) issue_qk(t, 0);
                    umma_commit(&slot_empty[used % kRing]);   // K_0 read
                }
                for (int j = 0; ok && j < sh.all; ++j) {
                    // Per tile: PV_t(j) once the softmax has stored P_t(j) (p_full),
                    // then QK_t(j+1) into the same columns: MMAs of one thread run
                    // in issue order, so P_t(j) is read before S_t(j+1) lands.
                    const uint32_t v = used + 2 * j + 1;
                    if (!wait_load(v, 307)) break;
                    const bool next = j + 1 < sh.all;
                    if (next && !wait_load(v + 1, 308)) break;
#pragma unroll
                    for (int t = 0; t < 2; ++t) {
                        if (j >= skip(t)) {
                            if (!mbar_wait(&p_full[t], n_p[t] & 1, p.flag, 309 + t, &aborted)) {
                                ok = false;
                                break;
                            }
                            ++n_p[t];
                            tc_fence_after();
                            const uint32_t v_addr = smem_u32(sRing + v % kRing * L::TILE);
#pragma unroll
                            for (int kk = 0; kk < BKV / 16; ++kk)   // O_t (+)= P_t V_j: 16 keys = 8 packed columns per MMA
                                umma_f16_ts(tmem + 256 + t * 128, tmem + t * 128 + 64 + kk * 8,
                                            sdesc_sw128(v_addr + kk * 2048, L::HALF, 1024), idesc_pv,
                                            (j > skip(t) || kk > 0) ? 1u : 0u);
                        }
                        if (!next && sh.cnt[t] > 0) umma_commit(&pv_done[t]);
                        if (next && j + 1 >= skip(t)) issue_qk(t, j + 1);
                    }
                    if (!ok) break;
                    umma_commit(&slot_empty[v % kRing]);                     // V_j read
                    if (next) umma_commit(&slot_empty[(v + 1) % kRing]);     // K_{j+1} read
                    if (j + 2 == sh.all || sh.all == 1) umma_commit(q_empty);   // the last QK has been issued
                }
            }
        }
    } else {
        // Softmax warps: tile t = 0 (warps 2-5) or 1 (warps 6-9), row quad*32 + lane.
        const int t = (warp - 2) >> 2;
        const int quad = warp & 3;
        const int r_thread = quad * 32 + lane;
        const uint32_t s_tmem = tmem + ((uint32_t)(quad * 32) << 16) + t * 128, o_tmem = s_tmem + 256;
        RowScores<MODE> rs{};
        const float sc = rs.kCapped ? p.scale / p.softcap : p.scale * kLog2e;
        rs.sc = make_float2(sc, sc);
        if constexpr (rs.kCapped) rs.cap2 = p.softcap * kLog2e;
        uint32_t n_items = 0, phase = 0;   // of s_full[t] (bit 0) and pv_done[t] (bit 1)
        float m_ref = -INFINITY, l = 0.f;   // a row's maximum that P is taken against (log2 domain), its sum
        bool row_ok = false, any_o = false, other_o = false, join = false;
        __nv_bfloat16 *dst = nullptr;
        while (!aborted) {
            // The item stays in shared memory (volatile: read again behind the
            // tiles, not kept in registers through them).
            const volatile Item &it = s_item[n_items & 1];
            if (!warp_wait(&i_full[n_items & 1], (n_items >> 1) & 1, p.flag, 303, &aborted)) break;
            if (it.kvh < 0) break;
            const int r_in = fresh(r_thread);
            int n_mine, left, left_min, place, clean = BKV;   // keys a row sees in the tile at hand, the warp's least
            {
                const Item i{it.qs, it.lq, it.ks, it.lk, it.tile0, it.doc, it.kvh, 0};
                const Share sh(p, i, split);
                const int token = (i.tile0 + t) * tt + r_in / p.group;   // in the document
                const bool ok = t < sh.nt && r_in < tt * p.group && token < i.lq;
                n_mine = t ? sh.cnt[1] : sh.cnt[0];
                other_o = (t ? sh.cnt[0] : sh.cnt[1]) > 0;
                const int top = (sh.j0 + n_mine - 1) * BKV;       // first key of the tile to begin with
                row_ok = ok;
                if constexpr (rs.kCapped) {
                    rs.sc = ok ? make_float2(sc, sc) : make_float2(0.f, 0.f);
                    rs.ends = min(BKV, i.lk - top);
                }
                left = ok ? limit_of(p, i, token, sh.prefix) - top : kNoRow;
                left_min = __reduce_min_sync(0xffffffffu, left);
                place = key_beside(i.lq, i.lk, token) - top;
                if constexpr (MODE == kBias || rs.kCappedOnline)
                    rs.slope = p.slopes && ok ? p.slopes[i.kvh * p.group + r_in % p.group] * kLog2e : 0.f;
                // V rows behind the document's end, in the first tile loaded: tile
                // A's threads zero theirs, B's where A skips that tile
                if (top + BKV > i.lk && (t == 0 || sh.cnt[0] < sh.cnt[1])) clean = i.lk - top;
            }
            any_o = n_mine > 0;   // warp-uniform
            m_ref = -INFINITY;
            l = 0.f;
            const bool active = left_min != kNoRow;   // the warp holds rows
            for (; n_mine > 0; --n_mine, left += BKV, left_min += BKV, place += BKV) {
                // warp-uniform outcome: the tcgen05.ld/st below are warp-collective
                if (!warp_wait(&s_full[t], phase & 1, p.flag, 311, &aborted)) break;
                phase ^= 1;
                if (active) {
                    tc_fence_after();
                    rs.set_tile(place);
                    if constexpr (MODE == kCapFixed) softmax_tile_fixed(s_tmem, rs, left, left_min < BKV, m_ref, l);
                    else softmax_tile<D, VF16, MODE>(s_tmem, o_tmem, rs, left, left_min < BKV, m_ref, l);
                }
                if (clean < BKV) {
                    if (r_in >= clean) {
                        const uint32_t s = it.load0 + 1;
                        mbar_wait(&slot_full[s % kRing], (s / kRing) & 1, p.flag, 313, &aborted);
                        unsigned char *v = sRing + (s % kRing) * L::TILE + r_in * 128;
#pragma unroll
                        for (int x = 0; x < D / 64; ++x)
#pragma unroll
                            for (int c = 0; c < 8; ++c)
                                *reinterpret_cast<uint4 *>(v + x * L::HALF + c * 16) = make_uint4(0, 0, 0, 0);
                        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    }
                    aborted = __any_sync(0xffffffffu, aborted);
                    clean = BKV;
                }
                if constexpr (rs.kCapped) rs.ends = BKV;   // the last tile went first
                __syncwarp();
                if (lane == 0) mbar_arrive(&p_full[t]);
            }
            // O_t is final once the last P.V has completed; in a cluster (one item) the ring
            // is free once both tiles' have.  A tile without K/V tiles has no P.V: nothing
            // would hold the MMA thread back from the next item's phase of pv_done, which
            // p_full does where there are some.
            if (any_o) {
                warp_wait(&pv_done[t], phase >> 1, p.flag, 312, &aborted);
                phase ^= 2;
            }
            if (p.splits > 1 && other_o) warp_wait(&pv_done[t ^ 1], 0, p.flag, 314, &aborted);
            tc_fence_after();
            const int r_now = fresh(r_thread);
            dst = p.out + ((int64_t)it.qs + (it.tile0 + t) * tt + r_now / p.group) * p.ldo +
                  (it.kvh * p.group + r_now % p.group) * D;
            __syncwarp();
            if (lane == 0) mbar_arrive(&i_empty[n_items & 1]);
            ++n_items;
            if (p.splits > 1) {   // one item: joined below
                join = !aborted;
                break;
            }
            if (!aborted && any_o) {
                const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);   // a row that saw no key is 0, NaN stays
#pragma unroll
                for (int c = 0; c < D / 32; ++c) {
                    uint32_t r[32];
                    tmem_ld_32x32b_x32(o_tmem + c * 32, r);
                    tmem_ld_wait_regs(r);
                    if (!row_ok) continue;
#pragma unroll
                    for (int g = 0; g < 4; ++g) {
                        uint32_t w[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            w[e] = pack16<false>(make_float2(__uint_as_float(r[g * 8 + 2 * e]) * inv, __uint_as_float(r[g * 8 + 2 * e + 1]) * inv));
                        *reinterpret_cast<uint4 *>(dst + c * 32 + g * 8) = make_uint4(w[0], w[1], w[2], w[3]);
                    }
                }
            } else if (!aborted && row_ok) {   // no row of the tile sees a key
#pragma unroll
                for (int c = 0; c < D / 8; ++c) *reinterpret_cast<uint4 *>(dst + c * 8) = make_uint4(0, 0, 0, 0);
            }
            tc_fence_before();   // O_t has been read: the next item's first P.V, after p_full, may write it
        }
        if (p.splits > 1 && !join) {   // no item, or a wait that gave up: meet the others all the same
            cluster_sync();
            cluster_sync();
        } else if (p.splits > 1) {
            // Join the cluster's partial results.  Every CTA publishes its rows'
            // (maximum, sum); then it sends its O, weighted by all of them, to the
            // owners: rank s sums columns [s D/S, (s+1) D/S) over the ranks, in their
            // order, in the place of its ring, which no product reads any more.
            // (Stores: nothing waits for a peer's answer.  Loads from the peers took
            // 4 to 10 us.)
            s_ml[t * 128 + r_thread] = make_float2(m_ref, l);
            cluster_sync();
            float w_own = 0.f;
            if (row_ok) {
                float2 ml[kMaxSplits];   // every peer's answer is on its way before the first is used
#pragma unroll
                for (int s = 0; s < kMaxSplits; ++s)
                    ml[s] = s < p.splits ? ld_peer2(peer_addr(&s_ml[t * 128 + r_thread], s)) : make_float2(-INFINITY, 0.f);
                float top = -INFINITY, total = 0.f;
#pragma unroll
                for (int s = 0; s < kMaxSplits; ++s) top = fmaxf(top, ml[s].x);
#pragma unroll
                for (int s = 0; s < kMaxSplits; ++s) total += ml[s].y * (ml[s].x == -INFINITY ? 0.f : ex2(ml[s].x - top));
                // no key seen anywhere: all weights 0; a NaN sum stays NaN
                if (m_ref != -INFINITY) w_own = ex2(m_ref - top) / total;
                else if (l != l) w_own = l;
            }
            // [source][piece][256 rows]: a warp's lanes store 512 bytes in a row
            float4 *part = reinterpret_cast<float4 *>(sRing) + t * 128 + r_thread;
            const int per = D / 4 / p.splits, shift = __ffs(per) - 1;   // 16-byte pieces of a row for each rank
#pragma unroll
            for (int c = 0; c < D / 32; ++c) {
                uint32_t r[32] = {};
                if (any_o) {
                    tmem_ld_32x32b_x32(o_tmem + c * 32, r);
                    tmem_ld_wait_regs(r);
                }
                if (!row_ok) continue;
#pragma unroll
                for (int q = 0; q < 8; ++q) {
                    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
                    if (any_o && w_own != 0.f)
                        v = make_float4(__uint_as_float(r[4 * q]) * w_own, __uint_as_float(r[4 * q + 1]) * w_own,
                                        __uint_as_float(r[4 * q + 2]) * w_own, __uint_as_float(r[4 * q + 3]) * w_own);
                    const int i = c * 8 + q;
                    st_peer4(peer_addr(part + (split * per + (i & (per - 1))) * 256, i >> shift), v);
                }
            }
            cluster_sync();
            if (row_ok && !aborted) {
                for (int i = 0; i < per; i += 2) {
                    float4 a = make_float4(0.f, 0.f, 0.f, 0.f), b = a;
                    for (int s = 0; s < p.splits; ++s) {
                        const float4 x = part[(s * per + i) * 256], y = part[(s * per + i + 1) * 256];
                        a = make_float4(a.x + x.x, a.y + x.y, a.z + x.z, a.w + x.w);
                        b = make_float4(b.x + y.x, b.y + y.y, b.z + y.z, b.w + y.w);
                    }
                    *reinterpret_cast<uint4 *>(dst + (split * per + i) * 4) =
                        make_uint4(pack16<false>(make_float2(a.x, a.y)), pack16<false>(make_float2(a.z, a.w)),
                                   pack16<false>(make_float2(b.x, b.y)), pack16<false>(make_float2(b.z, b.w)));
                }
            }
        }
    }
    if (p.splits > 1 && warp < 2) {   // the softmax warps' two
        cluster_sync();
        cluster_sync();
    }

    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

template <int D>
cudaError_t launch_packed(const ltx_ctx *ctx, bool f16, Mode mode, const CUtensorMap &tq, const CUtensorMap &tk, const CUtensorMap &tv,
                          const PackedParams &p) {
    auto kern = f16 ? (mode == kCap      ? packed_kernel<D, true, kCap>
                       : mode == kCapFar ? packed_kernel<D, true, kCapFar>
                       : mode == kBias ? packed_kernel<D, true, kBias>
                                       : packed_kernel<D, true, kPlain>)
                    : (mode == kCap        ? packed_kernel<D, false, kCap>
                       : mode == kCapFixed ? packed_kernel<D, false, kCapFixed>
                       : mode == kCapFar   ? packed_kernel<D, false, kCapFar>
                       : mode == kBias     ? packed_kernel<D, false, kBias>
                                           : packed_kernel<D, false, kPlain>);
    cudaError_t e = allow_smem(ctx, reinterpret_cast<const void *>(kern), Smem<D>::BYTES);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)((int64_t)p.pairs * p.kv_heads * p.splits));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = Smem<D>::BYTES;
    cfg.stream = ctx->stream;
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

extern "C" int ltx_attention_packed_fwd(ltx_ctx *ctx, const ltx_packed_attention *args) {
    using namespace ltx;
    if (!ctx) return LTX_ERR_INVALID_ARG;
    const char *w = "attention_packed";
    if (!args) return fail(ctx, LTX_ERR_INVALID_ARG, "%s: null arguments", w);
    const auto &[q_dev, k_dev, v_dev, out_dev, q_offsets_dev, k_offsets_dev, prefix_dev, slopes_dev, ldq, ldk, ldv, ldo, v_dtype,
                 docs, rows_q, rows_k, heads, kv_heads, head_dim, causal, scale, softcap] = *args;
    if (v_dtype != LTX_BF16 && v_dtype != LTX_F16) return fail(ctx, LTX_ERR_DTYPE, "%s: V must be BF16 or F16", w);
    if (head_dim != 64 && head_dim != 128)
        return fail(ctx, LTX_ERR_UNSUPPORTED, "%s: head_dim %d (64 or 128)", w, head_dim);
    if (docs < 0 || rows_q < 0 || rows_k < 0 || heads < 1 || kv_heads < 1 || heads % kv_heads)
        return fail(ctx, LTX_ERR_SHAPE, "%s: %d documents, %d x %d rows, %d heads over %d key heads", w, docs, rows_q,
                    rows_k, heads, kv_heads);
    if (rows_q > 1 << 29 || rows_k > 1 << 29) return fail(ctx, LTX_ERR_UNSUPPORTED, "%s: more than 2^29 rows", w);
    // a search through the offsets, 32 documents at a time, has to stay well under the 2 s that the others wait for it
    if (docs > 1 << 24) return fail(ctx, LTX_ERR_UNSUPPORTED, "%s: more than 2^24 documents", w);
    if (heads / kv_heads > 128) return fail(ctx, LTX_ERR_UNSUPPORTED, "%s: more than 128 heads per key head", w);
    if (!(scale > 0.f) || !std::isfinite(scale) || !(softcap >= 0.f) || !std::isfinite(softcap))
        return fail(ctx, LTX_ERR_INVALID_ARG, "%s: scale must be finite and > 0, softcap finite and >= 0", w);
    if (!std::isfinite(scale * kLog2e) || !std::isfinite(softcap * kLog2e) ||
        (softcap > 0.f && (!std::isnormal(scale / softcap) || !std::isnormal(softcap))))
        return fail(ctx, LTX_ERR_INVALID_ARG, "%s: scale, softcap or their quotient leaves f32", w);
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
                   docs, rows_q, rows_k, kv_heads, group, tokens, causal, 0, 1, 1, 2, scale, softcap, ctx->timeout_flag};
    // Few rows per document over many keys, by their averages (the host does
    // not see the offsets): the kernel whose tiles have keys as rows and whose
    // CTAs share every document.  Under some 512 keys its join and its start
    // cost more than it saves.  Averages do badly by a batch of both kinds: 512
    // rows and 64 single ones over 4000 keys x 32/8 heads take 636 us together, in
    // tiles of 64 rows, 20 + 174 in two calls.
    const int some = std::min(docs, rows_q);
    const int64_t rows_per_doc = (int64_t)((rows_q + some - 1) / some) * group;
    if (rows_per_doc <= kMaxFewRows && rows_k / docs >= 512)
        return attention_packed_few(ctx, tk, tv, q_dev, ldq, p, heads, head_dim, v_dtype == LTX_F16, (int)rows_per_doc);
    // Items over all documents: sum ceil(lq / per) <= (rows + docs (per - 1)) / per.
    auto items_of = [&p, some](int64_t per) { return (p.rows_q + (int64_t)some * (per - 1)) / per; };
    // Too few CTAs for the SMs: split the keys over a cluster, at least one K/V tile
    // each if one document had them all (two: 25.1 us for 546 x 913 capped causal
    // rows x 2/1 heads, one: 20.7).
    auto splits_of = [&p, ctx](int64_t items) {
        int s = 1;
        while (s < kMaxSplits && items * s * 2 <= ctx->sm_count && (int64_t)s * 2 * BKV <= p.rows_k) s *= 2;
        return s;
    };
    // Two query tiles to an item share its K and V; where that leaves half of the
    // SMs without work even so, a tile each: half the exponentials on a CTA's way
    // (the same rows 20.7 -> 17.0; 148 x 148 capped with slopes x 8/1 heads 21 -> 17).
    // Where it does not, a tile each means fewer shares of the keys: 4887 capped causal
    // rows of 7 documents x 1 head took 28.6 us instead of 19.9.
    const int64_t twos = items_of(2 * tokens) * kv_heads;
    if (twos * splits_of(twos) * 2 <= ctx->sm_count) p.item_tiles = 1;
    const int64_t pairs = items_of(p.item_tiles * tokens), items = pairs * kv_heads;
    if (items > 0x7fffffff / 8) return fail(ctx, LTX_ERR_UNSUPPORTED, "%s: more than 2^28 tiles", w);
    p.splits = splits_of(items);
    p.pairs = (int)pairs;
    // Key heads that go together, the longest pairs of all of them first: as many
    // as keep K and V within 32 MB of L2.  (5 x 820 capped causal rows x 16/4 heads:
    // 44.7 us a head at a time, 35.3 all four together.  8192 x 32 heads: 892 a head
    // at a time, 942 all together, 900 in eights.)
    p.head_group = (int)std::clamp<int64_t>((32 << 20) / std::max<int64_t>(1, (int64_t)rows_k * head_dim * 4), 1, kv_heads);
    const bool fixed = !slopes_dev && v_dtype == LTX_BF16 && softcap * kLog2e <= kFixedCap;
    const bool far = softcap * kLog2e > kExpCap;
    const Mode mode = softcap > 0.f ? (fixed ? kCapFixed : far ? kCapFar : kCap) : slopes_dev ? kBias : kPlain;
    const cudaError_t e = head_dim == 64 ? launch_packed<64>(ctx, v_dtype == LTX_F16, mode, tq, tk, tv, p)
                                         : launch_packed<128>(ctx, v_dtype == LTX_F16, mode, tq, tk, tv, p);
    return e == cudaSuccess ? LTX_OK : cuda_fail(ctx, e, w);
}
