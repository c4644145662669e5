// Attention of many rows (prompts) over the paged e4m3 cache, on the 5th-generation tensor cores.
//
//   t_ij = scale (q_i . kcode_j) ks[block(j)] log2 e + log2 vs[block(j)],   w = 2^(t - max t)
//   out_i = sum_j w_ij vcode_j / sum_j (w_ij / vs[block(j)])
//
// The codes are the operands as they lie in memory: no conversion of K or V.  tcgen05's 8-bit products run at twice the
// 16-bit rate, and the two left-hand operands, which are not 8-bit, are split into sums of e4m3 values: a value of 8
// significant bits (bfloat16 q) is the sum of two (4 bits each), one of 11 (binary16 q) of three.  Two products at the 8-bit rate take
// the time of one at the 16-bit rate, with half the shared memory for K and V.  The value scales go into the exponent
// (the running maximum is that of t), so a block's scales cost nothing for each score but the constants of one FMA, and the sum
// of the softmax takes them out again for each block of 16 keys.
//
// A tile is 128 rows: `tpt` tokens x the query heads of one kv head.  Key tiles are 128 keys.  Bound by the tensor pipe: 2 * PARTS *
// 128 * 128 * D multiply-adds for each tile at 8192 a clock and SM.  Roles: eight softmax warps (two threads for each row, 64
// keys each), four warps that bring a tile's Q rows, one warp each for the K/V copies, the products and the scales.
#include <algorithm>

#include "paged_sched.cuh"
#include "umma.cuh"

namespace saetta {

constexpr int kPpRows = 128, kPpKeys = 128, kPpThreads = 512;
constexpr float kPpShift = 6.f;   // w is kept times 2^6: e4m3 ends at 448 = 2^8.8, and its smallest steps should lie low
constexpr float kPpRescale = 2.f; // O follows the running maximum only past this many doublings: w stays below 2^8
constexpr int kPpScaleRing = 4;

template <int D, int PARTS>
struct PpLayout {
    static constexpr int kSlabs = D / 128;
    static constexpr int kQPart = kPpRows * D;
    static constexpr int kStage = kPpKeys * D; // K or V of a tile
    static constexpr int kStages = D == 256 ? (PARTS == 2 ? 5 : 4) : 8;
    static constexpr int kRing = kStages * kStage;
    static constexpr int kSmem = 1024 /* alignment */ + PARTS * kQPart + kRing + 2048 /* statistics, scales, barriers */;
    static constexpr int kPBufs = D == 256 && PARTS == 3 ? 1 : 2;
    static constexpr int kPCols = 32 * PARTS;
    static constexpr int kTmemO = 0, kTmemS = D, kTmemP = D + 128;
    static_assert(kTmemP + kPBufs * kPCols <= 512, "fits tensor memory");
    static_assert(kSmem <= 227 * 1024, "fits a CTA's shared memory");
};

__device__ __forceinline__ void tc_mma8(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(d_tmem), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
}
// A from tensor memory: row m in lane m, four e4m3 values in a column.
__device__ __forceinline__ void tc_mma8_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], [%1], %2, %3, p;\n\t}"
        ::"r"(d_tmem), "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};"
        ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
          "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(taddr)
        : "memory");
}
__device__ __forceinline__ uint32_t f2_to_e4m3x2(float lo, float hi) {
    uint16_t d;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(d) : "f"(hi), "f"(lo));
    return d;
}
__device__ __forceinline__ uint32_t h2_to_e4m3x2(uint32_t h) {
    uint16_t d;
    asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;" : "=h"(d) : "r"(h));
    return d;
}
__device__ __forceinline__ uint32_t e4m3x2_as_h2(uint32_t w) {
    uint32_t h;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(uint16_t(w)));
    return h;
}
// Four values as sums of PARTS e4m3 values each: word p holds the four p-th terms.  Every remainder is exact (a value less its
// rounding to fewer bits), so the sum is off by the last term's rounding alone: 2^-8 of the value with two, 2^-12 with three,
// and 2^-10 of a unit below e4m3's normal range.
template <int PARTS>
__device__ __forceinline__ void split4(float a, float b, float c, float d, uint32_t (&w)[PARTS]) {
    if constexpr (PARTS == 2) {
        // by way of binary16, whose 11 bits hold the two terms
        const uint32_t h0 = pack_half2(a, b), h1 = pack_half2(c, d);
        const uint32_t t0 = h2_to_e4m3x2(h0), t1 = h2_to_e4m3x2(h1);
        w[0] = t0 | t1 << 16;
        w[1] = h2_to_e4m3x2(hsub2_u32(h0, e4m3x2_as_h2(t0))) | h2_to_e4m3x2(hsub2_u32(h1, e4m3x2_as_h2(t1))) << 16;
    } else {
#pragma unroll
        for (int p = 0; p < PARTS; p++) {
            const uint32_t t0 = f2_to_e4m3x2(a, b), t1 = f2_to_e4m3x2(c, d);
            w[p] = t0 | t1 << 16;
            const float2 f0 = h2f2(e4m3x2_as_h2(t0)), f1 = h2f2(e4m3x2_as_h2(t1));
            a -= f0.x, b -= f0.y, c -= f1.x, d -= f1.y;
        }
    }
}
__device__ __forceinline__ void pair_sync(uint32_t quarter) { asm volatile("bar.sync %0, 64;" ::"r"(quarter + 1) : "memory"); }
__device__ __forceinline__ void softmax_sync() { asm volatile("bar.sync 5, 256;" ::: "memory"); }
__device__ __forceinline__ float lg2_approx(float x) {
    float y;
    asm("lg2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

template <int D, int PARTS>
__global__ void __launch_bounds__(kPpThreads, 1)
paged_prefill_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const PagedArgs a, const uint32_t tpt) {
    using L = PpLayout<D, PARTS>;
    constexpr int kSlabs = L::kSlabs, NST = L::kStages, NP = L::kPBufs;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t *sQ = smem;                                  // [part][slab][128 rows][128 dims]
    uint8_t *ring = sQ + PARTS * L::kQPart;              // [stage][slab][128 keys][128 dims], K and V by turns
    __nv_bfloat16 *xch = reinterpret_cast<__nv_bfloat16 *>(ring + L::kRing); // [2][2 halves][128 rows] maxima, rounded up
    float *lx = reinterpret_cast<float *>(xch);              // at a tile's end: [2 halves][128 rows] sums
    float4 *scl = reinterpret_cast<float4 *>(lx + 256);      // [kPpScaleRing][8]: key scale, log2 and reciprocal of the value scale, bad
    uint64_t *bars = reinterpret_cast<uint64_t *>(scl + kPpScaleRing * 8);
    uint64_t *full = bars, *empty = bars + 8, *sc_full = bars + 16, *sc_empty = bars + 20, *q_full = bars + 24, *q_empty = bars + 25,
             *s_full = bars + 26, *s_free = bars + 27, *p_full = bars + 28, *pv_done = bars + 30, *o_final = bars + 32, *o_empty = bars + 33;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + 34);
    volatile uint32_t *abort_flag = tmem_slot + 1, *never_set = tmem_slot + 2, *arrived = tmem_slot + 3;
    // the share's scratch is the Q area, free until the roles begin
    uint64_t *scratch = reinterpret_cast<uint64_t *>(sQ);
    PagedShare *share = reinterpret_cast<PagedShare *>(scratch + 40);
    uint8_t *row_e = reinterpret_cast<uint8_t *>(bars + 40); // [128]: the power of two (biased) that undoes what a row of Q was scaled by

    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int s = 0; s < NST; s++) mbar_init(&full[s], 1), mbar_init(&empty[s], 1);
        for (int s = 0; s < kPpScaleRing; s++) mbar_init(&sc_full[s], 1), mbar_init(&sc_empty[s], 9);
        mbar_init(q_full, 4), mbar_init(q_empty, 9), mbar_init(s_full, 1), mbar_init(s_free, 8), mbar_init(o_final, 1), mbar_init(o_empty, 8);
        for (int s = 0; s < 2; s++) mbar_init(&p_full[s], 8), mbar_init(&pv_done[s], 1);
        *abort_flag = 0, *never_set = 0;
        mbar_fence_init();
    }
    pdl_wait();
    paged_share<kPpKeys>(a, tpt, kPpThreads, 1, scratch, share);
    const PagedShare sh = *share;
    if (sh.x0 >= sh.x1) return; // (the whole CTA)
    if (warp == 13) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(tmem_slot)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    const uint32_t tmem_o = tmem + L::kTmemO, tmem_s = tmem + L::kTmemS, tmem_p = tmem + L::kTmemP;
    auto give_up = [&](uint32_t bit) {
        atomicOr(a.words, bit);
        *abort_flag = 1;
    };
    const uint32_t G = a.group;
    PagedWalk<kPpKeys> walk(a, sh, tpt);
    PagedItem it;

    if (warp >= 12) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
        if (warp == 12) {
            // ------------------------------------------------------------ K and V copies, in the order of the products: K0 K1 V0 K2 V1 ...
            const uint32_t bt = min(a.block_tokens, uint32_t(kPpKeys)), per_tile = kPpKeys / bt;
            uint32_t r = 0;
            bool ok = true;
            while (ok && walk.next(it)) {
                const int32_t *table = a.tables + size_t(it.seq) * a.table_stride;
                const uint32_t keys = walk.tiles.keys(it.q, it.rtile), page = lane / kSlabs, slab = lane % kSlabs;
                auto block_of = [&](uint32_t kt) -> int32_t {
                    const uint32_t key = kt * kPpKeys + page * bt;
                    return page < per_tile && key < keys ? table[key / a.block_tokens] : -2;
                };
                auto load = [&](int32_t block, bool values) {
                    const uint32_t st = r % NST, ph = (r / NST) & 1;
                    if (!mbar_wait(&empty[st], ph ^ 1, abort_flag)) { give_up(kStatusEmptyTimeout); return false; }
                    const bool good = block != -2 && uint32_t(block) < a.blocks;
                    const uint32_t copies = __popc(__ballot_sync(0xffffffffu, good));
                    if (lane == 0) mbar_expect_tx(&full[st], copies * bt * 128);
                    __syncwarp();
                    if (good)
                        tma_load_3d(ring + st * L::kStage + slab * (kPpKeys * 128) + page * bt * 128, values ? &map_v : &map_k, &full[st], 0,
                                    int((uint32_t(block) * a.kv_heads + it.head) * a.block_tokens), int(slab));
                    r++;
                    return true;
                };
                int32_t cur = block_of(it.kt0), prev = -2;
                for (uint32_t kt = it.kt0; ok && kt < it.kt1; kt++) {
                    const int32_t next = kt + 1 < it.kt1 ? block_of(kt + 1) : -2;
                    ok = load(cur, false);
                    if (ok && kt > it.kt0) ok = load(prev, true);
                    prev = cur, cur = next;
                }
                if (ok) ok = load(prev, true);
            }
            for (uint32_t k = r > NST ? r - NST : 0; k < r; k++) mbar_wait(&full[k % NST], (k / NST) & 1, never_set, 200000u);
        } else if (warp == 13) {
            // ------------------------------------------------------------ products
            constexpr uint32_t idesc_s = (1u << 4) | (uint32_t(kPpKeys >> 3) << 17) | (uint32_t(kPpRows >> 4) << 24);
            constexpr uint32_t idesc_o = (1u << 4) | (1u << 16) | (uint32_t(D >> 3) << 17) | (uint32_t(kPpRows >> 4) << 24);
            uint32_t r = 0, g = 0, tc = 0; // ring places, tiles, items so far
            bool ok = true;
            while (ok && walk.next(it)) {
                const uint32_t nb = it.kt1 - it.kt0;
                const int32_t vis = min(int32_t(it.q.kv), it.lim0 + int32_t(it.ntok) - 1);
                if (!mbar_wait(q_full, tc & 1, abort_flag)) { give_up(kStatusFullTimeout); break; }
                auto values = [&](uint32_t j) { // O += P V of tile j
                    const uint32_t st = r % NST, ph = (r / NST) & 1, gj = g + j, pb = gj % NP, ss = gj % kPpScaleRing;
                    if (!mbar_wait(&full[st], ph, abort_flag)) { give_up(kStatusFullTimeout); return false; }
                    if (!mbar_wait(&sc_full[ss], (gj / kPpScaleRing) & 1, abort_flag)) { give_up(kStatusFullTimeout); return false; }
                    // rows behind the last key, and of bad blocks, may hold NaN, which a weight of 0 does not silence
                    const int32_t key0 = int32_t((it.kt0 + j) * kPpKeys);
                    const uint32_t bad = __ballot_sync(0xffffffffu, lane < 8 && scl[ss * 8 + lane].w != 0.f);
                    if (key0 + kPpKeys > vis || bad) {
                        for (uint32_t i = lane; i < kPpKeys * 8 * kSlabs; i += 32) {
                            const uint32_t key = (i >> 3) % kPpKeys, slab = i / (kPpKeys * 8);
                            if (key0 + int32_t(key) >= vis || (bad >> (key >> 4) & 1))
                                *reinterpret_cast<uint4 *>(ring + st * L::kStage + slab * (kPpKeys * 128) + key * 128 + (i & 7) * 16) = make_uint4(0, 0, 0, 0);
                        }
                        fence_async_smem();
                    }
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&sc_empty[ss]);
                    if (j == 0 && !mbar_wait(o_empty, (tc & 1) ^ 1, abort_flag)) { give_up(kStatusMmaTimeout); return false; }
                    if (!mbar_wait(&p_full[pb], (gj / NP) & 1, abort_flag)) { give_up(kStatusMmaTimeout); return false; }
                    tc_fence_after();
                    if (lane == 0) {
                        const uint64_t bd = umma_desc(smem_u32(ring) + st * L::kStage, kPpKeys * 128, 1024);
#pragma unroll
                        for (int p = 0; p < PARTS; p++)
#pragma unroll
                            for (int ks = 0; ks < kPpKeys / 32; ks++)
                                tc_mma8_ts(tmem_o, tmem_p + pb * L::kPCols + p * 32 + ks * 8, bd + uint64_t((ks * 4096) >> 4), idesc_o, j > 0 || p > 0 || ks > 0);
                        tc_commit(&empty[st]);
                        tc_commit(&pv_done[pb]);
                        if (j + 1 == nb) tc_commit(o_final);
                    }
                    __syncwarp();
                    r++;
                    return true;
                };
                for (uint32_t j = 0; ok && j < nb; j++) {
                    const uint32_t st = r % NST, ph = (r / NST) & 1, gj = g + j;
                    if (!mbar_wait(&full[st], ph, abort_flag)) { give_up(kStatusFullTimeout); ok = false; break; }
                    if (!mbar_wait(s_free, (gj & 1) ^ 1, abort_flag)) { give_up(kStatusMmaTimeout); ok = false; break; }
                    tc_fence_after();
                    if (lane == 0) {
                        const uint64_t ad = umma_desc(smem_u32(sQ), 16, 1024), bd = umma_desc(smem_u32(ring) + st * L::kStage, 16, 1024);
#pragma unroll
                        for (int p = 0; p < PARTS; p++)
#pragma unroll
                            for (int ks = 0; ks < D / 32; ks++) {
                                const uint32_t off = (ks >> 2) * (128 * 128) + (ks & 3) * 32;
                                tc_mma8(tmem_s, ad + uint64_t((p * L::kQPart + off) >> 4), bd + uint64_t(off >> 4), idesc_s, p > 0 || ks > 0);
                            }
                        tc_commit(&empty[st]);
                        tc_commit(s_full);
                        if (j + 1 == nb) tc_commit(q_empty);
                    }
                    __syncwarp();
                    r++;
                    if (j > 0) ok = values(j - 1);
                }
                if (ok) ok = values(nb - 1);
                g += nb, tc++;
            }
        } else if (warp == 14) {
            // ------------------------------------------------------------ scales of each 16 keys
            uint32_t g = 0;
            bool ok = true;
            while (ok && walk.next(it)) {
                const int32_t *table = a.tables + size_t(it.seq) * a.table_stride;
                const uint32_t keys = walk.tiles.keys(it.q, it.rtile);
                for (uint32_t kt = it.kt0; kt < it.kt1; kt++, g++) {
                    const uint32_t ss = g % kPpScaleRing, key = kt * kPpKeys + lane * 16;
                    float4 v = make_float4(1.f, 0.f, 1.f, 0.f); // behind the last key: masked whatever stands here
                    if (lane < 8 && key < keys) {
                        const int32_t block = table[key / a.block_tokens];
                        if (uint32_t(block) < a.blocks) {
                            const float2 s = *reinterpret_cast<const float2 *>(a.scales + (size_t(block) * a.kv_heads + it.head) * 2);
                            v = make_float4(s.x, lg2_approx(s.y), 1.f / s.y, 0.f);
                        } else {
                            v.w = 1.f;
                            atomicOr(a.words, kStatusBadBlock);
                        }
                    }
                    if (!mbar_wait(&sc_empty[ss], ((g / kPpScaleRing) & 1) ^ 1, abort_flag)) { give_up(kStatusEmptyTimeout); ok = false; break; }
                    if (lane < 8) scl[ss * 8 + lane] = v;
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&sc_full[ss]);
                }
            }
        }
    } else if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 104;");
        // ------------------------------------------------------------ a tile's Q rows, a thread for each
        const uint32_t row = threadIdx.x - 256, tok = row / G, hq = row % G;
        uint32_t tc = 0;
        while (walk.next(it)) {
            const bool live = tok < it.ntok && row < tpt * G;
            const size_t at = live ? size_t(it.q.row0 + it.tok0 + tok) * a.q_stride + size_t(it.head * G + hq) * D : 0;
            float top = 0.f;
            if (live) {
#pragma unroll 8
                for (int c = 0; c < D; c += 8) {
                    float x[8];
                    paged_load_q8(a, at + c, x);
#pragma unroll
                    for (int e = 0; e < 8; e++) top = fmaxf(top, fabsf(x[e]));
                }
            }
            // a power of two brings the row's largest to [128, 256)
            const int e = min(max(int(__float_as_uint(top) >> 23), 8), 247) - 134;
            const float up = __uint_as_float(uint32_t(127 - e) << 23);
            // the products of the tile before have read the old Q, and its softmax the old factors
            if (!mbar_wait(q_empty, (tc & 1) ^ 1, abort_flag)) { give_up(kStatusMmaTimeout); break; }
            row_e[row] = uint8_t(127 + e);
#pragma unroll 2
            for (int c = 0; c < D; c += 16) {
                float x[2][8];
                if (live) {
                    paged_load_q8(a, at + c, x[0]), paged_load_q8(a, at + c + 8, x[1]);
                } else {
#pragma unroll
                    for (int k = 0; k < 8; k++) x[0][k] = x[1][k] = 0.f;
                }
                uint32_t w[4][PARTS];
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const float *y = &x[k >> 1][(k & 1) * 4];
                    split4<PARTS>(y[0] * up, y[1] * up, y[2] * up, y[3] * up, w[k]);
                }
                uint8_t *dst = sQ + (c >> 7) * (kPpRows * 128) + row * 128 + ((((c >> 4) & 7) ^ (row & 7)) << 4);
#pragma unroll
                for (int p = 0; p < PARTS; p++) *reinterpret_cast<uint4 *>(dst + p * L::kQPart) = make_uint4(w[0][p], w[1][p], w[2][p], w[3][p]);
            }
            fence_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(q_full);
            tc++;
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 168;");
        // ------------------------------------------------------------ softmax; a tile's end
        const uint32_t quarter = warp & 3, half = warp >> 2, row = quarter * 32 + lane;
        const uint32_t lane_addr = (quarter * 32) << 16;
        const uint32_t tok = row / G, hq = row % G;
        uint32_t g = 0, tc = 0;
        bool ok = true;
        while (walk.next(it)) {
            const bool live = tok < it.ntok && row < tpt * G;
            const int32_t lim = it.lim0 + int32_t(tok);
            if (ok && !mbar_wait(q_full, tc & 1, abort_flag)) { give_up(kStatusFullTimeout); ok = false; }
            const float rs = __uint_as_float(uint32_t(row_e[row]) << 23) * a.scale_log2;
            __syncwarp();
            if (lane == 0) mbar_arrive(q_empty); // the factor has been read
            float m = -INFINITY, l = 0.f;
            for (uint32_t kt = it.kt0; kt < it.kt1; kt++, g++) {
                const int32_t key0 = int32_t(kt * kPpKeys + half * 64);
                const uint32_t ss = g % kPpScaleRing, pb = g % NP;
                if (ok && !mbar_wait(&sc_full[ss], (g / kPpScaleRing) & 1, abort_flag)) { give_up(kStatusFullTimeout); ok = false; }
                float c[4], lv[4], iv[4];
                bool bad = false;
#pragma unroll
                for (int b = 0; b < 4; b++) {
                    const float4 v = scl[ss * 8 + half * 4 + b];
                    c[b] = v.x * rs, lv[b] = v.y, iv[b] = v.z;
                    bad |= v.w != 0.f;
                }
                uint32_t badmask = 0;
                if (bad) {
#pragma unroll
                    for (int b = 0; b < 4; b++) badmask |= (scl[ss * 8 + half * 4 + b].w != 0.f ? 1u : 0u) << b;
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(&sc_empty[ss]);
                if (ok && !mbar_wait(s_full, g & 1, abort_flag)) { give_up(kStatusFullTimeout); ok = false; }
                tc_fence_after();
                uint32_t sr[2][32];
                tmem_ld32(tmem_s + lane_addr + half * 64, sr[0]);
                tmem_ld32(tmem_s + lane_addr + half * 64 + 32, sr[1]);
                tmem_wait_ld();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(s_free); // the scores are in registers
                float s[64];
#pragma unroll
                for (int k = 0; k < 64; k++) s[k] = __uint_as_float(sr[k >> 5][k & 31]);
                if (key0 + 64 > it.lim0 || badmask) {
#pragma unroll
                    for (int k = 0; k < 64; k++)
                        if (key0 + k >= lim || (badmask >> (k >> 4) & 1)) s[k] = -INFINITY;
                }
                float mx = -INFINITY;
#pragma unroll
                for (int b = 0; b < 4; b++) {
                    float t[4] = {s[b * 16], s[b * 16 + 1], s[b * 16 + 2], s[b * 16 + 3]};
#pragma unroll
                    for (int k = 4; k < 16; k++) t[k & 3] = fmaxf(t[k & 3], s[b * 16 + k]);
                    mx = fmaxf(mx, fmaf(fmaxf(fmaxf(t[0], t[1]), fmaxf(t[2], t[3])), c[b], lv[b]));
                }
                // the two threads of a row agree on one maximum; rounded up it is still one that no score passes
                __nv_bfloat16 *x = xch + (g & 1) * 256;
                const __nv_bfloat16 up = __float2bfloat16_ru(mx);
                x[half * 128 + row] = up;
                pair_sync(quarter);
                mx = fmaxf(__bfloat162float(up), __bfloat162float(x[(half ^ 1) * 128 + row]));
                const bool need = mx > m + kPpRescale;
                float f = 1.f;
                if (need) {
                    f = ex2_approx(m - mx); // 0 for the first
                    m = mx;
                    l *= f;
                }
                if (kt > it.kt0 && __any_sync(0xffffffffu, need)) {
                    // the product of the tile before must have landed in O
                    const uint32_t gp = g - 1;
                    if (ok && !mbar_wait(&pv_done[gp % NP], (gp / NP) & 1, abort_flag)) { give_up(kStatusMmaTimeout); ok = false; }
                    tc_fence_after();
#pragma unroll 1
                    for (int k = 0; k < D / 2; k += 32) {
                        uint32_t o[32];
                        tmem_ld32(tmem_o + lane_addr + half * (D / 2) + k, o);
                        tmem_wait_ld();
#pragma unroll
                        for (int j = 0; j < 32; j++) o[j] = __float_as_uint(__uint_as_float(o[j]) * f);
                        tmem_st32(tmem_o + lane_addr + half * (D / 2) + k, o);
                    }
                    tmem_wait_st();
                }
                const float base = kPpShift - (m == -INFINITY ? 0.f : m);
                uint32_t pw[PARTS][16];
#pragma unroll
                for (int b = 0; b < 4; b++) {
                    const float d = lv[b] + base;
                    float sum[2] = {0.f, 0.f};
#pragma unroll
                    for (int k = 0; k < 16; k += 4) {
                        float e[4];
#pragma unroll
                        for (int j = 0; j < 4; j++) e[j] = ex2_approx(fmaf(s[b * 16 + k + j], c[b], d));
                        sum[0] += e[0] + e[1], sum[1] += e[2] + e[3];
                        uint32_t w[PARTS];
                        split4<PARTS>(e[0], e[1], e[2], e[3], w);
#pragma unroll
                        for (int p = 0; p < PARTS; p++) pw[p][b * 4 + k / 4] = w[p];
                    }
                    l = fmaf(sum[0] + sum[1], iv[b], l);
                }
                // P buffer: the product of NP tiles ago has read it
                if (ok && !mbar_wait(&pv_done[pb], ((g / NP) & 1) ^ 1, abort_flag)) { give_up(kStatusMmaTimeout); ok = false; }
                tc_fence_after();
#pragma unroll
                for (int p = 0; p < PARTS; p++) tmem_st16(tmem_p + lane_addr + pb * L::kPCols + p * 32 + half * 16, pw[p]);
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&p_full[pb]);
            }
            // ---- the tile's end: two halves of a row's sum become one, O leaves tensor memory
            softmax_sync(); // every warp has read its last maxima: the sums take their place
            lx[half * 128 + row] = l;
            softmax_sync();
            l += lx[(half ^ 1) * 128 + row];
            softmax_sync();
            if (ok && !mbar_wait(o_final, tc & 1, abort_flag)) { give_up(kStatusMmaTimeout); ok = false; }
            tc_fence_after();
            const bool whole = it.kt0 == 0 && it.kt1 == it.tiles;
            const size_t orow = live ? size_t(it.q.row0 + it.tok0 + tok) * a.heads + it.head * G + hq : 0;
            auto finish = [&](int d, float4 v, float inv) { // dims d .. d + 3 of this thread's row
                v.x *= inv, v.y *= inv, v.z *= inv, v.w *= inv;
                if (a.q_and_gate) {
                    const float4 gt = *reinterpret_cast<const float4 *>(a.q_and_gate + orow * 2 * D + D + d);
                    v.x *= sigmoid(gt.x), v.y *= sigmoid(gt.y), v.z *= sigmoid(gt.z), v.w *= sigmoid(gt.w);
                }
                paged_store4(a, orow * D + d, v.x, v.y, v.z, v.w);
            };
            auto inverse = [](float sum) { return sum > 0.f ? 1.f / sum : (sum == 0.f ? 0.f : sum); }; // no key: 0; NaN stays
            float *part = a.parts + (size_t(blockIdx.x) * 2 + (it.kt0 == 0 ? 1 : 0)) * a.part_floats;
            const float inv = inverse(l);
#pragma unroll 1
            for (int k = 0; k < D / 2; k += 32) {
                uint32_t o[32];
                tmem_ld32(tmem_o + lane_addr + half * (D / 2) + k, o);
                tmem_wait_ld();
                if (k + 32 >= D / 2) {
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(o_empty);
                }
                if (live) {
#pragma unroll
                    for (int j = 0; j < 32; j += 4) {
                        const float4 v = make_float4(__uint_as_float(o[j]), __uint_as_float(o[j + 1]), __uint_as_float(o[j + 2]), __uint_as_float(o[j + 3]));
                        const int d = half * (D / 2) + k + j;
                        if (whole) finish(d, v, inv);
                        else *reinterpret_cast<float4 *>(part + size_t(row) * D + d) = v;
                    }
                }
            }
            if (!whole) {
                if (half == 0) *reinterpret_cast<float2 *>(part + kPpRows * D + row * 2) = make_float2(m, l);
                // the last CTA of the item to arrive joins the parts, in the order of the CTAs
                const uint32_t c0 = paged_cta_of(sh, it.first), c1 = paged_cta_of(sh, it.first + it.tiles - 1), parts = c1 - c0 + 1;
                uint32_t *counter = a.words + kPagedCounters + c0;
                __threadfence();
                softmax_sync();
                if (threadIdx.x == 0) {
                    const uint32_t n = atomicAdd(counter, 1);
                    if (n + 1 == parts) *counter = 0;
                    *arrived = n + 1;
                }
                softmax_sync();
                if (*arrived == parts) {
                    __threadfence();
                    if (live) {
                        auto part_of = [&](uint32_t p) { return a.parts + (size_t(c0 + p) * 2 + (p == 0 ? 1 : 0)) * a.part_floats; };
                        float top = -INFINITY, sum = 0.f;
                        for (uint32_t p = 0; p < parts; p++) top = fmaxf(top, __ldcg(part_of(p) + kPpRows * D + row * 2));
                        const float mu = top == -INFINITY ? 0.f : top;
                        for (uint32_t p = 0; p < parts; p++) {
                            const float2 ml = __ldcg(reinterpret_cast<const float2 *>(part_of(p) + kPpRows * D + row * 2));
                            sum += ml.y * ex2_approx(ml.x - mu);
                        }
                        const float is = inverse(sum);
#pragma unroll 1
                        for (int k = 0; k < D / 2; k += 16) {
                            const int d = half * (D / 2) + k;
                            float4 v[4];
#pragma unroll
                            for (int j = 0; j < 4; j++) v[j] = make_float4(0.f, 0.f, 0.f, 0.f);
                            for (uint32_t p = 0; p < parts; p++) {
                                const float *pp = part_of(p);
                                const float wt = ex2_approx(__ldcg(pp + kPpRows * D + row * 2) - mu);
#pragma unroll
                                for (int j = 0; j < 4; j++) {
                                    const float4 u = __ldcg(reinterpret_cast<const float4 *>(pp + size_t(row) * D + d + 4 * j));
                                    v[j].x = fmaf(u.x, wt, v[j].x), v[j].y = fmaf(u.y, wt, v[j].y), v[j].z = fmaf(u.z, wt, v[j].z), v[j].w = fmaf(u.w, wt, v[j].w);
                                }
                            }
#pragma unroll
                            for (int j = 0; j < 4; j++) finish(d + 4 * j, v[j], is);
                        }
                    }
                }
                softmax_sync(); // `arrived` has been read
            }
            tc++;
        }
    }

    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 13) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
}

template <int D, int PARTS>
static int prefill_configure_one() {
    SAETTA_CUDA(cudaFuncSetAttribute(paged_prefill_kernel<D, PARTS>, cudaFuncAttributeMaxDynamicSharedMemorySize, PpLayout<D, PARTS>::kSmem));
    return SAETTA_OK;
}

int paged_prefill_configure(int) {
    int rc = prefill_configure_one<128, 2>();
    if (!rc) rc = prefill_configure_one<128, 3>();
    if (!rc) rc = prefill_configure_one<256, 2>();
    if (!rc) rc = prefill_configure_one<256, 3>();
    return rc;
}

int launch_paged_prefill(const PagedArgs &a, const saetta_paged_cache *cache, int ctas, cudaStream_t stream) {
    CUtensorMap mk, mv;
    const uint32_t box = std::min<uint32_t>(a.block_tokens, kPpKeys);
    if (int rc = paged_map(&mk, cache->keys, cache, box, 1)) return rc;
    if (int rc = paged_map(&mv, cache->values, cache, box, 1)) return rc;
    const bool two = a.q_dtype == SAETTA_BF16; // 8 significant bits: two e4m3 terms
    const uint32_t tpt = kPpRows / a.group;
    void (*kernel)(CUtensorMap, CUtensorMap, PagedArgs, uint32_t) = nullptr;
    size_t smem = 0;
    if (cache->head_dim == 256) {
        kernel = two ? paged_prefill_kernel<256, 2> : paged_prefill_kernel<256, 3>;
        smem = two ? PpLayout<256, 2>::kSmem : PpLayout<256, 3>::kSmem;
    } else {
        kernel = two ? paged_prefill_kernel<128, 2> : paged_prefill_kernel<128, 3>;
        smem = two ? PpLayout<128, 2>::kSmem : PpLayout<128, 3>::kSmem;
    }
    SAETTA_CUDA(launch_pdl(kernel, dim3(unsigned(ctas)), dim3(kPpThreads), smem, stream, mk, mv, a, tpt));
    return SAETTA_OK;
}

} // namespace saetta
