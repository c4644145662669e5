// Attention of many rows (prompts) over the paged e4m3 cache, on the 5th-generation tensor cores.
//
//   s_ij = scale (q_i . kcode_j) ks[block(j)] log2 e,   r_j = vs[block(j)] / vref,   w = 2^(s + log2 r - m),  m some max(s + log2 r)
//   out_i = vref sum_j w_ij vcode_j / sum_j (w_ij / r_j)
//
// The codes are the operands as they lie in memory: no conversion of K or V.  tcgen05's 8-bit products run at twice the
// 16-bit rate, and the two left-hand operands, which are not 8-bit, are split into sums of e4m3 values: a value of 8
// significant bits (bfloat16 q) is the sum of two (4 bits each), one of 11 (binary16 q) of three; of a weight's terms all but the first are e5m2.  Two products at the 8-bit rate take
// the time of one at the 16-bit rate, with half the shared memory for K and V.  The value scales go into the exponent,
// relative to the largest so far (vref, by which O is kept), so a block's scales cost nothing for each score but the constants of one FMA, and
// the sum of the softmax takes them out again for each 16 keys.  (r is not let below 2^-60: a block of zeros, whose scale is
// 2^-126, still counts in the sum; what the bound adds to values is below 2^-60 of the largest.)
//
// A tile is 128 rows: `tpt` tokens x the query heads of one kv head.  Key tiles are 128 keys.  Bound by the tensor pipe: 2 * PARTS *
// 128 * 128 * D multiply-adds for each tile at 8192 a clock and SM.  Roles: sixteen softmax warps in two teams that take
// tiles by turns (two threads for each row, 64 keys each), four warps that bring a tile's Q rows, one warp each for the K/V copies, the score
// products, the scales and the value products.
//
// Measured (bfloat16, 16 query and 2 kv heads of 256, 4096 rows at 28672 keys): 1.85 ms in a stream of calls under the power limit (1.12 PFLOP/s counted as
// 16-bit products).  With head dim 128 a tile has half the products and the same softmax, which then bounds it: a warp needs 5000
// clocks for its tile, two teams so 2600 a tile (1024 of products); binary16 queries 3600 (1536).  7 prompts of 425 to 2554 keys, 32 over 8
// heads of 128, binary16: 683 us (18 of them so that NaN stays with the rows that see it).  Beside the tiles: 14,000 clocks before a CTA's first item (its code and share come cold), 10,000 for the first Q rows (later
// ones come under the tiles before), 12,000 between items, up to 24,000 where the last CTA joins an item's parts.  (A second Q buffer, tried
// for head dim 128: 688 us against 640.  Q rows four at a time, each read by 8 lanes: 900, from spills.)
#include <algorithm>
#include <cfloat>

#include "paged_sched.cuh"
#include "umma.cuh"

namespace saetta {

constexpr int kPpRows = 128, kPpKeys = 128, kPpThreads = 768;
constexpr int kPpWarps = 16;  // of the softmax: two teams of eight, which take the tiles by turns
constexpr int kPpAhead = 2;   // keys are copied this many tiles ahead of the values
// A weight's first term is e4m3, which ends at 448 = 2^8.8: w is kept times 2^6, against a maximum that O follows only when a row's scores pass it by
// 2.5 doublings (w stays below 2^8.5); then all 32 rows of the warp are brought up to date, with one doubling to spare: a
// whole one, so that the weight it stands by is a power of two and not rounded (a key of nearly all weight, or a row's only one).  (With each row
// following for itself past 2 doublings, some row of a CTA did so in every other tile of a random prompt of 8192 keys, and the products wait for
// it; now in one of ten.)
constexpr float kPpShift = 6.f, kPpRescale = 2.5f;
constexpr float kPpHalf = -8.f /* see split_weights */, kPpSpare = 1.f;
// The reference falls where a tile's largest lies 8 doublings below it: kept at 2^-2 at least, that weight and those to 2^-4 of it have all their bits.
constexpr float kPpFall = 8.f, kPpReach = 40.f;
// Largest |log2 of a weight| that f32 holds to an eighth: past it the difference to the maximum, in one FMA, may pass what a first term holds.  Such rows get NaN.
constexpr float kPpMaxScore = 1048576.f;
constexpr uint32_t kPpGroup = 8;  // parts of an item that one CTA joins by itself
constexpr int kPpScaleRing = 4, kPpScales = 9;

// What the roles of a CTA need of an item: one warp walks the items and leaves this in a small ring of shared memory.  (With a walk in
// each role's registers they spilled, and of the 256 KB an SM has for L1 and shared memory this kernel leaves L1 so little that the spills
// missed it: every step of every role took hundreds of clocks.)
struct PpItem {
    uint32_t kt0, kt1;      // key tiles; kt0 == kt1: no more items
    int32_t lim0;           // keys that the first token sees
    uint32_t seq, head;
    uint32_t row0, ntok;    // first row of q, tokens
    uint32_t keys;          // that the last token sees: those to be copied
    uint32_t span;          // the CTAs it lies in: the first, and how many << 16
    float vref;             // by which O is kept after the last tile (written with that tile's scales)
};
constexpr int kPpItems = 3;
constexpr int kPpItemReaders = 2 /* products */ + 1 /* scales */ + 4 /* Q rows */ + kPpWarps;

template <int D, int PARTS>
struct PpLayout {
    static constexpr int kSlabs = D / 128;
    static constexpr int kQPart = kPpRows * D;
    static constexpr int kStage = kPpKeys * D; // K or V of a tile
    static constexpr int kKStages = D == 256 ? 2 : 4, kVStages = D == 256 ? 2 : 4;
    static constexpr int kRing = (kKStages + kVStages) * kStage;
    // the statistics' area: maxima, scales, items, the share, barriers, four words, the rows' exponents
    static constexpr int kBarriers = 2 * (kKStages + kVStages) + 2 * kPpScaleRing + 2 * kPpItems + 3 * 2 + 6 + 16;
    static constexpr int kStats = 4 * kPpRows * 4 + kPpScaleRing * kPpScales * 8 + kPpItems * int(sizeof(PpItem)) + int(sizeof(PagedShare)) + kBarriers * 8 + 16 + kPpRows;
    static_assert((kPpItems * sizeof(PpItem)) % 8 == 0 && sizeof(PagedShare) % 8 == 0, "barriers stand at multiples of 8 bytes");
    static constexpr int kSmem = PARTS * kQPart + kRing + kStats;
    // O; the scores of one tile; the weights' buffers, one or two
    static constexpr int kPBufs = D == 256 && PARTS == 3 ? 1 : 2;
    static constexpr int kPCols = 32 * PARTS;
    static constexpr int kTmemO = 0, kTmemS = D, kTmemP = D + 128;
    static_assert(kTmemP + kPBufs * kPCols <= 512, "fits tensor memory");
    static_assert(kSmem <= 227 * 1024, "fits a CTA's shared memory");
};

// The products are issued under elect.sync's predicate, which the compiler knows to be one lane of a warp in step: five instructions each,
// from uniform registers.  (Under `lane == 0`, or with the predicate inside the instruction, 15 to 27, and 120 clocks for each product, of which the
// pipe needs 64.)
// Descriptors come as their low words; the high word, the same for all (stride 1024 bytes, 128-byte swizzle), is an immediate.
constexpr uint32_t kDescHigh = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t uniform(uint32_t x) { return __shfl_sync(0xffffffffu, x, 0); }
__device__ __forceinline__ void tc_mma8(uint32_t d_tmem, uint32_t adesc, uint32_t bdesc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\tsetp.ne.b32 p, %4, 0;\n\tmov.b64 a, {%1, %5};\n\tmov.b64 b, {%2, %5};\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], a, b, %3, p;\n\t}"
        ::"r"(d_tmem), "r"(adesc), "r"(bdesc), "r"(idesc), "r"(accumulate), "n"(kDescHigh)
        : "memory");
}
// A from tensor memory: row m in lane m, four e4m3 values in a column.
__device__ __forceinline__ void tc_mma8_ts(uint32_t d_tmem, uint32_t a_tmem, uint32_t bdesc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 b;\n\tsetp.ne.b32 p, %4, 0;\n\tmov.b64 b, {%2, %5};\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], [%1], b, %3, p;\n\t}"
        ::"r"(d_tmem), "r"(a_tmem), "r"(bdesc), "r"(idesc), "r"(accumulate), "n"(kDescHigh)
        : "memory");
}
__device__ __forceinline__ uint32_t desc_low(uint32_t saddr, uint32_t lbo_bytes) { return ((saddr & 0x3ffffu) >> 4) | (lbo_bytes >> 4) << 16; }
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t (&r)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%8], {%0,%1,%2,%3,%4,%5,%6,%7};"
                 ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(taddr)
                 : "memory");
}
// Scores from the `see`-th on belong to keys that the row does not see.
__device__ __forceinline__ void mask32(uint32_t (&s)[32], int32_t see) {
    if (see < 32) {
#pragma unroll
        for (int k = 0; k < 32; k++)
            if (k >= see) s[k] = 0xff800000u; // -infinity
    }
}
// Two FMAs, two additions, in one instruction each; the largest of three.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\t"
        "fma.rn.f32x2 x, x, y, z;\n\tmov.b64 {%0, %1}, x;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 d;
    asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tadd.rn.f32x2 x, x, y;\n\tmov.b64 {%0, %1}, x;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
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
// N values as sums of PARTS e4m3 values each: w[p] holds the p-th terms, four to a word.  Every remainder is exact (a value less its
// rounding to fewer bits), so the sum is off by the last term's rounding alone: 2^-8 of the value with two, 2^-12 with three,
// and 2^-10 of a unit below e4m3's normal range.  Stage by stage over all values: each step has the latency of a conversion.
template <int PARTS, int N>
__device__ __forceinline__ void split(float (&x)[N], uint32_t (&w)[PARTS][N / 4]) {
    uint32_t t[N / 2];
    if constexpr (PARTS == 2) {
        // by way of binary16, whose 11 bits hold the two terms
        uint32_t h[N / 2];
#pragma unroll
        for (int i = 0; i < N / 2; i++) h[i] = pack_half2(x[2 * i], x[2 * i + 1]);
#pragma unroll
        for (int i = 0; i < N / 2; i++) t[i] = h2_to_e4m3x2(h[i]);
#pragma unroll
        for (int i = 0; i < N / 4; i++) w[0][i] = prmt(t[2 * i], t[2 * i + 1], 0x5410);
#pragma unroll
        for (int i = 0; i < N / 2; i++) h[i] = hsub2_u32(h[i], e4m3x2_as_h2(t[i]));
#pragma unroll
        for (int i = 0; i < N / 2; i++) t[i] = h2_to_e4m3x2(h[i]);
#pragma unroll
        for (int i = 0; i < N / 4; i++) w[1][i] = prmt(t[2 * i], t[2 * i + 1], 0x5410);
    } else {
#pragma unroll
        for (int p = 0; p < PARTS; p++) {
#pragma unroll
            for (int i = 0; i < N / 2; i++) t[i] = f2_to_e4m3x2(x[2 * i], x[2 * i + 1]);
#pragma unroll
            for (int i = 0; i < N / 4; i++) w[p][i] = prmt(t[2 * i], t[2 * i + 1], 0x5410);
            if (p + 1 < PARTS) {
#pragma unroll
                for (int i = 0; i < N / 2; i++) {
                    const float2 f = h2f2(e4m3x2_as_h2(t[i]));
                    x[2 * i] -= f.x, x[2 * i + 1] -= f.y;
                }
            }
        }
    }
}
// The same for weights, which are not negative, in a third of the time and with more range: the first term is e4m3, those after it are e5m2 (the instruction
// descriptor of each product says which), whose grid ends at 2^-16 where e4m3's ends at 2^-9.  Weights come times 2^-8 (kPpHalf), where the
// exponent field of a binary16 value is that of its e4m3 code, subnormals included, so that the rounded value's bits 14 .. 7 are the code.  What remains,
// exact, is taken back times 2^8, where its upper byte is its e5m2 code, sign included.  The last term is rounded, halves up for odd keys and
// down for even ones (small weights have few bits left and are often halves: all up, 4096 keys under one of nine tenths of the weight came out 0.0002 too
// large), one between is cut.  Off by
// 2^-8 of a weight from 2^-6 up, 2^-14 below (two terms); 2^-11, 2^-17 (three).
template <int PARTS>
__device__ __forceinline__ void split_weights(const float *x, uint32_t (&w)[PARTS]) { // of four
    const uint32_t h0 = pack_half2(x[0], x[1]), h1 = pack_half2(x[2], x[3]);
    const uint32_t t0 = (h0 + 0x00400040u) & 0xff80ff80u, t1 = (h1 + 0x00400040u) & 0xff80ff80u;
    w[0] = prmt(t0 * 2, t1 * 2, 0x7531); // the codes stand in the upper bytes
    uint32_t r0 = hmul2_u32(hsub2_u32(h0, t0), 0x5c005c00u), r1 = hmul2_u32(hsub2_u32(h1, t1), 0x5c005c00u); // times 256
    if (PARTS == 3) {
        w[1] = prmt(r0, r1, 0x7531);
        r0 = hsub2_u32(r0, r0 & 0xff00ff00u), r1 = hsub2_u32(r1, r1 & 0xff00ff00u);
    }
    w[PARTS - 1] = prmt(r0 + 0x0080007fu, r1 + 0x0080007fu, 0x7531);
}
// Each byte of four codes that is NaN (0x7f or 0xff) as 0xff, the others as 0.
__device__ __forceinline__ uint32_t nan_codes(uint32_t w) { return ((((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) >> 7) * 255u; }
__device__ __forceinline__ void sts128(uint32_t addr, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
    asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}
// A bounded wait of a whole warp, in as few instructions as it takes (there are forty of them): polls that the hardware holds for up to a
// millisecond each, 2000 at most.
__device__ __forceinline__ bool short_wait(uint64_t *bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .u32 n;\n\tmov.u32 n, 2000;\n"
        "poll:\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, 1000000;\n\t@p bra over;\n\tsub.u32 n, n, 1;\n\t"
        "setp.ne.u32 p, n, 0;\n\t@p bra poll;\nover:\n\tmov.u32 %0, n;\n\t}"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity)
        : "memory");
    return __all_sync(0xffffffffu, ok != 0);
}
// An f32 value as an unsigned integer, of the same order (0 is below them all), for the largest of several by atomicMax; and back.
__device__ __forceinline__ uint32_t in_order(float x) {
    const uint32_t u = __float_as_uint(x);
    return u ^ (uint32_t(int32_t(u) >> 31) | 0x80000000u);
}
__device__ __forceinline__ float from_order(uint32_t u) { return __uint_as_float(u ^ (uint32_t(int32_t(~u) >> 31) | 0x80000000u)); }

template <int D, int PARTS>
__global__ void __launch_bounds__(kPpThreads, 1)
paged_prefill_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const PagedArgs a, const uint32_t tpt) {
    using L = PpLayout<D, PARTS>;
    constexpr int kSlabs = L::kSlabs, NK = L::kKStages, NV = L::kVStages, NP = L::kPBufs;
    extern __shared__ __align__(1024) uint8_t smem[];
    uint8_t *sQ = smem;                                  // [part][slab][128 rows][128 dims]
    uint8_t *ring = sQ + PARTS * L::kQPart;              // [K stages, V stages][slab][128 keys][128 dims]
    uint8_t *ring_v = ring + NK * L::kStage;
    // the statistics' area
    uint32_t *xch = reinterpret_cast<uint32_t *>(ring + L::kRing); // [4 tiles][128 rows]: maxima, as in_order gives them; 0: none yet
    float *lx = reinterpret_cast<float *>(xch);                    // at a tile's end: [4][128 rows] sums
    float2 *scl = reinterpret_cast<float2 *>(xch + 4 * kPpRows);   // [kPpScaleRing][8]: key scale (-1: bad block), log2 r; then
                                                                   // what vref falls by against the tile before
    PpItem *items = reinterpret_cast<PpItem *>(scl + kPpScaleRing * kPpScales);
    PagedShare *share = reinterpret_cast<PagedShare *>(items + kPpItems);
    uint64_t *bars = reinterpret_cast<uint64_t *>(share + 1);
    uint64_t *k_full = bars, *v_full = k_full + NK, *k_empty = v_full + NV, *v_empty = k_empty + NK, *sc_full = v_empty + NV, *sc_empty = sc_full + kPpScaleRing,
             *item_full = sc_empty + kPpScaleRing, *item_empty = item_full + kPpItems,
             *s_full = item_empty + kPpItems /* one for each team: a wait by parity must not find the other's phase */, *p_full = s_full + 2,
             *pv_done = p_full + 2, *q_full = pv_done + 2, *q_empty = q_full + 1, *s_free = q_full + 2, *o_final = s_free + 1, *o_empty = s_free + 2,
             *all_met = s_free + 3, *x_met = s_free + 4 /* [4 tiles][4 row quarters] */;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(x_met + 16);
    volatile uint32_t *never_set = tmem_slot + 1, *arrived = tmem_slot + 2;
    volatile uint32_t *nan_item = tmem_slot + 3; // bit ni & 1: item ni has NaN in values that some of its rows do not see (set before o_final)
    uint8_t *row_e = reinterpret_cast<uint8_t *>(tmem_slot + 4); // [128]: the power of two (biased) that undoes what a row of Q was scaled by

    const uint32_t warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (smem_u32(smem) & 1023) { // the swizzle and the descriptors count on it
        if (threadIdx.x == 0) atomicOr(a.words, kStatusMmaTimeout);
        return;
    }
    if (threadIdx.x < 4 * kPpRows) xch[threadIdx.x] = 0;
    if (threadIdx.x == 0) {
        for (int s = 0; s < NK; s++) mbar_init(&k_full[s], 1), mbar_init(&k_empty[s], 1);
        for (int s = 0; s < NV; s++) mbar_init(&v_full[s], 1), mbar_init(&v_empty[s], 1);
        for (int s = 0; s < kPpScaleRing; s++) mbar_init(&sc_full[s], 1), mbar_init(&sc_empty[s], 1);
        for (int s = 0; s < kPpItems; s++) mbar_init(&item_full[s], 1), mbar_init(&item_empty[s], kPpItemReaders);
        for (int s = 0; s < 2; s++) mbar_init(&s_full[s], 2), mbar_init(&p_full[s], kPpWarps / 2), mbar_init(&pv_done[s], 1);
        for (int s = 0; s < 16; s++) mbar_init(&x_met[s], 2);
        mbar_init(q_full, 4), mbar_init(q_empty, 1 + kPpWarps), mbar_init(s_free, kPpWarps / 2), mbar_init(o_final, 2), mbar_init(o_empty, kPpWarps);
        mbar_init(all_met, kPpWarps);
        *never_set = 0, *nan_item = 0;
        mbar_fence_init();
    }
    pdl_wait();
    paged_share<kPpKeys>(a, tpt, kPpThreads, reinterpret_cast<uint64_t *>(sQ), share); // (its scratch is the Q area, free until the roles begin)
    if (share->x0 >= share->x1) return; // (the whole CTA)
    if (warp == 21) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(tmem_slot)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    const uint32_t tmem_o = tmem + L::kTmemO, tmem_s = tmem + L::kTmemS, tmem_p = tmem + L::kTmemP;
    // Waits are bounded: one that gives up ends its role, which ends the others' waits the same way.  (No role waits at a named barrier, which
    // would have no bound.)
#define PP_WAIT(bar, parity) \
    if (!short_wait(bar, parity)) goto failed

    uint32_t copied_k = 0, copied_v = 0; // of the copying warp

    // registers: 512 x 96 + 256 x 48 = the 768 x 80 of the launch
    if (warp >= 20) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 48;");
        if (warp == 20) {
            // ------------------------------------------------------------ items; K and V copies: K0 K1 K2 V0 K3 V1 ... through all items
            // (A K stage is free once the scores that use it are done, and those wait for no value product later than the one two
            // tiles before them.)
            const uint32_t bt = min(a.block_tokens, uint32_t(kPpKeys)), per_tile = kPpKeys / bt;
            PagedWalk<kPpKeys> walk(a, *share, tpt);
            const uint32_t tiles = walk.end;
            uint32_t ni = 0, kk = 0, kk1 = 0, keys = 0, head = 0;
            int row[kPpAhead + 1] = {-1, -1, -1}; // of this lane's copy in the cache, of the tile at hand and those before; -1: none
            PagedPages pages;
            auto copy = [&](const CUtensorMap *map, uint64_t *full, uint8_t *dst, int mine) { // a lane for each page and slab
                const int r = __shfl_sync(0xffffffffu, mine, lane / kSlabs);
                const bool good = lane / kSlabs < per_tile && r >= 0;
                const uint32_t copies = __popc(__ballot_sync(0xffffffffu, good));
                if (lane == 0) mbar_expect_tx(full, copies * bt * 128);
                __syncwarp();
                if (good) tma_load_3d(dst + lane % kSlabs * (kPpKeys * 128) + lane / kSlabs * bt * 128, map, full, 0, r, int(lane % kSlabs));
            };
            for (uint32_t i = 0; i < tiles + kPpAhead; i++) {
#pragma unroll
                for (int k = kPpAhead; k > 0; k--) row[k] = row[k - 1];
                if (i < tiles) {
                    if (kk == kk1) {
                        PagedItem it;
                        walk.next(it);
                        kk = it.kt0, kk1 = it.kt1, keys = walk.tiles.keys(it.q, it.rtile), head = it.head;
                        pages.begin(a, it.seq, keys, bt, kk * per_tile);
                        PP_WAIT(&item_empty[ni % kPpItems], (ni / kPpItems & 1) ^ 1);
                        const uint2 span = it.kt0 == 0 && it.kt1 == it.tiles ? make_uint2(0, 1) : paged_ctas_of(*share, it);
                        if (lane == 0) {
                            items[ni % kPpItems] = PpItem{it.kt0, it.kt1, it.lim0, it.seq, it.head, it.q.row0 + it.tok0, it.ntok, keys, span.x | span.y << 16, 0.f};
                            mbar_arrive(&item_full[ni % kPpItems]);
                        }
                        __syncwarp();
                        ni++;
                    }
                    const uint32_t block = uint32_t(pages.of(kk * per_tile));
                    row[0] = lane < per_tile && kk * kPpKeys + lane * bt < keys && block < a.blocks ? int((block * a.kv_heads + head) * a.block_tokens) : -1;
                    kk++;
                    const uint32_t st = i % NK;
                    PP_WAIT(&k_empty[st], (i / NK & 1) ^ 1);
                    copied_k = i + 1;
                    copy(&map_k, &k_full[st], ring + st * L::kStage, row[0]);
                }
                if (i >= kPpAhead) {
                    const uint32_t g = i - kPpAhead, st = g % NV;
                    PP_WAIT(&v_empty[st], (g / NV & 1) ^ 1);
                    copied_v = g + 1;
                    copy(&map_v, &v_full[st], ring_v + st * L::kStage, row[kPpAhead]);
                }
            }
            PP_WAIT(&item_empty[ni % kPpItems], (ni / kPpItems & 1) ^ 1);
            if (lane == 0) {
                items[ni % kPpItems].kt0 = items[ni % kPpItems].kt1 = 0;
                mbar_arrive(&item_full[ni % kPpItems]);
            }
        } else if (warp == 21) {
            // ------------------------------------------------------------ score products
            constexpr uint32_t idesc = (1u << 4) | (uint32_t(kPpKeys >> 3) << 17) | (uint32_t(kPpRows >> 4) << 24);
            const uint32_t ad = uniform(desc_low(smem_u32(sQ), 16)), bd0 = uniform(desc_low(smem_u32(ring), 16)), ts = uniform(tmem_s);
            uint32_t g = 0;
            for (uint32_t ni = 0;; ni++) {
                PP_WAIT(&item_full[ni % kPpItems], ni / kPpItems & 1);
                const uint32_t end = g + uniform(items[ni % kPpItems].kt1 - items[ni % kPpItems].kt0);
                if (g == end) break;
                __syncwarp();
                if (lane == 0) mbar_arrive(&item_empty[ni % kPpItems]);
                PP_WAIT(q_full, ni & 1);
                for (; g < end; g++) {
                    const uint32_t st = g % NK;
                    PP_WAIT(&k_full[st], g / NK & 1);
                    PP_WAIT(&sc_full[g % kPpScaleRing], g / kPpScaleRing & 1);
                    PP_WAIT(s_free, (g & 1) ^ 1);
                    if (lane == 0) mbar_arrive(&s_full[g & 1]); // hands the tile's scales on; the scores follow
                    tc_fence_after();
                    __syncwarp();
                    const uint32_t bd = bd0 + st * (L::kStage >> 4);
                    if (elect_one()) {
#pragma unroll
                        for (uint32_t k = 0; k < PARTS * D / 32; k++) // 32 dims of one term; slabs of 128 dims lie 16 KB apart, the terms of Q behind one another
                            tc_mma8(ts, ad + (k >> 2) * 1024 + (k & 3) * 2, bd + (k >> 2) % kSlabs * 1024 + (k & 3) * 2, idesc, k > 0);
                        tc_commit(&s_full[g & 1]);
                        tc_commit(&k_empty[st]);
                        if (g + 1 == end) tc_commit(q_empty);
                    }
                }
            }
        } else if (warp == 22) {
            // ------------------------------------------------------------ scales of each 16 keys
            uint32_t g = 0;
            for (uint32_t ni = 0;; ni++) {
                PP_WAIT(&item_full[ni % kPpItems], ni / kPpItems & 1);
                const PpItem &it = items[ni % kPpItems];
                const uint32_t keys = it.keys, head = it.head, kt1 = it.kt1;
                uint32_t kt = it.kt0;
                const int32_t *table = a.tables + size_t(it.seq) * a.table_stride;
                if (kt == kt1) break;
                float vref = 0.f;
                for (; kt < kt1; kt++, g++) {
                    const uint32_t ss = g % kPpScaleRing, key = kt * kPpKeys + lane * 16;
                    float2 v = make_float2(1.f, 0.f); // behind the last key: masked whatever stands here
                    bool good = false;
                    if (lane < 8 && key < keys) {
                        const int32_t block = table[key / a.block_tokens];
                        if (uint32_t(block) < a.blocks) {
                            const float2 s = *reinterpret_cast<const float2 *>(a.scales + (size_t(block) * a.kv_heads + head) * 2);
                            v = make_float2(fmaxf(s.x, FLT_MIN), s.y);
                            good = true;
                        } else {
                            v.x = -1.f;
                            atomicOr(a.words, kStatusBadBlock);
                        }
                    }
                    float top = v.y;
#pragma unroll
                    for (int d = 4; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
                    top = fmaxf(fmaxf(__shfl_sync(0xffffffffu, top, 0), FLT_MIN), vref);
                    v.y = good ? fmaxf(lg2_approx(v.y / top), -60.f) : 0.f;
                    if (lane == 8) v = make_float2(vref > 0.f ? vref / top : 1.f, top);
                    vref = top;
                    PP_WAIT(&sc_empty[ss], (g / kPpScaleRing & 1) ^ 1);
                    if (lane < kPpScales) scl[ss * kPpScales + lane] = v;
                    if (lane == 0 && kt + 1 == kt1) items[ni % kPpItems].vref = vref;
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&sc_full[ss]);
                }
                if (lane == 0) mbar_arrive(&item_empty[ni % kPpItems]);
            }
        } else {
            // ------------------------------------------------------------ value products
            constexpr uint32_t idesc = (1u << 4) | (1u << 16) | (uint32_t(D >> 3) << 17) | (uint32_t(kPpRows >> 4) << 24), a_e5m2 = 1u << 7;
            const uint32_t bd0 = uniform(desc_low(smem_u32(ring_v), kPpKeys * 128)), to = uniform(tmem_o), tp = uniform(tmem_p);
            uint32_t g = 0;
            for (uint32_t ni = 0;; ni++) {
                PP_WAIT(&item_full[ni % kPpItems], ni / kPpItems & 1);
                const int32_t keys = int32_t(items[ni % kPpItems].keys);
                const uint32_t kt0 = uniform(items[ni % kPpItems].kt0), kt1 = uniform(items[ni % kPpItems].kt1);
                const int32_t lim0 = items[ni % kPpItems].lim0;
                uint32_t nan_found = 0;
                if (kt0 == kt1) break;
                __syncwarp();
                if (lane == 0) mbar_arrive(&item_empty[ni % kPpItems]);
                for (uint32_t kt = kt0; kt < kt1; kt++, g++) {
                    const uint32_t st = g % NV, pb = g % NP, ss = g % kPpScaleRing;
                    PP_WAIT(&v_full[st], g / NV & 1);
                    PP_WAIT(&sc_full[ss], g / kPpScaleRing & 1);
                    // rows behind the last key, and of bad blocks, may hold NaN, which a weight of 0 does not silence
                    const int32_t key0 = int32_t(kt * kPpKeys);
                    const uint32_t bad = __ballot_sync(0xffffffffu, lane < 8 && scl[ss * kPpScales + (lane & 7)].x < 0.f);
                    const uint32_t tile = smem_u32(ring_v) + st * L::kStage;
                    if (key0 + kPpKeys > keys || bad) {
#pragma unroll 1
                        for (uint32_t slab = 0; slab < kSlabs; slab++) {
                            const uint32_t end = tile + (slab + 1) * (kPpKeys * 128);
#pragma unroll 1
                            for (uint32_t at = end - kPpKeys * 128 + lane * 16, key = lane >> 3; bad && at < end; at += 512, key += 4)
                                if (bad >> (key >> 4) & 1) sts128(at, 0, 0, 0, 0);
#pragma unroll 1
                            for (uint32_t at = end - min(uint32_t(key0 + kPpKeys - keys), 128u) * 128 + lane * 16; key0 + kPpKeys > keys && at < end; at += 512) sts128(at, 0, 0, 0, 0);
                        }
                        fence_async_smem();
                        __syncwarp();
                    }
                    if (lim0 < keys && key0 + kPpKeys > lim0) {
                        // Keys that some rows do not see, and a weight of 0 does not silence NaN either: it becomes 0 to the products, and NaN again at the tile's end in
                        // the rows that see the key.
                        const uint32_t hi = tile + uint32_t(min(keys - key0, kPpKeys)) * 128;
                        bool found = false;
#pragma unroll
                        for (uint32_t slab = 0; slab < kSlabs; slab++)
#pragma unroll 2
                            for (uint32_t at = tile + uint32_t(max(lim0 - key0, 0)) * 128 + lane * 16; at < hi; at += 512) {
                                const uint4 v = lds128(at + slab * (kPpKeys * 128));
                                const uint32_t x = nan_codes(v.x), y = nan_codes(v.y), z = nan_codes(v.z), w = nan_codes(v.w);
                                if (x | y | z | w) {
                                    sts128(at + slab * (kPpKeys * 128), v.x & ~x, v.y & ~y, v.z & ~z, v.w & ~w);
                                    found = true;
                                }
                            }
                        if (__any_sync(0xffffffffu, found)) {
                            fence_async_smem();
                            __syncwarp();
                            nan_found = 1;
                        }
                    }
                    if (kt == kt0) PP_WAIT(o_empty, (ni & 1) ^ 1);
                    // (Behind that wait: it shows that the item before has had both its arrivals, so that this one counts for its own.)
                    if (kt + 1 == kt1 && lane == 0) {
                        *nan_item = (*nan_item & ~(1u << (ni & 1))) | nan_found << (ni & 1);
                        mbar_arrive(o_final);
                    }
                    PP_WAIT(&p_full[pb], g / NP & 1);
                    tc_fence_after();
                    __syncwarp();
                    const uint32_t bd = bd0 + st * (L::kStage >> 4), ap = tp + pb * L::kPCols;
                    if (elect_one()) {
#pragma unroll
                        for (uint32_t k = 0; k < PARTS * kPpKeys / 32; k++) // 32 keys of one term
                            tc_mma8_ts(to, ap + k * 8, bd + (k & 3) * 256, k < kPpKeys / 32 ? idesc : idesc | a_e5m2, k ? 1u : kt - kt0);
                        tc_commit(&pv_done[g & 1]);
                        tc_commit(&v_empty[st]);
                        tc_commit(&sc_empty[ss]); // (its softmax is over too)
                        if (kt + 1 == kt1) tc_commit(o_final);
                    }
                }
            }
        }
    } else if (warp >= 16) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 48;");
        // ------------------------------------------------------------ a tile's Q rows, a thread for each
        const uint32_t row = threadIdx.x - 512, tok = row / a.group, hq = row % a.group;
        for (uint32_t ni = 0;; ni++) {
            PP_WAIT(&item_full[ni % kPpItems], ni / kPpItems & 1);
            const PpItem &it = items[ni % kPpItems];
            if (it.kt0 == it.kt1) break;
            const bool live = tok < it.ntok && row < tpt * a.group;
            const size_t at = live ? size_t(it.row0 + tok) * a.q_stride + size_t(it.head * a.group + hq) * D : 0;
            __syncwarp();
            if (lane == 0) mbar_arrive(&item_empty[ni % kPpItems]);
            float top = 0.f;
            if (live) {
#pragma unroll 2
                for (int c = 0; c < D; c += 8) {
                    float x[8];
                    paged_load_q8(a, at + c, x);
#pragma unroll
                    for (int e = 0; e < 8; e++) top = fmaxf(top, fabsf(x[e]));
                }
            }
            // a power of two brings the row's largest to [128, 256)
            const int e = min(max(int(__float_as_uint(top) >> 23), 8), 254) - 134;
            const float up = __uint_as_float(uint32_t(127 - e) << 23);
            // the products of the tile before have read the old Q, and its softmax the old factors
            PP_WAIT(q_empty, (ni & 1) ^ 1);
            row_e[row] = uint8_t(127 + e);
#pragma unroll 1
            for (int c = 0; c < D; c += 16) {
                uint8_t *dst = sQ + (c >> 7) * (kPpRows * 128) + row * 128 + ((((c >> 4) & 7) ^ (row & 7)) << 4);
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    float x[8];
                    if (live) {
                        paged_load_q8(a, at + c + 8 * h, x);
                    } else {
#pragma unroll
                        for (int k = 0; k < 8; k++) x[k] = 0.f;
                    }
                    uint32_t w[PARTS][2];
#pragma unroll
                    for (int k = 0; k < 8; k++) x[k] = fmaf(x[k], up, x[k] * 0.f); // (an infinity becomes NaN: e4m3 has none)
                    split<PARTS, 8>(x, w);
#pragma unroll
                    for (int p = 0; p < PARTS; p++) *reinterpret_cast<uint2 *>(dst + p * L::kQPart + 8 * h) = make_uint2(w[p][0], w[p][1]);
                }
            }
            fence_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(q_full);
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 96;");
        // ------------------------------------------------------------ softmax; a tile's end
        // Two teams of eight warps take the tiles by turns, so that one team's loads, maxima and hand-overs run under the other's exponentials
        // and the products.  A team takes its 128 x 128 scores into registers at once, which frees their place for the next tile's.  What a
        // tile needs of the one before it is only the running maximum.
        // (At 4096 rows by 32768 keys, when it was tried: one tile at a time by eight warps 2.25 ms, by sixteen 2.2; two teams with the scores left in
        // tensor memory, the weights written over them: 1.94, the two teams in step and the products between them; as it is: 1.55.)
        const uint32_t quarter = warp & 3, half = warp >> 2 & 1, team = warp >> 3, row = quarter * 32 + lane;
        const uint32_t lane_addr = (quarter * 32) << 16;
        uint32_t g = 0, all = 0; // tiles, meetings of all warps, so far
        for (uint32_t ni = 0;; ni++) {
            PP_WAIT(&item_full[ni % kPpItems], ni / kPpItems & 1);
            const uint32_t kt0 = items[ni % kPpItems].kt0, kt1 = items[ni % kPpItems].kt1;
            if (kt0 == kt1) break;
            const int32_t lim0 = items[ni % kPpItems].lim0;
            const int32_t lim = lim0 + int32_t(row / a.group);
            PP_WAIT(q_full, ni & 1);
            const float rs = __uint_as_float(uint32_t(row_e[row]) << 23) * a.scale_log2;
            __syncwarp();
            if (lane == 0) mbar_arrive(q_empty); // the factor has been read
            float m = -INFINITY, l = 0.f, hi = -INFINITY;
            // What a tile's weights stand against, after a tile whose largest is 2^top (the same in all four warps that share the rows).  `top` is of
            // s + log2 r over the keys that the row sees: of what they put into O, so that a block of large values which the row hardly or not
            // yet sees takes no bits from the others.  It goes down as well, so that neither does a key of much weight in an earlier tile, but for
            // no more than 2^kPpReach below the largest so far: l, the sum without r, stays below 2^(kPpReach + 60 + 31).
            auto follow = [&](float was, float top) {
                hi = fmaxf(hi, top);
                const float low = fmaxf(top + kPpSpare, hi - kPpReach);
                const bool down = low < was - kPpFall && top > -INFINITY;
                if (!__any_sync(0xffffffffu, top > was + kPpRescale || down)) return was;
                return down ? low : fmaxf(was, top + kPpSpare);
            };
            for (uint32_t kt = kt0; kt < kt1; kt++, g++) {
                if ((g & 1) != team) continue;
                const int32_t key0 = int32_t(kt * kPpKeys + half * 64);
                const uint32_t ss = g % kPpScaleRing, pb = g % NP;
                const float2 *sc = scl + ss * kPpScales + half * 4;
                PP_WAIT(&s_full[team], g >> 1 & 1);
                tc_fence_after();
                uint32_t s[2][32];
                tmem_ld32(tmem_s + lane_addr + half * 64, s[0]);
                tmem_ld32(tmem_s + lane_addr + half * 64 + 32, s[1]);
                tmem_wait_ld();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(s_free); // the scores are in registers
                if (key0 + 64 > lim0) {
                    mask32(s[0], lim - key0);
                    mask32(s[1], lim - key0 - 32);
                }
                float mx = -INFINITY;
#pragma unroll
                for (int b = 0; b < 4; b++) {
                    const float f = sc[b].x;
                    if (f < 0.f) { // a bad block: what its place in shared memory held before
#pragma unroll
                        for (int k = 0; k < 16; k++) s[b >> 1][(b & 1) * 16 + k] = 0xff800000u;
                    }
                    const float *x = reinterpret_cast<const float *>(&s[b >> 1][(b & 1) * 16]);
                    float t[2] = {max3(x[0], x[1], x[2]), max3(x[3], x[4], x[5])};
                    t[0] = max3(t[0], x[6], x[7]), t[1] = max3(t[1], x[8], x[9]), t[0] = max3(t[0], x[10], x[11]), t[1] = max3(t[1], x[12], x[13]);
                    mx = fmaxf(mx, fmaf(fmaxf(max3(t[0], x[14], x[15]), t[1]), fmaxf(fabsf(f) * rs, FLT_MIN), sc[b].y)); // (not 0: that times a masked key's -infinity is NaN)
                }
                // The two threads of a row agree on one maximum.  Every warp follows the running maximum through all tiles: the other team's tile first,
                // then its own.  (The maxima go through shared memory in f32: in bfloat16, whatever way it is rounded, one of 1000 is off by
                // several doublings, and the weights with it.)  A slot is cleared three tiles after its own, by the other team: waiting for the
                // tile before this one has shown that all four warps of these rows are past the two tiles in which they read it.
                const uint32_t xs = g & 3;
                float m_was = -INFINITY;
                if (kt > kt0) {
                    const uint32_t xo = (g - 1) & 3;
                    PP_WAIT(&x_met[xo * 4 + quarter], (g - 1) >> 2 & 1);
                    m_was = follow(m, from_order(xch[xo * kPpRows + row]));
                }
                if (half == 0) xch[((g + 1) & 3) * kPpRows + row] = 0;
                atomicMax(&xch[xs * kPpRows + row], in_order(mx));
                __syncwarp();
                if (lane == 0) mbar_arrive(&x_met[xs * 4 + quarter]);
                PP_WAIT(&x_met[xs * 4 + quarter], g >> 2 & 1);
                const float mt = follow(m_was, from_order(xch[xs * kPpRows + row]));
                if (mt != m) {
                    l *= ex2_approx(m - mt); // 0 for the first
                    m = mt;
                }
                const bool need = __any_sync(0xffffffffu, mt != m_was);
                const float fv = scl[ss * kPpScales + 8].x;
                if (kt > kt0 && (need || fv != 1.f)) {
                    // The product of the tile before must have landed in O.  (That of two tiles before first: it shares no barrier with it, and
                    // once it is done the barrier waited for next is in the phase asked for or the one before.)
                    if (g >= 2 && NP == 2) PP_WAIT(&pv_done[g & 1], (g - 2) >> 1 & 1);
                    PP_WAIT(&pv_done[(g - 1) & 1], (g - 1) >> 1 & 1);
                    tc_fence_after();
                    const float f = (mt != m_was ? ex2_approx(m_was - mt) : 1.f) * fv;
#pragma unroll 1
                    for (int k = 0; k < D / 2; k += 16) {
                        uint32_t o[16];
                        tmem_ld16(tmem_o + lane_addr + half * (D / 2) + k, o);
                        tmem_wait_ld();
#pragma unroll
                        for (int j = 0; j < 16; j++) o[j] = __float_as_uint(__uint_as_float(o[j]) * f);
                        tmem_st16(tmem_o + lane_addr + half * (D / 2) + k, o);
                    }
                    tmem_wait_st();
                }
                const float base = kPpShift + kPpHalf - (m == -INFINITY ? 0.f : m);
                float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
                for (int h = 0; h < 3; h++) {
                    // the exponentials of 32 keys, and between them the terms of the 32 before: the two run on different units
                    uint32_t pw[PARTS][8];
#pragma unroll
                    for (int q = 0; q < 8; q++) {
                        if (h < 2) {
                            float *e = reinterpret_cast<float *>(&s[h][q * 4]);
                            const float2 f = sc[h * 2 + (q >> 2)];
                            const float c = fmaxf(fabsf(f.x) * rs, FLT_MIN), d = f.y + base;
                            const float2 t0 = fma2(make_float2(e[0], e[1]), make_float2(c, c), make_float2(d, d));
                            const float2 t1 = fma2(make_float2(e[2], e[3]), make_float2(c, c), make_float2(d, d));
                            e[0] = ex2_approx(t0.x), e[1] = ex2_approx(t0.y), e[2] = ex2_approx(t1.x), e[3] = ex2_approx(t1.y);
                        }
                        if (h > 0) {
                            const float *e = reinterpret_cast<const float *>(&s[h - 1][q * 4]);
                            uint32_t w[PARTS];
                            split_weights<PARTS>(e, w);
#pragma unroll
                            for (int p = 0; p < PARTS; p++) pw[p][q] = w[p];
                            sum[q & 1] = add2(sum[q & 1], add2(make_float2(e[0], e[1]), make_float2(e[2], e[3])));
                            if (q & 2 && q & 1) {
                                const float2 t = add2(sum[0], sum[1]);
                                l = fmaf(t.x + t.y, ex2_approx(-sc[(h - 1) * 2 + (q >> 2)].y), l);
                                sum[0] = sum[1] = make_float2(0.f, 0.f);
                            }
                        }
                    }
                    if (h == 1 && g >= uint32_t(NP)) { // the product of NP tiles ago has read this buffer (pv_done: a barrier for even and one for odd tiles)
                        PP_WAIT(&pv_done[(g - NP) & 1], (g - NP) >> 1 & 1);
                        tc_fence_after();
                    }
                    if (h > 0) {
#pragma unroll
                        for (int p = 0; p < PARTS; p++) tmem_st8(tmem_p + lane_addr + pb * L::kPCols + p * 32 + half * 16 + (h - 1) * 8, pw[p]);
                    }
                }
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&p_full[pb]);
            }
            // ---- the tile's end: the four sums of a row become one, O leaves tensor memory
#define PP_MEET_ALL()                                      \
    __syncwarp();                                          \
    if (lane == 0) mbar_arrive(all_met);                   \
    PP_WAIT(all_met, all++ & 1)
            if (((g - 1) & 1) != team) { // the last tile was the other team's
                PP_WAIT(&x_met[((g - 1) & 3) * 4 + quarter], (g - 1) >> 2 & 1);
                const float mt = follow(m, from_order(xch[((g - 1) & 3) * kPpRows + row]));
                if (mt != m) l *= ex2_approx(m - mt);
                m = mt;
            }
            PP_MEET_ALL(); // all maxima have been read: the sums take their place
            lx[(team * 2 + half) * 128 + row] = l;
            PP_MEET_ALL();
            l = ((lx[row] + lx[128 + row]) + (lx[256 + row] + lx[384 + row])) * 256.f; // (the weights' sums were taken times 2^-8)
            if (fabsf(hi) > kPpMaxScore && hi > -INFINITY) l = __uint_as_float(0x7fc00000u);
            PP_MEET_ALL();
            const PpItem &it = items[ni % kPpItems];
            const uint32_t cq = warp >> 2, tok = row / a.group, hq = row % a.group;
            const bool live = tok < it.ntok && row < tpt * a.group;
            const uint32_t c0 = it.span & 0xffff, parts = it.span >> 16;
            const size_t orow = live ? size_t(it.row0 + tok) * a.heads + it.head * a.group + hq : 0;
            const float vref = it.vref;
            PP_WAIT(o_final, ni & 1);
            tc_fence_after();
            auto finish = [&](int d, float4 v, float inv) { // dims d .. d + 3 of this thread's row
                v.x *= inv, v.y *= inv, v.z *= inv, v.w *= inv;
                if (a.q_and_gate) {
                    const float4 gt = *reinterpret_cast<const float4 *>(a.q_and_gate + orow * 2 * D + D + d);
                    v.x *= sigmoid(gt.x), v.y *= sigmoid(gt.y), v.z *= sigmoid(gt.z), v.w *= sigmoid(gt.w);
                }
                paged_store4(a, orow * D + d, v.x, v.y, v.z, v.w);
            };
            auto inverse = [](float sum) { return sum > 0.f ? 1.f / sum : (sum == 0.f ? 0.f : sum); }; // no key: 0; NaN stays
            float *part = a.parts + (size_t(blockIdx.x) * 2 + (kt0 == 0 ? 1 : 0)) * a.part_floats;
            const float inv = inverse(l) * vref;
#pragma unroll 1
            for (int k = 0; k < D / 4; k += 16) {
                uint32_t o[16];
                tmem_ld16(tmem_o + lane_addr + cq * (D / 4) + k, o);
                tmem_wait_ld();
                if (k + 16 >= D / 4) {
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(o_empty);
                }
                if (live) {
#pragma unroll
                    for (int j = 0; j < 16; j += 4) {
                        const float4 v = make_float4(__uint_as_float(o[j]), __uint_as_float(o[j + 1]), __uint_as_float(o[j + 2]), __uint_as_float(o[j + 3]));
                        const int d = cq * (D / 4) + k + j;
                        if (parts == 1) finish(d, v, inv);
                        else *reinterpret_cast<float4 *>(part + size_t(row) * D + d) = v;
                    }
                }
            }
            if (*nan_item >> (ni & 1) & 1) { // dims that some rows see as NaN
                const uint32_t bt = a.block_tokens;
                const int32_t end = min(lim, int32_t(min(it.keys, kt1 * kPpKeys)));
#pragma unroll 1
                for (int32_t key = max(lim0, int32_t(kt0 * kPpKeys)); live && key < end; key++) {
                    const uint32_t block = uint32_t(a.tables[size_t(it.seq) * a.table_stride + uint32_t(key) / bt]);
                    if (block >= a.blocks) continue;
                    const uint8_t *code = a.values + ((size_t(block) * a.kv_heads + it.head) * bt + uint32_t(key) % bt) * D;
#pragma unroll 1
                    for (uint32_t d = cq * (D / 4); d < (cq + 1) * (D / 4); d++) {
                        if ((code[d] & 0x7f) != 0x7f) continue;
                        if (parts > 1) part[size_t(row) * D + d] = __uint_as_float(0x7fc00000u);
                        else if (a.out_dtype == SAETTA_F32) static_cast<uint32_t *>(a.out)[orow * D + d] = 0x7fc00000u;
                        else static_cast<uint16_t *>(a.out)[orow * D + d] = a.out_dtype == SAETTA_F16 ? 0x7e00 : 0x7fc0;
                    }
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&item_empty[ni % kPpItems]);
            if (parts > 1) {
                if (cq == 0) *reinterpret_cast<float2 *>(part + kPpRows * D + row * 2) = make_float2(m, l);
                if (warp == 0 && lane == 0) part[kPpRows * (D + 2)] = vref;
                // The parts are joined by the last CTA to arrive, in the order of the CTAs; many of them in two rounds, groups of some first.
                uint32_t per = parts;
                if (parts > kPpGroup) {
                    per = 2;
                    while (per * per < parts) per++;
                }
                const uint32_t groups = (parts + per - 1) / per, mine = (blockIdx.x - c0) / per;
                uint32_t lo = mine * per, step = 1, n = min(per, parts - lo);
                // a group's counter: by its first CTA, which may begin another item's tail as well
                uint32_t *counter = a.words + kPagedCounters + (mine ? gridDim.x : 0) + c0 + lo;
                auto part_of = [&](uint32_t p) { return a.parts + (size_t(c0 + lo + p * step) * 2 + (lo + p * step == 0 ? 1 : 0)) * a.part_floats; };
#pragma unroll 1
                for (bool last = groups == 1;; last = true) {
                    PP_MEET_ALL();
                    if (warp == 0 && lane == 0) {
                        __threadfence(); // (the others' writes too: they came before the meeting)
                        const uint32_t k = atomicAdd(counter, 1) + 1;
                        if (k == n) *counter = 0;
                        __threadfence();
                        *arrived = k;
                    }
                    PP_MEET_ALL();
                    const bool mine_to_do = *arrived == n;
                    PP_MEET_ALL(); // `arrived` has been read
                    if (!mine_to_do) break;
                    // each row's maximum and sum; the weights take the place of the parts' maxima
                    float top = -INFINITY, sum = 0.f, vtop = 0.f;
                    if (cq == 0 && live) {
#pragma unroll 4
                        for (uint32_t p = 0; p < n; p++) {
                            top = fmaxf(top, __ldcg(part_of(p) + kPpRows * D + row * 2));
                            vtop = fmaxf(vtop, __ldcg(part_of(p) + kPpRows * (D + 2)));
                        }
                        const float mu = top == -INFINITY ? 0.f : top;
#pragma unroll 4
                        for (uint32_t p = 0; p < n; p++) {
                            float2 *ml = reinterpret_cast<float2 *>(part_of(p) + kPpRows * D + row * 2);
                            const float2 x = __ldcg(ml);
                            const float w = ex2_approx(x.x - mu);
                            sum = fmaf(x.y, w, sum);
                            __stcg(&ml->x, w * (__ldcg(part_of(p) + kPpRows * (D + 2)) / vtop));
                        }
                        lx[row] = inverse(sum) * vtop;
                        __threadfence();
                    }
                    PP_MEET_ALL();
                    if (live) {
                        const float is = lx[row];
#pragma unroll 1
                        for (int k = 0; k < D / 4; k += 8) {
                            const int d = cq * (D / 4) + k;
                            float4 v[2] = {make_float4(0.f, 0.f, 0.f, 0.f), make_float4(0.f, 0.f, 0.f, 0.f)};
#pragma unroll 4
                            for (uint32_t p = 0; p < n; p++) {
                                const float *pp = part_of(p);
                                const float wt = __ldcg(pp + kPpRows * D + row * 2);
#pragma unroll
                                for (int j = 0; j < 2; j++) {
                                    const float4 u = __ldcg(reinterpret_cast<const float4 *>(pp + size_t(row) * D + d + 4 * j));
                                    v[j].x = fmaf(u.x, wt, v[j].x), v[j].y = fmaf(u.y, wt, v[j].y), v[j].z = fmaf(u.z, wt, v[j].z), v[j].w = fmaf(u.w, wt, v[j].w);
                                }
                            }
#pragma unroll
                            for (int j = 0; j < 2; j++) {
                                if (last) finish(d + 4 * j, v[j], is);
                                else *reinterpret_cast<float4 *>(part_of(0) + size_t(row) * D + d + 4 * j) = v[j];
                            }
                        }
                    }
                    if (last) break;
                    PP_MEET_ALL(); // the weights have been read
                    if (cq == 0 && live) *reinterpret_cast<float2 *>(part_of(0) + kPpRows * D + row * 2) = make_float2(top, sum);
                    if (warp == 0 && lane == 0) part_of(0)[kPpRows * (D + 2)] = vtop; // (row 0 is always live)
                    lo = 0, step = per, n = groups, counter = a.words + kPagedCounters + 2 * gridDim.x + c0;
                }
                PP_MEET_ALL(); // the joined sums have been read
            }
            xch[threadIdx.x] = 0; // the next item's maxima take the sums' place
            PP_MEET_ALL();
        }
    }
    goto done;
failed:
    if (lane == 0) atomicOr(a.words, kStatusMmaTimeout);
done:
    if (warp == 20) { // what was issued lands before the shared memory goes (it has, unless a wait gave up)
        for (uint32_t k = copied_k > NK ? copied_k - NK : 0; k < copied_k; k++) mbar_wait(&k_full[k % NK], (k / NK) & 1, never_set, 200000u);
        for (uint32_t k = copied_v > NV ? copied_v - NV : 0; k < copied_v; k++) mbar_wait(&v_full[k % NV], (k / NV) & 1, never_set, 200000u);
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    __syncwarp();
    if (warp == 21) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
#undef PP_WAIT
#undef PP_MEET_ALL
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
