// Attention of few rows (single tokens, verify rows) over the paged e4m3 cache.
//
//   s_ij = scale (q_i . kcode_j) ks[block(j)],  out_i = sum_j p_ij vs[block(j)] vcode_j / sum_j p_ij,  p = exp(s - max)
//
// A block's scales leave the products: they multiply a score, and a probability, of a whole block, so the codes go to the
// tensor cores as they are (an e4m3 value is a binary16 value).  Bound by the cache's bytes, 2 * head_dim for each key and
// kv head; the rest is arranged so that these stream without a pause:
//
//  * One CTA for each SM takes an equal share of all key tiles (paged_sched.cuh); producer warps keep a ring of
//    tiles of K and V in flight (64 keys with head dim 256, 128 with 128; TMA tensor copies of whole pages, 128-byte
//    swizzle: 160 KB on the way) and the pages' scales beside them (8-byte asynchronous copies).
//  * Eight consumer warps, four for each tile, 16 or 32 keys a warp, each with its own running maximum, sum and accumulators: no
//    barrier between tiles.  Keys are the 16 rows of mma.m16n8k16, query rows its 8 columns (a group of 8 heads fills them).
//    The order of dims inside a product is free, so a lane feeds 16 consecutive bytes of a key to four products; with the
//    swizzle, chunk 2 t + j for lane t of a key makes these 128-bit loads free of bank conflicts, and chunk g for lane
//    group g those of the values.
//  * Values enter as pairs of keys of one dim: two byte permutes for four dims, then the conversion to binary16.
//  * P is rounded to binary16 (11 bits; with the value scale in it, relative to the largest of the warp's so far; the maximum it stands against is of both, over the
//    keys that the row sees), scores, sums and accumulators are f32.  Queries enter as binary16 after a power of two for each row, so bfloat16's range
//    fits; f32 queries are rounded to 11 bits there.
//
// Measured: one sequence of 131072 keys (bfloat16, 16 query and 2 kv heads of 256) 40.5 us (3.3 TB/s; the bytes alone take 20.5), 61 sequences of up to
// 8192 keys (binary16, 32 over 8 heads of 128) 125 us (3.8 TB/s), 701 keys 12.6 us.  What is left beyond the bytes is the start of a CTA (its share, the
// first pages, the first bytes: 6 us), the change of items, and the parts' joining (3 to 4 us a round).  (One warp for keys, values and scales together: 61 sequences 139 us; copies issued page
// by page from one lane: 173; scores of two products for 32 rows in place of the many-rows kernel: 138 against 96.)
#include <algorithm>
#include <cfloat>

#include "paged_sched.cuh"
#include "umma.cuh"

namespace saetta {

constexpr int kPdThreads = 384;  // 8 consumer warps; items and keys, values, scales; one warp that makes up the group of 4
constexpr uint32_t kPdGroup = 12; // parts of an item that one CTA joins by itself; one more in each of two rounds
static_assert((kPdGroup + 1) * (kPdGroup + 1) >= uint32_t(kPagedMaxCtas), "two rounds join the parts of every CTA");
constexpr float kPdRescale = 8.f; // the accumulators follow the running maximum only past this many doublings
constexpr float kPdShift = 7.f;   // weights are kept times this many doublings: binary16 ends at 2^16, and is whole down to 2^-14

template <int D, int NT>
struct PdLayout {
    static constexpr int kRows = 8 * NT;
    static constexpr int kSub = D == 256 ? 1 : 2;  // 16-key pieces that a warp takes of a tile
    static constexpr int kTile = 64 * kSub;        // keys of a tile
    static constexpr int kSide = kTile * D;
    static constexpr int kStage = 2 * kSide;       // 32 KB
    static constexpr int kStages = 5;
    // Barriers of landed tiles, two for each stage.  The teams take tiles by turns and the stages are odd in number, so a stage goes from team to team: on
    // one barrier a team would see every other phase, always of one parity, and take an older use of its own for the tile it waits for.
    static constexpr int kFull = 2 * kStages;
    static constexpr int kPages = kTile / 16;      // of a tile, at most
    static_assert(kRows * D / 4 >= 256, "every consumer has values to join");
    static constexpr int kRow = 128 + 4;                      // floats of one row of the exchange buffer
    static constexpr int kExchange = 8 * 8 * kRow * 4;        // 8 warps x 8 rows of 128 dims
    static constexpr int kRing = kStages * kStage;
    static constexpr int kSmem = 1024 + kRing + kExchange + kStages * kPages * 8 /*scales*/ + 3 * 1024 /*barriers, items, statistics*/;
};
static_assert(PdLayout<256, 2>::kSmem <= 227 * 1024 && PdLayout<128, 2>::kSmem <= 227 * 1024, "fits a CTA's shared memory");

__device__ __forceinline__ uint32_t e4m3x2_to_h2(uint32_t w) {
    uint32_t h;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(uint16_t(w)));
    return h;
}
__device__ __forceinline__ void cp_async8(void *dst, const void *src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
// Arrives on `bar` once this thread's asynchronous copies so far have landed (at once if there are none).
__device__ __forceinline__ void cp_async_arrive(uint64_t *bar) {
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void consumers_sync() { asm volatile("bar.sync 1, 256;" ::: "memory"); }

// All consumers: whether `yes` holds for each of them.
__device__ __forceinline__ bool consumers_all(bool yes) {
    uint32_t r;
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbarrier.cta.red.and.pred q, 1, 256, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
                 : "=r"(r)
                 : "r"(uint32_t(yes))
                 : "memory");
    return r;
}

// What the consumers need of an item; the producer walks the items and leaves this in a ring of shared memory.
struct PdItem {
    uint32_t kt0, kt1;    // key tiles; kt0 == kt1: no more items
    int32_t lim0, vis;    // keys that the first and the last token see
    uint32_t row0, ntok;  // first row of q, tokens
    uint32_t head;
    uint32_t c0, parts;   // the CTAs that the item lies in
    uint32_t pad;
};
constexpr int kPdItems = 4;

template <int D, int NT>
__global__ void __launch_bounds__(kPdThreads, 1)
paged_decode_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const PagedArgs a, const uint32_t tpt) {
    using L = PdLayout<D, NT>;
    constexpr int kSlabs = D / 128, R = L::kRows, kTile = L::kTile, U = L::kSub;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *ring = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    float *xch = reinterpret_cast<float *>(ring + L::kRing);                  // [8 warps][8 rows][kRow]
    float2 *scl = reinterpret_cast<float2 *>(ring + L::kRing + L::kExchange); // [stage][page]
    uint64_t *full = reinterpret_cast<uint64_t *>(scl + L::kStages * L::kPages), *empty = full + L::kFull;
    uint64_t *item_full = empty + L::kStages, *item_empty = item_full + kPdItems;
    uint64_t *scratch = item_empty + kPdItems; // 40 words
    PagedShare *share = reinterpret_cast<PagedShare *>(scratch + 40);
    PdItem *items = reinterpret_cast<PdItem *>(share + 1);
    float *wm = reinterpret_cast<float *>(items + kPdItems); // [8][R] maxima, then sums, then weights; [R] joint maximum and sum
    float *wl = wm + 8 * 16, *ww = wl + 8 * 16, *rm = ww + 8 * 16, *rl = rm + 16, *wv = rl + 16;
    volatile uint32_t *abort_flag = reinterpret_cast<volatile uint32_t *>(wv + 8);
    volatile uint32_t *never_set = abort_flag + 1;
    volatile uint32_t *arrived = abort_flag + 2;

    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (tid == 0) {
        for (int s = 0; s < L::kFull; s++) mbar_init(&full[s], 34);
        for (int s = 0; s < L::kStages; s++) mbar_init(&empty[s], 4);
        for (int s = 0; s < kPdItems; s++) mbar_init(&item_full[s], 1), mbar_init(&item_empty[s], 8);
        *abort_flag = 0, *never_set = 0;
        mbar_fence_init();
    }
    if (tid == kPdThreads - 1) prefetch_map(&map_k), prefetch_map(&map_v);
    pdl_wait();
    paged_share<kTile>(a, tpt, kPdThreads, scratch, share);
    if (share->x0 >= share->x1) return;
    auto give_up = [&](uint32_t bit) {
        atomicOr(a.words, bit);
        *abort_flag = 1;
    };
    const uint32_t bt = min(a.block_tokens, uint32_t(kTile)); // keys of one copy
    const uint32_t G = a.group;

    // registers: 256 x 232 + 128 x 40 = the 384 x 168 of the launch
    if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
        if (warp == 11) return;
        // ------------------------------------------------------------ producers: warp 8 the items and the keys, 9 the values, 10 the scales
        // (One warp for all three took 2200 clocks for a tile of 8 pages, which the memory delivers in 1400.)
        PagedWalk<kTile> walk(a, *share, tpt);
        PagedItem it;
        uint32_t g = 0, ni = 0;
        bool ok = true;
        const uint32_t per_tile = kTile / bt;
        PagedPages pages;
        while (ok && walk.next(it)) {
            const uint32_t keys = walk.tiles.keys(it.q, it.rtile);
            pages.begin(a, it.seq, keys, bt, it.kt0 * per_tile);
            if (warp == 8 && !mbar_wait(&item_empty[ni % kPdItems], (ni / kPdItems & 1) ^ 1, abort_flag)) { give_up(kStatusEmptyTimeout); break; }
            PdItem *item = &items[ni % kPdItems];
            if (warp == 8 && lane == 0) {
                *item = PdItem{it.kt0, it.kt1, it.lim0, paged_visible(it), it.q.row0 + it.tok0, it.ntok, it.head, 0, 1, 0};
                mbar_arrive(&item_full[ni % kPdItems]);
            }
            __syncwarp();
            ni++;
            for (uint32_t tk = 0; warp == 9 && tk < it.ntok; tk++) { // the query rows on their way to L2
                const uint32_t el = a.q_dtype == SAETTA_F32 ? 4 : 2;
                const char *row = static_cast<const char *>(a.q) + (size_t(it.q.row0 + it.tok0 + tk) * a.q_stride + size_t(it.head) * G * D) * el;
                for (uint32_t at = lane * 128; at < G * D * el; at += 32 * 128) prefetch_l2(row + at);
            }
            for (uint32_t kt = it.kt0; kt < it.kt1; kt++, g++) {
                const uint32_t st = g % L::kStages, ph = (g / L::kStages) & 1, key0 = kt * kTile;
                uint64_t *landed = &full[g % L::kFull];
                const int32_t block = pages.of(kt * per_tile); // of this lane's copy
                const bool want = lane < per_tile && key0 + lane * bt < keys, good = want && uint32_t(block) < a.blocks;
                if (warp == 8 && kt + 1 == it.kt1 && it.kt1 - it.kt0 < it.tiles) { // where the parts are (read after the last tile)
                    const uint2 span = paged_ctas_of(*share, it);
                    if (lane == 0) item->c0 = span.x, item->parts = span.y;
                }
                if (!mbar_wait(&empty[st], ph ^ 1, abort_flag)) { give_up(kStatusEmptyTimeout); ok = false; break; }
                if (warp == 10) {
                    if (want && !good) atomicOr(a.words, kStatusBadBlock);
                    if (want) // a bad block's keys are marked by its scales
                        cp_async8(&scl[st * L::kPages + lane], good ? a.scales + (size_t(block) * a.kv_heads + it.head) * 2
                                                                    : reinterpret_cast<const float *>(a.words + kPagedBadScale));
                    cp_async_arrive(landed);
                    continue;
                }
                const uint32_t copies = __popc(__ballot_sync(0xffffffffu, good));
                if (lane == 0) mbar_expect_tx(landed, copies * bt * D);
                __syncwarp();
                if (good)
                    tma_load_3d(ring + st * L::kStage + (warp == 9 ? L::kSide : 0) + lane * bt * D, warp == 9 ? &map_v : &map_k, landed, 0,
                                int((uint32_t(block) * a.kv_heads + it.head) * a.block_tokens + ((key0 + lane * bt) & (a.block_tokens - 1))), 0);
            }
        }
        if (warp == 8 && ok && mbar_wait(&item_empty[ni % kPdItems], (ni / kPdItems & 1) ^ 1, abort_flag) && lane == 0) {
            items[ni % kPdItems].kt0 = items[ni % kPdItems].kt1 = 0;
            mbar_arrive(&item_full[ni % kPdItems]);
        }
        // let what was issued land before the shared memory goes
        const uint32_t from = g > L::kStages ? g - L::kStages : 0;
        for (uint32_t k = from; k < g; k++) mbar_wait(&full[k % L::kFull], (k / L::kFull) & 1, never_set, 200000u);
        return;
    }

    asm volatile("setmaxnreg.inc.sync.aligned.u32 232;");
    // ------------------------------------------------------------ consumers
    const uint32_t gi = lane >> 2, t = lane & 3, sub = warp & 3, team = warp >> 2;
    uint32_t g = 0;
    bool ok = true;
    for (uint32_t ni = 0;; ni++) {
        // (the consumers agree whether there is another item: they meet at barriers that have no bound)
        if (!consumers_all(mbar_wait(&item_full[ni % kPdItems], ni / kPdItems & 1, abort_flag))) {
            give_up(kStatusFullTimeout);
            break;
        }
        const PdItem it = items[ni % kPdItems];
        if (it.kt0 == it.kt1) break;
        // the item's query rows as B fragments, binary16 after a power of two that brings the row's largest to [128, 256)
        uint32_t qf[NT][D / 16][2];
        float rs[NT][2]; // of rows 2 t and 2 t + 1: that power undone, times the softmax scale in log2 units
        int32_t lim[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            const uint32_t idx = nt * 8 + gi, tok = idx / G, hd = it.head * G + idx % G;
            const bool live = tok < it.ntok && idx < tpt * G;
            float x[kSlabs * 4][8];
            float top = 0.f;
#pragma unroll
            for (int c = 0; c < kSlabs * 4; c++) {
                // chunk 2 t + j of a slab, its two halves
                const uint32_t d = (c >> 2) * 128 + (2 * t + ((c >> 1) & 1)) * 16 + (c & 1) * 8;
                if (live) paged_load_q8(a, size_t(it.row0 + tok) * a.q_stride + size_t(hd) * D + d, x[c]);
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    if (!live) x[c][e] = 0.f;
                    top = fmaxf(top, fabsf(x[c][e]));
                }
            }
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            const int e = min(max(int(__float_as_uint(top) >> 23), 8), 254) - 134; // 2^(e + 7) <= top < 2^(e + 8)
            const float up = __uint_as_float(uint32_t(127 - e) << 23);
#pragma unroll
            for (int c = 0; c < kSlabs * 4; c++) {
                // a quarter chunk (4 dims) for each product: dims 0, 1 its columns 2 t, dims 2, 3 its columns 2 t + 8
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const int ks = (c >> 2) * 8 + ((c >> 1) & 1) * 4 + (c & 1) * 2 + h;
                    qf[nt][ks][0] = pack_half2(x[c][4 * h] * up, x[c][4 * h + 1] * up);
                    qf[nt][ks][1] = pack_half2(x[c][4 * h + 2] * up, x[c][4 * h + 3] * up);
                }
            }
            // (an infinity in a row makes its scores NaN, whatever the keys' signs: all of them -infinity would look like a row without keys)
            const float undo = top < INFINITY ? __uint_as_float(uint32_t(127 + e) << 23) * a.scale_log2 : __uint_as_float(0x7fc00000u);
#pragma unroll
            for (int j = 0; j < 2; j++) {
                rs[nt][j] = __shfl_sync(0xffffffffu, undo, (2 * t + j) * 4);
                lim[nt][j] = it.lim0 + int32_t((nt * 8 + 2 * t + j) / G);
            }
        }
        float o[NT][kSlabs * 8][4];
        float m[NT][2], l[NT][2], vref = 0.f;
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            m[nt][0] = m[nt][1] = -INFINITY, l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
            for (int i = 0; i < kSlabs * 8; i++)
#pragma unroll
                for (int e = 0; e < 4; e++) o[nt][i][e] = 0.f;
        }
        const int32_t vis = it.vis;
        for (uint32_t kt = it.kt0; kt < it.kt1; kt++, g++) {
            if ((g & 1) != team) continue;
            const uint32_t st = g % L::kStages;
            if (ok && !mbar_wait(&full[g % L::kFull], (g / L::kFull) & 1, abort_flag)) { give_up(kStatusFullTimeout); ok = false; }
            if (!ok) continue;
            const int32_t key0 = int32_t(kt * kTile + sub * 16 * U);
            if (key0 < vis) {
                uint32_t kbase[U], in[U];
                float2 sc[U];
                bool use[U];
#pragma unroll
                for (int u = 0; u < U; u++) {
                    const uint32_t at = (sub * U + u) * 16, page = at / bt;
                    in[u] = at % bt;
                    kbase[u] = smem_u32(ring) + st * L::kStage + page * bt * D;
                    sc[u] = scl[st * L::kPages + page];
                    use[u] = key0 + u * 16 < vis && sc[u].x >= 0.f; // not behind the last key, not of a bad block
                    if (!use[u]) sc[u] = make_float2(1.f, 0.f);
                }
                // four chains of products: one after the other they would wait for one another
                constexpr int kChains = kSlabs * 2;
                float acc[U][kChains][NT][4];
#pragma unroll
                for (int u = 0; u < U; u++)
#pragma unroll
                    for (int c = 0; c < kChains; c++)
#pragma unroll
                        for (int nt = 0; nt < NT; nt++) acc[u][c][nt][0] = acc[u][c][nt][1] = acc[u][c][nt][2] = acc[u][c][nt][3] = 0.f;
#pragma unroll
                for (int u = 0; u < U; u++)
#pragma unroll
                    for (int c = 0; c < kChains; c++) {
                        const uint32_t row = in[u] + gi, at = kbase[u] + (c >> 1) * bt * 128 + row * 128 + (((2 * t + (c & 1)) ^ (row & 7)) << 4);
                        const uint4 lo = lds128(at), hi = lds128(at + 8 * 128); // key gi, key gi + 8 (the same swizzle)
                        const uint32_t wl4[4] = {lo.x, lo.y, lo.z, lo.w}, wh4[4] = {hi.x, hi.y, hi.z, hi.w};
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            const uint32_t a0 = e4m3x2_to_h2(wl4[e]), a1 = e4m3x2_to_h2(wh4[e]);
                            const uint32_t a2 = e4m3x2_to_h2(wl4[e] >> 16), a3 = e4m3x2_to_h2(wh4[e] >> 16);
#pragma unroll
                            for (int nt = 0; nt < NT; nt++) mma_f16(acc[u][c][nt], a0, a1, a2, a3, qf[nt][c * 4 + e][0], qf[nt][c * 4 + e][1]);
                        }
                    }
                const bool edge = key0 + 16 * U > it.lim0;
                float vnew = vref;
                bool all_used = true;
#pragma unroll
                for (int u = 0; u < U; u++) vnew = fmaxf(vnew, sc[u].y), all_used &= use[u];
                vnew = fmaxf(vnew, FLT_MIN);
                float s[U][NT][4];
                uint32_t pb[U][NT][2];
                bool need = vnew != vref;
                float f[NT][2], d[U];
#pragma unroll
                for (int u = 0; u < U; u++) d[u] = fmaxf(lg2_approx(sc[u].y / vnew), -60.f);
                // A larger value scale: O keeps its place by the maximum's falling as much, so far as the sum l, which has no r in it, can follow.
                const float up = need && vref > 0.f ? lg2_approx(vnew / vref) : 0.f;
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
#pragma unroll
                    for (int j = 0; j < 2; j++) {
                        float mx = -INFINITY;
                        f[nt][j] = 1.f;
                        if (up > 0.f) {
                            const float by = fminf(up, float(max(0, 227 - max(127, int(__float_as_uint(l[nt][j]) >> 23))))); // l stays below 2^101
                            m[nt][j] -= by, l[nt][j] *= ex2_approx(by), f[nt][j] = ex2_approx(by - up);
                        }
#pragma unroll
                        for (int u = 0; u < U; u++) {
                            const float c = sc[u].x * rs[nt][j];
#pragma unroll
                            for (int k = 0; k < 2; k++) { // key gi, key gi + 8
                                float x = acc[u][0][nt][2 * k + j] + acc[u][1][nt][2 * k + j];
                                if (kChains == 4) x += acc[u][kChains - 2][nt][2 * k + j] + acc[u][kChains - 1][nt][2 * k + j];
                                x = fmaf(x, c, d[u]); // of what the key puts into O: the value scale is in it
                                if ((edge && key0 + u * 16 + int32_t(gi) + 8 * k >= lim[nt][j]) || !use[u]) x = -INFINITY;
                                s[u][nt][2 * k + j] = x;
                                mx = fmaxf(mx, x);
                            }
                        }
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
                        if (mx > m[nt][j] + kPdRescale) {
                            const float g1 = ex2_approx(m[nt][j] - mx); // 0 for the first
                            m[nt][j] = mx;
                            l[nt][j] *= g1, f[nt][j] *= g1;
                            need = true;
                        }
                    }
                }
                if (__any_sync(0xffffffffu, need)) {
#pragma unroll
                    for (int nt = 0; nt < NT; nt++)
#pragma unroll
                        for (int i = 0; i < kSlabs * 8; i++) {
                            o[nt][i][0] *= f[nt][0], o[nt][i][1] *= f[nt][1];
                            o[nt][i][2] *= f[nt][0], o[nt][i][3] *= f[nt][1];
                        }
                    vref = vnew;
                }
#pragma unroll
                for (int u = 0; u < U; u++) {
                    const float ir = ex2_approx(-d[u]);
#pragma unroll
                    for (int nt = 0; nt < NT; nt++) {
                        float p[4];
#pragma unroll
                        for (int j = 0; j < 2; j++) {
                            const float mu = m[nt][j] == -INFINITY ? 0.f : m[nt][j] - kPdShift;
                            p[j] = ex2_approx(s[u][nt][j] - mu), p[2 + j] = ex2_approx(s[u][nt][2 + j] - mu);
                            l[nt][j] = fmaf(p[j] + p[2 + j], ir, l[nt][j]);
                        }
                        pb[u][nt][0] = movmatrix_trans(pack_half2(p[0], p[1]));
                        pb[u][nt][1] = movmatrix_trans(pack_half2(p[2], p[3]));
                    }
                }
                if (edge && it.lim0 < vis) {
                    // The tokens see different keys of this piece, and a weight of 0 does not silence NaN: its dims become NaN in the rows that see the key, and 0
                    // in shared memory (which this warp alone reads) for the products of all.
#pragma unroll 1
                    for (int32_t j = max(it.lim0, key0); j < min(vis, key0 + 16 * U); j++) {
                        const uint32_t at = sub * U * 16 + uint32_t(j - key0), page = at / bt, row = at % bt;
                        if (scl[st * L::kPages + page].x < 0.f) continue; // of a bad block
#pragma unroll
                        for (int sl = 0; sl < kSlabs; sl++) {
                            const uint32_t addr = smem_u32(ring) + st * L::kStage + L::kSide + page * bt * D + sl * bt * 128 + row * 128 + ((gi ^ (row & 7)) << 4);
                            const uint4 v = lds128(addr);
                            uint32_t w[4] = {v.x, v.y, v.z, v.w}, nan[4];
#pragma unroll
                            for (int e = 0; e < 4; e++) nan[e] = (((w[e] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) >> 7; // the codes 0x7f and 0xff
                            if (!__any_sync(0xffffffffu, nan[0] | nan[1] | nan[2] | nan[3])) continue;
#pragma unroll
                            for (int e = 0; e < 4; e++) {
#pragma unroll
                                for (int b = 0; b < 4; b++)
#pragma unroll
                                    for (int nt = 0; nt < NT; nt++)
#pragma unroll
                                        for (int c = 0; c < 2; c++) // dim 16 gi + 4 e + b of row 2 t + c
                                            if ((nan[e] >> 8 * b & 1) && j < lim[nt][c]) o[nt][sl * 8 + 2 * e + (b >> 1)][2 * (b & 1) + c] = __uint_as_float(0x7fc00000u);
                                w[e] &= ~(nan[e] * 255u);
                            }
                            if (t == 0) asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]) : "memory");
                            fence_async_smem(); // (the next tile is copied here)
                            __syncwarp();
                        }
                    }
                }
                const bool tail = key0 + 16 * U > vis || !all_used; // what lies behind the last key is any byte, NaN too: no product may read it
#pragma unroll
                for (int u = 0; u < U; u++)
#pragma unroll
                    for (int sl = 0; sl < kSlabs; sl++) {
                        uint4 v[4];
#pragma unroll
                        for (int k = 0; k < 4; k++) {
                            const uint32_t key = 2 * t + (k & 1) + (k >> 1) * 8, row = in[u] + key;
                            v[k] = lds128(kbase[u] + L::kSide + sl * bt * 128 + row * 128 + ((gi ^ (row & 7)) << 4));
                            if (tail && (key0 + u * 16 + int32_t(key) >= vis || !use[u])) v[k] = make_uint4(0, 0, 0, 0);
                        }
                        const uint32_t w[4][4] = {{v[0].x, v[0].y, v[0].z, v[0].w}, {v[1].x, v[1].y, v[1].z, v[1].w},
                                                  {v[2].x, v[2].y, v[2].z, v[2].w}, {v[3].x, v[3].y, v[3].z, v[3].w}};
#pragma unroll
                        for (int e = 0; e < 4; e++)
#pragma unroll
                            for (int h = 0; h < 2; h++) {
                                const uint32_t x = prmt(w[0][e], w[1][e], h ? 0x7362 : 0x5140), y = prmt(w[2][e], w[3][e], h ? 0x7362 : 0x5140);
                                const uint32_t a0 = e4m3x2_to_h2(x), a1 = e4m3x2_to_h2(x >> 16), a2 = e4m3x2_to_h2(y), a3 = e4m3x2_to_h2(y >> 16);
#pragma unroll
                                for (int nt = 0; nt < NT; nt++) mma_f16(o[nt][sl * 8 + e * 2 + h], a0, a1, a2, a3, pb[u][nt][0], pb[u][nt][1]);
                            }
                    }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&empty[st]);
        }

        // ---- the eight warps' results become one: weights first, then 128 dims of 8 rows at a time
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int j = 0; j < 2; j++) {
                float x = l[nt][j];
                x += __shfl_xor_sync(0xffffffffu, x, 4), x += __shfl_xor_sync(0xffffffffu, x, 8), x += __shfl_xor_sync(0xffffffffu, x, 16);
                if (gi == 0) wm[warp * R + nt * 8 + 2 * t + j] = m[nt][j], wl[warp * R + nt * 8 + 2 * t + j] = x;
            }
        if (lane == 0) wv[warp] = vref;
        consumers_sync();
        if (tid < 8 * R) {
            const uint32_t w = tid / R, row = tid % R;
            float top = -INFINITY, sum = 0.f;
#pragma unroll
            for (int k = 0; k < 8; k++) top = fmaxf(top, wm[k * R + row]);
            const float mu = (top == -INFINITY ? 0.f : top) + kPdShift; // the parts' values are without it
#pragma unroll
            for (int k = 0; k < 8; k++) sum += wl[k * R + row] * ex2_approx(wm[k * R + row] - mu);
            ww[w * R + row] = ex2_approx(wm[w * R + row] - mu) * wv[w];
            if (w == 0) rm[row] = top, rl[row] = sum;
        }
        const uint32_t c0 = items[ni % kPdItems].c0, parts = items[ni % kPdItems].parts;
        const bool whole = parts == 1;
        float *part = a.parts + (size_t(blockIdx.x) * 2 + (it.kt0 == 0 ? 1 : 0)) * a.part_floats;
        auto finish = [&](uint32_t row, uint32_t d, float4 v, float sum) { // one row's dims d .. d + 3, unnormalised
            const uint32_t tok = row / G, hd = it.head * G + row % G;
            if (tok >= it.ntok || row >= tpt * G) return;
            const size_t at = size_t(it.row0 + tok) * a.heads + hd;
            const float inv = sum > 0.f ? 1.f / sum : (sum == 0.f ? 0.f : sum); // no key: 0; NaN stays
            v.x *= inv, v.y *= inv, v.z *= inv, v.w *= inv;
            if (a.q_and_gate) {
                const float4 gt = *reinterpret_cast<const float4 *>(a.q_and_gate + at * 2 * D + D + d);
                v.x *= sigmoid(gt.x), v.y *= sigmoid(gt.y), v.z *= sigmoid(gt.z), v.w *= sigmoid(gt.w);
            }
            paged_store4(a, at * D + d, v.x, v.y, v.z, v.w);
        };
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int sl = 0; sl < kSlabs; sl++) {
                if (nt || sl) consumers_sync(); // the exchange buffer has been read
#pragma unroll
                for (int j = 0; j < 2; j++)
#pragma unroll
                    for (int c = 0; c < 4; c++) {
                        // dims gi * 16 + 4 q .. + 3 of row 2 t + j; starting at q = gi keeps the lanes on different banks
                        const uint32_t q4 = (c + gi) & 3;
                        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                        for (int k = 0; k < 4; k++)
                            if (q4 == uint32_t(k)) v = make_float4(o[nt][sl * 8 + 2 * k][j], o[nt][sl * 8 + 2 * k][2 + j], o[nt][sl * 8 + 2 * k + 1][j], o[nt][sl * 8 + 2 * k + 1][2 + j]);
                        *reinterpret_cast<float4 *>(xch + (warp * 8 + 2 * t + j) * L::kRow + gi * 16 + q4 * 4) = v;
                    }
                consumers_sync();
                const uint32_t row = nt * 8 + warp, d = lane * 4;
                float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                for (int w = 0; w < 8; w++) {
                    const float4 x = *reinterpret_cast<const float4 *>(xch + (w * 8 + warp) * L::kRow + d);
                    const float wt = ww[w * R + row];
                    // a warp that saw no key has weight 0 and accumulators 0
                    v.x = fmaf(x.x, wt, v.x), v.y = fmaf(x.y, wt, v.y), v.z = fmaf(x.z, wt, v.z), v.w = fmaf(x.w, wt, v.w);
                }
                if (whole) finish(row, sl * 128 + d, v, rl[row]);
                else *reinterpret_cast<float4 *>(part + row * D + sl * 128 + d) = v;
            }
        if (!whole) {
            float *ml = part + R * D;
            if (tid < R) ml[tid * 2] = rm[tid], ml[tid * 2 + 1] = rl[tid];
            // The parts are joined by the last CTA to arrive, in the order of the CTAs; many of them in two rounds, groups of some first, because one CTA
            // reads no more than some 100 bytes a clock.
            uint32_t per = parts; // parts of a group
            if (parts > kPdGroup) {
                per = 2;
                while (per * per < parts) per++;
            }
            const uint32_t groups = (parts + per - 1) / per, mine = (blockIdx.x - c0) / per;
            auto part_of = [&](uint32_t p) { return a.parts + (size_t(c0 + p) * 2 + (p == 0 ? 1 : 0)) * a.part_floats; };
            // parts lo, lo + step, ... (n of them) are joined: into part lo, or the output
            uint32_t lo = mine * per, step = 1, n = min(per, parts - lo);
            // a group's counter: by its first CTA, which may begin another item's tail as well
            uint32_t *counter = a.words + kPagedCounters + (mine ? gridDim.x : 0) + c0 + lo;
#pragma unroll 1
            for (bool last = groups == 1;; last = true) {
                consumers_sync();
                if (tid == 0) {
                    __threadfence(); // (the others' writes too: they came before the barrier)
                    const uint32_t k = atomicAdd(counter, 1) + 1;
                    if (k == n) *counter = 0;
                    __threadfence();
                    *arrived = k;
                }
                consumers_sync();
                if (*arrived != n) break;
                float4 x[kPdGroup + 1];
                float2 *in = reinterpret_cast<float2 *>(xch); // [n][R] maxima and sums; the maxima become weights
                for (uint32_t i = tid; i < n * R; i += 256) in[i] = __ldcg(reinterpret_cast<const float2 *>(part_of(lo + i / R * step) + R * D) + i % R);
                float top = -INFINITY, sum = 0.f;
#pragma unroll 1
                for (uint32_t i = tid; i < R * D / 4; i += 256) {
                    const uint32_t row = i * 4 / D, d = i * 4 % D;
#pragma unroll
                    for (uint32_t p = 0; p <= kPdGroup; p++)
                        if (p < n) x[p] = __ldcg(reinterpret_cast<const float4 *>(part_of(lo + p * step)) + i);
                    if (i == tid) { // the weights, while the first values are on their way
                        consumers_sync();
                        if (tid < R) {
#pragma unroll 4
                            for (uint32_t p = 0; p < n; p++) top = fmaxf(top, in[p * R + tid].x);
                            const float mu = top == -INFINITY ? 0.f : top;
#pragma unroll 4
                            for (uint32_t p = 0; p < n; p++) {
                                const float2 y = in[p * R + tid];
                                const float w = ex2_approx(y.x - mu);
                                in[p * R + tid].x = w;
                                sum = fmaf(y.y, w, sum);
                            }
                            rl[tid] = sum;
                        }
                        consumers_sync();
                    }
                    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                    for (uint32_t p = 0; p <= kPdGroup; p++)
                        if (p < n) {
                            const float wt = in[p * R + row].x;
                            v.x = fmaf(x[p].x, wt, v.x), v.y = fmaf(x[p].y, wt, v.y), v.z = fmaf(x[p].z, wt, v.z), v.w = fmaf(x[p].w, wt, v.w);
                        }
                    if (last) finish(row, d, v, rl[row]);
                    else reinterpret_cast<float4 *>(part_of(lo))[i] = v;
                }
                if (last) break;
                if (tid < R) *reinterpret_cast<float2 *>(part_of(lo) + R * D + tid * 2) = make_float2(top, sum);
                lo = 0, step = per, n = groups, counter = a.words + kPagedCounters + 2 * gridDim.x + c0;
            }
        }
        consumers_sync(); // statistics and exchange buffer are free for the next item
        if (lane == 0) mbar_arrive(&item_empty[ni % kPdItems]);
    }
}

template <int D, int NT>
static int decode_configure() {
    SAETTA_CUDA(cudaFuncSetAttribute(paged_decode_kernel<D, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, PdLayout<D, NT>::kSmem));
    return SAETTA_OK;
}

int paged_decode_configure(int) {
    int rc = decode_configure<128, 1>();
    if (!rc) rc = decode_configure<128, 2>();
    if (!rc) rc = decode_configure<256, 1>();
    if (!rc) rc = decode_configure<256, 2>();
    return rc;
}

int launch_paged_decode(const PagedArgs &a, const saetta_paged_cache *cache, uint32_t rows, int ctas, cudaStream_t stream) {
    CUtensorMap mk, mv;
    const uint32_t box = std::min<uint32_t>(a.block_tokens, cache->head_dim == 256 ? PdLayout<256, 1>::kTile : PdLayout<128, 1>::kTile), slabs = uint32_t(cache->head_dim / 128);
    if (int rc = paged_map(&mk, cache->keys, cache, box, slabs)) return rc;
    if (int rc = paged_map(&mv, cache->values, cache, box, slabs)) return rc;
    const bool two = rows > 8; // a product's columns hold 8 rows; two products for each piece of keys rather than two passes over the keys
    const uint32_t tpt = (two ? 16 : 8) / a.group; // tokens whose heads fill the product's columns
    void (*kernel)(CUtensorMap, CUtensorMap, PagedArgs, uint32_t) = nullptr;
    size_t smem = 0;
    if (cache->head_dim == 256) {
        kernel = two ? paged_decode_kernel<256, 2> : paged_decode_kernel<256, 1>;
        smem = two ? PdLayout<256, 2>::kSmem : PdLayout<256, 1>::kSmem;
    } else {
        kernel = two ? paged_decode_kernel<128, 2> : paged_decode_kernel<128, 1>;
        smem = two ? PdLayout<128, 2>::kSmem : PdLayout<128, 1>::kSmem;
    }
    SAETTA_CUDA(launch_pdl(kernel, dim3(unsigned(ctas)), dim3(kPdThreads), smem, stream, mk, mv, a, tpt));
    return SAETTA_OK;
}

} // namespace saetta
