// How an attention launch over the paged cache divides its work: the tiles of all (sequence, kv head, row tile) items,
// one after the other, are cut into equal shares, a share for each CTA, on the device from the lengths there (so a
// captured launch serves every length).  An item that a cut crosses leaves partials; the last CTA of it to arrive joins them.
#pragma once

#include "paged.hpp"
#include "umma.cuh"

namespace saetta {

// sum over i < n of floor((a i + b) / T), T a power of two, a > 0: the numerators' sum less that of their remainders, by T.  With g the largest power
// of two that divides a (T at most), the remainders of T / g numerators in a row are, in some order, b mod g and every step of g above it up
// to T: whole periods cost nothing, and fewer than T / g terms are left to be added one by one.
template <uint32_t T>
__host__ __device__ __forceinline__ uint64_t tile_sum(uint32_t n, uint32_t a, uint64_t b) {
    static_assert((T & (T - 1)) == 0 && T > 1, "a power of two");
    const uint32_t low = a & (0u - a), g = low < T ? low : T, period = T / g, left = n & (period - 1);
    uint64_t rest = uint64_t(n / period) * (period * (uint32_t(b) & (g - 1)) + T / 2 * (period - 1));
    uint32_t x = uint32_t(b);
#pragma unroll 1
    for (uint32_t i = 0; i < left; i++, x += a) rest += x & (T - 1);
    return (uint64_t(n) * (n - 1) / 2 * a + uint64_t(n) * b - rest) / T;
}

// A sequence as the kernels read it: its rows [row0, row0 + n) of q, its keys [0, kv).
struct PagedSeq {
    uint32_t row0, n, kv;
};

__device__ __forceinline__ PagedSeq paged_seq(const PagedArgs &a, uint32_t s) {
    PagedSeq q;
    const uint32_t lo = min(a.row_starts[s], a.rows), hi = min(a.row_starts[s + 1], a.rows);
    q.row0 = lo, q.n = hi > lo ? hi - lo : 0;
    q.kv = min(a.kv_lens[s], a.table_stride * a.block_tokens);
    return q;
}

// Key tiles (of T keys) of a sequence's row tiles (of `tpt` tokens): tile r needs the keys its last token sees.
template <int T>
struct PagedTiles {
    uint32_t tpt;
    __device__ __forceinline__ uint32_t row_tiles(const PagedSeq &q) const { return (q.n + tpt - 1) / tpt; }
    __device__ __forceinline__ uint32_t keys(const PagedSeq &q, uint32_t r) const {
        // more rows than keys: the first rows see nothing; every tile is given all keys
        return q.kv < q.n ? q.kv : min(q.kv, q.kv - q.n + (r + 1) * tpt);
    }
    // at least one tile, so that rows that see no key are written too
    __device__ __forceinline__ uint32_t count(const PagedSeq &q, uint32_t r) const { return max(1u, (keys(q, r) + T - 1) / T); }
    __device__ __forceinline__ uint64_t before(const PagedSeq &q, uint32_t r) const { // of row tiles 0 .. r - 1
        if (!r) return 0;
        if (q.kv < q.n) return uint64_t(r) * count(q, 0);
        const uint32_t full = r == row_tiles(q) ? r - 1 : r;
        uint64_t sum = full ? tile_sum<T>(full, tpt, q.kv - q.n + tpt + T - 1) : 0;
        if (full != r) sum += count(q, r - 1);
        return sum;
    }
    __device__ __forceinline__ uint64_t per_head(const PagedSeq &q) const { return q.n <= tpt ? count(q, 0) : before(q, row_tiles(q)); }
};

// One CTA's part of one item.
struct PagedItem {
    uint32_t seq, head, rtile;  // which item
    PagedSeq q;
    uint32_t tok0, ntok;        // tokens of the row tile, in the sequence
    int32_t lim0;               // keys the tile's first token sees (<= 0: none)
    uint32_t tiles, kt0, kt1;   // key tiles of the item, and this CTA's [kt0, kt1)
    uint32_t at;                // tile kt0's place in the CTA's share
};

struct PagedShare {
    uint64_t total, x0, x1; // tiles of the launch, this CTA's
    uint64_t head_base;     // flat index of (seq, head 0, row tile 0)
    uint64_t per_head;      // tiles of `seq` for each kv head
    uint32_t ctas;          // that have a share
    uint32_t seq, head, rtile, kt0; // where it begins
    PagedSeq q;             // of `seq`
};

// The CTAs that get a share.
__device__ __forceinline__ uint32_t paged_ctas(uint64_t total) { return uint32_t(min(uint64_t(gridDim.x), max(uint64_t(1), total))); }
// total * c / n for a CTA number c <= n < 256.  No division of 64-bit numbers: that is a call, and this and what follows run in warps that have given
// registers back, where a callee compiled for the launch's number may use some that are gone.  In 32 bits where that holds; else 16 bits
// of the dividend at a time (a remainder and 16 bits stay below 2^24).
__host__ __device__ __forceinline__ uint64_t paged_cut(uint64_t total, uint32_t c, uint32_t n) {
    if (total < (1u << 24)) return uint32_t(total) * c / n;
    const uint64_t x = total * c;
    uint64_t q = 0;
    uint32_t rest = 0;
#pragma unroll 1
    for (int at = 48; at >= 0; at -= 16) {
        const uint32_t y = rest << 16 | (uint32_t(x >> at) & 0xffffu);
        q = q << 16 | y / n, rest = y % n;
    }
    return q;
}

// Walks the items of a share; every role of a CTA walks the same ones.
template <int T>
struct PagedWalk {
    const PagedArgs &a;
    PagedTiles<T> tiles;
    uint32_t at, end; // places in the share
    uint32_t seq, head, rtile, rtiles, kt0;
    PagedSeq q;

    __device__ __forceinline__ PagedWalk(const PagedArgs &args, const PagedShare &s, uint32_t tpt) : a(args), tiles{tpt} {
        at = 0, end = uint32_t(s.x1 - s.x0), seq = s.seq, head = s.head, rtile = s.rtile, kt0 = s.kt0, q = s.q;
        rtiles = tiles.row_tiles(q);
    }
    __device__ __forceinline__ bool next(PagedItem &it) {
        if (at >= end) return false;
        it.seq = seq, it.head = head, it.rtile = rtile, it.q = q;
        it.tok0 = rtile * tiles.tpt, it.ntok = min(tiles.tpt, q.n - it.tok0);
        it.lim0 = int32_t(q.kv) - int32_t(q.n) + int32_t(it.tok0) + 1;
        it.tiles = tiles.count(q, rtile);
        it.kt0 = kt0;
        it.kt1 = kt0 + min(it.tiles - kt0, end - at);
        it.at = at;
        at += it.kt1 - it.kt0;
        kt0 = 0;
        if (++rtile == rtiles) {
            rtile = 0;
            if (++head == a.kv_heads) {
                head = 0;
                if (at < end)
                    do q = paged_seq(a, ++seq);
                    while (!q.n && seq + 1 < a.seqs);
                rtiles = tiles.row_tiles(q);
            }
        }
        return true;
    }
};

// Keys that an item's last token sees.
__device__ __forceinline__ int32_t paged_visible(const PagedItem &it) { return min(int32_t(it.q.kv), it.lim0 + int32_t(it.ntok) - 1); }

// The CTA whose share holds tile x.
__host__ __device__ __forceinline__ uint32_t paged_cta_of(uint64_t total, uint32_t ctas, uint64_t x) {
    if (total < (1u << 24)) { // the quotient is the CTA or the one after it, whose share would begin behind x
        const uint32_t c = uint32_t(x) * ctas / uint32_t(total);
        return c + (c + 1 < ctas && uint32_t(total) * (c + 1) / ctas <= uint32_t(x));
    }
    uint32_t lo = 0, hi = ctas;
#pragma unroll 1
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) / 2;
        if (paged_cut(total, mid, ctas) <= x) lo = mid;
        else hi = mid;
    }
    return lo;
}
// The CTAs that an item's tiles lie in: the first, and how many.
__device__ __forceinline__ uint2 paged_ctas_of(const PagedShare &s, const PagedItem &it) {
    const uint64_t first = s.x0 + it.at - it.kt0;
    const uint32_t c0 = paged_cta_of(s.total, s.ctas, first);
    return make_uint2(c0, paged_cta_of(s.total, s.ctas, first + it.tiles - 1) - c0 + 1);
}

// Finds this CTA's share.  All `threads` threads of the block call it; `scratch` (40 words of 8 bytes) and `share` are shared memory.
template <int T>
__device__ __forceinline__ void paged_share(const PagedArgs &a, uint32_t tpt, uint32_t threads, uint64_t *scratch, PagedShare *share) {
    const PagedTiles<T> tiles{tpt};
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, warps = threads / 32;
    uint64_t total = 0, x0 = 0;
    // The sum of all sequences' tiles first, then which one holds x0; with no more sequences than threads the sums at hand serve both.
    const bool once = a.seqs <= threads;
#pragma unroll 1
    for (int pass = once ? 1 : 0; pass < 2; pass++) {
        uint64_t carry = 0;
#pragma unroll 1
        for (uint32_t base = 0; base < a.seqs; base += threads) {
            const uint32_t s = base + tid;
            uint64_t cost = 0, per = 0;
            PagedSeq q;
            q.row0 = q.n = q.kv = 0;
            if (s < a.seqs) {
                q = paged_seq(a, s);
                if (blockIdx.x == 0 && pass == 1 && (a.row_starts[s + 1] > a.rows || a.row_starts[s] > a.row_starts[s + 1] ||
                                                      (q.n && a.kv_lens[s] > a.table_stride * a.block_tokens)))
                    atomicOr(a.words, kStatusCut); // (the length of a sequence without rows is not read)
                if (q.n) cost = a.kv_heads * (per = tiles.per_head(q));
            }
            uint64_t v = cost;
            if (a.seqs > 1) {
#pragma unroll
                for (int d = 1; d < 32; d <<= 1) {
                    const uint64_t y = __shfl_up_sync(0xffffffffu, v, d);
                    if (lane >= uint32_t(d)) v += y;
                }
            }
            if (a.seqs == 1 ? tid == 0 : lane == 31) scratch[warp] = v;
            __syncthreads();
            uint64_t before = carry, all = 0;
            if (a.seqs == 1) {
                all = scratch[0];
            } else {
#pragma unroll 1
                for (uint32_t w = 0; w < warps; w++) {
                    if (w < warp) before += scratch[w];
                    all += scratch[w];
                }
            }
            v += before; // inclusive
            if (once || pass == 0) total = carry + all;
            if (once) {
                const uint32_t ctas = paged_ctas(total);
                x0 = blockIdx.x < ctas ? paged_cut(total, blockIdx.x, ctas) : total;
            }
            if (pass == 1 && cost && v - cost <= x0 && x0 < v) share->seq = s, share->head_base = v - cost, share->q = q, share->per_head = per;
            carry += all;
            __syncthreads();
        }
        const uint32_t ctas = paged_ctas(total);
        x0 = blockIdx.x < ctas ? paged_cut(total, blockIdx.x, ctas) : total;
        if (tid == 0) {
            share->total = total, share->ctas = ctas, share->x0 = x0;
            share->x1 = blockIdx.x < ctas ? paged_cut(total, blockIdx.x + 1, ctas) : total;
        }
    }
    __syncthreads();
    if (warp == 0 && x0 < total) {
        const PagedSeq q = share->q;
        const uint64_t per = share->per_head, rest_all = x0 - share->head_base;
        const uint32_t head = rest_all >> 32 || per >> 32 ? uint32_t(rest_all / per) : uint32_t(rest_all) / uint32_t(per);
        const uint64_t rest = rest_all - uint64_t(head) * per;
        uint32_t lo = 0, hi = tiles.row_tiles(q); // the last r with before(r) <= rest, 32 candidates at a time
        while (hi - lo > 1) {
            const uint32_t step = (hi - lo + 31) / 32, r = lo + lane * step;
            const uint32_t le = __ballot_sync(0xffffffffu, r < hi && tiles.before(q, r) <= rest);
            lo += (__popc(le) - 1) * step;
            hi = min(hi, lo + step);
        }
        const uint32_t kt0 = uint32_t(rest - (lo ? tiles.before(q, lo) : 0));
        if (lane == 0) share->head = head, share->rtile = lo, share->kt0 = kt0;
    }
    __syncthreads();
}

// The pages of an item's tiles, for the warp that copies them: 32 table entries at a time in a register of each lane, and the 32 after them on
// their way (an entry is some 800 clocks away, and the copies of a tile take 200).
struct PagedPages {
    const int32_t *table;
    uint32_t entries, base, shift; // entries of the table in use; first one in `now`; log2 of the copies to an entry
    int32_t now, next;             // -1: none
    __device__ __forceinline__ int32_t load(uint32_t first) const {
        const uint32_t i = first + (threadIdx.x & 31);
        return i < entries ? table[i] : -1;
    }
    // `copy`: number of the first copy (of bt keys) that will be asked for
    __device__ __forceinline__ void begin(const PagedArgs &a, uint32_t seq, uint32_t keys, uint32_t bt, uint32_t copy) {
        table = a.tables + size_t(seq) * a.table_stride;
        entries = (keys + a.block_tokens - 1) / a.block_tokens;
        shift = a.block_tokens > bt ? __ffs(int(a.block_tokens / bt)) - 1 : 0;
        base = (copy >> shift) & ~31u;
        now = load(base), next = load(base + 32);
    }
    // The block of copy number `copy` + lane: asked for in rising order; a tile's copies lie within one such group of 32.
    __device__ __forceinline__ int32_t of(uint32_t copy) {
        const uint32_t first = copy >> shift;
        if (first >= base + 32) {
            base += 32;
            now = next, next = load(base + 32);
        }
        return __shfl_sync(0xffffffffu, now, ((copy + (threadIdx.x & 31)) >> shift) - base);
    }
};

// Four values of an output row.
__device__ __forceinline__ void paged_store4(const PagedArgs &a, size_t i, float x, float y, float z, float w) {
    if (a.out_dtype == SAETTA_F32) {
        *reinterpret_cast<float4 *>(static_cast<float *>(a.out) + i) = make_float4(x, y, z, w);
    } else if (a.out_dtype == SAETTA_F16) {
        *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(a.out) + i) = make_uint2(pack_half2(x, y), pack_half2(z, w));
    } else {
        const __nv_bfloat162 p = __floats2bfloat162_rn(x, y), r = __floats2bfloat162_rn(z, w);
        *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(a.out) + i) =
            make_uint2(*reinterpret_cast<const uint32_t *>(&p), *reinterpret_cast<const uint32_t *>(&r));
    }
}
__device__ __forceinline__ uint4 lds128(uint32_t addr) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
    return v;
}
__device__ __forceinline__ float lg2_approx(float x) {
    float y;
    asm("lg2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float sigmoid(float g) { return __fdividef(1.f, 1.f + __expf(-g)); }

// 8 consecutive values of q.
__device__ __forceinline__ void paged_load_q8(const PagedArgs &a, size_t i, float (&x)[8]) {
    if (a.q_dtype == SAETTA_F32) {
        const float4 *p = reinterpret_cast<const float4 *>(static_cast<const float *>(a.q) + i);
        const float4 u = p[0], v = p[1];
        x[0] = u.x, x[1] = u.y, x[2] = u.z, x[3] = u.w, x[4] = v.x, x[5] = v.y, x[6] = v.z, x[7] = v.w;
    } else {
        const uint4 w = *reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(a.q) + i);
        const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int j = 0; j < 4; j++) {
            if (a.q_dtype == SAETTA_BF16) {
                x[2 * j] = __uint_as_float(u[j] << 16), x[2 * j + 1] = __uint_as_float(u[j] & 0xffff0000u);
            } else {
                const float2 f = h2f2(u[j]);
                x[2 * j] = f.x, x[2 * j + 1] = f.y;
            }
        }
    }
}

// ----------------------------------------------------------------- host side

// Keys or values as [slab of 128 dims][token rows][128 bytes]: a copy brings `box_slabs` slabs of `box_rows` rows.
inline int paged_map(CUtensorMap *map, const void *base, const saetta_paged_cache *c, uint32_t box_rows, uint32_t box_slabs) {
    EncodeTiledFn enc = encode_fn();
    if (!enc) return fail(SAETTA_ERR_CUDA, "paged attention: cuTensorMapEncodeTiled is not available");
    const cuuint64_t rows = cuuint64_t(c->blocks) * c->kv_heads * c->block_tokens;
    const cuuint64_t dims[3] = {128, rows, cuuint64_t(c->head_dim / 128)};
    const cuuint64_t strides[2] = {cuuint64_t(c->head_dim), 128};
    const cuuint32_t box[3] = {128, box_rows, box_slabs}, el[3] = {1, 1, 1};
    const CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void *>(base), dims, strides, box, el, CU_TENSOR_MAP_INTERLEAVE_NONE,
                           CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(SAETTA_ERR_CUDA, "paged attention: tensor map for the cache rejected");
    return SAETTA_OK;
}

} // namespace saetta
