// The paged 8-bit cache: its objects, block assignment on the device, and the quantising append.
//
// The cache holds e4m3 values in blocks of 16 to 128 tokens, [block][kv head][token][dim], and one scale for each
// (block, kv head, side).  A scale is a power of two: e4m3 is a floating-point format, so within its range the scale
// costs no precision whatever its value, x / s only places the range, and raising a block's scale when a larger row is
// appended re-scales the codes it holds without rounding them again, except those that fall among e4m3's subnormals.
// No counterpart in the reference (its quantised rows carry a scale and a bias for 64 channels of one token,
// src/kv_quant.rs:54-105, in one buffer per sequence).
#include <cooperative_groups.h>

#include <algorithm>
#include <cmath>
#include <new>

#include "paged.hpp"

namespace saetta {

// ----------------------------------------------------------------- block assignment

constexpr int kAssignThreads = 1024;

struct AssignArgs {
    const uint32_t *kv_lens, *new_tokens, *finished; // finished may be null
    int32_t *free_blocks;
    const uint32_t *free_count;
    int32_t *tables;
    uint32_t *row_starts;
    int32_t *slots, *positions; // positions may be null
    uint32_t *kv_lens_out, *free_count_out, *status;
    uint32_t seqs, table_stride, block_shift, free_cap, rows_cap;
};

// Sums that saturate stay above every capacity (which are below 2^31): no count of tokens wraps round to a valid one.
__device__ __forceinline__ uint32_t add_sat(uint32_t a, uint32_t b) { return a + b < a ? 0xffffffffu : a + b; }

// The largest s with a[s] <= x; a ascends, a[0] <= x.
__device__ __forceinline__ uint32_t last_at_or_below(const uint32_t *a, uint32_t n, uint32_t x) {
    uint32_t lo = 0, hi = n;
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) >> 1;
        if (a[mid] <= x) lo = mid;
        else hi = mid;
    }
    return lo;
}

// One scheduling step.  Every CTA of the (single) cluster scans the lengths of all sequences by itself -- three sums:
// blocks given back, blocks taken, rows -- into shared memory, and then the cluster's threads deal out table entries and
// rows, each finding its sequence by a binary search over the sums.  Nothing is written before every CTA has read its
// inputs (cluster barrier), so lengths and count may be updated in place.  Bound by latency: the chain is lengths ->
// scan -> free stack -> tables and slots.  1024 prompts of 133,000 rows in all 14.2 us a call, one behind the other (a cluster of 8 CTAs above 4096
// rows: the rows' writes then weigh more than the cluster's start); 1 sequence and 509 of one token each 10.2, which is the host's call (from
// cold caches 5.0 and 13.0).
__global__ void __launch_bounds__(kAssignThreads) paged_assign_kernel(const AssignArgs a) {
    namespace cg = cooperative_groups;
    cg::cluster_group cluster = cg::this_cluster();
    extern __shared__ uint32_t assign_smem[];
    uint32_t *row0 = assign_smem, *take0 = row0 + a.seqs + 1, *back0 = take0 + a.seqs + 1, *len0 = back0 + a.seqs + 1;
    __shared__ uint32_t warp_sum[3][32];
    __shared__ uint32_t bad_word;
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const uint32_t gtid = blockIdx.x * kAssignThreads + tid, gthreads = gridDim.x * kAssignThreads;
    const uint32_t B = 1u << a.block_shift;
    const uint64_t width_tokens = uint64_t(a.table_stride) << a.block_shift;
    if (tid == 0) bad_word = 0;
    pdl_wait();
    const uint32_t count = *a.free_count;
    __syncthreads();

    uint32_t carry[3] = {0, 0, 0}; // rows, taken, given back before this chunk
    uint32_t bad = 0;
    for (uint32_t base = 0; base < a.seqs; base += kAssignThreads) {
        const uint32_t s = base + tid;
        uint32_t v[3] = {0, 0, 0};
        uint32_t len = 0;
        if (s < a.seqs) {
            const uint32_t was = a.kv_lens[s], n = a.new_tokens[s];
            const bool done = a.finished && a.finished[s];
            if (was > width_tokens || n > width_tokens || (done ? 0 : was) + uint64_t(n) > width_tokens) {
                bad |= SAETTA_PAGED_TABLE_FULL;
            } else {
                len = done ? 0 : was;
                v[0] = n;
                v[1] = ((len + n + B - 1) >> a.block_shift) - ((len + B - 1) >> a.block_shift);
                v[2] = done ? (was + B - 1) >> a.block_shift : 0;
            }
        }
        uint32_t x[3];
#pragma unroll
        for (int k = 0; k < 3; k++) {
            x[k] = v[k];
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const uint32_t y = __shfl_up_sync(0xffffffffu, x[k], d);
                if (lane >= uint32_t(d)) x[k] = add_sat(x[k], y);
            }
            if (lane == 31) warp_sum[k][warp] = x[k];
        }
        __syncthreads();
        if (warp < 3) {
            uint32_t w = warp_sum[warp][lane];
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const uint32_t y = __shfl_up_sync(0xffffffffu, w, d);
                if (lane >= uint32_t(d)) w = add_sat(w, y);
            }
            warp_sum[warp][lane] = w;
        }
        __syncthreads();
        uint32_t *dst[3] = {row0, take0, back0};
#pragma unroll
        for (int k = 0; k < 3; k++) {
            const uint32_t before = add_sat(add_sat(carry[k], warp ? warp_sum[k][warp - 1] : 0), x[k]) - v[k];
            if (s < a.seqs) dst[k][s] = before;
            carry[k] = add_sat(carry[k], warp_sum[k][31]);
        }
        if (s < a.seqs) len0[s] = len;
        __syncthreads();
    }
    if (carry[0] > a.rows_cap) bad |= SAETTA_PAGED_ROWS_FULL;
    if (count > a.free_cap || uint64_t(count) + carry[2] > a.free_cap || carry[1] > uint64_t(count) + carry[2]) bad |= SAETTA_PAGED_NO_BLOCKS;
    if (bad) atomicOr(&bad_word, bad);
    if (tid == 0) row0[a.seqs] = carry[0], take0[a.seqs] = carry[1], back0[a.seqs] = carry[2];
    if (gridDim.x > 1) cluster.sync(); // every input has been read
    else __syncthreads();
    bad = bad_word;

    if (bad) { // nothing is assigned
        for (uint32_t r = gtid; r < a.rows_cap; r += gthreads) {
            a.slots[r] = -1;
            if (a.positions) a.positions[r] = -1;
        }
        for (uint32_t s = gtid; s <= a.seqs; s += gthreads) a.row_starts[s] = 0;
        if (a.kv_lens_out != a.kv_lens)
            for (uint32_t s = gtid; s < a.seqs; s += gthreads) a.kv_lens_out[s] = a.kv_lens[s];
        if (gtid == 0) *a.free_count_out = count, *a.status = bad;
        return;
    }

    const uint32_t back = carry[2], take = carry[1], rows = carry[0], top = count + back;
    if (back) {
        for (uint32_t e = gtid; e < back; e += gthreads) {
            const uint32_t s = last_at_or_below(back0, a.seqs, e);
            a.free_blocks[count + e] = a.tables[size_t(s) * a.table_stride + (e - back0[s])];
        }
        if (gridDim.x > 1) cluster.sync(); // the stack is whole, the tables of finished sequences have been read
        else __syncthreads();
    }
    for (uint32_t e = gtid; e < take; e += gthreads) {
        const uint32_t s = last_at_or_below(take0, a.seqs, e);
        const uint32_t have = (len0[s] + B - 1) >> a.block_shift;
        a.tables[size_t(s) * a.table_stride + have + (e - take0[s])] = a.free_blocks[top - 1 - e];
    }
    // Four rows a thread, one search for them, where the rows are more than the threads (133,000 rows: 14.5 us; one row a thread: 21).
    const uint32_t per = a.rows_cap > gthreads ? 4 : 1;
    const bool quads = per == 4 && (reinterpret_cast<uintptr_t>(a.slots) | reinterpret_cast<uintptr_t>(a.positions)) % 16 == 0;
    for (uint32_t r0 = gtid * per; r0 < a.rows_cap; r0 += gthreads * per) {
        int32_t slot[4], pos[4];
        uint32_t s = r0 < rows ? last_at_or_below(row0, a.seqs, r0) : 0, end = r0 < rows ? row0[s + 1] : 0;
#pragma unroll
        for (uint32_t j = 0; j < 4; j++) {
            const uint32_t r = r0 + j;
            slot[j] = pos[j] = -1;
            if (r >= rows || j >= per) continue;
            while (r >= end) end = row0[++s + 1];
            pos[j] = int32_t(len0[s] + (r - row0[s]));
            const uint32_t have = (len0[s] + B - 1) >> a.block_shift, idx = uint32_t(pos[j]) >> a.block_shift;
            // the block is one the sequence had, or one of those taken above (read from the stack: no wait for the table)
            const int32_t block = idx < have ? a.tables[size_t(s) * a.table_stride + idx] : a.free_blocks[top - 1 - (take0[s] + idx - have)];
            slot[j] = int32_t((uint32_t(block) << a.block_shift) + (uint32_t(pos[j]) & (B - 1)));
        }
        if (quads && r0 + 4 <= a.rows_cap) {
            *reinterpret_cast<int4 *>(a.slots + r0) = make_int4(slot[0], slot[1], slot[2], slot[3]);
            if (a.positions) *reinterpret_cast<int4 *>(a.positions + r0) = make_int4(pos[0], pos[1], pos[2], pos[3]);
        } else {
            for (uint32_t j = 0; j < per && r0 + j < a.rows_cap; j++) {
                a.slots[r0 + j] = slot[j];
                if (a.positions) a.positions[r0 + j] = pos[j];
            }
        }
    }
    for (uint32_t s = gtid; s <= a.seqs; s += gthreads) {
        a.row_starts[s] = row0[s];
        if (s < a.seqs) a.kv_lens_out[s] = len0[s] + (row0[s + 1] - row0[s]);
    }
    if (gtid == 0) *a.free_count_out = top - take, *a.status = 0;
}

// ----------------------------------------------------------------- append

struct StoreArgs {
    const void *k, *v;
    const int32_t *slots;
    uint8_t *keys, *values;
    float *scales;
    uint32_t *status; // may be null
    size_t k_stride, v_stride;
    uint32_t rows, kv_heads, block_shift, total_slots;
};

// 8 consecutive values as f32.
template <int DT>
__device__ __forceinline__ void load8(const void *base, size_t i, float (&x)[8]) {
    if constexpr (DT == SAETTA_F32) {
        const float4 *p = reinterpret_cast<const float4 *>(static_cast<const float *>(base) + i);
        const float4 a = p[0], b = p[1];
        x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
    } else {
        const uint4 w = *reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(base) + i);
        const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int j = 0; j < 4; j++) {
            if constexpr (DT == SAETTA_BF16) {
                x[2 * j] = __uint_as_float(u[j] << 16), x[2 * j + 1] = __uint_as_float(u[j] & 0xffff0000u);
            } else {
                const float2 f = h2f2(u[j]);
                x[2 * j] = f.x, x[2 * j + 1] = f.y;
            }
        }
    }
}

// Two values to e4m3, round to nearest even, saturating at +-448 (NaN stays NaN).
__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
    uint16_t d;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(d) : "f"(hi), "f"(lo));
    return d;
}
__device__ __forceinline__ float2 e4m3x2_to_f2(uint32_t w) {
    uint32_t h;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(uint16_t(w)));
    return h2f2(h);
}

// The smallest power of two, 2^-126 at least, by which amax lies within e4m3: 448 = 1.75 * 2^8.
__device__ __forceinline__ float pow2_scale(float amax) {
    const uint32_t u = __float_as_uint(amax);
    const int e = int(u >> 23) - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
    return __uint_as_float(uint32_t(max(e, 1)) << 23);
}

// A CTA for each (16 rows of the call, kv head, side): it takes the runs (rows of one block, one behind the other) that begin there, long ones with all
// of its warps, short ones with a warp each; a row leads a run where the row before it lies in another block.  Bound by memory: rows
// in, codes out, each once (the second pass over a run, which needs its largest value, hits the caches).  17413 bfloat16 rows of 2 x 256
// in blocks of 64: 21.0 us, 2.55 TB/s (a run's two passes and their meeting are what is left); a warp for each run took 45: too few loads on
// their way.  One row, and 253 rows of as many sequences: 7.9 us, the host's call (from cold caches 4.0 and 7.5 to 8.1).
template <int DT, int D>
__global__ void __launch_bounds__(256) paged_store_kernel(const StoreArgs a) {
    constexpr uint32_t kLanes = D / 8;      // lanes of one row
    constexpr uint32_t kRows = 32 / kLanes; // rows a warp takes at once
    __shared__ float red[8];
    const uint32_t per_row = a.kv_heads * 2, rest = blockIdx.x % per_row, head = rest >> 1, side = rest & 1;
    const uint32_t row0 = blockIdx.x / per_row * 16, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t B = 1u << a.block_shift;
    pdl_wait();
    uint32_t leads, follows; // of the 16 rows
    int32_t slot = -1;
    {
        const uint32_t row = row0 + lane;
        const bool in = lane < 16 && row < a.rows;
        slot = in ? a.slots[row] : -1;
        const int32_t prev = in && row ? a.slots[row - 1] : -1;
        const bool real = slot >= 0 && uint32_t(slot) < a.total_slots;
        const bool same = real && prev >= 0 && uint32_t(prev) >> a.block_shift == uint32_t(slot) >> a.block_shift;
        leads = __ballot_sync(0xffffffffu, real && !same);
        follows = __ballot_sync(0xffffffffu, same && prev + 1 == slot);
        // a slot outside the cache, or one that does not follow its predecessor in the same block
        const bool bad = slot >= 0 && (!real || (same && prev + 1 != slot));
        if (rest == 0 && warp == 0 && bad && a.status) atomicOr(a.status, uint32_t(SAETTA_PAGED_BAD_SLOT));
    }
    const void *x = side ? a.v : a.k;
    const size_t stride = side ? a.v_stride : a.k_stride;
    const uint32_t sub = lane / kLanes, col = (lane % kLanes) * 8;
    uint32_t turn = 0; // whose short run is next
    for (; leads; leads &= leads - 1) {
        const uint32_t k = uint32_t(__ffs(int(leads)) - 1), row = row0 + k;
        const uint32_t first = uint32_t(__shfl_sync(0xffffffffu, slot, k)), block = first >> a.block_shift, off = first & (B - 1);
        uint32_t n = 1 + uint32_t(__ffs(int(~(follows >> (k + 1)))) - 1); // rows of the run, within these 16
        while (k + n >= 16) { // and behind them
            const uint32_t r = row + n + lane;
            const uint32_t ballot = __ballot_sync(0xffffffffu, r < a.rows && off + n + lane < B && a.slots[r] == int32_t(first + n + lane));
            const uint32_t more = ballot == 0xffffffffu ? 32 : uint32_t(__ffs(int(~ballot)) - 1);
            n += more;
            if (more < 32) break;
        }
        const bool wide = n > 2 * kRows; // all warps take part
        if (!wide && turn++ % 8 != warp) continue;
        const uint32_t i0 = (wide ? warp * kRows : 0) + sub, di = wide ? 8 * kRows : kRows;
        const size_t x0 = size_t(row) * stride + size_t(head) * D + col;
        float amax = 0.f;
#pragma unroll 4
        for (uint32_t i = i0; i < n; i += di) {
            float f[8];
            load8<DT>(x, x0 + size_t(i) * stride, f);
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const float m = fabsf(f[j]);
                amax = m < INFINITY ? fmaxf(amax, m) : amax; // an infinity saturates, a NaN stays one: neither places the range
            }
        }
#pragma unroll
        for (int d = 16; d; d >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, d));
        float *sp = a.scales + (size_t(block) * a.kv_heads + head) * 2 + side;
        const float was = off ? *sp : 0.f;
        if (wide) {
            if (lane == 0) red[warp] = amax;
            __syncthreads(); // (and `was` has been read)
#pragma unroll
            for (int w = 0; w < 8; w++) amax = fmaxf(amax, red[w]);
        } else {
            __syncwarp(); // `was` has been read by every lane
        }
        uint8_t *page = (side ? a.values : a.keys) + (size_t(block) * a.kv_heads + head) * B * D;
        const float fresh = pow2_scale(amax), scale = off ? fmaxf(fresh, was) : fresh;
        if (off && scale != was) { // a block that goes on: its scale never falls, and what it holds follows it
            const float f = was / scale;
            for (uint32_t i = wide ? threadIdx.x : lane; i < off * D / 8; i += wide ? 256 : 32) {
                uint2 *p = reinterpret_cast<uint2 *>(page) + i;
                uint2 w = *p;
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    uint32_t &u = h ? w.y : w.x;
                    const float2 lo = e4m3x2_to_f2(u & 0xffff), hi = e4m3x2_to_f2(u >> 16);
                    u = e4m3x2(lo.x * f, lo.y * f) | e4m3x2(hi.x * f, hi.y * f) << 16;
                }
                *p = w;
            }
        }
        if (lane == 0 && (!wide || warp == 0)) *sp = scale;
        const float inv = 1.f / scale;
#pragma unroll 4
        for (uint32_t i = i0; i < n; i += di) {
            float f[8];
            load8<DT>(x, x0 + size_t(i) * stride, f);
            uint2 w;
            w.x = e4m3x2(f[0] * inv, f[1] * inv) | e4m3x2(f[2] * inv, f[3] * inv) << 16;
            w.y = e4m3x2(f[4] * inv, f[5] * inv) | e4m3x2(f[6] * inv, f[7] * inv) << 16;
            *reinterpret_cast<uint2 *>(page + size_t(off + i) * D + col) = w;
        }
        if (wide) __syncthreads(); // `red` may be written again
    }
}

static bool aligned(const void *p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

static int block_shift(size_t block_tokens) {
    for (int s = 4; s <= 7; s++)
        if (block_tokens == size_t(1) << s) return s;
    return -1;
}

static int paged_cache_check(size_t kv_heads, size_t head_dim, size_t block_tokens, size_t blocks) {
    if (head_dim != 128 && head_dim != 256) return fail(SAETTA_ERR_BAD_SHAPE, "PagedKvCache: head dim must be 128 or 256");
    if (!kv_heads || kv_heads > 1024) return fail(SAETTA_ERR_BAD_SHAPE, "PagedKvCache: 1 to 1024 kv heads");
    if (block_shift(block_tokens) < 0) return fail(SAETTA_ERR_BAD_SHAPE, "PagedKvCache: blocks hold 16, 32, 64 or 128 tokens");
    // slots are 32-bit, and the tensor copies' row coordinate (block, kv head, token) is too
    if (!blocks || blocks > size_t(0x7fffffff) / (kv_heads * block_tokens))
        return fail(SAETTA_ERR_BAD_SHAPE, "PagedKvCache: blocks * kv_heads * block_tokens must lie in 1 .. 2^31 - 1");
    return SAETTA_OK;
}

static int attend_check(const saetta_paged_attention *op, const saetta_paged_cache *c, const saetta_paged_batch &b, const void *q,
                        int q_dtype, size_t q_stride, const float *gate, const void *out, int out_dtype, float scale) {
    if (!op || !c) return fail(SAETTA_ERR_BAD_ARG, "paged attention: null handle");
    if (c->device != op->device) return fail(SAETTA_ERR_BAD_ARG, "paged attention: the cache lives on another device than the op");
    if (c->kv_heads != op->kv_heads || c->head_dim != op->head_dim)
        return fail(SAETTA_ERR_BAD_SHAPE, "paged attention: the cache's kv heads or head dim differ from the op's");
    for (int dt : {q_dtype, out_dtype})
        if (dt != SAETTA_F32 && dt != SAETTA_F16 && dt != SAETTA_BF16) return fail(SAETTA_ERR_BAD_ARG, "paged attention: unknown dtype");
    if (b.seqs > kPagedMaxSeqs) return fail(SAETTA_ERR_BAD_SHAPE, "paged attention: at most 8192 sequences");
    if (b.rows > 0x7fffffff / (op->heads * 2 * op->head_dim)) return fail(SAETTA_ERR_BAD_SHAPE, "paged attention: too many rows for one call");
    if (b.rows && (!q || !out)) return fail(SAETTA_ERR_BAD_ARG, "paged attention: null pointer");
    if (b.seqs && (!b.row_starts_dev || !b.kv_lens_dev || !b.block_tables_dev)) return fail(SAETTA_ERR_BAD_ARG, "paged attention: null pointer");
    if (b.seqs && !b.table_stride) return fail(SAETTA_ERR_BAD_SHAPE, "paged attention: block tables without columns");
    if (b.table_stride > size_t(0x7fffffff) / c->block_tokens) return fail(SAETTA_ERR_BAD_SHAPE, "paged attention: block tables too wide");
    if (q_stride < op->heads * op->head_dim || q_stride > 0xffffffffu) return fail(SAETTA_ERR_BAD_SHAPE, "paged attention: q_stride is below a row's values");
    const size_t el = q_dtype == SAETTA_F32 ? 4 : 2;
    if (!aligned(q, 16) || q_stride * el % 16) return fail(SAETTA_ERR_BAD_ARG, "paged attention: rows of q must be 16-byte aligned");
    if (!aligned(out, 16)) return fail(SAETTA_ERR_BAD_ARG, "paged attention: out must be 16-byte aligned");
    if (!aligned(gate, 16)) return fail(SAETTA_ERR_BAD_ARG, "paged attention: q_and_gate must be 16-byte aligned");
    if (!(scale > 0.f) || !(scale < INFINITY)) return fail(SAETTA_ERR_BAD_ARG, "paged attention: scale must be positive and finite");
    return SAETTA_OK;
}

} // namespace saetta

using namespace saetta;

extern "C" {

int saetta_paged_cache_wrap(int device, size_t kv_heads, size_t head_dim, size_t block_tokens, size_t blocks, void *keys_dev,
                            void *values_dev, float *scales_dev, saetta_paged_cache **out) {
    if (!out || !keys_dev || !values_dev || !scales_dev) return fail(SAETTA_ERR_BAD_ARG, "PagedKvCache wrap: null pointer");
    if (int rc = paged_cache_check(kv_heads, head_dim, block_tokens, blocks)) return rc;
    if (!aligned(keys_dev, 16) || !aligned(values_dev, 16) || !aligned(scales_dev, 16))
        return fail(SAETTA_ERR_BAD_ARG, "PagedKvCache wrap: buffers must be 16-byte aligned");
    auto *c = new (std::nothrow) saetta_paged_cache();
    if (!c) return fail(SAETTA_ERR_NO_MEM, "PagedKvCache wrap: host allocation");
    c->device = device, c->kv_heads = kv_heads, c->head_dim = head_dim, c->block_tokens = block_tokens, c->blocks = blocks;
    c->keys = static_cast<uint8_t *>(keys_dev), c->values = static_cast<uint8_t *>(values_dev), c->scales = scales_dev;
    *out = c;
    return SAETTA_OK;
}

int saetta_paged_cache_create(int device, size_t kv_heads, size_t head_dim, size_t block_tokens, size_t blocks, saetta_paged_cache **out) {
    if (!out) return fail(SAETTA_ERR_BAD_ARG, "PagedKvCache: out is null");
    if (int rc = paged_cache_check(kv_heads, head_dim, block_tokens, blocks)) return rc;
    DeviceGuard guard(device);
    if (!guard.ok) return fail(SAETTA_ERR_CUDA, "PagedKvCache: cannot select the device");
    auto *c = new (std::nothrow) saetta_paged_cache();
    if (!c) return fail(SAETTA_ERR_NO_MEM, "PagedKvCache: host allocation");
    c->device = device, c->kv_heads = kv_heads, c->head_dim = head_dim, c->block_tokens = block_tokens, c->blocks = blocks, c->owns = true;
    void *p[3] = {};
    const size_t bytes[3] = {c->side_bytes(), c->side_bytes(), blocks * kv_heads * 2 * sizeof(float)};
    cudaError_t e = cudaSuccess;
    for (int i = 0; i < 3 && e == cudaSuccess; i++) {
        e = cudaMalloc(&p[i], bytes[i]);
        if (e == cudaSuccess) e = cudaMemset(p[i], 0, bytes[i]);
    }
    if (e == cudaSuccess) e = cudaStreamSynchronize(nullptr); // zero before a call on any stream
    c->keys = static_cast<uint8_t *>(p[0]), c->values = static_cast<uint8_t *>(p[1]), c->scales = static_cast<float *>(p[2]);
    if (e != cudaSuccess) {
        const int rc = cuda_fail(e, "PagedKvCache: device allocation");
        cudaGetLastError();
        saetta_paged_cache_destroy(c);
        return rc;
    }
    *out = c;
    return SAETTA_OK;
}

void saetta_paged_cache_destroy(saetta_paged_cache *c) {
    if (!c) return;
    if (c->owns) {
        DeviceGuard guard(c->device);
        cudaFree(c->keys), cudaFree(c->values), cudaFree(c->scales);
    }
    delete c;
}

int saetta_paged_cache_buffers(const saetta_paged_cache *c, void **keys_dev, void **values_dev, float **scales_dev) {
    if (!c) return fail(SAETTA_ERR_BAD_ARG, "PagedKvCache: null handle");
    if (keys_dev) *keys_dev = c->keys;
    if (values_dev) *values_dev = c->values;
    if (scales_dev) *scales_dev = c->scales;
    return SAETTA_OK;
}

int saetta_paged_assign(int device, size_t seqs, size_t block_tokens, const uint32_t *kv_lens_dev, const uint32_t *new_tokens_dev,
                        const uint32_t *finished_dev, int32_t *free_blocks_dev, size_t free_cap, const uint32_t *free_count_dev,
                        int32_t *block_tables_dev, size_t table_stride, uint32_t *row_starts_dev, int32_t *slots_dev,
                        int32_t *positions_dev, size_t rows_cap, uint32_t *kv_lens_out_dev, uint32_t *free_count_out_dev,
                        uint32_t *status_dev, void *stream) {
    if (!free_count_dev || !row_starts_dev || !free_count_out_dev || !status_dev) return fail(SAETTA_ERR_BAD_ARG, "paged assign: null pointer");
    if (seqs && (!kv_lens_dev || !new_tokens_dev || !block_tables_dev || !kv_lens_out_dev)) return fail(SAETTA_ERR_BAD_ARG, "paged assign: null pointer");
    if ((rows_cap && !slots_dev) || (free_cap && !free_blocks_dev)) return fail(SAETTA_ERR_BAD_ARG, "paged assign: null pointer");
    const int shift = block_shift(block_tokens);
    if (shift < 0) return fail(SAETTA_ERR_BAD_SHAPE, "paged assign: blocks hold 16, 32, 64 or 128 tokens");
    if (seqs > kPagedMaxSeqs) return fail(SAETTA_ERR_BAD_SHAPE, "paged assign: at most 8192 sequences");
    if (seqs && !table_stride) return fail(SAETTA_ERR_BAD_SHAPE, "paged assign: block tables without columns");
    if (table_stride > size_t(0x7fffffff) / block_tokens) return fail(SAETTA_ERR_BAD_SHAPE, "paged assign: block tables too wide");
    if (free_cap > size_t(0x7fffffff) / block_tokens) return fail(SAETTA_ERR_BAD_SHAPE, "paged assign: slots are 32-bit: free_cap * block_tokens must stay below 2^31");
    if (rows_cap > 0x7fffffff) return fail(SAETTA_ERR_BAD_SHAPE, "paged assign: rows_cap must stay below 2^31");
    DeviceGuard guard(device);
    if (!guard.ok) return fail(SAETTA_ERR_CUDA, "paged assign: cannot select the device");
    const AssignArgs a{kv_lens_dev, new_tokens_dev, finished_dev, free_blocks_dev, free_count_dev, block_tables_dev, row_starts_dev,
                       slots_dev, positions_dev, kv_lens_out_dev, free_count_out_dev, status_dev, uint32_t(seqs), uint32_t(table_stride),
                       uint32_t(shift), uint32_t(free_cap), uint32_t(rows_cap)};
    const size_t smem = 4 * (seqs + 1) * sizeof(uint32_t);
    // 48 KB hold what a launch has without asking, the kernel's static shared memory (some 400 bytes) included
    if (smem > 47 * 1024) SAETTA_CUDA(cudaFuncSetAttribute(paged_assign_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(4 * (kPagedMaxSeqs + 1) * 4)));
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[2];
    const unsigned ctas = rows_cap > 4096 ? 8 : 1;
    cfg.gridDim = dim3(ctas), cfg.blockDim = dim3(kAssignThreads), cfg.dynamicSmemBytes = smem, cfg.stream = cudaStream_t(stream);
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = ctas, attr[0].val.clusterDim.y = 1, attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr, cfg.numAttrs = 2;
    SAETTA_CUDA(cudaLaunchKernelEx(&cfg, paged_assign_kernel, a));
    return SAETTA_OK;
}

int saetta_paged_store(saetta_paged_cache *c, const void *k_dev, const void *v_dev, int dtype, size_t rows, size_t k_stride,
                       size_t v_stride, const int32_t *slots_dev, uint32_t *status_dev, void *stream) {
    if (!c) return fail(SAETTA_ERR_BAD_ARG, "paged store: null handle");
    if (dtype != SAETTA_F32 && dtype != SAETTA_F16 && dtype != SAETTA_BF16) return fail(SAETTA_ERR_BAD_ARG, "paged store: unknown dtype");
    if (rows && (!k_dev || !v_dev || !slots_dev)) return fail(SAETTA_ERR_BAD_ARG, "paged store: null pointer");
    const size_t el = dtype == SAETTA_F32 ? 4 : 2, values = c->kv_heads * c->head_dim;
    if (k_stride < values || v_stride < values) return fail(SAETTA_ERR_BAD_SHAPE, "paged store: a stride is below a row's values");
    if (!aligned(k_dev, 16) || !aligned(v_dev, 16) || k_stride * el % 16 || v_stride * el % 16)
        return fail(SAETTA_ERR_BAD_ARG, "paged store: rows of k and v must be 16-byte aligned");
    if (rows > 0x7fffffff / (c->kv_heads * 2)) return fail(SAETTA_ERR_BAD_SHAPE, "paged store: too many rows for one call");
    if (!rows) return SAETTA_OK;
    DeviceGuard guard(c->device);
    if (!guard.ok) return fail(SAETTA_ERR_CUDA, "paged store: cannot select the device");
    const StoreArgs a{k_dev, v_dev, slots_dev, c->keys, c->values, c->scales, status_dev, k_stride, v_stride, uint32_t(rows),
                      uint32_t(c->kv_heads), uint32_t(block_shift(c->block_tokens)), uint32_t(c->blocks * c->block_tokens)};
    const size_t ctas = (rows + 15) / 16 * c->kv_heads * 2;
    void (*kernel)(StoreArgs) = nullptr;
    if (c->head_dim == 256) kernel = dtype == SAETTA_F32 ? paged_store_kernel<SAETTA_F32, 256> : dtype == SAETTA_F16 ? paged_store_kernel<SAETTA_F16, 256> : paged_store_kernel<SAETTA_BF16, 256>;
    else kernel = dtype == SAETTA_F32 ? paged_store_kernel<SAETTA_F32, 128> : dtype == SAETTA_F16 ? paged_store_kernel<SAETTA_F16, 128> : paged_store_kernel<SAETTA_BF16, 128>;
    SAETTA_CUDA(launch_pdl(kernel, dim3(unsigned(ctas)), dim3(256), 0, cudaStream_t(stream), a));
    return SAETTA_OK;
}

int saetta_paged_attention_create(int device, size_t heads, size_t kv_heads, size_t head_dim, saetta_paged_attention **out) {
    if (!out) return fail(SAETTA_ERR_BAD_ARG, "PagedAttention: out is null");
    if (head_dim != 128 && head_dim != 256) return fail(SAETTA_ERR_BAD_SHAPE, "PagedAttention: head dim must be 128 or 256");
    if (!kv_heads || kv_heads > 1024 || !heads || heads % kv_heads || heads / kv_heads > size_t(kPagedMaxGroup))
        return fail(SAETTA_ERR_BAD_SHAPE, "PagedAttention: heads must be 1 to 16 times the kv heads");
    DeviceGuard guard(device);
    if (!guard.ok) return fail(SAETTA_ERR_CUDA, "PagedAttention: cannot select the device");
    if (int rc = paged_decode_configure(device)) return rc;
    if (int rc = paged_prefill_configure(device)) return rc;
    auto *op = new (std::nothrow) saetta_paged_attention();
    if (!op) return fail(SAETTA_ERR_NO_MEM, "PagedAttention: host allocation");
    op->device = device, op->heads = heads, op->kv_heads = kv_heads, op->head_dim = head_dim;
    op->ctas = std::min(sm_count(device), kPagedMaxCtas);
    op->part_floats = 128 * (head_dim + 2) + 4; // 128 rows: the largest tile; (m, l) of each; the value scale O is kept by
    void *p = nullptr, *w = nullptr;
    const size_t words = size_t(kPagedCounters) + 3 * size_t(op->ctas);
    cudaError_t e = cudaMalloc(&p, size_t(op->ctas) * 2 * op->part_floats * sizeof(float));
    op->parts = static_cast<float *>(p);
    if (e == cudaSuccess) e = cudaMalloc(&w, words * sizeof(uint32_t));
    op->words = static_cast<uint32_t *>(w);
    if (e == cudaSuccess) e = cudaMemset(w, 0, words * sizeof(uint32_t));
    const float bad[2] = {-1.f, -1.f};
    if (e == cudaSuccess) e = cudaMemcpy(op->words + kPagedBadScale, bad, sizeof bad, cudaMemcpyHostToDevice);
    if (e == cudaSuccess) e = cudaStreamSynchronize(nullptr); // the words are set before a call on any stream
    if (e != cudaSuccess) {
        const int rc = cuda_fail(e, "PagedAttention: device allocation");
        cudaGetLastError();
        saetta_paged_attention_destroy(op);
        return rc;
    }
    *out = op;
    return SAETTA_OK;
}

void saetta_paged_attention_destroy(saetta_paged_attention *op) {
    if (!op) return;
    DeviceGuard guard(op->device);
    cudaFree(op->parts), cudaFree(op->words);
    delete op;
}

int saetta_paged_attention_status(saetta_paged_attention *op, void *stream, uint32_t *status) {
    if (!op || !status) return fail(SAETTA_ERR_BAD_ARG, "paged attention: null pointer");
    DeviceGuard guard(op->device);
    SAETTA_CUDA(cudaMemcpyAsync(status, op->words, sizeof *status, cudaMemcpyDeviceToHost, cudaStream_t(stream)));
    SAETTA_CUDA(cudaStreamSynchronize(cudaStream_t(stream)));
    return SAETTA_OK;
}

int saetta_paged_attend(saetta_paged_attention *op, const saetta_paged_cache *cache, saetta_paged_batch batch, const void *q_dev,
                        int q_dtype, size_t q_stride, const float *q_and_gate_dev, void *out_dev, int out_dtype, float scale,
                        void *stream) {
    if (int rc = attend_check(op, cache, batch, q_dev, q_dtype, q_stride, q_and_gate_dev, out_dev, out_dtype, scale)) return rc;
    if (!batch.rows || !batch.seqs) return SAETTA_OK;
    DeviceGuard guard(op->device);
    if (!guard.ok) return fail(SAETTA_ERR_CUDA, "paged attention: cannot select the device");
    PagedArgs a{};
    a.q = q_dev, a.q_and_gate = q_and_gate_dev, a.out = out_dev;
    a.row_starts = batch.row_starts_dev, a.kv_lens = batch.kv_lens_dev, a.tables = batch.block_tables_dev;
    a.scales = cache->scales, a.parts = op->parts, a.words = op->words, a.values = cache->values, a.part_floats = op->part_floats;
    a.q_stride = uint32_t(q_stride), a.rows = uint32_t(batch.rows), a.seqs = uint32_t(batch.seqs);
    a.table_stride = uint32_t(batch.table_stride), a.blocks = uint32_t(cache->blocks);
    a.heads = uint32_t(op->heads), a.kv_heads = uint32_t(op->kv_heads), a.group = uint32_t(op->heads / op->kv_heads);
    a.block_tokens = uint32_t(cache->block_tokens);
    a.q_dtype = q_dtype, a.out_dtype = out_dtype;
    a.scale_log2 = scale * 1.4426950408889634f;
    // which kernel: see kPagedFewRows
    const size_t rows = std::max<size_t>(1, std::min(batch.max_rows, batch.rows)) * a.group;
    if (rows <= kPagedFewRows) return launch_paged_decode(a, cache, uint32_t(rows), op->ctas, cudaStream_t(stream));
    return launch_paged_prefill(a, cache, op->ctas, cudaStream_t(stream));
}

} // extern "C"
