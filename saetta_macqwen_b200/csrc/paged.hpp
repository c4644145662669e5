// Host objects and launchers of the paged 8-bit cache (paged.cu, paged_attend.cu).  No counterpart in the
// reference, whose caches are one contiguous buffer per sequence (src/gpu_layers.rs:179-293).
#pragma once

#include "host.hpp"

struct saetta_paged_cache {
    int device = 0;
    size_t kv_heads = 0, head_dim = 0, block_tokens = 0, blocks = 0;
    uint8_t *keys = nullptr, *values = nullptr; // e4m3 [blocks][kv_heads][block_tokens][head_dim]
    float *scales = nullptr;                    // [blocks][kv_heads][2]: of the keys, of the values
    bool owns = false;
    size_t side_bytes() const { return blocks * kv_heads * block_tokens * head_dim; }
};

struct saetta_paged_attention {
    int device = 0;
    size_t heads = 0, kv_heads = 0, head_dim = 0;
    int ctas = 0;              // of a launch: one for each SM
    float *parts = nullptr;    // [ctas][2] partials: O rows, then (m, l) of each row
    size_t part_floats = 0;    // floats of one partial
    uint32_t *words = nullptr; // [0] status, [1] pad, [2..3] the scale pair that marks a bad block, [kPagedCounters ..) arrival counters
};

namespace saetta {

constexpr uint32_t kStatusBadBlock = 16u; // a block table entry outside the cache was met
constexpr uint32_t kStatusCut = 32u;      // a length behind its row of the block table, or rows behind the call's, were cut off
constexpr int kPagedBadScale = 2;         // word index of the (-1, -1) pair
constexpr int kPagedCounters = 8;
constexpr int kPagedMaxGroup = 16;        // query heads of one kv head
constexpr size_t kPagedMaxSeqs = 8192;
// CTAs of an attention launch, at most.  Parts of an item are joined in two rounds of groups of ceil(sqrt(parts)): 13 is what the few-rows
// kernel has registers for.  (paged_cut's 32-bit steps hold up to 255.)
constexpr int kPagedMaxCtas = 13 * 13;
// Rows (tokens x heads of a kv head) of a sequence up to which the few-rows kernel runs: what two products' columns hold.  Measured, few-rows against
// many-rows kernel: 24 sequences of 4700 keys, heads of 256, 8 rows 39 us and 63, 16 rows 71 and 67; heads of 128, 8 rows 63 and 110, 16 rows 75 and
// 117; one sequence of 700 keys, 16 rows 21 and 35; 24 sequences of some 3000 keys, 32 rows 138 (in two passes over the keys) and 96.
constexpr size_t kPagedFewRows = 16;

// What an attention launch reads and writes.
struct PagedArgs {
    const void *q;
    const float *q_and_gate; // may be null
    void *out;
    const uint32_t *row_starts, *kv_lens;
    const int32_t *tables;
    const float *scales;
    float *parts;
    uint32_t *words;
    const uint8_t *values;
    size_t part_floats;
    uint32_t q_stride; // values between the rows of q
    uint32_t rows, seqs, table_stride, blocks;
    uint32_t heads, kv_heads, group, block_tokens;
    int q_dtype, out_dtype;
    float scale_log2;
};

int launch_paged_decode(const PagedArgs &a, const saetta_paged_cache *cache, uint32_t rows, int ctas, cudaStream_t stream); // rows of a sequence x its heads per kv head, at most
int paged_decode_configure(int device);
int launch_paged_prefill(const PagedArgs &a, const saetta_paged_cache *cache, int ctas, cudaStream_t stream);
int paged_prefill_configure(int device);

} // namespace saetta
