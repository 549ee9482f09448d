// Rotary positions over several axes, and the append of rotated keys to a paged cache.
#pragma once

#include "common.cuh"

namespace abx {

constexpr int kRotaryAxes = 4;
constexpr int kPairs = kHeadDim / 2;

// One tensor of a launch: rows (batch, head, token) of 128 elements, read at
// `src` and written at `dst` with strides in elements.
struct RotaryJob {
    const void* src;
    void* dst;
    int64_t s_batch, s_head, s_token;
    int64_t d_batch, d_head, d_token;  // paged: d_batch steps pages, d_token steps tokens of a page
    int32_t heads;
    int32_t turn;   // 0: copied
    int32_t paged;  // dst is found through the page table
};

struct RotaryArgs {
    RotaryJob job[3];
    double freq[kPairs];  // of each pair of dims: angle / pi for one step of its axis
    uint8_t axis[kPairs];
    const int32_t* positions;  // [batch or 1, tokens, axes]
    int64_t p_batch;           // 0: one set of positions for the batch
    int32_t axes, jobs, heads;  // heads: of all jobs
    int32_t batch, tokens;
    int32_t slices;  // the heads of a token are shared out to this many thread groups
    int32_t halves;  // 1: pairs (i, i + 64), 0: pairs (2i, 2i + 1)
    float sign;      // -1: the turn back
    // paged jobs
    const int32_t *starts, *lengths, *table;
    int32_t seqs, table_width, page_size, pages;
    int* error;
};

// dtype: 0 bf16, 1 fp16, 2 f32
cudaError_t launch_rotary(const RotaryArgs& args, int dtype, cudaStream_t stream);

}  // namespace abx
