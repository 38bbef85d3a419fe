// A 4-bit product as its C entries take it, handed to the tensor-core kernel (int4_tc.cu).
#pragma once
#include "common.cuh"

namespace p2p {

constexpr int kInt4TileTokens = 272;    // most tokens of a tile: its accumulator and three A tiles fill tensor memory

struct Int4Call {
    const void* x;
    int dtype;
    int64_t tokens, cols, ldx;          // dense
    const void* layout;
    bool has_zeros;
    int64_t rows;
    int group, gated;
    void* y;
    int64_t ldy;
    const int32_t *items, *n_items;     // routed: x's rows are the places
    int64_t max_items, item_tokens, pairs;
    const int32_t* routed;              // not null: y's rows from *routed to pairs become zero
    int hold = -1;                      // a test's withheld x load (each CTA's load of that number is never issued), or -1
    uint64_t wait_ns = 2000000000ull;   // how long a pipeline wait may take before the launch gives up
};

// Bytes of workspace int4_tc_run needs for a dense call.
size_t int4_tc_workspace(int64_t tokens, int64_t rows, int64_t cols, int gated);
// x: 16-byte aligned rows (ldx and the start).
int int4_tc_run(const Int4Call& call, void* workspace, cudaStream_t st, const char* what);

// The site of that kernel's first wait that gave up (0: none); reset != 0 clears it. Syncs the stream.
int int4_tc_error(int* site, int reset, cudaStream_t st);

}  // namespace p2p
