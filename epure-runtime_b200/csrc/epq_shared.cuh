// Attention of rows that share a prefix, in four launches: a plan (which tokens are shared by
// which rows) and the shared tokens (k_paged_shared.cu), each row's other tokens
// (k_paged_attn_shared.cu), and the join of both (k_paged_shared.cu).  What they hand on.
#pragma once

#include "epq_paged.cuh"

namespace epq {
namespace paged {

constexpr int kSharedTokens = 128;         // of a block of the shared part
constexpr int kSharedLanes = 128;          // query rows (row, head of the group) of a tensor-core tile

// Rows [row0, row0 + rows) of the batch, all of which (but the empty ones) see tokens [0, tokens) of sequence seq.
// A unit is a tile and a key head; its blocks are dealt out from place first + head * blocks on.
struct SharedTile {
    int row0, rows, seq, tokens, blocks, reserved0;
    int64_t first;
};
struct SharedHead {
    int64_t total;                         // blocks of all units
    int run;                               // blocks a CTA: it takes places [run * cta, run * cta + run)
    int tiles;
};

// Where they lie.  A record is a query row's sums over a part of the shared tokens, pitch floats: head_dim values
// (in the kernels' own dimension dim), then the maximum m (log2) and the sum of 2^(score - m) in two parts.  A unit's first piece
// leaves its records in `own` [2][batch * heads]; one that goes on into another CTA in that CTA's `cut` [grid][2][128].
// `rest` [batch * heads] holds the sums over the rows' other tokens.
struct SharedD {
    SharedHead* head;
    SharedTile* tiles;
    int32_t* row_tile;                     // [batch], -1: none
    int32_t* row_from;                     // [batch]: tokens that the row's tile took care of
    float* own;
    float* cut;
    float* rest;
    int64_t own_records;                   // batch * heads
    int pitch, slots, lane_rows;           // slots: tensor-core tiles of a unit; lane_rows: rows that one holds
};

// Whether a unit's blocks go to two accumulators in turn (its rows fill one tensor-core tile at most).
__host__ __device__ inline bool shared_alternates(int rows, int lane_rows, int slots) { return slots == 2 && rows <= lane_rows; }

}  // namespace paged
}  // namespace epq
