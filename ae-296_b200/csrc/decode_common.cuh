// Shared definitions of the operators around the delta: append, attention, 4-bit products (sm_100a).
#pragma once

#include "b200_decode.h"
#include "entry_common.cuh"
#include "lora_common.cuh"

namespace b200lora {

// ---- append ---------------------------------------------------------------------------------
cudaError_t launch_kv_append(const b200_append& a, const b200_kv_cache& c, int dtype, bool vectors, int n_sm, cudaStream_t s);

// ---- attention ------------------------------------------------------------------------------
// The work of a call is cut into units: one unit is kKeys keys of one row tile (at most kRows query rows that read
// the same keys) of one cache head.  Entities (groups first, then requests) follow one another, in an entity its
// cache heads, in a head its row tiles, in a tile its keys: unit u of all U belongs to worker ceil((u + 1) W / U) - 1,
// so a worker has a contiguous range and leaves one partial result per item (tile of a head of an entity) that it
// touches.  Items and workers both only ascend, so slot item + worker is a place of its own.
constexpr int kAttnKeys = 16;
constexpr int kAttnRows = 16;
constexpr int kAttnMaxWorkers = 2048;
// Groups of more than kWideFrom rows go to the wide kernel: units of kWideKeys keys for tiles of kWideRows rows, one
// worker per SM.  With 64 heads over 8 of 128, 32 groups of 4 requests (32 rows) over prefixes of 2048 tokens take 103 us in the split kernel
// (two tiles, of which the second finds the keys in L2) and 121 us in the wide one, 32 groups of 8 (64 rows) 190 and 141 us; one group
// over 16384 tokens 32 and 35 us (32 rows), 55 and 43 us (64 rows); all measured when the two kernels still ran side by side.
constexpr int kWideFrom = 32;                     // a multiple of kAttnRows
constexpr int kWideKeys = 128;
constexpr int kWideRows = 256;
constexpr int kWideMaxWorkers = 256;

struct AttnParams {
    b200_attention a;
    b200_kv_cache c;
    int per;               // query heads of a cache head
    unsigned per_inverse;  // 2^32 / per, rounded up
    int page_shift;
    int req_tiles;         // row tiles of a request
    int req_rows;          // rows of a request's partial result
    int max_group_tiles;   // of all groups together
    int grid;              // blocks of the wide and of the split kernel: SMs
    int wide_tiles;        // at most, of all groups together; 0: no group can be that large
    float scale_log2;
    int* units;            // [n_groups + n_requests + 1] units of a cache head before each entity
    int* tiles;            // [n_groups + 1] row tiles before each group
    int *wide_units, *wide_tile;   // the same of the wide kernel, [n_groups + 1] both
    float* part;           // partial results: rows of head_dim sums, then of (maximum, sum)
    float2* part_ml;
};
// rows of partial results: those of the groups' items, of the requests', of the wide kernel's
__host__ __device__ inline size_t attn_group_rows(const AttnParams& p) {
    return p.max_group_tiles == 0 ? 0 : ((size_t)p.max_group_tiles * p.c.n_kv_heads + kAttnMaxWorkers) * kAttnRows;
}
__host__ __device__ inline size_t attn_request_rows(const AttnParams& p) {
    return ((size_t)p.a.n_requests * p.req_tiles * p.c.n_kv_heads + kAttnMaxWorkers) * p.req_rows;
}
__host__ __device__ inline size_t attn_wide_rows(const AttnParams& p) {
    return p.wide_tiles == 0 ? 0 : ((size_t)p.wide_tiles * p.c.n_kv_heads + kWideMaxWorkers) * kWideRows;
}
cudaError_t launch_attention_wide(const AttnParams& p, int dtype, cudaStream_t s);
cudaError_t launch_attention(const AttnParams& p, int dtype, int n_sm, cudaStream_t s);

// ---- products with 4-bit weights --------------------------------------------------------------
cudaError_t launch_int4(const b200_int4& a, int dtype, int y_f32, int n_sm, cudaStream_t s);

}  // namespace b200lora
