// Internal launcher declarations of the paged cache (include/cactus_hip_paged.h).  Operands are checked by paged_api.hip.
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace cactus_hip {

struct PagedCache {
    int8_t* k;
    int8_t* v;
    float* ks;
    float* vs;
    const int32_t* tables;
    int num_pages, table_width, page_shift, kv_heads;
};

// rotation frequencies of a head in turns per position: theta^(-2i / D) / (2 pi).  They travel as a kernel argument
struct RopeTurns {
    double turn[128];
};

struct PagedAppendArgs {
    PagedCache c;
    const int32_t* positions;
    const int32_t* cu;         // null: one row per sequence
    int batch, tokens;
    const uint16_t *k, *v, *q;
    size_t k_stride, v_stride, q_stride;
    uint16_t* q_out;
    int q_heads;
    const uint16_t *q_weight, *k_weight;
    float eps;
    int rotate;
    int kv_per_part, kv_parts, q_per_part;      // items of a workgroup, workgroups of a page's items, query heads of one (the launcher's)
    RopeTurns rope;
};
hipError_t launch_kv_append_paged(int head_dim, const PagedAppendArgs& a, hipStream_t st);

struct PagedReadArgs {
    PagedCache c;
    const int32_t* starts;
    const int32_t* cu;
    int batch, rows;
    uint16_t *k_out, *v_out;
};
hipError_t launch_kv_read_paged(int head_dim, const PagedReadArgs& a, hipStream_t st);

struct PagedAttnArgs {
    PagedCache c;              // paged attention
    const int32_t* contexts;
    const uint16_t *k, *v;     // ragged attention
    size_t k_stride, v_stride;
    const int32_t* cu;         // null: one row per sequence
    int batch, tokens;
    const uint16_t* q;
    size_t q_stride;
    uint16_t* out;
    int q_heads, kv_heads;
    float scale;
    int window, sink;
    float* work;               // split records: per (item, split) work_rows x (maximum, sum) and work_rows x [head_dim]
    int work_rows;
    int min_rows;              // tile kernel: sequences with at most that many rows per kv head are not its
};
// attention_paged.hip: up to 16 rows (query rows x group) per sequence and kv head.  row tiles per (sequence, kv head), rows
// kept per record, key splits
struct StepShape {
    int row_tiles, rows, splits;
};
StepShape step_shape(size_t head_dim, size_t batch, size_t max_context, size_t q_heads, size_t kv_heads, size_t window, size_t sink,
                     bool one_row_each);
hipError_t launch_attention_step(int head_dim, const PagedAttnArgs& a, const StepShape& s, hipStream_t st);
// attention_tiles.hip: 128 rows at a time, over the pages or over FP16 rows.  blocks: workgroups, records: split records, joined:
// workgroups of the join (times the rows)
struct TileShape {
    int slots, splits, groups;
    size_t blocks, records, joined;
};
TileShape tile_shape(size_t head_dim, bool paged, size_t batch, size_t tokens, size_t max_context, size_t q_heads, size_t kv_heads,
                     size_t window, size_t sink, bool beside);
size_t tile_record_floats(size_t head_dim);
hipError_t launch_attention_tiles(int head_dim, bool paged, const PagedAttnArgs& a, const TileShape& s, hipStream_t st);

}  // namespace cactus_hip
