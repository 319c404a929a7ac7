// C ABI of the paged cache (include/cactus_hip_paged.h): argument checks and launches.
#include "../../include/cactus_hip_paged.h"

#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdio>

#include "paged.h"

namespace cactus_hip {
void set_last_error(const char* msg);   // api.hip
}  // namespace cactus_hip

using namespace cactus_hip;

namespace {

int refuse(const char* who, const char* what) {
    char buf[256];
    snprintf(buf, sizeof buf, "%s: %s", who, what);
    set_last_error(buf);
    return CACTUS_HIP_EINVAL;
}
int launched(const char* who, hipError_t e) {
    if (e == hipSuccess) return CACTUS_HIP_OK;
    char buf[256];
    snprintf(buf, sizeof buf, "%s launch: %s", who, hipGetErrorString(e));
    set_last_error(buf);
    return CACTUS_HIP_ERUNTIME;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// rows, sequences, pages and table entries are indexed with 32-bit integers on the device (elements with 64)
constexpr size_t MAX_ROWS = size_t(1) << 26, MAX_BATCH = size_t(1) << 20, MAX_PAGES = size_t(1) << 30, MAX_HEADS = 4096;

const char* bad_head_dim(size_t D) {
    return D == 64 || D == 128 || D == 256 ? nullptr : "head_dim must be 64, 128 or 256";
}

const char* bad_cache(const cactus_hip_paged_kv* c, const int32_t* tables, size_t width) {
    if (!c || !c->k || !c->v || !c->k_scales || !c->v_scales) return "null cache";
    if (!tables || width == 0) return "null block table";
    if (const char* e = bad_head_dim(c->head_dim)) return e;
    if (c->page_size != 16 && c->page_size != 32 && c->page_size != 64 && c->page_size != 128)
        return "page_size must be 16, 32, 64 or 128";
    if (c->kv_heads == 0 || c->kv_heads > MAX_HEADS) return "kv_heads must be 1 .. 4096";
    if (c->num_pages == 0 || c->num_pages > MAX_PAGES || width > MAX_PAGES / 128) return "too many pages, or none";
    if (!aligned16(c->k) || !aligned16(c->v)) return "the pages must be 16-byte aligned";
    return nullptr;
}

const char* bad_rows(const void* p, size_t stride, size_t heads, size_t D) {
    if (!p) return "null rows";
    if (!aligned16(p) || stride % 8 != 0) return "rows must be 16-byte aligned, their stride a multiple of 8 elements";
    if (stride < heads * D) return "row stride below heads * head_dim";
    if (stride >= size_t(1) << 24) return "row stride of 2^24 elements or more";
    return nullptr;
}

const char* bad_batch(const int32_t* cu, size_t batch, size_t tokens) {
    if (batch > MAX_BATCH || tokens > MAX_ROWS) return "more than 2^20 sequences or 2^26 rows";
    if (!cu && tokens != batch) return "without cu_seqlens there is one row per sequence";
    return nullptr;
}

// workgroups of a launch: a grid holds less than 2^32 threads, 512 to a workgroup at most
constexpr size_t MAX_ITEMS = size_t(1) << 23;
const char* too_many = "too many rows for one launch";

const char* bad_groups(size_t q_heads, size_t kv_heads) {
    if (q_heads == 0 || kv_heads == 0 || q_heads % kv_heads != 0 || q_heads > MAX_HEADS)
        return "num_q_heads must be a multiple of the kv heads, at most 4096";
    return nullptr;
}

// The kernels' running maximum starts at -1e30: rows of halves (and what append makes of them) have products of 1e14 at most, so
// scores stay above that.
const char* bad_scale(float scale) {
    return std::fabs(scale) <= 1e15f ? nullptr : "scale must be finite, 1e15 at most";
}

const char* bad_window(size_t window, size_t sink) {
    return window > 0x7fffffff || sink > 0x7fffffff ? "window and sink must be below 2^31" : nullptr;
}

// Positions lie below 2^30 (a table holds at most 2^30 tokens): a larger window or sink sees the same, and differences of two
// of them stay in an int.
int reach(size_t n) { return n < (size_t(1) << 30) ? (int)n : 1 << 30; }

PagedCache view(const cactus_hip_paged_kv& c, const int32_t* tables, size_t width) {
    PagedCache v{};
    v.k = c.k;
    v.v = c.v;
    v.ks = c.k_scales;
    v.vs = c.v_scales;
    v.tables = tables;
    v.num_pages = (int)c.num_pages;
    v.table_width = (int)width;
    v.page_shift = c.page_size == 16 ? 4 : c.page_size == 32 ? 5 : c.page_size == 64 ? 6 : 7;
    v.kv_heads = (int)c.kv_heads;
    return v;
}

// How a call of the paged attention is cut.  One row per sequence: the step kernel.  A ragged batch: sequences of at most 16
// rows per kv head are the step kernel's, longer ones the tile kernel's; which of them a batch holds only the device knows, so
// both are launched - except when the average is 64 rows or more (a batch of prompt chunks), where a launch that finds nothing to
// do costs about 3 us.  An odd short sequence costs less than that in the tile kernel while its context is a few key tiles; a long
// one is walked by one workgroup per kv head (one row on 32k keys beside a prompt of 4096 tokens: 853 us for both, 126 and 19 apart).
struct PagedPlan {
    bool by_step, by_tile;
    StepShape step;
    TileShape tile;
    size_t step_items, tile_items, step_bytes, tile_bytes;
    size_t bytes() const { return step_bytes + tile_bytes; }
    size_t items() const { return step_items > tile_items ? step_items : tile_items; }
};
PagedPlan paged_plan(const cactus_hip_paged_kv& c, size_t batch, size_t tokens, size_t max_context, size_t q_heads, size_t window,
                     size_t sink, bool one_row_each) {
    PagedPlan p{};
    p.by_step = one_row_each || tokens * (q_heads / c.kv_heads) < 64 * batch;
    p.by_tile = !one_row_each;
    if (p.by_step) {
        p.step = step_shape(c.head_dim, batch, max_context, q_heads, c.kv_heads, window, sink, one_row_each);
        p.step_items = batch * c.kv_heads * p.step.row_tiles * p.step.splits;
        if (p.step.splits > 1) p.step_bytes = p.step_items * p.step.rows * (c.head_dim + 2) * sizeof(float);
    }
    if (p.by_tile) {
        p.tile = tile_shape(c.head_dim, true, batch, tokens, max_context, q_heads, c.kv_heads, window, sink, p.by_step);
        p.tile_items = p.tile.blocks;
        p.tile_bytes = p.tile.records * tile_record_floats(c.head_dim) * sizeof(float);
    }
    return p;
}

// theta^(-2i/D) / (2 pi) for the pairs of a head; a decode loop asks for the same two numbers every step
const RopeTurns& rope_turns(size_t D, float theta) {
    thread_local RopeTurns table;
    thread_local size_t have_d = 0;
    thread_local float have_theta = 0.0f;
    if (have_d != D || have_theta != theta) {
        for (size_t i = 0; i < D / 2; i++)
            table.turn[i] = std::pow((double)theta, -2.0 * (double)i / (double)D) / 6.283185307179586476925286766559;
        have_d = D;
        have_theta = theta;
    }
    return table;
}

}  // namespace

#define REFUSE_IF(bad)                                    \
    do {                                                  \
        if (const char* why_ = (bad)) return refuse(who, why_); \
    } while (0)

extern "C" {

int cactus_hip_kv_append_paged_f16_dev(const cactus_hip_paged_kv* cache, const int32_t* block_tables, size_t table_width,
                                       const int32_t* positions, const int32_t* cu_seqlens, size_t batch, size_t tokens,
                                       const cactus_half_t* k, size_t k_stride, const cactus_half_t* v, size_t v_stride,
                                       const cactus_half_t* q, size_t q_stride, cactus_half_t* q_output,
                                       size_t num_q_heads, const cactus_half_t* q_weight, const cactus_half_t* k_weight,
                                       float eps, float theta, void* stream) {
    const char* who = "kv_append_paged";
    REFUSE_IF(bad_batch(cu_seqlens, batch, tokens));
    if (batch == 0 || tokens == 0) return CACTUS_HIP_OK;
    REFUSE_IF(bad_cache(cache, block_tables, table_width));
    if (!positions) return refuse(who, "null positions");
    REFUSE_IF(bad_rows(k, k_stride, cache->kv_heads, cache->head_dim));
    REFUSE_IF(bad_rows(v, v_stride, cache->kv_heads, cache->head_dim));
    if (q) {
        REFUSE_IF(bad_groups(num_q_heads, cache->kv_heads));
        REFUSE_IF(bad_rows(q, q_stride, num_q_heads, cache->head_dim));
        REFUSE_IF(bad_rows(q_output, num_q_heads * cache->head_dim, num_q_heads, cache->head_dim));
    }
    if ((q_weight && !aligned16(q_weight)) || (k_weight && !aligned16(k_weight)))
        return refuse(who, "norm weights must be 16-byte aligned");
    if (!(theta >= 0.0f) || std::isinf(theta)) return refuse(who, "theta must be finite and not negative");
    if (!(eps >= 0.0f) || std::isinf(eps)) return refuse(who, "eps must be finite and not negative");
    PagedAppendArgs a{};
    a.c = view(*cache, block_tables, table_width);
    a.positions = positions;
    a.cu = cu_seqlens;
    a.batch = (int)batch;
    a.tokens = (int)tokens;
    a.k = k;
    a.v = v;
    a.q = q;
    a.k_stride = k_stride;
    a.v_stride = v_stride;
    a.q_stride = q_stride;
    a.q_out = q_output;
    a.q_heads = (int)num_q_heads;
    a.q_weight = q_weight;
    a.k_weight = k_weight;
    a.eps = eps;
    a.rotate = theta > 0.0f;
    if (a.rotate) a.rope = rope_turns(cache->head_dim, theta);
    return launched(who, launch_kv_append_paged((int)cache->head_dim, a, (hipStream_t)stream));
}

int cactus_hip_kv_read_paged_f16_dev(const cactus_hip_paged_kv* cache, const int32_t* block_tables, size_t table_width,
                                     const int32_t* starts, const int32_t* cu_seqlens, size_t batch, size_t rows,
                                     cactus_half_t* k_output, cactus_half_t* v_output, void* stream) {
    const char* who = "kv_read_paged";
    if (batch == 0 || rows == 0) return CACTUS_HIP_OK;
    REFUSE_IF(bad_cache(cache, block_tables, table_width));
    if (!cu_seqlens || !starts) return refuse(who, "null starts or cu_seqlens");
    REFUSE_IF(bad_batch(cu_seqlens, batch, rows));
    if (!k_output || !v_output || !aligned16(k_output) || !aligned16(v_output))
        return refuse(who, "outputs must be 16-byte aligned");
    if (rows * cache->kv_heads * (cache->head_dim / 16) >= size_t(1) << 32) return refuse(who, too_many);
    PagedReadArgs a{view(*cache, block_tables, table_width), starts, cu_seqlens, (int)batch, (int)rows, k_output, v_output};
    return launched(who, launch_kv_read_paged((int)cache->head_dim, a, (hipStream_t)stream));
}

size_t cactus_hip_attention_paged_workspace_bytes(const cactus_hip_paged_kv* cache, size_t batch, size_t tokens,
                                                  size_t max_context, size_t num_q_heads, size_t window, size_t sink,
                                                  int one_row_each) {
    if (!cache || batch == 0 || tokens == 0 || bad_groups(num_q_heads, cache->kv_heads) || batch > MAX_BATCH || tokens > MAX_ROWS)
        return 0;
    return paged_plan(*cache, batch, tokens, max_context, num_q_heads, window, sink, one_row_each != 0).bytes();
}

int cactus_hip_attention_paged_f16_dev(const cactus_hip_paged_kv* cache, const int32_t* block_tables, size_t table_width,
                                       const int32_t* context_lens, const int32_t* cu_seqlens, size_t batch, size_t tokens,
                                       size_t max_context, const cactus_half_t* q, size_t q_stride, cactus_half_t* output,
                                       size_t num_q_heads, float scale, size_t window, size_t sink, void* workspace,
                                       size_t workspace_bytes, void* stream) {
    const char* who = "attention_paged";
    REFUSE_IF(bad_batch(cu_seqlens, batch, tokens));
    if (batch == 0 || tokens == 0) return CACTUS_HIP_OK;
    REFUSE_IF(bad_cache(cache, block_tables, table_width));
    REFUSE_IF(bad_groups(num_q_heads, cache->kv_heads));
    REFUSE_IF(bad_window(window, sink));
    if (tokens * (num_q_heads / cache->kv_heads) > MAX_ROWS * 8) return refuse(who, too_many);
    if (!context_lens) return refuse(who, "null context_lens");
    REFUSE_IF(bad_rows(q, q_stride, num_q_heads, cache->head_dim));
    REFUSE_IF(bad_rows(output, num_q_heads * cache->head_dim, num_q_heads, cache->head_dim));
    REFUSE_IF(bad_scale(scale));
    PagedAttnArgs a{};
    a.c = view(*cache, block_tables, table_width);
    a.contexts = context_lens;
    a.cu = cu_seqlens;
    a.batch = (int)batch;
    a.tokens = (int)tokens;
    a.q = q;
    a.q_stride = q_stride;
    a.out = output;
    a.q_heads = (int)num_q_heads;
    a.kv_heads = (int)cache->kv_heads;
    a.scale = scale == 0.0f ? 1.0f / std::sqrt((float)cache->head_dim) : scale;
    a.window = reach(window);
    a.sink = reach(sink);
    const PagedPlan p = paged_plan(*cache, batch, tokens, max_context, num_q_heads, window, sink, cu_seqlens == nullptr);
    if (p.bytes() > 0 && (!workspace || workspace_bytes < p.bytes() || !aligned16(workspace)))
        return refuse(who, "workspace missing, too small or not 16-byte aligned");
    if (p.items() >= MAX_ITEMS) return refuse(who, too_many);
    a.work = static_cast<float*>(workspace);
    if (p.by_step) {
        a.work_rows = p.step.rows;
        const int rc = launched(who, launch_attention_step((int)cache->head_dim, a, p.step, (hipStream_t)stream));
        if (rc != CACTUS_HIP_OK) return rc;
        a.work += p.step_bytes / sizeof(float);
        a.min_rows = 16;
    }
    if (p.by_tile) return launched(who, launch_attention_tiles((int)cache->head_dim, true, a, p.tile, (hipStream_t)stream));
    return CACTUS_HIP_OK;
}

int cactus_hip_attention_ragged_f16_dev(const cactus_half_t* q, size_t q_stride, const cactus_half_t* k, size_t k_stride,
                                        const cactus_half_t* v, size_t v_stride, cactus_half_t* output,
                                        const int32_t* cu_seqlens, size_t batch, size_t tokens, size_t num_q_heads,
                                        size_t num_kv_heads, size_t head_dim, float scale, size_t window, size_t sink,
                                        void* stream) {
    const char* who = "attention_ragged";
    if (batch == 0 || tokens == 0) return CACTUS_HIP_OK;
    REFUSE_IF(bad_head_dim(head_dim));
    if (!cu_seqlens) return refuse(who, "null cu_seqlens");
    REFUSE_IF(bad_batch(cu_seqlens, batch, tokens));
    REFUSE_IF(bad_groups(num_q_heads, num_kv_heads));
    REFUSE_IF(bad_window(window, sink));
    if (tokens * (num_q_heads / num_kv_heads) > MAX_ROWS * 8) return refuse(who, too_many);
    REFUSE_IF(bad_rows(q, q_stride, num_q_heads, head_dim));
    REFUSE_IF(bad_rows(k, k_stride, num_kv_heads, head_dim));
    REFUSE_IF(bad_rows(v, v_stride, num_kv_heads, head_dim));
    REFUSE_IF(bad_rows(output, num_q_heads * head_dim, num_q_heads, head_dim));
    REFUSE_IF(bad_scale(scale));
    PagedAttnArgs a{};
    a.k = k;
    a.v = v;
    a.k_stride = k_stride;
    a.v_stride = v_stride;
    a.cu = cu_seqlens;
    a.batch = (int)batch;
    a.tokens = (int)tokens;
    a.q = q;
    a.q_stride = q_stride;
    a.out = output;
    a.q_heads = (int)num_q_heads;
    a.kv_heads = (int)num_kv_heads;
    a.scale = scale == 0.0f ? 1.0f / std::sqrt((float)head_dim) : scale;
    a.window = reach(window);
    a.sink = reach(sink);
    const TileShape s = tile_shape(head_dim, false, batch, tokens, 0, num_q_heads, num_kv_heads, window, sink, false);
    if (s.blocks >= MAX_ITEMS) return refuse(who, too_many);
    return launched(who, launch_attention_tiles((int)head_dim, false, a, s, (hipStream_t)stream));
}

}  // extern "C"
