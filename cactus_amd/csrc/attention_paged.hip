// Attention over the paged INT8 cache (include/cactus_hip_paged.h) for few query rows: a decode step, or sequences of a
// mixed batch with at most 16 rows per kv head.
//
//   o = sum_j w_j v_j s_v[page(j)] / sum_j w_j,   w_j = exp(scale * s_k[page(j)] * q . k_j)
//
// Bound: HBM, 2 * context * kv_heads * head_dim bytes; a cached byte is loaded once for all query heads of its kv head.
//
// A workgroup is four waves on one (sequence, kv head, 16 rows, key range); a wave takes every fourth block of 32 keys.
// Nothing but the last merge goes through LDS: everything is computed transposed, so that a lane owns a row (lane % 16),
//   S^T = K Q^T   v_mfma_f32_16x16x32_f16, A = 16 keys: lane (key, g) holds 16-byte pieces of its key's row as they lie in
//                 memory (the contraction order is free as long as Q is laid out the same way)
//   O^T = V^T P^T A = 16 dims: lane (n, g) loads head_dim / 16 neighbouring bytes of 8 keys, and v_perm picks a byte of two
//                 keys at a time, so the transposition costs nothing; B = the weights where the scores left them.
// INT8 to binary16: a byte b ^ 0x80 under a zero byte is the subnormal half (b + 128) 2^-24 (one v_xor per four values, one
// v_perm per two), which the matrix cores multiply exactly (measured).  Keys stay like that: 2^24 and the 128 come back
// as one fma per score.  Values take one v_pk_fma_f16 per two more, to b 2^-9 (exact): left with the offset the output would be
// a small difference of large sums.
// A page has one scale per head.  Its key scale multiplies the scores of 16 keys at once; its value scale is added to the
// scores as a logarithm, so that weights (exp2(s + log2 s_v - running maximum + LIFT), rounded to binary16 against the maximum
// of all of them) never leave binary16's range whatever the scales are, and the sum of the plain weights takes the
// fp32 weights over s_v back.
// The next block's rows are requested before the current one is computed (registers, two blocks deep).  The output is
// rescaled only when a maximum has grown by more than 2^LAG.
// Measured (16 heads over 8, D = 128; a read-only kernel reaches 6.75 TB/s): 256 sequences of 300 to 700 keys 50.8 us = 5.2 TB/s; 4 of
// 32k, 32 heads over 8, 48.2 us with the join.  Kernels alone: 4 of 32k 45.7 us = 5.6 TB/s and 4.6 for the join; one of 4096 5.8 + 3.2
// us; 64 of window 508 + 4, 4 heads over 1, D = 256, 11.0 + 3.9 us (13.4 in a row).
#include "paged.hip.h"

#include <math.h>

namespace cactus_hip {

namespace {

constexpr float LOG2E = 1.4426950408889634f;
constexpr int STEP_ROWS = 16, STEP_WAVES = 4, STEP_KEYS = 32;

typedef int v2i __attribute__((ext_vector_type(2)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));

__device__ __forceinline__ v8h as_halves(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    const v4i v = {(int)a, (int)b, (int)c, (int)d};
    return __builtin_bit_cast(v8h, v);
}
// bytes 0, 1 (2, 3) of a word as two subnormal halves
__device__ __forceinline__ uint32_t low_pair(uint32_t x) { return __builtin_amdgcn_perm(0u, x, 0x0c010c00u); }
__device__ __forceinline__ uint32_t high_pair(uint32_t x) { return __builtin_amdgcn_perm(0u, x, 0x0c030c02u); }
// byte C of two words (each ^ 0x80) as two halves value * 2^-9
template <int C>
__device__ __forceinline__ uint32_t byte_pair(uint32_t x, uint32_t y) {
    const uint32_t u = __builtin_amdgcn_perm(y, x, 0x0c000c00u | ((4u + C) << 16) | (uint32_t)C);
    const _Float16 up = (_Float16)32768.0f, down = (_Float16)-0.25f;
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(__builtin_bit_cast(v2h, u), v2h{up, up}, v2h{down, down}));
}

// lanes l % 16 + {0, 16, 32, 48} combine a value
__device__ __forceinline__ float rows_max(float x) {
    unsigned u = __float_as_uint(x);
    auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    x = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
    u = __float_as_uint(x);
    r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float rows_sum(float x) {
    unsigned u = __float_as_uint(x);
    auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    x = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    u = __float_as_uint(x);
    r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

template <int W>
struct Words {
    uint32_t w[W];
};
template <int W>
__device__ __forceinline__ Words<W> load_words(const int8_t* p) {
    Words<W> r;
    if constexpr (W == 1) {
        r.w[0] = __builtin_nontemporal_load(reinterpret_cast<const uint32_t*>(p));
    } else if constexpr (W == 2) {
        const v2i v = __builtin_nontemporal_load(reinterpret_cast<const v2i*>(p));
        r.w[0] = v[0];
        r.w[1] = v[1];
    } else {
        const v4i v = __builtin_nontemporal_load(reinterpret_cast<const v4i*>(p));
        for (int i = 0; i < 4; i++) r.w[i] = v[i];
    }
    return r;
}

// a block of 32 keys as it lies in memory, and what its two halves need beside it
template <int D>
struct StepBlock {
    v4i k[2][D / 64];
    Words<D / 64> v[2][4];
    float ks[2], vs[2];
    size_t at[2];     // element offset of a half's first key
    int page[2];      // -1: none of these 16 keys is seen
    int key;          // first key
};

template <int D>
__global__ __launch_bounds__(64 * STEP_WAVES) __attribute__((amdgpu_waves_per_eu(D == 64 ? 4 : D == 128 ? 3 : 2)))
void attention_step_kernel(const PagedAttnArgs a, const int splits, const int row_tiles) {
    constexpr int KP = D / 64, DT = D / 16, DC = D < 128 ? D : 128;
    extern __shared__ float s_o[];               // [waves][rows][DC]
    __shared__ float s_m[STEP_WAVES][STEP_ROWS], s_l[STEP_WAVES][STEP_ROWS];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n = lane & 15, g = lane >> 4;
    const int split = blockIdx.x % splits, item = blockIdx.x / splits;
    const int tile = item % row_tiles, head = item / row_tiles % a.kv_heads, b = item / row_tiles / a.kv_heads;
    const int group = a.q_heads / a.kv_heads;
    const Rows rows = rows_of(a.cu, b, a.tokens);
    const int R = min(rows.count * group - tile * STEP_ROWS, STEP_ROWS);       // rows of this tile
    // a ragged batch: sequences with more rows are the chunk kernel's
    if (R <= 0 || (a.cu && rows.count * group > STEP_ROWS)) return;
    const int context = context_of(a, b);
    const int row = tile * STEP_ROWS + min(n, R - 1);                          // lanes past the last row repeat it
    const int token = rows.first + row / group, qh = head * group + row % group;
    const int pos = context - rows.count + row / group;
    const int pos_first = context - rows.count + tile * STEP_ROWS / group;
    const int pos_last = context - rows.count + (tile * STEP_ROWS + R - 1) / group;
    const TilePlan plan = plan_tiles(pos_first, pos_last, a.window, a.sink, STEP_KEYS);
    // this workgroup's blocks: whole rounds of its waves, so that a short sequence uses few splits
    const int rounds = (plan.tiles + STEP_WAVES - 1) / STEP_WAVES, per = (rounds + splits - 1) / splits * STEP_WAVES;
    const int u0 = split * per + wave, u1 = min(split * per + per, plan.tiles);

    // Q^T: step 2 i + c contracts bytes 64 i + 16 g + 8 c .. of a key row
    v8h q[2 * KP];
    float bias = 0.0f;
    {
        const uint16_t* qr = a.q + (size_t)token * a.q_stride + (size_t)qh * D;
#pragma unroll
        for (int i = 0; i < 2 * KP; i++) {
            q[i] = *reinterpret_cast<const v8h*>(qr + 64 * (i >> 1) + 16 * g + 8 * (i & 1));
#pragma unroll
            for (int e = 0; e < 8; e++) bias += (float)q[i][e];
        }
        bias = rows_sum(bias) * -128.0f;
    }

    const auto block_of = [&](int u) { return u < plan.sinks ? u : u - plan.sinks + plan.first; };
    const auto fetch_keys = [&](StepBlock<D>& t, int u) {
        t.key = block_of(u) * STEP_KEYS;
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const int key0 = t.key + 16 * h;
            int page = key0 <= pos_last ? page_of(a.c, b, key0 >> a.c.page_shift) : -1;
            page = __builtin_amdgcn_readfirstlane(page);
            t.page[h] = page;
            const size_t ph = (size_t)max(page, 0) * a.kv_heads + head;
            t.at[h] = ((ph << a.c.page_shift) + (key0 & ((1 << a.c.page_shift) - 1))) * D;
            t.ks[h] = a.c.ks[ph];
            t.vs[h] = a.c.vs[ph];
            const int8_t* kr = a.c.k + t.at[h] + n * D + 16 * g;
#pragma unroll
            for (int i = 0; i < KP; i++) t.k[h][i] = __builtin_nontemporal_load(reinterpret_cast<const v4i*>(kr + 64 * i));
        }
    };
    const auto fetch_values = [&](StepBlock<D>& t) {
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const int8_t* vr = a.c.v + t.at[h] + (4 * g) * D + n * DT;
#pragma unroll
            for (int r = 0; r < 4; r++) t.v[h][r] = load_words<KP>(vr + r * D);
        }
    };

    float m = -1e30f, l = 0.0f;
    v4f o[DT];
#pragma unroll
    for (int i = 0; i < DT; i++) o[i] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    const float c0 = a.scale * LOG2E;

    float s[8], inv_vs[2];
    const auto scores = [&](StepBlock<D>& t) {
        const bool whole = t.page[0] >= 0 && t.page[1] >= 0 && t.key + 31 <= pos_first &&
                           (!a.window || t.key >= pos_last - a.window || t.key + 31 < a.sink);
#pragma unroll
        for (int h = 0; h < 2; h++) {
            v4f acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int i = 0; i < KP; i++) {
                uint32_t x[4];
#pragma unroll
                for (int e = 0; e < 4; e++) x[e] = (uint32_t)t.k[h][i][e] ^ 0x80808080u;
                acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(as_halves(low_pair(x[0]), high_pair(x[0]), low_pair(x[1]), high_pair(x[1])),
                                                             q[2 * i], acc, 0, 0, 0);
                acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(as_halves(low_pair(x[2]), high_pair(x[2]), low_pair(x[3]), high_pair(x[3])),
                                                             q[2 * i + 1], acc, 0, 0, 0);
            }
            // scale * log2 e * s_k * (2^24 acc - 128 sum q) + log2 s_v
            const float vs = fmaxf(page_scale(t.vs[h]), 1e-20f), c = c0 * page_scale(t.ks[h]), up = c * 16777216.0f, add = fmaf(c, bias, __log2f(vs));
            inv_vs[h] = 1.0f / vs;
#pragma unroll
            for (int r = 0; r < 4; r++) s[4 * h + r] = fmaf(acc[r], up, add);
        }
        if (!whole) {
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const int key = t.key + 16 * (e >> 2) + 4 * g + (e & 3);
                const bool seen = t.page[e >> 2] >= 0 && key <= pos && (!a.window || pos - key <= a.window || key < a.sink);
                s[e] = seen ? s[e] : -INFINITY;
            }
            inv_vs[0] = t.page[0] >= 0 ? inv_vs[0] : 0.0f;
            inv_vs[1] = t.page[1] >= 0 ? inv_vs[1] : 0.0f;
        }
    };
    const auto values = [&](StepBlock<D>& t) {
        float top = fmaxf(fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3])), fmaxf(fmaxf(s[4], s[5]), fmaxf(s[6], s[7])));
        top = rows_max(top);
        if (__any(top > m + LAG)) {
            const float to = fmaxf(m, top), f = __builtin_amdgcn_exp2f(m - to);
            m = to;
            l *= f;
#pragma unroll
            for (int i = 0; i < DT; i++) o[i] *= f;
        }
        float w[8];
        const float unit = m - LIFT;
#pragma unroll
        for (int e = 0; e < 8; e++) w[e] = __builtin_amdgcn_exp2f(s[e] - unit);
        l = fmaf((w[0] + w[1]) + (w[2] + w[3]), inv_vs[0], l);
        l = fmaf((w[4] + w[5]) + (w[6] + w[7]), inv_vs[1], l);
        v8h p;
#pragma unroll
        for (int e = 0; e < 8; e++) p[e] = (_Float16)w[e];
        uint32_t x[8][KP];
#pragma unroll
        for (int e = 0; e < 8; e++)
#pragma unroll
            for (int i = 0; i < KP; i++) x[e][i] = t.v[e >> 2][e & 3].w[i] ^ 0x80808080u;
#define STEP_PV(C)                                                                                                           \
    o[4 * i + C] = __builtin_amdgcn_mfma_f32_16x16x32_f16(as_halves(byte_pair<C>(x[0][i], x[1][i]), byte_pair<C>(x[2][i], x[3][i]), \
                                                                    byte_pair<C>(x[4][i], x[5][i]), byte_pair<C>(x[6][i], x[7][i])), \
                                                          p, o[4 * i + C], 0, 0, 0)
#pragma unroll
        for (int i = 0; i < KP; i++) {
            STEP_PV(0);
            STEP_PV(1);
            STEP_PV(2);
            STEP_PV(3);
        }
#undef STEP_PV
    };

    if constexpr (D == 256) {
        // a block is 64 registers: the next keys are requested into the same ones as soon as the scores have used them, the
        // next values after the output has
        StepBlock<D> t;
        if (u0 < u1) {
            fetch_keys(t, u0);
            fetch_values(t);
        }
        for (int u = u0; u < u1; u += STEP_WAVES) {
            scores(t);
            if (u + STEP_WAVES < u1) fetch_keys(t, u + STEP_WAVES);
            values(t);
            if (u + STEP_WAVES < u1) fetch_values(t);
        }
    } else {
        StepBlock<D> t0, t1;
        const auto fetch = [&](StepBlock<D>& t, int u) {
            if (u >= u1) return;
            fetch_keys(t, u);
            fetch_values(t);
        };
        fetch(t0, u0);
        for (int u = u0; u < u1; u += 2 * STEP_WAVES) {
            fetch(t1, u + STEP_WAVES);
            scores(t0);
            values(t0);
            if (u + STEP_WAVES >= u1) break;
            fetch(t0, u + 2 * STEP_WAVES);
            scores(t1);
            values(t1);
        }
    }

    // the four waves' (maximum, sum, output) become one
    l = rows_sum(l);
    if (g == 0) {
        s_m[wave][n] = m;
        s_l[wave][n] = l;
    }
    __syncthreads();
    float top = s_m[0][n];
#pragma unroll
    for (int w = 1; w < STEP_WAVES; w++) top = fmaxf(top, s_m[w][n]);
    const float up = __builtin_amdgcn_exp2f(m - top) * 512.0f;
    float* record = splits > 1 ? a.work + (size_t)blockIdx.x * a.work_rows * (D + 2) : nullptr;
    // a lane's dims are the contiguous quarter g of the row; 128 of them at a time keep the exchange at 32 KB
#pragma unroll 1
    for (int d0 = 0; d0 < D; d0 += DC) {
        if (d0 > 0) __syncthreads();
        if (n < R && 4 * g * DT >= d0 && 4 * g * DT < d0 + DC) {
            float* mine = s_o + ((size_t)wave * R + n) * DC + 4 * g * DT - d0;
#pragma unroll
            for (int r = 0; r < 4; r++)
#pragma unroll
                for (int i = 0; i < DT; i += 4) {
                    v4f v;
#pragma unroll
                    for (int e = 0; e < 4; e++) v[e] = o[i + e][r] * up;
                    *reinterpret_cast<v4f*>(mine + r * DT + i) = v;
                }
        }
        __syncthreads();
        for (int i = threadIdx.x; i < R * DC / 4; i += 64 * STEP_WAVES) {
            const int rw = i / (DC / 4), d = i % (DC / 4) * 4;
            float mm = s_m[0][rw];
#pragma unroll
            for (int w = 1; w < STEP_WAVES; w++) mm = fmaxf(mm, s_m[w][rw]);
            float sum = 0.0f;
            v4f v = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int w = 0; w < STEP_WAVES; w++) {
                sum += s_l[w][rw] * __builtin_amdgcn_exp2f(s_m[w][rw] - mm);
                v += *reinterpret_cast<const v4f*>(s_o + ((size_t)w * R + rw) * DC + d);
            }
            const int orow = tile * STEP_ROWS + rw;
            if (record) {
                if (d == 0 && d0 == 0) {
                    record[2 * rw] = mm;
                    record[2 * rw + 1] = sum;
                }
                *reinterpret_cast<v4f*>(record + 2 * a.work_rows + rw * D + d0 + d) = v;
            } else {
                const float inv = sum > 0.0f || sum != sum ? 1.0f / sum : 0.0f;
                v4h h;
#pragma unroll
                for (int e = 0; e < 4; e++) h[e] = (_Float16)(v[e] * inv);
                *reinterpret_cast<v4h*>(a.out + ((size_t)(rows.first + orow / group) * a.q_heads + head * group + orow % group) * D +
                                        d0 + d) = h;
            }
        }
    }
}

// Joins the splits of a row: four waves per row, each every fourth split, lanes = dims; latency is all there is to it.
template <int D>
__global__ __launch_bounds__(256) void attention_join_kernel(const PagedAttnArgs a, const int splits, const int row_tiles) {
    constexpr int W = D / 64;
    __shared__ float s_l[4], s_o[4][D];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), item = blockIdx.x, rw = blockIdx.y;
    const int tile = item % row_tiles, head = item / row_tiles % a.kv_heads, b = item / row_tiles / a.kv_heads;
    const int group = a.q_heads / a.kv_heads;
    const Rows rows = rows_of(a.cu, b, a.tokens);
    const int orow = tile * STEP_ROWS + rw;
    if (orow >= rows.count * group || (a.cu && rows.count * group > STEP_ROWS)) return;
    const size_t step = (size_t)a.work_rows * (D + 2);
    const float* rec = a.work + (size_t)item * splits * step;
    float m = -1e30f, l = 0.0f, o[W];
#pragma unroll
    for (int i = 0; i < W; i++) o[i] = 0.0f;
    for (int s = lane; s < splits; s += 64) m = fmaxf(m, rec[s * step + 2 * rw]);
    m = wave_max(m);
#pragma unroll 8
    for (int s = wave; s < splits; s += 4) {
        const float f = __builtin_amdgcn_exp2f(rec[s * step + 2 * rw] - m);
        l = fmaf(rec[s * step + 2 * rw + 1], f, l);
        const float* x = rec + s * step + 2 * a.work_rows + rw * D + lane * W;
#pragma unroll
        for (int i = 0; i < W; i++) o[i] = fmaf(x[i], f, o[i]);
    }
    if (lane == 0) s_l[wave] = l;
#pragma unroll
    for (int i = 0; i < W; i++) s_o[wave][lane * W + i] = o[i];
    __syncthreads();
    const int d = threadIdx.x;
    if (d >= D) return;
    l = (s_l[0] + s_l[1]) + (s_l[2] + s_l[3]);
    const float inv = l > 0.0f || l != l ? 1.0f / l : 0.0f;
    a.out[((size_t)(rows.first + orow / group) * a.q_heads + head * group + orow % group) * D + d] =
        f2h(((s_o[0][d] + s_o[1][d]) + (s_o[2][d] + s_o[3][d])) * inv);
}

template <int D>
hipError_t launch_step(const PagedAttnArgs& a, const StepShape& s, hipStream_t st) {
    const int items = a.batch * a.kv_heads * s.row_tiles;
    attention_step_kernel<D><<<dim3((unsigned)((size_t)items * s.splits)), dim3(64 * STEP_WAVES),
                               (size_t)STEP_WAVES * s.rows * (D < 128 ? D : 128) * sizeof(float), st>>>(a, s.splits, s.row_tiles);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || s.splits == 1) return e;
    attention_join_kernel<D><<<dim3((unsigned)items, (unsigned)s.rows), dim3(256), 0, st>>>(a, s.splits, s.row_tiles);
    return hipGetLastError();
}

}  // namespace

// The split rule.  Keys are split until as many workgroups are there as keep about 16 MB of cache requested, which is what the
// memory's latency needs: 256 of four waves and two blocks each (one at head_dim 256), 512 at head_dim 64, whose blocks are half as
// large.  More only make records: 4 sequences of 32k, 4 heads over 1 of 256: 18 us with 256, 29 with 1024; 4 of 32k, 32 heads over 8 of
// 64: 37 and 28 with 512, 27 with 1024.  A round of a workgroup's waves takes 128 keys, and a split that saves fewer than three
// rounds does not pay for the join (300 keys in 64 sequences, 16 heads over 8 of 128: 18 us in two splits, 10 in one).
StepShape step_shape(size_t head_dim, size_t batch, size_t max_context, size_t q_heads, size_t kv_heads, size_t window, size_t sink,
                     bool one_row_each) {
    StepShape s;
    const size_t group = q_heads / kv_heads;
    s.rows = one_row_each && group < STEP_ROWS ? (int)((group + 1) & ~size_t(1)) : STEP_ROWS;   // even: records stay aligned
    s.row_tiles = one_row_each ? (int)((group + STEP_ROWS - 1) / STEP_ROWS) : 1;
    const size_t items = batch * kv_heads * s.row_tiles;
    size_t keys = max_context;
    if (window && window + sink < keys) keys = window + sink;
    const size_t rounds = (keys + STEP_WAVES * STEP_KEYS - 1) / (STEP_WAVES * STEP_KEYS);
    const size_t fill = head_dim == 64 ? 512 : 256, want = items >= fill ? 1 : fill / items, most = rounds < want ? rounds : want;
    s.splits = most > 1 && rounds - (rounds + most - 1) / most >= 3 ? (int)most : 1;
    return s;
}

hipError_t launch_attention_step(int D, const PagedAttnArgs& a, const StepShape& s, hipStream_t st) {
    return D == 64 ? launch_step<64>(a, s, st) : D == 128 ? launch_step<128>(a, s, st) : launch_step<256>(a, s, st);
}

}  // namespace cactus_hip
