// Attention over the paged INT8 cache and over packed FP16 prompts (include/cactus_hip_paged.h): one wave per query row
// and head, 64 keys at a time.  Lane = key for the scores, lane = dims for the output; online softmax on base-2 scores.
#include "paged.hip.h"

#include <math.h>

namespace cactus_hip {

namespace {

template <int D, bool PAGED>
__global__ __launch_bounds__(256) void attention_rows_kernel(const PagedAttnArgs a) {
    __shared__ float s_q[4][D];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const long long item = (long long)blockIdx.x * 4 + w;
    if (item >= (long long)a.tokens * a.q_heads) return;
    const int row = (int)(item / a.q_heads), h = (int)(item % a.q_heads), kvh = h / (a.q_heads / a.kv_heads);
    const int b = a.cu ? owner_of(row, a.batch, [&](int i) { return min(max(a.cu[i], 0), a.tokens); }) : row;
    const Rows rows = rows_of(a.cu, b, a.tokens);
    if (row < rows.first || row >= rows.first + rows.count) return;
    long long context = rows.count;
    if (PAGED) context = min((long long)a.contexts[b], (long long)a.c.table_width << a.c.page_shift);
    const long long pos = context - rows.count + (row - rows.first);
    const uint16_t* qr = a.q + (size_t)row * a.q_stride + (size_t)h * D;
    for (int d = lane; d < D; d += 64) s_q[w][d] = h2f(qr[d]);
    __builtin_amdgcn_wave_barrier();

    constexpr int DPL = D / 64;
    float o[DPL], m = -INFINITY, l = 0.0f;
    for (int i = 0; i < DPL; i++) o[i] = 0.0f;
    const long long low = a.window ? max(0LL, pos - a.window) : 0;
    for (long long k0 = 0; k0 <= pos; k0 += 64) {
        if (k0 + 64 <= low && k0 >= a.sink) {      // nothing here is seen
            continue;
        }
        const long long key = k0 + lane;
        bool seen = key <= pos && (!a.window || pos - key <= a.window || key < a.sink);
        int page = -1;
        size_t ph = 0;
        if (PAGED) {
            if (seen) page = page_of(a.c, b, (int)(key >> a.c.page_shift));
            seen = seen && page >= 0;
            ph = (size_t)max(page, 0) * a.kv_heads + kvh;
        }
        float s = -INFINITY, vscale = 1.0f;
        if (seen) {
            s = 0.0f;
            if (PAGED) {
                const int8_t* kr = a.c.k + ((ph << a.c.page_shift) + (key & ((1 << a.c.page_shift) - 1))) * D;
                for (int d = 0; d < D; d++) s = fmaf(s_q[w][d], (float)kr[d], s);
                s *= a.c.ks[ph];
                vscale = a.c.vs[ph];
            } else {
                const uint16_t* kr = a.k + (size_t)(rows.first + key) * a.k_stride + (size_t)kvh * D;
                for (int d = 0; d < D; d++) s = fmaf(s_q[w][d], h2f(kr[d]), s);
            }
            s *= a.scale;
        }
        const float mn = fmaxf(m, wave_max(s));
        if (mn == -INFINITY) continue;
        const float p = seen ? __expf(s - mn) : 0.0f, f = __expf(m - mn);
        m = mn;
        l = l * f + wave_sum(p);
        for (int i = 0; i < DPL; i++) o[i] *= f;
        for (int t = 0; t < 64; t++) {
            const float pt = __shfl(p, t);
            if (pt == 0.0f) continue;
            if (PAGED) {
                const size_t ph_t = (size_t)__shfl(page, t) * a.kv_heads + kvh;
                const float pv = pt * __shfl(vscale, t);
                const int8_t* vr = a.c.v + ((ph_t << a.c.page_shift) + ((k0 + t) & ((1 << a.c.page_shift) - 1))) * D;
                for (int i = 0; i < DPL; i++) o[i] = fmaf(pv, (float)vr[lane + 64 * i], o[i]);
            } else {
                const uint16_t* vr = a.v + (size_t)(rows.first + k0 + t) * a.v_stride + (size_t)kvh * D;
                for (int i = 0; i < DPL; i++) o[i] = fmaf(pt, h2f(vr[lane + 64 * i]), o[i]);
            }
        }
    }
    const float inv = l > 0.0f ? 1.0f / l : 0.0f;
    uint16_t* out = a.out + ((size_t)row * a.q_heads + h) * D;
    for (int i = 0; i < DPL; i++) out[lane + 64 * i] = f2h(o[i] * inv);
}

template <bool PAGED>
hipError_t launch_rows(int D, const PagedAttnArgs& a, hipStream_t st) {
    const dim3 grid((unsigned)(((size_t)a.tokens * a.q_heads + 3) / 4));
    if (D == 64)
        attention_rows_kernel<64, PAGED><<<grid, dim3(256), 0, st>>>(a);
    else if (D == 128)
        attention_rows_kernel<128, PAGED><<<grid, dim3(256), 0, st>>>(a);
    else
        attention_rows_kernel<256, PAGED><<<grid, dim3(256), 0, st>>>(a);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_attention_paged(int D, const PagedAttnArgs& a, hipStream_t st) { return launch_rows<true>(D, a, st); }
hipError_t launch_attention_ragged(int D, const PagedAttnArgs& a, hipStream_t st) { return launch_rows<false>(D, a, st); }

}  // namespace cactus_hip
