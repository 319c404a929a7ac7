// The paged INT8 key/value cache (include/cactus_hip_paged.h): appending the rows of a step, reading tokens back.
//
// Append.  k' = rope(rms_norm(k)), q' = rope(rms_norm(q)); the page's scale of k' (and of v) is the running
// max(|x|) / 127 of its tokens, q = rne(x / scale).  Bound: HBM for prompts (rows in, INT8 and the q rows out: every byte
// moves once), launch latency for a decode step.
//
// A workgroup takes the part of ONE page that the call writes, either for some of its items (a kv head's keys or its values: their
// maximum never leaves the workgroup) or for some query heads; the launch cuts finer the fewer pages there are.  D / 16 lanes
// hold a row: lane j the 8 elements from 8 j and their rotation partners from D / 2 + 8 j, two 16-byte loads, no exchange for
// the rotation.  The row slots of a workgroup are (token of the page) x (head): STEP (one row per sequence) gives them all to
// heads, otherwise tokens come first.  A lane keeps its tokens while it walks the heads, so an angle is computed once per
// workgroup: in fp64 as turns (pos * theta^(-2i/D) / 2 pi, only the fraction kept), because an fp32 product at position 30000
// is off by 1e-3; v_sin_f32 / v_cos_f32 take turns and are off by 2^-23 at most (measured).
// Measured: 7 prompts of 500 to 1900 tokens, 32 + 2 x 8 heads of 64: 25 us = 4.5 TB/s (a large copy reaches 5.16); a step of one
// sequence 4.9 us, of 256 6.8 us; 5 chunks of 100 to 256 tokens, 4 + 2 x 1 heads of 256 in pages of 128: 11.4 us, a chain of
// row, maximum, store and requantization in 96 workgroups.
#include "paged.hip.h"

#include <math.h>

namespace cactus_hip {

namespace {

__device__ __forceinline__ float finite_half(float x) {
    return x != x ? 0.0f : fminf(fmaxf(x, -65504.0f), 65504.0f);
}

template <int LPR>
__device__ __forceinline__ float row_sum(float v) {
#pragma unroll
    for (int o = LPR / 2; o > 0; o >>= 1) v += __shfl_xor(v, o, LPR);
    return v;
}
template <int LPR>
__device__ __forceinline__ float row_max(float v) {
#pragma unroll
    for (int o = LPR / 2; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, LPR));
    return v;
}

struct Row16 {
    float lo[8], hi[8];   // elements 8 j .. and D / 2 + 8 j ..
};

template <int D>
__device__ __forceinline__ Row16 load_row(const uint16_t* __restrict__ row, int j) {
    const v8h a = *reinterpret_cast<const v8h*>(row + 8 * j), b = *reinterpret_cast<const v8h*>(row + D / 2 + 8 * j);
    Row16 r;
#pragma unroll
    for (int e = 0; e < 8; e++) {
        r.lo[e] = (float)a[e];
        r.hi[e] = (float)b[e];
    }
    return r;
}

// rms_norm with an optional weight, then the rotation by the angle whose cosine and sine the lane holds
template <int D>
__device__ __forceinline__ void norm_rotate(Row16& r, bool norm, const Row16& w, float eps, bool rotate, const float (&cs)[8],
                                            const float (&sn)[8]) {
    if (norm) {
        float ss = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; e++) ss = fmaf(r.hi[e], r.hi[e], fmaf(r.lo[e], r.lo[e], ss));
        ss = row_sum<D / 16>(ss);
        const float inv = 1.0f / sqrtf(ss * (1.0f / D) + eps);
#pragma unroll
        for (int e = 0; e < 8; e++) {
            r.lo[e] = r.lo[e] * inv * w.lo[e];
            r.hi[e] = r.hi[e] * inv * w.hi[e];
        }
    }
    if (rotate) {
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const float a = r.lo[e], b = r.hi[e];
            r.lo[e] = a * cs[e] - b * sn[e];
            r.hi[e] = b * cs[e] + a * sn[e];
        }
    }
}

__device__ __forceinline__ float absmax(const Row16& r) {
    float m = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; e++) m = fmaxf(m, fmaxf(fabsf(r.lo[e]), fabsf(r.hi[e])));
    return m;
}

// x / scale rounded to an integer, as a byte.  |x| <= 127 scale.  One step of refinement makes the product with the reciprocal the
// quotient: without it one value in 10^5 falls on the other side of a half.
__device__ __forceinline__ uint32_t code(float x, float scale, float inv) {
    const float y = x * inv;
    return (uint32_t)rne_i32(fmaf(fmaf(-y, scale, x), inv, y)) & 0xFFu;
}
template <int D>
__device__ __forceinline__ void store_i8(int8_t* __restrict__ row, int j, const Row16& r, float scale) {
    const float inv = 1.0f / scale;
    uint32_t o[4] = {0, 0, 0, 0};
#pragma unroll
    for (int e = 0; e < 8; e++) {
        o[e >> 2] |= code(r.lo[e], scale, inv) << (8 * (e & 3));
        o[2 + (e >> 2)] |= code(r.hi[e], scale, inv) << (8 * (e & 3));
    }
    *reinterpret_cast<uint2*>(row + 8 * j) = make_uint2(o[0], o[1]);
    *reinterpret_cast<uint2*>(row + D / 2 + 8 * j) = make_uint2(o[2], o[3]);
}

constexpr int MAX_SLOTS = 256;   // row slots of a workgroup (1024 threads, 4 lanes a row)

// RPL: tokens a lane holds
template <int D, bool STEP, int RPL>
__global__ __launch_bounds__(1024) void append_paged_kernel(const PagedAppendArgs a) {
    constexpr int LPR = D / 16;
    __shared__ uint32_t s_max[MAX_SLOTS];
    __shared__ float s_again[MAX_SLOTS];         // old / new scale of a head whose earlier tokens are requantized, else -1

    const int tid = threadIdx.x, slot = tid / LPR, j = tid % LPR, slots = blockDim.x / LPR;
    const int P = 1 << a.c.page_shift;

    // which sequence, which page of it, which of the page's slots
    int b, seg = 0;
    if constexpr (STEP) {
        b = blockIdx.x;
    } else {
        const auto begin = [&](int i) { return slot_begin(a.cu, i, a.tokens, 1, P, 2); };
        b = owner_of((int)blockIdx.x, a.batch, begin);
        seg = (int)blockIdx.x - begin(b);
    }
    const Rows rows = rows_of(STEP ? nullptr : a.cu, b, a.tokens);
    const long long pos0 = a.positions[b];
    if (pos0 < 0 || seg < 0 || rows.count == 0) return;
    const long long index = (pos0 >> a.c.page_shift) + seg, base = index << a.c.page_shift;   // page of the sequence, its first position
    if (base >= pos0 + rows.count) return;
    const int e_lo = (int)max(pos0 - base, 0LL), e_hi = (int)min(pos0 + rows.count - base, (long long)P);
    const int row0 = rows.first + (int)(base - pos0);          // packed row of page slot 0

    const int TP = STEP ? 1 : min(P, slots), HP = slots / TP;  // tokens x heads of a pass
    const int ts = slot % TP, hs = slot / TP;
    // items of a page: its heads' keys, then their values
    const int item0 = blockIdx.y * a.kv_per_part, items = min(a.kv_per_part, 2 * a.c.kv_heads - item0);
    const bool turns = a.rotate && ((int)blockIdx.y >= a.kv_parts || item0 < a.c.kv_heads);
    float cs[RPL][8], sn[RPL][8];
    int e[RPL];
    bool live[RPL];
#pragma unroll
    for (int r = 0; r < RPL; r++) {
        e[r] = STEP ? e_lo : ts + r * TP;
        live[r] = e[r] >= e_lo && e[r] < e_hi;
        if (turns && live[r]) {
            const double pos = (double)(base + e[r]);
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const double t = pos * a.rope.turn[8 * j + i];
                const float turn = (float)(t - rint(t));
                sn[r][i] = __builtin_amdgcn_sinf(turn);
                cs[r][i] = __builtin_amdgcn_cosf(turn);
            }
        }
    }

    if ((int)blockIdx.y >= a.kv_parts) {         // query heads
        Row16 w{};
        if (a.q_weight) w = load_row<D>(a.q_weight, j);
        const int q0 = ((int)blockIdx.y - a.kv_parts) * a.q_per_part, qn = min(a.q_per_part, a.q_heads - q0);
        for (int h0 = hs; h0 < qn; h0 += HP) {
#pragma unroll
            for (int r = 0; r < RPL; r++) {
                if (!live[r]) continue;          // the same for all lanes of a row
                const size_t row = (size_t)(row0 + e[r]);
                Row16 x = load_row<D>(a.q + row * a.q_stride + (size_t)(q0 + h0) * D, j);
                norm_rotate<D>(x, a.q_weight != nullptr, w, a.eps, a.rotate, cs[r], sn[r]);
                v8h lo, hi;
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    lo[i] = (_Float16)x.lo[i];
                    hi[i] = (_Float16)x.hi[i];
                }
                uint16_t* out = a.q_out + (row * a.q_heads + q0 + h0) * D;
                *reinterpret_cast<v8h*>(out + 8 * j) = lo;
                *reinterpret_cast<v8h*>(out + D / 2 + 8 * j) = hi;
            }
        }
        return;
    }

    const int page = index < a.c.table_width ? page_of(a.c, b, (int)index) : -1;
    if (page < 0) return;
    Row16 w{};
    if (a.k_weight) w = load_row<D>(a.k_weight, j);
    for (int i0 = 0; i0 < items; i0 += HP) {
        const int item = item0 + i0 + hs;
        const bool on = i0 + hs < items, value = item >= a.c.kv_heads;
        const int kv_head = value ? item - a.c.kv_heads : item;
        const size_t ph = (size_t)page * a.c.kv_heads + kv_head;
        float* scale = (value ? a.c.vs : a.c.ks) + ph;
        const float old = on && e_lo > 0 ? page_scale(*scale) : 0.0f;
        if constexpr (!STEP) {
            for (int i = tid; i < HP; i += blockDim.x) s_max[i] = 0;
            __syncthreads();
        }
        Row16 x[RPL];
        float top = 0.0f;
#pragma unroll
        for (int r = 0; r < RPL; r++) {
            if (!on || !live[r]) continue;
            const size_t row = (size_t)(row0 + e[r]), head = (size_t)kv_head * D;
            x[r] = load_row<D>((value ? a.v + row * a.v_stride : a.k + row * a.k_stride) + head, j);
#pragma unroll
            for (int i = 0; i < 8; i++) {
                x[r].lo[i] = finite_half(x[r].lo[i]);
                x[r].hi[i] = finite_half(x[r].hi[i]);
            }
            if (!value) norm_rotate<D>(x[r], a.k_weight != nullptr, w, a.eps, a.rotate, cs[r], sn[r]);
            top = fmaxf(top, absmax(x[r]));
        }
        top = row_max<LPR>(top);
        if constexpr (!STEP) {
            // bits of non-negative floats order as the floats do: the maximum is the same in any order
            if (j == 0 && on) atomicMax(&s_max[hs], __float_as_uint(top));
            __syncthreads();
            top = __uint_as_float(s_max[hs]);
        }
        const float now = fmaxf(old, fmaxf(top / 127.0f, 1e-10f));
#pragma unroll
        for (int r = 0; r < RPL; r++) {
            if (!on || !live[r]) continue;
            store_i8<D>((value ? a.c.v : a.c.k) + ((ph << a.c.page_shift) + e[r]) * D, j, x[r], now);
        }
        if (on && ts == 0 && j == 0) {
            *scale = now;
            s_again[hs] = now > old ? old / now : -1.0f;
        }
        if (e_lo > 0) {                          // the page held tokens before: bring them to a scale that has grown
            __syncthreads();
            for (int c = 0; c < min(HP, items - i0); c++) {
                const float f = s_again[c];
                if (f < 0.0f) continue;
                const int it = item0 + i0 + c;
                const bool val = it >= a.c.kv_heads;
                const size_t first = (((size_t)page * a.c.kv_heads + (val ? it - a.c.kv_heads : it)) << a.c.page_shift) * D;
                int8_t* codes = (val ? a.c.v : a.c.k) + first;
                for (int i = tid * 16; i < e_lo * D; i += blockDim.x * 16) {
                    v4i q = *reinterpret_cast<const v4i*>(codes + i);
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        uint32_t o = 0;
#pragma unroll
                        for (int s = 0; s < 4; s++)
                            o |= (uint32_t)(rne_i32((float)(int8_t)((uint32_t)q[k] >> (8 * s)) * f) & 0xFF) << (8 * s);
                        q[k] = (int)o;
                    }
                    *reinterpret_cast<v4i*>(codes + i) = q;
                }
            }
        }
        __syncthreads();
    }
}

// Read: a lane turns 16 bytes of a token into 32.  A wave walks the 16-byte pieces of its tokens in memory order; it looks up
// the sequence of its first token and moves on from there.
// Bound: HBM; 53 MB in 12.4 us = 4.3 TB/s, a few tokens 2.6 us.
template <int D>
__global__ __launch_bounds__(256) void read_paged_kernel(const PagedReadArgs a) {
    const int chunks = a.c.kv_heads * (D / 16);              // 16-byte pieces of a token, keys or values
    const long long total = (long long)a.rows * chunks;
    const long long first = ((long long)blockIdx.x * 4 + (threadIdx.x >> 6)) * 64;
    if (first >= total) return;
    int b = owner_of((int)(first / chunks), a.batch, [&](int i) { return min(max(a.cu[i], 0), a.rows); });
    const long long at = first + (threadIdx.x & 63);
    if (at >= total) return;
    const int row = (int)(at / chunks), piece = (int)(at % chunks), h = piece / (D / 16), d = piece % (D / 16) * 16;
    while (b < a.batch && row >= a.cu[b + 1]) b++;
    if (b >= a.batch || row < a.cu[b]) return;
    const long long token = (long long)a.starts[b] + row - a.cu[b];
    const int page = token < 0 || (token >> a.c.page_shift) >= a.c.table_width ? -1 : page_of(a.c, b, (int)(token >> a.c.page_shift));
    const size_t ph = (size_t)max(page, 0) * a.c.kv_heads + h;
    const size_t src = ((ph << a.c.page_shift) + (size_t)(token & ((1 << a.c.page_shift) - 1))) * D + d;
#pragma unroll
    for (int which = 0; which < 2; which++) {
        uint16_t* out = (which ? a.v_out : a.k_out) + ((size_t)row * a.c.kv_heads + h) * D + d;
        v8h lo{}, hi{};
        if (page >= 0) {
            const float s = page_scale((which ? a.c.vs : a.c.ks)[ph]);
            const v4i q = *reinterpret_cast<const v4i*>((which ? a.c.v : a.c.k) + src);
#pragma unroll
            for (int e = 0; e < 8; e++) {
                lo[e] = (_Float16)((float)(int8_t)((uint32_t)q[e >> 2] >> (8 * (e & 3))) * s);
                hi[e] = (_Float16)((float)(int8_t)((uint32_t)q[2 + (e >> 2)] >> (8 * (e & 3))) * s);
            }
        }
        *reinterpret_cast<v8h*>(out) = lo;
        *reinterpret_cast<v8h*>(out + 8) = hi;
    }
}

template <int D>
hipError_t append_paged(const PagedAppendArgs& args, hipStream_t st) {
    PagedAppendArgs a = args;
    const int P = 1 << a.c.page_shift, LPR = D / 16;
    const bool step = a.cu == nullptr;
    // A row slot for every token of the page in 256 threads, else two tokens a lane (a lane's second token costs 35 registers, a
    // larger workgroup longer waits for each other: prompts of 8000 tokens, 32 heads of 64, pages of 32: 23.4 us with two, 22.2 with
    // one; 16 heads of 128, pages of 64: 25.2 in 256 threads, 28.1 in 512).  A step's row slots are its heads.
    const int rpl = P * LPR > 256 ? 2 : 1, threads = step || P * LPR < 256 ? 256 : P * LPR / rpl;
    const size_t pieces = step ? (size_t)a.batch : ((size_t)a.tokens >> a.c.page_shift) + 2 * (size_t)a.batch;
    // heads per workgroup: all of them when there are pages enough to fill the chip (about 1024 workgroups), one pass at least
    const int at_once = step ? 256 / LPR : 1;
    const auto cut = [&](int heads, int least) {
        const size_t want = (1024 + pieces - 1) / pieces;
        const int most = (heads + least - 1) / least, parts = want < (size_t)most ? (int)want : most;
        return (heads + parts - 1) / parts;
    };
    a.kv_per_part = cut(2 * a.c.kv_heads, at_once);
    a.kv_parts = (2 * a.c.kv_heads + a.kv_per_part - 1) / a.kv_per_part;
    int q_parts = 0;
    if (a.q) {
        a.q_per_part = cut(a.q_heads, at_once);
        q_parts = (a.q_heads + a.q_per_part - 1) / a.q_per_part;
    }
    const dim3 grid((unsigned)pieces, (unsigned)(a.kv_parts + q_parts));
    if (step)
        append_paged_kernel<D, true, 1><<<grid, dim3(threads), 0, st>>>(a);
    else if (rpl == 1)
        append_paged_kernel<D, false, 1><<<grid, dim3(threads), 0, st>>>(a);
    else
        append_paged_kernel<D, false, 2><<<grid, dim3(threads), 0, st>>>(a);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_kv_append_paged(int head_dim, const PagedAppendArgs& a, hipStream_t st) {
    return head_dim == 64 ? append_paged<64>(a, st) : head_dim == 128 ? append_paged<128>(a, st) : append_paged<256>(a, st);
}

hipError_t launch_kv_read_paged(int head_dim, const PagedReadArgs& a, hipStream_t st) {
    const size_t pieces = (size_t)a.rows * a.c.kv_heads * (head_dim / 16);
    const dim3 grid((unsigned)((pieces + 255) / 256));
    if (head_dim == 64)
        read_paged_kernel<64><<<grid, dim3(256), 0, st>>>(a);
    else if (head_dim == 128)
        read_paged_kernel<128><<<grid, dim3(256), 0, st>>>(a);
    else
        read_paged_kernel<256><<<grid, dim3(256), 0, st>>>(a);
    return hipGetLastError();
}

}  // namespace cactus_hip
