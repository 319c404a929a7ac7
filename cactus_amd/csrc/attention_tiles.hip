// Attention of many query rows (include/cactus_hip_paged.h): packed FP16 prompts, and prompt chunks over the paged INT8
// cache.  Bound: the matrix cores, the softmax's vector instructions and the LDS reads together, none of them alone: of the
// 4800 cycles that two waves of a SIMD take for a key tile each (D = 128, in-kernel stamps) the matrix cores work 2050.  Over
// a whole launch (prompt of 4096, counters) they are busy 33% of the cycles, vector instructions 31%, both at once 9%.
//
// A workgroup is four waves on 128 consecutive rows (64 at head_dim 256) of one (sequence, kv head); a row is (token, query head
// of the group), so a key tile in LDS serves all query heads of its kv head.  A wave owns 32 rows (16) and computes everything
// transposed, a lane owning a row (lane % 32):
//   S^T = K Q^T   v_mfma_f32_32x32x16_f16, K rows from LDS, the wave's Q in registers for the whole kernel
//   O^T = V^T P^T V^T through the transposing LDS read (ds_read_b64_tr_b16); P is the lane's own scores, in the key order the
//                 first product left them in (the contraction order is free)
// so the softmax's maximum and sum are in-lane work plus one exchange with lane ^ 32, and weights never move.  The rest is the
// online softmax in base 2; (l, O) move to a new maximum only when it has grown by more than 2^LAG.
// Key tiles (64 keys, 32 at head_dim 256) are double-buffered: the next one's loads go out between the products of the scores (a
// burst of them holds every wave up) and it is stored to the other buffer behind the output's products, one barrier per tile.
// Loads past a sequence's last row are cut off by the buffer's length and give zeros, so no tile needs a branch.  16-byte chunks
// of a row are swizzled so that neither the row reads of K (16 rows, one chunk) nor the transposed reads of V (4 rows, 4 chunks)
// meet on a bank.
// INT8 pages become halves on the way into LDS: keys as the subnormal (b + 128) 2^-24 (one v_perm per two; the offset leaves
// with the score's fma), values as b 2^-9.  Page scales enter as in attention_paged.hip.
// Weights are rounded to binary16 (2^-11 of each, averaged over the keys that count, down to 2^-25 of the largest: LIFT); everything
// else is fp32.
//
// Measured: one prompt of 4096 tokens, 16 heads over 8, D = 128: 84 us, 815 TFLOP/s (a large FP16 matrix product reaches
// 1139 to 1334).  Prompts of 4001 to 8190 tokens, 4 heads over 1, D = 256, window 508: 88 us, 480.  24 prompts of 17 to 300 tokens,
// D = 64: 18.0 us.  Three chunks of 131 to 256 tokens over 4000 cached ones: 44 us, 8 of them the join's.
// Slower were: values stored transposed, one 16-byte read for two transposing 8-byte ones (99 and 60 us instead of 90 and 55 then:
// turning them takes 8-byte loads, twice as many); two groups of waves half a tile apart instead of in step (101 instead of 97).
#include "paged.hip.h"

#include <math.h>

#include <type_traits>

namespace cactus_hip {

namespace {

constexpr float LOG2E = 1.4426950408889634f;
// rows of a wave: 32 (v_mfma_f32_32x32x16_f16), at head_dim 256 16 (v_mfma_f32_16x16x32_f16): 32 rows' output and queries alone
// are 192 registers there, which leaves one wave per SIMD and every latency in the open
constexpr int wave_rows(int D) { return D == 256 ? 16 : 32; }
constexpr int tile_rows(int D) { return 4 * wave_rows(D); }
// products that the LDS reads run ahead of (3 measures the same, 6 up to 1% slower, 2 up to 4%)
constexpr int READ_AHEAD = 4;

typedef float v16f __attribute__((ext_vector_type(16)));
typedef float v2f __attribute__((ext_vector_type(2)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef short v4s __attribute__((ext_vector_type(4)));
typedef short v8s __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) v4s* lds_v4s;

template <int RW>
struct Product;
template <>
struct Product<32> {
    typedef v16f Acc;
    static __device__ __forceinline__ Acc mul(v8h x, v8h y, Acc c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(x, y, c, 0, 0, 0); }
};
template <>
struct Product<16> {
    typedef v4f Acc;
    static __device__ __forceinline__ Acc mul(v8h x, v8h y, Acc c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(x, y, c, 0, 0, 0); }
};

// lanes n, n + RW, .. combine a value
__device__ __forceinline__ float pair_max(float x) {
    const unsigned u = __float_as_uint(x);
    const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float pair_sum(float x) {
    const unsigned u = __float_as_uint(x);
    const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

__device__ __forceinline__ float half_max(float x) {
    const unsigned u = __float_as_uint(x);
    const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float half_sum(float x) {
    const unsigned u = __float_as_uint(x);
    const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
template <int RW>
__device__ __forceinline__ float row_max(float x) { return pair_max(RW == 16 ? half_max(x) : x); }
template <int RW>
__device__ __forceinline__ float row_sum(float x) { return pair_sum(RW == 16 ? half_sum(x) : x); }

// 16-byte chunk at which chunk c of a row lies in LDS
template <int D>
__device__ __forceinline__ int k_chunk(int row, int c) { return D == 64 ? c ^ ((row >> 1) & 7) : c ^ (row & 15); }
template <int D>
__device__ __forceinline__ int v_chunk(int row, int c) {
    return D == 64 ? c ^ ((row & 2) << 1) : D == 128 ? c ^ ((row & 3) << 2) : c ^ ((row & 7) << 1);
}

// four bytes, each ^ 0x80, as halves (b + 128) 2^-24
__device__ __forceinline__ void offset_halves(uint32_t x, uint32_t& lo, uint32_t& hi) {
    lo = __builtin_amdgcn_perm(0u, x, 0x0c010c00u);
    hi = __builtin_amdgcn_perm(0u, x, 0x0c030c02u);
}
// (b + 128) 2^-24 -> b 2^-9
__device__ __forceinline__ uint32_t centred(uint32_t u) {
    const _Float16 up = (_Float16)32768.0f, down = (_Float16)-0.25f;
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(__builtin_bit_cast(v2h, u), v2h{up, up}, v2h{down, down}));
}

// One key tile on its way from memory to LDS: 16-byte pieces, and (paged) the scales of its 16-key groups
template <int D, bool PAGED>
struct TileLoad {
    static constexpr int BK = D == 256 ? 32 : 64;
    static constexpr int PIECES = BK * D * (PAGED ? 1 : 2) / 16 / 256;      // per thread and operand
    v4i k[PIECES], v[PIECES];
    float scale;         // lane 2 g + (0 key, 1 value): the scale of 16-key group g, and its page
    int page;
};

// The slot of a workgroup.  A causal tile's work grows with its position, so late slots go first and the light ones fill the gaps.
// Workgroups go round the 8 XCDs, and so do the kv heads: with 8 of them a head's rows stay in one L2.  With fewer, ranks are
// dealt to the XCDs that share a head 8 neighbours at a time, because neighbours read the same keys (windowed prompts of one
// kv head 121 -> 103 us; 4 to 32 neighbours measure the same).
__device__ __forceinline__ int slot_of(int rank, int slots, int kv_heads) {
    constexpr int NEIGHBOURS = 8;
    const int share = kv_heads % 8 == 0 ? 1 : kv_heads % 4 == 0 ? 2 : kv_heads % 2 == 0 ? 4 : 8, block = share * NEIGHBOURS;
    const int base = rank / block * block, in = rank - base;
    if (share > 1 && base + block <= slots) rank = base + in % share * NEIGHBOURS + in / share;
    return slots - 1 - rank;
}

// Which tile of whose rows a workgroup takes, and how many splits its keys have.
//
// How many row tiles a batch has depends on lengths that only the device knows.  For up to COUNTED sequences a wave counts them, a
// lane for every 64th part of the batch, and numbers them without gaps.  As many workgroups as the registers hold (resident) fill the
// chip, and a few more cost a second round (three chunks with 80 row tiles x heads, D = 128, take 47.4 us in 6 splits = 480
// workgroups, 50.2 in 5 and 62 in 7; at D = 64 768 take 54 us and 512 60, at 256 103 and 86), so the keys get the largest number of
// splits that stays within them.  Above, slots lie as slot_begin has them, and there are more than the chip holds at once whatever the
// lengths: keys are not split.
constexpr int resident(int D) { return D == 64 ? 768 : 512; }       // three waves per SIMD, or two
constexpr int COUNTED = 1024;
struct Place {
    int b, tile, split, splits, id;      // id: of the (tile, head) pair; tile < 0: nothing to do
};
// sum over lanes 0 .. this one
__device__ __forceinline__ int sum_upto(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, true);       // row_shr:1, 2, 4, 8
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, true);       // row_bcast:15 into rows 1 and 3
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, true);       // row_bcast:31 into rows 2 and 3
    return v;
}
template <int D, bool JOIN>
__device__ __forceinline__ Place place_of(const PagedAttnArgs& a, int block, int most, int slots, int group) {
    constexpr int size = tile_rows(D);
    Place p;
    p.tile = -1;
    if (a.batch > COUNTED) {
        p.splits = 1;
        p.id = block;
        p.split = 0;
        const auto begin = [&](int i) { return slot_begin(a.cu, i, a.tokens, group, size, 1); };
        const int slot = slot_of(p.id / a.kv_heads, slots, a.kv_heads);
        p.b = owner_of(slot, a.batch, begin);
        if (rows_of(a.cu, p.b, a.tokens).count * group > a.min_rows) p.tile = slot - begin(p.b);
        return p;
    }
    const int lane = threadIdx.x & 63, per = (a.batch + 63) >> 6;
    const auto tiles_of = [&](int b) {
        const int n = b < a.batch ? rows_of(a.cu, b, a.tokens).count * group : 0;
        return n > a.min_rows ? (n + size - 1) / size : 0;
    };
    int count = 0;
    for (int i = 0; i < per; i++) count += tiles_of(lane * per + i);
    count = min(count, 1 << 23);         // offsets that are none can count rows many times over: no sum of these passes an int
    const int upto = sum_upto(count), tiles = __builtin_amdgcn_readlane(upto, 63), pairs = min(tiles, resident(D)) * a.kv_heads;
    p.splits = min(max(resident(D) / max(pairs, 1), 1), most);
    p.id = JOIN ? block : block / p.splits;
    p.split = JOIN ? 0 : block % p.splits;
    const int rank = p.id / a.kv_heads;
    if (rank >= tiles) return p;
    const int slot = slot_of(rank, tiles, a.kv_heads);
    const int part = min(__popcll(__ballot(upto <= slot)), 63);
    p.b = part * per;
    p.tile = slot - __builtin_amdgcn_readlane(upto - count, part);
    if (per > 1) {                       // the sequence in the lane's part
        const int c = lane < per ? tiles_of(p.b + lane) : 0, u = sum_upto(c), i = min(__popcll(__ballot(u <= p.tile)), per - 1);
        p.tile -= __builtin_amdgcn_readlane(u - c, i);
        p.b += i;
    }
    p.b = min(p.b, a.batch - 1);
    return p;
}

// NG: groups of four waves.  Two groups take every second key tile each and join their (maximum, sum, output) at the end.
template <int D, bool PAGED, int NG>
__global__ __launch_bounds__(256 * NG) __attribute__((amdgpu_waves_per_eu(2)))
void attention_tile_kernel(const PagedAttnArgs a, const int most_splits, const int slots) {
    using Load = TileLoad<D, PAGED>;
    // RW rows a wave, lane n + RW h.  An accumulator holds AR values of a lane, quads of four neighbouring keys (dims): key (dim)
    // QUAD (r / 4) + 4 h + r % 4 of a tile of RW.  Two quads make the eight contracted keys of a lane: FRAGS fragments of FK keys.
    constexpr int RW = wave_rows(D), LG = 64 / RW, AR = RW * RW / 64, QUAD = 4 * LG, TILE_ROWS = tile_rows(D);
    constexpr int BK = Load::BK, KT = BK / RW, GROUPS = BK / 16, FK = 8 * LG, FRAGS = BK / FK, NST = D / (8 * LG), NDT = D / RW, ROW = D * 2;
    typedef typename Product<RW>::Acc Acc;
    __shared__ __attribute__((aligned(1024))) unsigned char s_kv[NG][4][BK * ROW];      // of a group: K, K, V, V
    // INT8, per 16-key group: factor of the score, (unused), log2 of the value scale, its reciprocal.  A group without a page has the
    // logarithm -inf, which is all the masking it needs.  The factor is above zero, so that a masked score stays -inf.
    __shared__ __attribute__((aligned(16))) float s_scales[NG][2][GROUPS][4];
    // FP16 rows: a value that is not finite must not reach a row that does not see its key, and 0 * inf is NaN.  So tiles that some
    // row does not see whole get zeros in their place (s_odd: there were any), and where they belong is looked up at the end.
    // s_marks: +inf, -inf, NaN bits of every row's dims
    __shared__ int s_odd;
    __shared__ uint32_t s_marks[PAGED ? 1 : 3][PAGED ? 1 : TILE_ROWS][D / 32];

    const int tid = threadIdx.x & 255, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);     // in the group
    const int grp = NG == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x >> 8);
    const int n = lane % RW, h = lane / RW;
    float(*const s_scale)[GROUPS][4] = s_scales[grp];
    const int group = a.q_heads / a.kv_heads;
    const Place at = place_of<D, false>(a, blockIdx.x, most_splits, slots, group);
    const int tile = at.tile, b = at.b, splits = PAGED ? at.splits : 1, split = PAGED ? at.split : 0, head = at.id % a.kv_heads;
    if (tile < 0) return;
    const Rows rows = rows_of(a.cu, b, a.tokens);
    const int R = min(rows.count * group - tile * TILE_ROWS, TILE_ROWS);
    if (R <= 0) return;
    int context = rows.count;
    if (PAGED) context = context_of(a, b);
    const int pos0 = context - rows.count;                    // position of the sequence's first row
    const auto pos_of = [&](int r) { return pos0 + (tile * TILE_ROWS + r) / group; };
    const int row = min(wave * RW + n, R - 1);                       // lanes past the last row repeat it
    const int orow = tile * TILE_ROWS + row, token = rows.first + orow / group, qh = head * group + orow % group;
    const int pos = pos0 + orow / group;
    const int wpos_first = pos_of(min(wave * RW, R - 1)), wpos_last = pos_of(min(wave * RW + RW - 1, R - 1));
    const int last = pos_of(R - 1);
    const TilePlan plan = plan_tiles(pos_of(0), last, a.window, a.sink, BK);
    const int per = (plan.tiles + splits - 1) / splits, u0 = split * per, u1 = min(u0 + per, plan.tiles);

    // Q^T; a negative scale is moved into Q, so that the largest score is the largest product
    v8h q[NST];
    float bias = 0.0f;
    {
        const uint16_t* qr = a.q + (size_t)token * a.q_stride + (size_t)qh * D;
        const uint32_t flip = a.scale < 0.0f ? 0x80008000u : 0u;
#pragma unroll
        for (int s = 0; s < NST; s++) {
            v4i x = *reinterpret_cast<const v4i*>(qr + 8 * LG * s + 8 * h);
#pragma unroll
            for (int e = 0; e < 4; e++) x[e] ^= (int)flip;
            q[s] = __builtin_bit_cast(v8h, x);
            if (PAGED)
#pragma unroll
                for (int e = 0; e < 8; e++) bias += (float)q[s][e];
        }
        if (PAGED) bias = row_sum<RW>(bias) * (-128.0f / 16777216.0f);
    }
    const float c0 = fabsf(a.scale) * LOG2E;

    // tile u of the plan starts at key BK * u (the sinks) or BK * (u + jump)
    const int jump = plan.first - plan.sinks;
    const auto key_of = [&](int u) { return (u < plan.sinks ? u : u + jump) * BK; };
    // What of the plan the wave looks at.  Of the tiles behind the sinks: [seen_lo, seen_hi) hold keys some row sees, [whole_lo,
    // whole_hi) are seen whole by all its rows.  Of the sinks: all are looked at, the first whole_sinks are seen whole.
    const auto up = [](int x) { return x <= 0 ? 0 : (x + BK - 1) / BK; };
    const int seen_hi = wpos_last < 0 ? 0 : wpos_last / BK + 1 - jump;
    const int whole_hi = wpos_first < 0 ? -jump : (wpos_first + 1) / BK - jump;
    int seen_lo = plan.sinks, whole_lo = plan.sinks, whole_sinks = 0;
    if (a.window) {
        if (a.sink <= plan.first * BK) seen_lo = max(seen_lo, up(wpos_first - a.window - BK + 1) - jump);
        whole_lo = max(whole_lo, up(wpos_last - a.window) - jump);
        whole_sinks = min(plan.sinks, a.sink / BK);
    }
    // page of the 16 keys from `key0`, or -1
    const auto page_at = [&](int key0) { return key0 <= last ? page_of(a.c, b, key0 >> a.c.page_shift) : -1; };
    int pages[Load::PIECES] = {}, my_page = -1;                      // of the tile after the next
    const auto look_up = [&](int u) {
        if constexpr (PAGED) {
            if (u >= u1) return;
            const int key = key_of(u);
#pragma unroll
            for (int i = 0; i < Load::PIECES; i++) {
                const int r = (i * 256 + wave * 64) / (D / 16);      // the wave's rows lie in one 16-key group
                pages[i] = page_at(key + (r & ~15));
            }
            my_page = page_at(key + 16 * (tid % (2 * GROUPS) >> 1));
        }
    };
    // FP16: byte offsets of the lane's pieces in a tile (strides are below 2^24)
    const uint32_t k_next = 512 / (D / 8) * a.k_stride, v_next = 512 / (D / 8) * a.v_stride;
    const uint32_t k_lane = 2 * (tid / (D / 8) * (uint32_t)a.k_stride + tid % (D / 8) * 8);
    const uint32_t v_lane = 2 * (tid / (D / 8) * (uint32_t)a.v_stride + tid % (D / 8) * 8);
    const auto fetch = [&](Load& t, int u) {
        const int key = key_of(u);
        if constexpr (PAGED) {
#pragma unroll
            for (int i = 0; i < Load::PIECES; i++) {
                const int p = i * 256 + tid, r = p / (D / 16), d = p % (D / 16) * 16, page = __builtin_amdgcn_readfirstlane(pages[i]);
                const int at = (key + r) & ((1 << a.c.page_shift) - 1);
                const size_t from = ((((size_t)max(page, 0) * a.kv_heads + head) << a.c.page_shift) + at) * D + d;
                t.k[i] = *reinterpret_cast<const v4i*>(a.c.k + from);
                t.v[i] = *reinterpret_cast<const v4i*>(a.c.v + from);
            }
            t.scale = (tid & 1 ? a.c.vs : a.c.ks)[(size_t)max(my_page, 0) * a.kv_heads + head];
            t.page = my_page;
        } else {
            // a tile's base is the same for all lanes; rows past the last key read as zero
            const int most = u < u1 ? min(last - key, BK - 1) : -1;
            const auto rows_from = [&](const uint16_t* x, size_t stride) {
                return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(x) + (size_t)(rows.first + key) * stride + (size_t)head * D, 0,
                                                         most < 0 ? 0 : 2 * (most * (int)stride + D), 0x00027000);
            };
            const auto kb = rows_from(a.k, a.k_stride), vb = rows_from(a.v, a.v_stride);
#pragma unroll
            for (int i = 0; i < Load::PIECES; i++)
                t.k[i] = __builtin_bit_cast(v4i, __builtin_amdgcn_raw_buffer_load_b128(kb, k_lane + i * k_next, 0, 0));
#pragma unroll
            for (int i = 0; i < Load::PIECES; i++)
                t.v[i] = __builtin_bit_cast(v4i, __builtin_amdgcn_raw_buffer_load_b128(vb, v_lane + i * v_next, 0, 0));
        }
    };
    // the tiles that every row of the workgroup sees whole
    const int all_whole_hi = pos_of(0) < 0 ? -jump : (pos_of(0) + 1) / BK - jump;
    const int all_whole_lo = a.window ? max(plan.sinks, up(last - a.window) - jump) : 0;
    // where the lane's pieces go: piece i lies a fixed number of rows below piece 0, at the same place of the swizzle (a chunk pair
    // of INT8 starts at an even chunk, so its second one is the other of the pair)
    constexpr int CHUNKS = PAGED ? D / 16 : D / 8, STEP_BYTES = 256 / CHUNKS * ROW;
    const int to_row = tid / CHUNKS, to_chunk = tid % CHUNKS * (PAGED ? 2 : 1);
    const uint32_t to_base = grp * 4 * BK * ROW + to_row * ROW;
    const uint32_t k_to = to_base + k_chunk<D>(to_row, to_chunk) * 16, v_to = to_base + v_chunk<D>(to_row, to_chunk) * 16;
    const auto stash = [&](auto buf, Load& t, int u) __attribute__((always_inline)) {
        if constexpr (!PAGED) {
            if (u >= all_whole_hi || (u < all_whole_lo && u >= whole_sinks)) {
                uint32_t odd = 0;
#pragma unroll
                for (int i = 0; i < Load::PIECES; i++)
#pragma unroll
                    for (int e = 0; e < 4; e++) odd |= (((uint32_t)t.v[i][e] & 0x7fff7fffu) + 0x04000400u) & 0x80008000u;
                if (odd) {
                    s_odd = 1;
#pragma unroll
                    for (int i = 0; i < Load::PIECES; i++)
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            const uint32_t x = (uint32_t)t.v[i][e];
                            t.v[i][e] = (int)(((x & 0x7c00u) == 0x7c00u ? 0u : x & 0xffffu) |
                                              ((x & 0x7c000000u) == 0x7c000000u ? 0u : x & 0xffff0000u));
                        }
                }
            }
        }
#pragma unroll
        for (int i = 0; i < Load::PIECES; i++) {
            if constexpr (PAGED) {
#pragma unroll
                for (int w = 0; w < 2; w++) {
                    v4i x, y;
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        uint32_t lo, hi;
                        offset_halves((uint32_t)t.k[i][2 * w + e] ^ 0x80808080u, lo, hi);
                        x[2 * e] = (int)lo;
                        x[2 * e + 1] = (int)hi;
                        offset_halves((uint32_t)t.v[i][2 * w + e] ^ 0x80808080u, lo, hi);
                        y[2 * e] = (int)centred(lo);
                        y[2 * e + 1] = (int)centred(hi);
                    }
                    *reinterpret_cast<v4i*>(&s_kv[0][buf][i * STEP_BYTES] + (k_to ^ (16 * w))) = x;
                    *reinterpret_cast<v4i*>(&s_kv[0][2 + buf][i * STEP_BYTES] + (v_to ^ (16 * w))) = y;
                }
            } else {
                const uint32_t turn = D == 256 && (i & 1) ? 8 * 16 : 0;      // 8 rows on: the other half of K's swizzle
                *reinterpret_cast<v4i*>(&s_kv[0][buf][i * STEP_BYTES] + (k_to ^ turn)) = t.k[i];
                *reinterpret_cast<v4i*>(&s_kv[0][2 + buf][i * STEP_BYTES] + v_to) = t.v[i];
            }
        }
        if (PAGED && tid < 2 * GROUPS) {         // worked out once here, not by every wave
            const float x = t.page < 0 ? 0.0f : page_scale(t.scale), v = fmaxf(x, 1e-20f);
            const v2f two = tid & 1 ? v2f{t.page < 0 ? -INFINITY : __log2f(v), t.page < 0 ? 0.0f : __builtin_amdgcn_rcpf(v)}
                                    : v2f{fmaxf(x * c0 * 16777216.0f, 1e-30f), 0.0f};
            *reinterpret_cast<v2f*>(&s_scale[buf][tid >> 1][2 * (tid & 1)]) = two;
        }
    };

    float m = -1e30f, l = 0.0f;
    Acc o[NDT];
#pragma unroll
    for (int i = 0; i < NDT; i++)
#pragma unroll
        for (int r = 0; r < AR; r++) o[i][r] = 0.0f;

    // Lane addresses in a buffer; which buffer, tile or fragment is an immediate offset.  K: row n of RW, chunk LG s + h.  V: key
    // 4 h + tq of QUAD, dims 4 tp .. of 16 (16 gi on where a tile has 32).
    const int tq = (lane >> 2) & 3, tp = lane & 3, gi = RW == 32 ? (lane >> 4) & 1 : 0;
    uint32_t k_at[NST], v_at[NDT];
#pragma unroll
    for (int i = 0; i < NST; i++) k_at[i] = grp * 4 * BK * ROW + n * ROW + k_chunk<D>(n, LG * i + h) * 16;
#pragma unroll
    for (int i = 0; i < NDT; i++)
        v_at[i] = grp * 4 * BK * ROW + (4 * h + tq) * ROW + v_chunk<D>(4 * h + tq, RW / 8 * i + 2 * gi + (tp >> 1)) * 16 + (tp & 1) * 8;
    // the eight keys of fragment f that a lane holds for its dim of dim tile i
    const auto value_frag = [&](auto buf, int i, int f) __attribute__((always_inline)) {
        const unsigned char* at = &s_kv[0][2 + buf][FK * f * ROW] + v_at[i];
        const v4s v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s)(at));
        const v4s v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s)(at + QUAD * ROW));
        return __builtin_bit_cast(v8h, v8s{v0[0], v0[1], v0[2], v0[3], v1[0], v1[1], v1[2], v1[3]});
    };
    const auto compute = [&](auto buf, Load& t, int u, bool whole) __attribute__((always_inline)) {
        const int key = key_of(u);
        fetch(t, u + NG);
        Acc s[KT];
#pragma unroll
        for (int j = 0; j < KT; j++)
#pragma unroll
            for (int r = 0; r < AR; r++) s[j][r] = 0.0f;
#pragma unroll
        for (int st = 0; st < NST; st++)
#pragma unroll
            for (int t = 0; t < KT; t++) {
                const v8h kf = *reinterpret_cast<const v8h*>(&s_kv[0][buf][RW * t * ROW] + k_at[st]);
                s[t] = Product<RW>::mul(kf, q[st], s[t]);
            }
        // LDS reads run READ_AHEAD ahead of the products that use them
        __builtin_amdgcn_sched_group_barrier(0x100, READ_AHEAD, 0);
#pragma unroll
        for (int i = 0; i < KT * NST - READ_AHEAD; i++) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
            if (i < 2 * Load::PIECES) __builtin_amdgcn_sched_group_barrier(0x20, 1, 0);
        }
        __builtin_amdgcn_sched_group_barrier(0x008, READ_AHEAD, 0);
        const auto group_of = [](int t, int r) { return (RW * t + QUAD * (r >> 2)) / 16; };      // 16-key group of a score
        float inv_vs[GROUPS], up[GROUPS], add[GROUPS];       // INT8: a weight's exponent is score * up + add of its group
        if constexpr (PAGED) {
#pragma unroll
            for (int g = 0; g < GROUPS; g++) {
                const v4f x = *reinterpret_cast<const v4f*>(s_scale[buf][g]);
                up[g] = x[0];
                add[g] = fmaf(x[0], bias, x[2]);
                inv_vs[g] = x[3];
            }
        }
        if (!whole) {
            // a score's key against the row's own key, its first window key and the sinks
            const int to = pos - key - 4 * h;
            if (u >= whole_hi) {
#pragma unroll
                for (int t = 0; t < KT; t++)
#pragma unroll
                    for (int r = 0; r < AR; r++) s[t][r] = RW * t + QUAD * (r >> 2) + (r & 3) <= to ? s[t][r] : -INFINITY;
            }
            if (u < whole_lo) {
                const int from = to - a.window, sinks = a.sink - key - 4 * h;
#pragma unroll
                for (int t = 0; t < KT; t++)
#pragma unroll
                    for (int r = 0; r < AR; r++) {
                        const int j = RW * t + QUAD * (r >> 2) + (r & 3);
                        s[t][r] = j >= from || j < sinks ? s[t][r] : -INFINITY;
                    }
            }
        }
        float top = -INFINITY;
        if constexpr (PAGED) {
            float most[GROUPS];
#pragma unroll
            for (int g = 0; g < GROUPS; g++) most[g] = -INFINITY;
#pragma unroll
            for (int t = 0; t < KT; t++)
#pragma unroll
                for (int r = 0; r < AR; r += 2) most[group_of(t, r)] = fmaxf(fmaxf(s[t][r], s[t][r + 1]), most[group_of(t, r)]);
#pragma unroll
            for (int g = 0; g < GROUPS; g++) top = fmaxf(top, fmaf(most[g], up[g], add[g]));
            top = row_max<RW>(top);
        } else {
#pragma unroll
            for (int t = 0; t < KT; t++)
#pragma unroll
                for (int r = 0; r < AR; r += 2) top = fmaxf(fmaxf(s[t][r], s[t][r + 1]), top);
            top = row_max<RW>(top) * c0;
        }
        if (__any(top > m + LAG)) {
            const float to = fmaxf(m, top), f = __builtin_amdgcn_exp2f(m - to);
            m = to;
            l *= f;
#pragma unroll
            for (int i = 0; i < NDT; i++)
#pragma unroll
                for (int r = 0; r < AR; r++) o[i][r] *= f;
        }
        const float lift = LIFT - m;
        if constexpr (PAGED) {
#pragma unroll
            for (int g = 0; g < GROUPS; g++) add[g] += lift;
        }
        // The wave that feeds the matrix cores goes before the one that is elsewhere in its tile: 2% at D = 128, nothing at 256; at
        // 64, where the products are short against the rest, it costs 4%.
        if constexpr (D > 64) __builtin_amdgcn_s_setprio(1);
        v8h p[FRAGS];
#pragma unroll
        for (int f = 0; f < FRAGS; f++) {
#pragma unroll
            for (int half = 0; half < 2; half++) {
                const int quad = 2 * f + half, t = quad / (AR / 4), r0 = quad % (AR / 4) * 4;
                float w[4];
#pragma unroll
                for (int e = 0; e < 4; e++) w[e] = __builtin_amdgcn_exp2f(PAGED ? fmaf(s[t][r0 + e], up[group_of(t, r0)], add[group_of(t, r0)]) : fmaf(s[t][r0 + e], c0, lift));
                const float sum = (w[0] + w[1]) + (w[2] + w[3]);
                l = PAGED ? fmaf(sum, inv_vs[group_of(t, r0)], l) : l + sum;
#pragma unroll
                for (int e = 0; e < 4; e += 2) {
                    const v2h two = __builtin_convertvector(v2f{w[e], w[e + 1]}, v2h);
                    p[f][4 * half + e] = two[0];
                    p[f][4 * half + e + 1] = two[1];
                }
            }
#pragma unroll
            for (int i = 0; i < NDT; i++) o[i] = Product<RW>::mul(value_frag(buf, i, f), p[f], o[i]);
        }
        // The first values are read while the first weights are computed; then every product is followed by the reads of one
        // READ_AHEAD further on and a share of the next fragment's exponentials, which run beside the matrix cores.
        constexpr int PER_FRAG = 28, SHARE = (PER_FRAG + NDT - 1) / NDT, PRODUCTS = FRAGS * NDT;
        __builtin_amdgcn_sched_group_barrier(0x100, 2 * READ_AHEAD, 1);
        __builtin_amdgcn_sched_group_barrier(0x402, PER_FRAG, 1);
#pragma unroll
        for (int i = 0; i < PRODUCTS; i++) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 1);
            if (i < PRODUCTS - READ_AHEAD) __builtin_amdgcn_sched_group_barrier(0x100, 2, 1);
            if (i < PRODUCTS - NDT) __builtin_amdgcn_sched_group_barrier(0x402, SHARE, 1);
        }
        if constexpr (D > 64) __builtin_amdgcn_s_setprio(0);
    };

    if (u0 < u1) {
        const std::integral_constant<int, 0> zero{};
        const std::integral_constant<int, 1> one{};
        Load t;
        // this group's tiles: first, first + NG, ..; every group takes part in every barrier
        const int first = u0 + grp;
        look_up(first);
        if (first < u1) fetch(t, first);
        look_up(first + NG);
        if constexpr (!PAGED) {
            if (threadIdx.x == 0) s_odd = 0;
            __syncthreads();
        }
        if (first < u1) stash(zero, t, first);
        __syncthreads();
        const auto step = [&](auto buf, auto other, int u) __attribute__((always_inline)) {
            const bool seen = u < seen_hi && (u >= seen_lo || u < plan.sinks) && (NG == 1 || u < u1);
            if (!seen && u + NG < u1) fetch(t, u + NG);
            if (seen) {
                compute(buf, t, u, (u >= whole_lo && u < whole_hi) || u < whole_sinks);
            }
            look_up(u + 2 * NG);
            if (u + NG < u1) stash(other, t, u + NG);
            __syncthreads();
        };
        for (int u = u0; u < u1; u += 2 * NG) {
            step(zero, one, u + grp);
            if (u + NG < u1) step(one, zero, u + NG + grp);
        }
    }

    l = row_sum<RW>(l);
    if constexpr (NG == 2) {
        // group 1 hands its state over through the tile buffers, 16 bytes a lane and register quad
        float* state = reinterpret_cast<float*>(&s_kv[0][0][0]) + (wave * NDT * (AR / 4) * 64 + lane) * 4;
        __shared__ float s_ml[TILE_ROWS][2];
        if (grp == 1) {
#pragma unroll
            for (int i = 0; i < NDT; i++)
#pragma unroll
                for (int r = 0; r < AR; r += 4)
                    *reinterpret_cast<v4f*>(state + (AR * i + r) * 64) = v4f{o[i][r], o[i][r + 1], o[i][r + 2], o[i][r + 3]};
            if (h == 0) {
                s_ml[wave * RW + n][0] = m;
                s_ml[wave * RW + n][1] = l;
            }
        }
        __syncthreads();
        if (grp == 1) return;
        const float m1 = s_ml[wave * RW + n][0], l1 = s_ml[wave * RW + n][1], to = fmaxf(m, m1);
        const float f0 = __builtin_amdgcn_exp2f(m - to), f1 = __builtin_amdgcn_exp2f(m1 - to);
        m = to;
        l = l * f0 + l1 * f1;
#pragma unroll
        for (int i = 0; i < NDT; i++)
#pragma unroll
            for (int r = 0; r < AR; r += 4) {
                const v4f x = *reinterpret_cast<const v4f*>(state + (AR * i + r) * 64);
#pragma unroll
                for (int e = 0; e < 4; e++) o[i][r + e] = fmaf(x[e], f1, o[i][r + e] * f0);
            }
    }
    if constexpr (!PAGED) {
        // Values that are not finite, once more.  In tiles that all rows see whole they have gone through the products: such a dim is
        // not finite, but what it is depends on roundings (weights of 0 in binary16, rescaling by 0 make NaN of an infinity).  In the
        // others they were left out.  If there are any of either kind, the wave looks through the values that its rows see, 4 KB at a
        // time, and every row that sees one has it in that dim, whatever it weighs.
        float zero = 0.0f;
#pragma unroll
        for (int i = 0; i < NDT; i++)
#pragma unroll
            for (int r = 0; r < AR; r++) zero = fmaf(o[i][r], 0.0f, zero);
        if (__any(zero != zero || s_odd != 0)) {
            constexpr int CHUNKS_ROW = D / 8, KEYS = 64 / CHUNKS_ROW, LOADS = 4, KIND = TILE_ROWS * (D / 32);
            uint32_t* const marks = &s_marks[0][wave * RW][0];
#pragma unroll 1
            for (int i = lane; i < RW * (D / 32); i += 64)
                for (int kind = 0; kind < 3; kind++) marks[kind * KIND + i] = 0;
            const auto scan = [&](int from, int to) {
#pragma unroll 1
                for (int key0 = from; key0 < to; key0 += LOADS * KEYS) {
                    v4i x[LOADS];            // keys past the last are the last one again
#pragma unroll
                    for (int j = 0; j < LOADS; j++) {
                        const int key = min(key0 + j * KEYS + lane / CHUNKS_ROW, to - 1);
                        x[j] = *reinterpret_cast<const v4i*>(a.v + (size_t)(rows.first + key) * a.v_stride + (size_t)head * D + lane % CHUNKS_ROW * 8);
                    }
#pragma unroll
                    for (int j = 0; j < LOADS; j++) {
                        uint32_t odd = 0;
#pragma unroll
                        for (int e = 0; e < 4; e++) odd |= (((uint32_t)x[j][e] & 0x7fff7fffu) + 0x04000400u) & 0x80008000u;
                        for (unsigned long long who = __ballot(odd != 0); who; who &= who - 1) {
                            const int src = __builtin_ctzll(who), key = min(key0 + j * KEYS + src / CHUNKS_ROW, to - 1), d0 = src % CHUNKS_ROW * 8;
                            const bool sees = key <= pos && (!a.window || pos - key <= a.window || key < a.sink);
#pragma unroll
                            for (int e = 0; e < 8; e++) {
                                const uint32_t y = ((uint32_t)__builtin_amdgcn_readlane(x[j][e >> 1], src) >> (16 * (e & 1))) & 0xffffu;
                                if ((y & 0x7c00u) != 0x7c00u) continue;
                                const int kind = y == 0x7c00u ? 0 : y == 0xfc00u ? 1 : 2;
                                if (sees && h == 0) atomicOr(&marks[kind * KIND + n * (D / 32) + ((d0 + e) >> 5)], 1u << ((d0 + e) & 31));
                            }
                        }
                    }
                }
            };
            const int low = a.window ? max(wpos_first - a.window, 0) : 0;
            scan(0, min(a.window ? a.sink : 0, low));
            scan(low, wpos_last + 1);
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");      // the rows' marks are the wave's own
#pragma unroll
            for (int i = 0; i < NDT; i++)
#pragma unroll
                for (int r = 0; r < AR; r++) {
                    const int d = RW * i + QUAD * (r >> 2) + (r & 3);           // and 4 h, which stays inside the word
                    const uint32_t* at = marks + n * (D / 32) + (d >> 5);
                    const int bit = (d & 31) + 4 * h;
                    const bool plus = (at[0] >> bit) & 1, minus = (at[KIND] >> bit) & 1, none = (at[2 * KIND] >> bit) & 1;
                    o[i][r] = none || (plus && minus) ? NAN : plus ? INFINITY : minus ? -INFINITY : o[i][r];
                }
        }
    }
    if (wave * RW + n >= R) return;
    const float unit = PAGED ? 512.0f : 1.0f;
    if (splits > 1) {
        float* record = a.work + (size_t)blockIdx.x * TILE_ROWS * (D + 2);
        if (h == 0) {
            record[2 * row] = m;
            record[2 * row + 1] = l;
        }
        float* out = record + 2 * TILE_ROWS + (size_t)row * D + 4 * h;
#pragma unroll
        for (int i = 0; i < NDT; i++)
#pragma unroll
            for (int r = 0; r < AR; r += 4) {
                v4f x;
#pragma unroll
                for (int e = 0; e < 4; e++) x[e] = o[i][r + e] * unit;
                *reinterpret_cast<v4f*>(out + RW * i + QUAD * (r >> 2)) = x;
            }
    } else {
        const float inv = l > 0.0f || l != l ? unit / l : 0.0f;
        uint16_t* out = a.out + ((size_t)token * a.q_heads + qh) * D + 4 * h;
#pragma unroll
        for (int i = 0; i < NDT; i++)
#pragma unroll
            for (int r = 0; r < AR; r += 4) {
                v4h x;
#pragma unroll
                for (int e = 0; e < 4; e++) x[e] = (_Float16)(o[i][r + e] * inv);
                *reinterpret_cast<v4h*>(out + RW * i + QUAD * (r >> 2)) = x;
            }
    }
}

// joins the splits of a tile's rows: a wave per row, lanes = dims
template <int D>
__global__ __launch_bounds__(256) void attention_tile_join_kernel(const PagedAttnArgs a, const int most_splits, const int slots) {
    constexpr int TILE_ROWS = tile_rows(D);
    const int lane = threadIdx.x & 63, row = blockIdx.y * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int group = a.q_heads / a.kv_heads;
    const Place at = place_of<D, true>(a, blockIdx.x, most_splits, slots, group);
    if (at.tile < 0 || at.splits == 1) return;       // one split: the tile kernel wrote the rows itself
    const int tile = at.tile, splits = at.splits, head = at.id % a.kv_heads;
    const Rows rows = rows_of(a.cu, at.b, a.tokens);
    const int orow = tile * TILE_ROWS + row;
    if (orow >= rows.count * group) return;
    constexpr size_t step = (size_t)TILE_ROWS * (D + 2);
    const float* rec = a.work + (size_t)at.id * splits * step;
    // Eight records at a time, all requested before the first is used: latency is what there is to hide.  Records that do not exist
    // are the last one again, with weight 0.
    constexpr int W = D / 64, AT_ONCE = 8;
    typedef float Dims __attribute__((ext_vector_type(W)));
    float m = -1e30f, l = 0.0f, o[W];
#pragma unroll
    for (int i = 0; i < W; i++) o[i] = 0.0f;
    for (int s0 = 0; s0 < splits; s0 += AT_ONCE) {
        v2f ml[AT_ONCE];
        Dims x[AT_ONCE];
#pragma unroll
        for (int s = 0; s < AT_ONCE; s++) {
            const float* from = rec + min(s0 + s, splits - 1) * step;
            ml[s] = *reinterpret_cast<const v2f*>(from + 2 * row);
            x[s] = *reinterpret_cast<const Dims*>(from + 2 * TILE_ROWS + (size_t)row * D + lane * W);
        }
        float to = m;
#pragma unroll
        for (int s = 0; s < AT_ONCE; s++) to = fmaxf(to, ml[s][0]);
        const float back = __builtin_amdgcn_exp2f(m - to);
        m = to;
        l *= back;
#pragma unroll
        for (int i = 0; i < W; i++) o[i] *= back;
#pragma unroll
        for (int s = 0; s < AT_ONCE; s++) {
            const float f = s0 + s < splits ? __builtin_amdgcn_exp2f(ml[s][0] - m) : 0.0f;
            l = fmaf(ml[s][1], f, l);
#pragma unroll
            for (int i = 0; i < W; i++) o[i] = fmaf(x[s][i], f, o[i]);
        }
    }
    const float inv = l > 0.0f || l != l ? 1.0f / l : 0.0f;
    uint16_t* out = a.out + ((size_t)(rows.first + orow / group) * a.q_heads + head * group + orow % group) * D + lane * W;
#pragma unroll
    for (int i = 0; i < W; i++) out[i] = f2h(o[i] * inv);
}

template <int D, bool PAGED>
hipError_t launch(const PagedAttnArgs& a, const TileShape& s, hipStream_t st) {
    constexpr int NG = D < 256 && !PAGED ? 2 : 1;            // the most groups that a launch may have
    if (s.groups == 2 && NG == 2)
        attention_tile_kernel<D, PAGED, NG><<<dim3((unsigned)s.blocks), dim3(256 * NG), 0, st>>>(a, s.splits, s.slots);
    else
        attention_tile_kernel<D, PAGED, 1><<<dim3((unsigned)s.blocks), dim3(256), 0, st>>>(a, s.splits, s.slots);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || s.splits == 1) return e;
    attention_tile_join_kernel<D><<<dim3((unsigned)s.joined, tile_rows(D) / 4), dim3(256), 0, st>>>(a, s.splits, s.slots);
    return hipGetLastError();
}

}  // namespace

// A tile kernel's launch: a slot per tile of a sequence's rows and kv head, and key splits where that leaves most of the chip
// idle, each of at least 128 keys, at head_dim 64, whose tiles are quick beside the join, 256 (256 rows on 344 keys, 16 heads over 8 of
// 128: 18.0 us with 128, 20.4 with 256, 22.7 with 512 at least; 4 heads over 1 of 256: 17, 23, 32; 4 x 100 rows on 900 keys, 32 heads
// over 8 of 64: 29.0, 29.5, 24.3, but 256 rows on 944 keys 26, 20, 25).  `beside` the step kernel, where most sequences and often
// all are not its, 512: the join is a launch for all of them (63 single tokens on 1000 keys 27.8 us, with 128 keys at least 34.0).
// FP16 prompts are not split; few row tiles of them get two groups of waves instead (one prompt of 4096 tokens 106 -> 95 us), which
// over pages cost more than two workgroups (50.4 against 53.2 us).
// Up to COUNTED sequences the kernel chooses the splits (place_of): more than one only while they are all resident, so that at
// most half as many row tiles x heads are joined.
TileShape tile_shape(size_t head_dim, bool paged, size_t batch, size_t tokens, size_t max_context, size_t q_heads, size_t kv_heads,
                     size_t window, size_t sink, bool beside) {
    TileShape s;
    const size_t rows = tokens * (q_heads / kv_heads), size = tile_rows((int)head_dim), least = (rows + size - 1) / size;
    s.slots = (int)(batch == 1 ? least : rows / size + batch);                        // slot_begin
    const size_t items = (size_t)s.slots * kv_heads;
    size_t keys = max_context;
    if (window && window + sink + size < keys) keys = window + sink + size;
    const size_t fill = resident((int)head_dim), most = keys / (beside ? 512 : head_dim == 64 ? 256 : 128);
    const size_t want = paged && batch <= (size_t)COUNTED ? fill / (least * kv_heads) : 1;
    s.splits = (int)(most < 1 || want < 1 ? 1 : most < want ? most : want);
    s.groups = !paged && head_dim < 256 && items <= 512 ? 2 : 1;
    s.blocks = s.splits > 1 && items < fill ? fill : items;
    s.records = s.splits > 1 ? fill : 0;
    s.joined = items < fill / 2 ? items : fill / 2;
    return s;
}
size_t tile_record_floats(size_t head_dim) { return tile_rows((int)head_dim) * (head_dim + 2); }

hipError_t launch_attention_tiles(int D, bool paged, const PagedAttnArgs& a, const TileShape& s, hipStream_t st) {
    if (paged) return D == 64 ? launch<64, true>(a, s, st) : D == 128 ? launch<128, true>(a, s, st) : launch<256, true>(a, s, st);
    return D == 64 ? launch<64, false>(a, s, st) : D == 128 ? launch<128, false>(a, s, st) : launch<256, false>(a, s, st);
}

}  // namespace cactus_hip
