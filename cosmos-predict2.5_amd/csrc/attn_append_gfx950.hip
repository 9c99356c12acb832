// New tokens on their way into a paged key-value cache, for gfx950: queries and keys normalised and turned by their positions, keys and values written into their pages: kernel and C ABI
// (cosmos_attn_cache_append).
//
// A row x of a query's or key's head, at position p:
//     n = x rsqrt(mean(x^2) + eps) w  (with a weight),   a_i = sum_axes p_axis freq_axis,i,   (u, v) -> (u cos a_i - v sin a_i, v cos a_i + u sin a_i)
// for its R pairs of channels, (i, i + R) or (2 i, 2 i + 1); what lies behind 2 R channels is not turned.  All of it in fp32, rounded once: to the 16-bit type, or as a code of 8 bits with its row's scale.
// Angles are formed in 64 bits, in quarters of a turn, and reduced there: at position 10^6 an angle in fp32 is off by 0.06.  Positions are the rows' places in their sequences, or given, several axes to a row.
#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>
#include <math.h>
#include <mutex>
#include <set>
#include <type_traits>
#include <utility>

#include "cosmos_attn_hip.h"

namespace {

#include "attn_common_gfx950.h"

constexpr int kThreads = 256;
#include "attn_cache_gfx950.h"

// Of the queries, keys or values: heads of a row, and workgroups.
struct Share { int heads; int64_t blocks; };
struct AppendParams : CacheParams {
    Share share[3];               // queries, keys, values
    const float* freqs;           // [axes, pairs]
    const int* positions;         // [rows, axes], or null: places in the sequences
    int64_t positions_row;
    const void* weight[2];        // of queries, of keys: fp32, or 16 bits; null: no norm
    int pairs, axes, weight_16;
    float eps;
};

// cos and sin of an angle: the nearest quarter turn off, in 64 bits (in 32 the rest would be off by as much as a rounding of 1), then Taylor's series on pi/4 to either side (their remainders are below 2^-33 and 2^-29)
__device__ __forceinline__ void turn(double angle, float& c, float& s) {
    const double quarters = angle * 0.63661977236758134308, whole = __builtin_rint(quarters);
    const float x = (float)((quarters - whole) * 1.57079632679489661923), y = x * x;
    float cx = __builtin_fmaf(y, -1.f / 3628800.f, 1.f / 40320.f);
    cx = __builtin_fmaf(y, cx, -1.f / 720.f);
    cx = __builtin_fmaf(y, cx, 1.f / 24.f);
    cx = __builtin_fmaf(y, cx, -0.5f);
    cx = __builtin_fmaf(y, cx, 1.f);
    float sx = __builtin_fmaf(y, 1.f / 362880.f, -1.f / 5040.f);
    sx = __builtin_fmaf(y, sx, 1.f / 120.f);
    sx = __builtin_fmaf(y, sx, -1.f / 6.f);
    sx = __builtin_fmaf(y * x, sx, x);
    const int q = (int)(int64_t)whole;
    const float a = q & 1 ? sx : cx, b = q & 1 ? cx : sx;
    c = (q + 1) & 2 ? -a : a;
    s = q & 2 ? -b : b;
}
template <int CTRL> __device__ __forceinline__ float dpp_sum(float v) {
    return v + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xF, 0xF, false));
}
// sum over the LANES (4 or 8) neighbouring lanes of a row
template <int LANES> __device__ __forceinline__ float row_sum(float v) {
    v = dpp_sum<0xB1>(v);       // quad_perm [1, 0, 3, 2]
    v = dpp_sum<0x4E>(v);       // quad_perm [2, 3, 0, 1]
    return LANES == 8 ? dpp_sum<0x141>(v) : v;      // row_half_mirror
}

// A lane has 16 channels of a row, two runs of 8, so that it has both of each of its 8 pairs; D / 16 lanes a row of a head.  Workgroups are the queries', the keys' or the values': which is theirs is
// the scalar unit's to find.  A workgroup's few rows' cosines and sines are formed once, by all threads, and read from LDS, each lane its own 8.
// Memory: 13069 rows of 32 + 8 + 8 heads to e4m3 with norms 63 us, 4.7 TB/s (a plain copy of the queries, norm and angles left out, 52, 5.6 TB/s: what is left are norms, turns and codes, the vector unit's); to
// 16 bits 62 us, 5.1 TB/s.  Angles in each lane for four heads after each other 72 us, shared for four heads 70, two 65; keys and values alone 28, 26.6, 24 and 21 us: the fewer registers, the more
// wavefronts there are.  Loads or stores past the caches: 65, but 25 % slower for 16 bits without norms.
template <typename T, int KIND, int D, bool INTERLEAVED>
__global__ void __launch_bounds__(kThreads) cache_append_kernel(const AppendParams p) {
#if defined(__HIP_DEVICE_COMPILE__)
    constexpr int LANES = D / 16, GROUPS = kThreads / LANES;
    __shared__ int position_of[GROUPS];                                                              // of the workgroup's rows
    __shared__ __attribute__((aligned(16))) float cos_of[GROUPS * D / 2], sin_of[GROUPS * D / 2];    // [row][pair]
    int64_t block = blockIdx.x;
    int what = 0;                 // 0 queries, 1 keys, 2 values
    for (; what < 2 && block >= p.share[what].blocks; ++what) block -= p.share[what].blocks;
    const Share& share = p.share[what];
    const int64_t unit = block * GROUPS, row0 = unit / share.heads;
    const unsigned u = (unsigned)(unit - row0 * share.heads) + threadIdx.x / LANES, r = u / (unsigned)share.heads;
    const int64_t row = row0 + r;
    const int head = (int)(u - r * share.heads), lane = threadIdx.x % LANES;
    const bool in = row < p.rows;
    // where this lane's two runs of channels begin, and its first pair (none from p.pairs on)
    const bool turned = what < 2 && 8 * lane < p.pairs;
    const int c0 = INTERLEAVED ? 16 * lane : 8 * lane < p.pairs ? 8 * lane : 16 * lane, c1 = INTERLEAVED || 8 * lane >= p.pairs ? c0 + 8 : c0 + p.pairs;
    const char* from = what == 0 ? p.q : p.side[what - 1].packed;
    const int64_t from_row = what == 0 ? p.q_row : p.side[what - 1].packed_row, from_head = what == 0 ? p.q_head : p.side[what - 1].packed_head;
    from += row * from_row + head * from_head;
    u32x4 w[2] = {u32x4{0, 0, 0, 0}, u32x4{0, 0, 0, 0}};
    if (in) {
        w[0] = *reinterpret_cast<const u32x4*>(from + 2 * c0);
        w[1] = *reinterpret_cast<const u32x4*>(from + 2 * c1);
    }
    // the row's sequence and place
    Place at(p, p.cu ? last_below(p.cu, 0, p.B, row0) : (int)(row0 < p.B ? row0 : p.B), true);
    if (in && row >= at.end && at.seq < p.B) at = Place(p, p.cu ? last_below(p.cu, at.seq + 1, p.B, row) : (int)row, true);
    const bool of = in && at.has(p, (int)row) && at.len >= at.end - at.start;
    const int position = of ? at.len - (at.end - (int)row) : 0;
    char* pages = nullptr;
    float* scales = nullptr;
    bool there = of;
    if (what) {
        const Side& side = p.side[what - 1];
        int page = -1;
        if (of && (position >> p.page_shift) < p.width) page = p.table[at.seq * p.table_row + (position >> p.page_shift)];
        there = page >= 0 && page < p.pages;
        const int place = position & ((1 << p.page_shift) - 1);
        pages = side.pages + (int64_t)(there ? page : 0) * side.page + place * side.row + head * side.head;
        if constexpr (KIND != SAME16) scales = side.scales + (int64_t)(there ? page : 0) * side.scale_page + head * side.scale_head + place;
    }
    float c[8], s[8], by[16];
    if (what < 2 && p.pairs) {
        const int first = (int)(unit - row0 * share.heads), rows = (first + GROUPS - 1) / share.heads + 1;      // the workgroup's, from row0 on
        if (lane == 0) position_of[r] = position;
        __syncthreads();
        for (int i = threadIdx.x; i < rows * p.pairs; i += kThreads) {
            const int at_row = i / p.pairs, pair = i - at_row * p.pairs;
            double angle = 0.0;
            for (int a = 0; a < p.axes; ++a) {
                int n = position_of[at_row];
                if (p.positions) n = row0 + at_row < p.rows ? p.positions[(row0 + at_row) * p.positions_row + a] : 0;
                angle = __builtin_fma((double)n, (double)p.freqs[a * p.pairs + pair], angle);
            }
            turn(angle, cos_of[i], sin_of[i]);
        }
        __syncthreads();
        if (turned) {
            __builtin_memcpy(c, __builtin_assume_aligned(cos_of + r * p.pairs + 8 * lane, 16), 32);
            __builtin_memcpy(s, __builtin_assume_aligned(sin_of + r * p.pairs + 8 * lane, 16), 32);
        }
    }
    const void* const weight = what < 2 ? p.weight[what] : nullptr;
    if (weight) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int channel = h ? c1 : c0;
            if (p.weight_16) {
                const u32x4 x = *reinterpret_cast<const u32x4*>((const char*)weight + 2 * channel);
#pragma unroll
                for (int j = 0; j < 4; ++j) { by[8 * h + 2 * j] = low<T>(x[j]); by[8 * h + 2 * j + 1] = high<T>(x[j]); }
            } else {
                __builtin_memcpy(by + 8 * h, __builtin_assume_aligned((const float*)weight + channel, 16), 32);
            }
        }
    }
    float x[16];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        x[2 * j] = low<T>(w[j / 4][j % 4]);
        x[2 * j + 1] = high<T>(w[j / 4][j % 4]);
    }
    if (weight) {
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < 16; ++j) sum = __builtin_fmaf(x[j], x[j], sum);
        const float mean = __builtin_fmaf(row_sum<LANES>(sum), 1.f / D, p.eps);
        float root = __builtin_amdgcn_rsqf(mean);
        if (mean > 0.f && mean < INFINITY) root = __builtin_fmaf(0.5f * root, __builtin_fmaf(-mean * root, root, 1.f), root);      // (a step of Newton's: the instruction is good to one unit in the last place)
#pragma unroll
        for (int j = 0; j < 16; ++j) x[j] *= root * by[j];
    }
    if (turned) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            float& a = x[INTERLEAVED ? 2 * j : j];
            float& b = x[INTERLEAVED ? 2 * j + 1 : 8 + j];
            const float A = __builtin_fmaf(a, c[j], -(b * s[j])), B = __builtin_fmaf(b, c[j], a * s[j]);
            a = A;
            b = B;
        }
    }
    if (what == 0 || KIND == SAME16) {
        u32x4 y[2];
#pragma unroll
        for (int j = 0; j < 8; ++j) y[j / 4][j % 4] = round2<T>(x[2 * j], x[2 * j + 1]);
        if (what == 0 && !of) y[0] = y[1] = u32x4{0, 0, 0, 0};
        char* const to = what == 0 ? p.o + row * p.o_row + head * p.o_head : pages;
        if (there || (what == 0 && in && p.fill)) {
            *reinterpret_cast<u32x4*>(to + 2 * c0) = y[0];
            *reinterpret_cast<u32x4*>(to + 2 * c1) = y[1];
        }
    } else {
        // the largest magnitude: floats without their signs as whole numbers, in whose order NaN comes behind infinity and that behind all others
        unsigned top = 0;
#pragma unroll
        for (int j = 0; j < 16; ++j) { const unsigned b = __builtin_bit_cast(unsigned, x[j]) & 0x7FFFFFFFu; top = top > b ? top : b; }
        top = row_max<LANES>(top);
        // (a row of zeros: divided by 1; one that is not finite: codes of no meaning)
        const float scale = top < 0x7F800000u ? __builtin_bit_cast(float, top) * (KIND == E4M3 ? 1.f / 448.f : 1.f / 127.f) : NAN;
        const Divide over(scale > 0.f ? scale : 1.f);
        if (__any(over.by != 1.f)) {
#pragma unroll
            for (int j = 0; j < 16; ++j) x[j] *= over.by;
        }
#pragma unroll
        for (int j = 0; j < 16; ++j) x[j] = over(x[j]);
        u32x2 y[2];
#pragma unroll
        for (int j = 0; j < 4; ++j) y[j / 2][j % 2] = code_word<KIND>(x[4 * j], x[4 * j + 1], x[4 * j + 2], x[4 * j + 3]);
        if (there) {
            *reinterpret_cast<u32x2*>(pages + c0) = y[0];
            *reinterpret_cast<u32x2*>(pages + c1) = y[1];
            if (lane == 0) *scales = scale;
        }
    }
#endif
}

// ---- C ABI
constexpr int kMostAxes = 8;
int check_rope(const cosmos_attn_cache_desc* d, const cosmos_attn_cache_rope* r) {
    if (!r || r->pairs < 0 || r->axes < 1 || !(r->eps >= 0.f && r->eps <= 3.0e38f)) return COSMOS_ATTN_BAD_ARG;
    if (r->pairs % 8 || 2 * (int64_t)r->pairs > d->D) return COSMOS_ATTN_BAD_SHAPE;
    if (r->axes > kMostAxes) return COSMOS_ATTN_UNSUPPORTED;
    if (r->pairs && (!r->freqs || (r->axes > 1 && d->rows && !r->positions))) return COSMOS_ATTN_BAD_ARG;
    if (!aligned16(r->freqs) || !aligned16(r->q_weight) || !aligned16(r->k_weight) || (reinterpret_cast<uintptr_t>(r->positions) & 3) || r->positions_stride < 0) return COSMOS_ATTN_BAD_STRIDE;
    return COSMOS_ATTN_OK;
}
int check_append(const cosmos_attn_cache_desc* d, const cosmos_attn_cache_rope* r) {
    int st = check(d);
    if (st == COSMOS_ATTN_OK) st = check_rope(d, r);
    if (st != COSMOS_ATTN_OK) return st;
    if (d->rows < 0 || d->rows > kMost || (d->q && d->Hq < 1)) return COSMOS_ATTN_BAD_ARG;
    if (!d->rows) return COSMOS_ATTN_OK;
    if (d->B && !d->lens) return COSMOS_ATTN_BAD_ARG;
    if (!d->cu && d->rows != d->B) return COSMOS_ATTN_BAD_SHAPE;
    st = check_written(d);
    if (st == COSMOS_ATTN_OK) st = check_rows(d->k_rows, d->k_rows_stride);
    if (st == COSMOS_ATTN_OK) st = check_rows(d->v_rows, d->v_rows_stride);
    if (st == COSMOS_ATTN_OK && d->q) st = check_rows(d->q, d->q_stride);
    if (st == COSMOS_ATTN_OK && d->q) st = check_out(d->o, d->o_stride, d->rows, d->Hq, d->D);
    return st;
}
Share share_of(const cosmos_attn_cache_desc* d, int heads) {
    const int groups = kThreads / (d->D / 16);
    return {heads, (d->rows * heads + groups - 1) / groups};
}

}  // namespace

extern "C" {

int cosmos_attn_cache_append(const cosmos_attn_cache_desc* desc, const cosmos_attn_cache_rope* rope, void* stream) {
    const int st = check_append(desc, rope);
    if (st != COSMOS_ATTN_OK || !desc->rows) return st;
    AppendParams p = {};
    static_cast<CacheParams&>(p) = params_of(desc);
    p.q = (const char*)desc->q; p.o = (char*)desc->o;
    p.q_row = 2 * desc->q_stride[0]; p.q_head = 2 * desc->q_stride[1]; p.o_row = 2 * desc->o_stride[0]; p.o_head = 2 * desc->o_stride[1];
    p.share[0] = desc->q ? share_of(desc, desc->Hq) : Share{1, 0};
    p.share[1] = p.share[2] = share_of(desc, desc->Hkv);
    const int64_t blocks = p.share[0].blocks + p.share[1].blocks + p.share[2].blocks;
    if (blocks > kMostBlocks) return COSMOS_ATTN_UNSUPPORTED;
    if (desc->q) {
        // (keys or values that queries have been written over would be what another workgroup reads)
        const Packed o = {desc->o, desc->o_stride, desc->Hq};
        if (check_in_place(desc, desc->rows) != COSMOS_ATTN_OK || meet_in_memory(o, {desc->k_rows, desc->k_rows_stride, desc->Hkv}, desc->rows, desc->D) ||
            meet_in_memory(o, {desc->v_rows, desc->v_rows_stride, desc->Hkv}, desc->rows, desc->D)) return COSMOS_ATTN_BAD_ARG;
    }
    if (!device_is_whole_mi355x()) return COSMOS_ATTN_WRONG_DEVICE;
    p.freqs = rope->freqs; p.positions = rope->positions; p.positions_row = rope->positions_stride;
    p.weight[0] = rope->q_weight; p.weight[1] = rope->k_weight; p.weight_16 = rope->weight_16 != 0;
    p.pairs = rope->pairs; p.axes = rope->axes; p.eps = rope->eps;
    return with_type(desc, [&](auto* t, auto dim, auto kind) {
        typedef std::remove_pointer_t<decltype(t)> T;
        constexpr int D = decltype(dim)::value, K = decltype(kind)::value;
        return rope->interleaved ? launch(cache_append_kernel<T, K, D, true>, blocks, 0, p, stream) : launch(cache_append_kernel<T, K, D, false>, blocks, 0, p, stream);
    });
}

}  // extern "C"
