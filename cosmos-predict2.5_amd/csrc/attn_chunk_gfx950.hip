// Attention of several new tokens of each sequence over a paged key-value cache, for gfx950: kernel and C ABI (cosmos_attn_cache_chunk).
//
// Sequence i has the rows cu[i] .. cu[i + 1] - 1 of q, Lq of them: the last Lq of its lens[i] positions, whose keys and values lie in the cache already.  With p = t + lens[i] - Lq the
// position of token t, c the scale:
//     s_tj = c q_t k_j,   visible: j <= p, and with a window j > p - window or j < sinks,   o_t = sum_j softmax_j(s_tj) v_j,   lse_t = log sum_j exp(s_tj)
// A row that sees no key (a position below 0): o = 0, lse = -inf.
//
// The rows, tiles, cuts and joins are those of packed sequences (attn_ragged_gfx950.h): the query heads of a key head are rows of one matrix, a workgroup has 128 of them and K and V go by in steps
// of 64 keys through LDS.  A step's 64 keys are four runs of 16, each within a page: wavefront w looks up run w's page, a step before it is needed, and brings its rows.
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
#include "attn_ragged_gfx950.h"
#include "attn_cache_gfx950.h"

struct ChunkParams : RaggedParams {
    Side side[2];                  // keys, values
    const int* table;
    int64_t table_row;
    int pages, page_shift;
    int short_blocks;              // workgroups of short sequences, behind the tiles'
    float* short_sums;             // what their parts leave: of part s of the i-th and key head h, at (i Hkv + h) short_parts + s
};

// ---- Sequences of few rows (a token or some, of which the query heads of a key head are 16 at most together): keys and values go by once, for a product or two, and what counts is how many bytes are
// under way.  A wavefront has 32 of 128 keys to a step, straight from memory into registers, as in cache_attention_kernel; rows are the columns of 16 x 16 x 32 products.  In the tiles' launch, behind
// these: 46 single tokens of 1 to 7939 keys beside pieces of 512 and 300 tokens, 16 heads of 128 on 8 in e4m3, 105 us; as tiles of 128 rows with 2 live ones 145.  (The single tokens alone 61 us, 4.1 TB/s, where
// cache_attention_kernel's three wavefronts on a SIMD take 46; the pieces alone 61.  Tiles and short sequences alternating, 119; first the short ones, 120.  What these bound each other by is the
// vector unit, which both need for codes.)
constexpr int kShortRows = 16, kShortStep = 128;
template <int D> constexpr int kShortFloats = kShortRows * (D + 2);       // of a part: its rows' D sums, then max and sum of exponentials
// the keys that a sequence's tokens see, in steps: those of the first keys and, behind the `gap` that none looks at, those from the first token's window on
template <bool WINDOW> struct Seen {
    int from, first, gap, steps;
    __device__ __forceinline__ Seen(const RaggedParams& p, Lengths n) {
        const int len = n.lk > 0 ? n.lk : 0;
        from = WINDOW && len - n.lq + 1 > p.window ? len - n.lq + 1 - p.window : 0;
        first = ((p.sinks < from ? p.sinks : from) + kShortStep - 1) / kShortStep;
        gap = WINDOW && from / kShortStep > first ? from / kShortStep - first : 0;
        steps = (len + kShortStep - 1) / kShortStep - gap;
    }
};
template <bool WINDOW> struct ShortTiles {
    const RaggedParams& p;
    __device__ __forceinline__ int keys_of(int i) const { return RowTilesOf<WINDOW, true>{p}.keys_of(i); }
    __device__ __forceinline__ Lengths lengths(int i) const { return RowTilesOf<WINDOW, true>{p}.lengths(i); }
    __device__ __forceinline__ int count(Lengths n) const { return n.lq > 0 && (int64_t)n.lq * p.group <= p.short_rows; }
    static __device__ __forceinline__ int at(int rank, int) { return rank; }
    __device__ __forceinline__ int steps(Lengths n, int) const { return Seen<WINDOW>(p, n).steps; }
    __device__ __forceinline__ int64_t all_steps(Lengths n, int) const { return steps(n, 0); }
    __device__ __forceinline__ int most_parts() const { return p.short_parts; }
    __device__ __forceinline__ int least() const { return p.short_least; }
    static constexpr bool OF_KEYS = false, IN_PAGES = true;
};
__device__ __forceinline__ float over_quarters_max(float x) {
    x = over_halves_max(x);
    return fmaxf(x, __shfl_xor(x, 16));
}
// row r of the sequence that begins at `start`: o and lse from its sums
template <typename T> __device__ __forceinline__ void store_row(const ChunkParams& p, int start, int head, int r, int c, const float (&f)[8], float top, float sum, bool bad) {
    const int token = r / p.group, hq = head * p.group + (r - token * p.group);
    float by = sum > 0.f ? 1.f / sum : sum == 0.f ? 0.f : sum, lse = sum > 0.f ? (top + __builtin_amdgcn_logf(sum)) * 0.693147180559945309f : sum == 0.f ? -INFINITY : sum;
    if (bad) by = lse = NAN;
    *reinterpret_cast<u32x4*>(p.o + (start + token) * p.o_row + hq * p.o_head + 2 * c) = u32x4{round2<T>(f[0] * by, f[1] * by), round2<T>(f[2] * by, f[3] * by), round2<T>(f[4] * by, f[5] * by), round2<T>(f[6] * by, f[7] * by)};
    if (p.lse && c == 0) p.lse[(start + token) * p.lse_row + hq] = lse;
}
// sums: two halves, of two wavefronts each
template <typename T, int KIND, int D, bool WINDOW>
__device__ __forceinline__ void short_sequence(const ChunkParams& p, const Found& f, int head, int index, int part, float* sums01, float* sums23, float* stat) {
#if defined(__HIP_DEVICE_COMPILE__)
    typedef typename VecOf<T>::v8 V8;
    constexpr bool CODES = KIND != SAME16;
    constexpr int BYTES = CODES ? 1 : 2, NC = D / 32, NB = D / 16;       // NC: products of 32 channels; NB: of 16 channels of the output, channels of a lane of V
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n16 = lane & 15, g = lane >> 4;
    const Range rq = rows_of_sequence(p.cu_q, f.seq, f.n.lq);
    const int rows = rq.length * p.group, len = f.n.lk > 0 ? f.n.lk : 0;
    const Seen<WINDOW> seen(p, f.n);
    const int from = (int)((int64_t)part * seen.steps / f.parts), to = (int)((int64_t)(part + 1) * seen.steps / f.parts);
    const int* const table = p.table + f.seq * p.table_row;
    const char* const kh = p.side[0].pages + head * p.side[0].head;
    const char* const vh = p.side[1].pages + head * p.side[1].head;
    const int mask = (1 << p.page_shift) - 1;
    // Q: row n16, the channels that this lane's K holds
    const int row = n16 < rows ? n16 : rows - 1, token = row / p.group, row_end = len - (rq.length - 1 - token);      // row_end: keys that it sees
    V8 qf[NC];
    {
        const char* const at = p.q + (rq.start + token) * p.q_row + (head * p.group + (row - token * p.group)) * p.q_head;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            u32x4 w = *reinterpret_cast<const u32x4*>(at + 2 * (CODES ? 64 * (c / 2) + 16 * g + 8 * (c % 2) : 32 * c + 8 * g));
            w ^= p.flip;
            qf[c] = __builtin_bit_cast(V8, w);
        }
    }
    f32x4 acc[NB];
    float m = kLowest, l = 0.f, R = 0.f;
#pragma unroll
    for (int b = 0; b < NB; ++b) acc[b] = f32x4{0.f, 0.f, 0.f, 0.f};
    // Steps of 32 keys.  A step's K is loaded behind the products of the one before, its V behind that one's, and its pages are looked up a step earlier still.  Keys past the end are the last
    // one's, keys that no token sees the first one that is looked back on.
    constexpr int KLOADS = CODES ? NC / 2 : NC, VWORDS = NB * BYTES / 4;
    const int most = len - 1, first_key = 32 * wave;
    auto base_of = [&](int u) { return (WINDOW && u >= seen.first ? u + seen.gap : u) * kShortStep + first_key; };
    auto is_seen = [&](int key) { return !WINDOW || key >= seen.from || key < p.sinks; };
    int end = (len - first_key + kShortStep - 1) / kShortStep - seen.gap;
    end = to < end ? to : end;
    u32x4 kw[2][KLOADS];
    unsigned vw[8][VWORDS];
    float ks[8], vs[8];
    // K: row n16 of key half u is key 8 (n16 / 4) + 4 u + n16 % 4, so that a lane's results of the two halves are those of 8 keys in order, 8 g .. 8 g + 7
    auto k_key = [&](int t, int u) { const int key = base_of(t) + 8 * (n16 >> 2) + 4 * u + (n16 & 3); return key >= most ? most : is_seen(key) ? key : seen.from; };
    // V: keys 8 g .. 8 g + 7, channels NB n16 .. NB n16 + NB - 1; 8 keys in order share a page
    auto v_key = [&](int t) { const int key = base_of(t) + 8 * g; return key >= (most & ~7) ? most & ~7 : is_seen(key) || is_seen(key + 7) ? key : seen.from & ~7; };
    int kp[2], vp;
    bool none = false, none_next = false;      // the page of this lane's keys of the step, and of the next one, is not there
    auto look_up = [&](int t) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < 2; ++u) kp[u] = table[k_key(t, u) >> p.page_shift];
        vp = table[v_key(t) >> p.page_shift];
    };
    auto is_there = [&](int page) { return page >= 0 && page < p.pages; };
    auto load_k = [&](int t) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const char* const at = kh + (int64_t)(is_there(kp[u]) ? kp[u] : 0) * p.side[0].page + (k_key(t, u) & mask) * p.side[0].row + 16 * g;
#pragma unroll
            for (int c = 0; c < KLOADS; ++c) kw[u][c] = *reinterpret_cast<const u32x4*>(at + 64 * c);
        }
    };
    auto load_v = [&](int t, int page) __attribute__((always_inline)) {
        const int key8 = v_key(t), in8 = key8 & mask;
        const char* const at = vh + page * p.side[1].page + in8 * p.side[1].row + NB * BYTES * n16;
#pragma unroll
        for (int i = 0; i < 8; ++i) __builtin_memcpy(vw[i], __builtin_assume_aligned(at + (key8 + i < most ? i : most - key8) * p.side[1].row, 4 * VWORDS), 4 * VWORDS);
        if constexpr (CODES) {
            __builtin_memcpy(ks, __builtin_assume_aligned(p.side[0].scales + page * p.side[0].scale_page + head * p.side[0].scale_head + in8, 16), 32);
            __builtin_memcpy(vs, __builtin_assume_aligned(p.side[1].scales + page * p.side[1].scale_page + head * p.side[1].scale_head + in8, 16), 32);
        }
    };
    if (from < end) {
        look_up(from);
        load_k(from);
        none = !is_there(vp);
        load_v(from, none ? 0 : vp);
        look_up(from + 1);
    }
    // (the last step loads nothing: a condition around the loads would have the compiler wait for all of them at the next use of any)
    auto step = [&](int t, auto more) __attribute__((always_inline)) {
        f32x4 s[2] = {f32x4{0.f, 0.f, 0.f, 0.f}, f32x4{0.f, 0.f, 0.f, 0.f}};
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                u32x4 w;
                if constexpr (CODES) {
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        w[2 * i] = code_pair<T, KIND, false>(kw[u][c / 2][2 * (c % 2) + i]);
                        w[2 * i + 1] = code_pair<T, KIND, true>(kw[u][c / 2][2 * (c % 2) + i]);
                    }
                } else {
                    w = kw[u][c];
                }
                s[u] = mfma16(__builtin_bit_cast(V8, w), qf[c], s[u]);
            }
        int vnext = 0;
        if constexpr (decltype(more)::value) {
            load_k(t + 1);
            none_next = !is_there(vp);
            vnext = none_next ? 0 : vp;
            look_up(t + 2);
        }
        const int at = base_of(t) + 8 * g, left = row_end - at, out = left - p.window, in = p.sinks - at;
        // keys that this lane's row sees; that some row does
        auto counts = [&](int i) { return i < left && (!WINDOW || i >= out || i < in); };
        auto any_sees = [&](int i) { return !none && i < len - at && (!WINDOW || i >= seen.from - at || i < in); };
        float by[8];                            // what V's weights are multiplied with
        if constexpr (CODES) {
#pragma unroll
            for (int i = 0; i < 8; ++i) by[i] = counts(i) ? vs[i] : 0.f;
            if constexpr (__is_same(T, _Float16)) {
                // (weights p scale in fp16 would leave its range where values are small: held relative to the largest scale so far of the keys that this lane's row sees, but for a factor of up to 64)
                float top = by[0];
#pragma unroll
                for (int i = 1; i < 8; ++i) top = fmaxf(top, by[i]);
                if (__any(top > 64.f * R)) {
                    top = fmaxf(fmaxf(R, over_quarters_max(top)), 0x1p-100f);
                    const float f = R / top;
#pragma unroll
                    for (int b = 0; b < NB; ++b) acc[b] *= f;
                    R = top;
                }
                const float over = R > 0.f ? 1.f / R : 1.f;
#pragma unroll
                for (int i = 0; i < 8; ++i) by[i] *= over;
            }
        }
        float x[8], top = -INFINITY;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            x[i] = s[i / 4][i % 4] * p.scale_log2;
            if constexpr (CODES) x[i] *= ks[i];
            x[i] = !counts(i) ? -INFINITY : none ? NAN : x[i];
            top = fmaxf(top, x[i]);
        }
        if (__any(top > m + kMaxSlack)) {
            top = fmaxf(m, over_quarters_max(top));
            const float f = __builtin_amdgcn_exp2f(m - top);
            m = top;
            l *= f;
#pragma unroll
            for (int b = 0; b < NB; ++b) acc[b] *= f;
        }
        V8 pf, pr;          // the weights, and what their rounding leaves off: there is time for both
        {
            u32x4 w, rest;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                x[i] = __builtin_amdgcn_exp2f(x[i] - m);
                l += x[i];
                if constexpr (CODES) x[i] *= by[i];
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = round2<T>(x[2 * i], x[2 * i + 1]);
            asm("" : "+v"(w));       // (what the product takes)
#pragma unroll
            for (int i = 0; i < 4; ++i) rest[i] = round2<T>(x[2 * i] - element<T>(w[i], 0), x[2 * i + 1] - element<T>(w[i], 1));
            pf = __builtin_bit_cast(V8, w);
            pr = __builtin_bit_cast(V8, rest);
        }
        // rows that no token sees may hold anything, which a weight of 0 would make NaN
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int j = 0; j < VWORDS; ++j) vw[i][j] = any_sees(i) ? vw[i][j] : 0u;
        // output rows NB n + b, n = 0 .. 15: what lane n16 holds of V, transposed in its registers
        unsigned vx[8][NB / 2];
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int j = 0; j < VWORDS; ++j) {
                if constexpr (CODES) {
                    vx[i][2 * j] = code_pair<T, KIND, false>(vw[i][j]);
                    vx[i][2 * j + 1] = code_pair<T, KIND, true>(vw[i][j]);
                } else {
                    vx[i][j] = vw[i][j];
                }
            }
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            u32x4 vt;
#pragma unroll
            for (int i = 0; i < 4; ++i) vt[i] = __builtin_amdgcn_perm(vx[2 * i + 1][b / 2], vx[2 * i][b / 2], b % 2 ? 0x07060302u : 0x05040100u);
            acc[b] = mfma16(__builtin_bit_cast(V8, vt), pf, acc[b]);
            acc[b] = mfma16(__builtin_bit_cast(V8, vt), pr, acc[b]);
        }
        if constexpr (decltype(more)::value) {
            load_v(t + 1, vnext);
            none = none_next;
        }
    };
    if (from < end) {
        for (int t = from; t + 1 < end; ++t) step(t, Int<1>{});
        step(end - 1, Int<0>{});
    }
    // ---- join the wavefronts: [wave][row][channel], and [wave][row] of max, sum
    auto sums_of = [&](int w) { return (w < 2 ? sums01 : sums23) + (w & 1) * kShortRows * D; };
    const float back = CODES && __is_same(T, _Float16) ? R : 1.f;
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    if (g == 0) {
        stat[2 * (wave * kShortRows + n16)] = m;
        stat[2 * (wave * kShortRows + n16) + 1] = l;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int b = 0; b < NB; b += 4) *reinterpret_cast<f32x4*>(sums_of(wave) + n16 * D + NB * (4 * g + e) + b) = f32x4{acc[b][e], acc[b + 1][e], acc[b + 2][e], acc[b + 3][e]} * back;
    __syncthreads();
    constexpr int LANES = D / 8, AT_ONCE = kThreads / LANES;
    for (int r = threadIdx.x / LANES; r < rows; r += AT_ONCE) {
        const int c = 8 * (threadIdx.x % LANES);
        float top = kLowest, sum = 0.f, o[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < 4; ++w) top = fmaxf(top, stat[2 * (w * kShortRows + r)]);
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float by = __builtin_amdgcn_exp2f(stat[2 * (w * kShortRows + r)] - top);
            sum += by * stat[2 * (w * kShortRows + r) + 1];
#pragma unroll
            for (int i = 0; i < 8; ++i) o[i] += by * sums_of(w)[r * D + c + i];
        }
        if (f.parts == 1) {
            store_row<T>(p, rq.start, head, r, c, o, top, sum, f.n.lk < 0);
        } else {
            float* const to_part = p.short_sums + (((int64_t)index * p.Hkv + head) * p.short_parts + part) * kShortFloats<D>;
            *reinterpret_cast<f32x4*>(to_part + r * D + c) = f32x4{o[0], o[1], o[2], o[3]};
            *reinterpret_cast<f32x4*>(to_part + r * D + c + 4) = f32x4{o[4], o[5], o[6], o[7]};
            if (c == 0) { to_part[kShortRows * D + 2 * r] = top; to_part[kShortRows * D + 2 * r + 1] = sum; }
        }
    }
#endif
}

// what was written to LDS is there and all reads have returned; then the workgroup meets, with loads to registers under way
__device__ __forceinline__ void meet_in_lds() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0xC07F);           // lgkmcnt 0 alone
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// ---- A workgroup: as ragged_fwd_kernel, with K and V out of pages.  2048 tokens on 16384 positions, 32 heads of 128 on 8: 500 us, 1.0 PFLOP/s, in 8 bits 595 to 620 (codes' conversions are 8 %, scales 11 % of that, measured
// without them; the matrix unit is busy 55 % of the time, as there with two wavefronts on a SIMD, whose maxima and exponentials it waits for).  A call of few tiles is as long as its longest part: a step of 64 keys takes 1.1 us in 16 bits and 1.7 in 8, all of it one chain.
// Hence parts of 4 steps at least, if there are more than 8 (64 tokens on 1280 positions, 8 heads on 2, us, bf16 / int8: whole 30 / 42, parts of 8 and more 24 / 30, of 6 21 / 26, of 4 18 / 21, with 5 for the second launch).
// 16 bits: rows go straight to LDS; what lies behind the last key, and runs that no row of the tile sees, come as zeros.  8 bits: codes are loaded into registers a step earlier, become exact
// 16-bit values on their way to LDS, K's scales multiply the scores and V's the weights, before these are rounded.
// A page that is not there: its keys are NaN, for the rows that see them.
template <typename T, int KIND, int D, bool WINDOW>
__global__ void __launch_bounds__(kThreads, 2) cache_chunk_kernel(const ChunkParams p) {
#if defined(__HIP_DEVICE_COMPILE__)
    typedef typename VecOf<T>::v8 V8;
    typedef Tile<D> L;
    typedef RowTilesOf<WINDOW, true> Rows;
    constexpr int NC = D / 16, NB = D / 32, RUN = kStep / 4;        // RUN: keys of a step that a wavefront brings
    constexpr bool CODES = KIND != SAME16;
    LDS_TILES(L);
    __shared__ __attribute__((aligned(16))) float scales0[CODES ? 2 * kStep : 4], scales1[CODES ? 2 * kStep : 4];      // of a step's keys, then of its values
    if ((int)blockIdx.x >= (int)gridDim.x - p.short_blocks) {
        // (first come the first parts of all short sequences, then the second ones)
        const int b = blockIdx.x - (gridDim.x - p.short_blocks), rest = b / p.Hkv, part = rest / p.n_seq, index = rest - part * p.n_seq;
        const Found f = find<ShortTiles<WINDOW>>(p, index);
        if (f.seq >= 0 && part < f.parts) short_sequence<T, KIND, D, WINDOW>(p, f, b - rest * p.Hkv, index, part, (float*)tile0, (float*)tile1, (float*)tile2);
        return;
    }
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5;
    const Block block = block_of(p, blockIdx.x);
    const int head = block.head;
    const Found f = find<Rows>(p, block.index);
    if (f.seq < 0) {
        if (p.fill && block.part == 0) clear_rows<D>(p.fill == COSMOS_ATTN_FILL_LSE ? nullptr : p.o, p.o_row, p.o_head, p.cu_q, p.n_seq, p.Tq, p.group, head * p.group, kRows, f, p.lse, p.lse_row, p.lse_head);
        return;
    }
    if (block.part >= f.parts) return;
    const int tile = f.tile;
    const Range rq = rows_of_sequence(p.cu_q, f.seq, f.n.lq);
    const int rows = rq.length * p.group, lk = f.n.lk > 0 ? f.n.lk : 0, shift = lk - rq.length;
    const int row = tile * kRows + 32 * wave + (lane & 31);
    const bool live = row < rows;
    const int token = row / p.group, hq = head * p.group + (row - token * p.group);
    // keys that this lane's row sees, the most of this wavefront's and of the workgroup's rows, the fewest of this wavefront's
    auto keys_of = [&](int t) { const int e = t + shift + 1; return e > lk ? lk : e < 0 ? 0 : e; };
    const int end = live ? keys_of(token) : 0;
    const int first = tile * kRows + 32 * wave;
    auto token_at = [&](int r) { return __builtin_amdgcn_readfirstlane((r < rows ? r : rows - 1) / p.group); };
    const int wave_end = first < rows ? keys_of(token_at(first + 31)) : 0, wave_all = keys_of(token_at(first));
    // (WINDOW: the first key that this lane's row looks back on, the last and the first of those of this wavefront's, the first of the tile's)
    const int from = WINDOW ? Rows{p}.first_key(f.n, row) : 0, wave_from = WINDOW ? __builtin_amdgcn_readfirstlane(Rows{p}.first_key(f.n, first + 31)) : 0,
              wave_first = WINDOW ? __builtin_amdgcn_readfirstlane(Rows{p}.first_key(f.n, first)) : 0, tile_first = WINDOW ? __builtin_amdgcn_readfirstlane(Rows{p}.first_key(f.n, tile * kRows)) : 0;
    // one behind the last key that a row of the tile sees: no page from there on is looked at
    const int tile_end = keys_of(token_at(tile * kRows + kRows - 1));
    // steps of this part; of step u, where its keys begin
    const int steps = Rows{p}.end_step(f.n, tile), sink_steps = Rows{p}.sink_steps(), gap = Rows{p}.gap(f.n, tile);
    auto at_step = [&](int u) { return WINDOW && u >= sink_steps ? u + gap : u; };
    const int t0 = (int)((int64_t)block.part * steps / f.parts), n = (int)((int64_t)(block.part + 1) * steps / f.parts);

    // (of constant memory, so that the scalar unit looks up: a vector load's result in scalar registers is waited for at once, with all loads in front of it; 160 -> 145 us, and 2048 + 512 + 77 tokens on
    // 16384, 9001 and 1301 positions in bf16 717 -> 653)
    typedef const __attribute__((address_space(4))) int* Table;
    const Table table = (Table)(uintptr_t)(p.table + f.seq * p.table_row);
    const int mask = (1 << p.page_shift) - 1;
    const char* const kh = p.side[0].pages + head * p.side[0].head;
    const char* const vh = p.side[1].pages + head * p.side[1].head;
    // this wavefront's run of step u: its first key, and whether some row of the tile sees some of it
    auto run_of = [&](int u) { return at_step(u) * kStep + RUN * wave; };
    auto is_seen = [&](int key) { return key < tile_end && (!WINDOW || key + RUN > tile_first || key < p.sinks); };
    auto look_up = [&](int u) { const int key = run_of(u); return table[(u < n && is_seen(key) ? key : tile_end - 1) >> p.page_shift]; };      // (there is a key: t0 < n)
    // WINDOW: keys of a run that no row of the tile sees, beside others that are seen
    auto is_hidden = [&](int key) { return WINDOW && key < tile_first && key >= p.sinks; };

    // 16 bits: a run straight to LDS
    int k_off[L::LOADS], v_off[L::LOADS];
    auto bring = [&](int u, int page, char* kt, char* vt) __attribute__((always_inline)) {
        const int key0 = run_of(u);
        const bool seen = is_seen(key0), there = page >= 0 && page < p.pages;
        const int left = seen && there ? (tile_end - key0 < RUN ? tile_end - key0 : RUN) : 0;
        const int64_t at = there ? page : 0;
        const auto kr = rows_of<D, RUN>(kh + at * p.side[0].page + (key0 & mask) * p.side[0].row, p.side[0].row, left);
        const auto vr = rows_of<D, RUN>(vh + at * p.side[1].page + (key0 & mask) * p.side[1].row, p.side[1].row, left);
        const bool partly = WINDOW && key0 < tile_first && key0 + RUN > p.sinks;
#pragma unroll
        for (int i = 0; i < L::LOADS; ++i) {
            const bool hidden = partly && is_hidden(key0 + L::load_row(lane, 0, i));
            if (seen && !there) {
                const unsigned none = round2<T>(NAN, NAN);
                *reinterpret_cast<u32x4*>(kt + L::load_to(wave, i) + 16 * lane) = u32x4{none, none, none, none};
            } else {
                load_to_lds(kr, kt + L::load_to(wave, i), hidden ? (int)0x80000000 : k_off[i]);
            }
            load_to_lds(vr, vt + L::load_to(wave, i), hidden ? (int)0x80000000 : v_off[i]);
        }
    };
    // 8 bits: 16 codes to a lane, CODE_ROWS rows at a time
    constexpr int CODE_LANES = D / 16, CODE_ROWS = 64 / CODE_LANES, CODE_LOADS = RUN / CODE_ROWS;
    struct Codes {
        u32x4 codes[2][CODES ? CODE_LOADS : 1];
        float scale[2];            // of row lane % RUN
        bool none;                 // its page is not there
    };
    int code_off[2][CODES ? CODE_LOADS : 1];
    // (Without a condition around the loads, whatever is there: behind a branch the compiler waits for all that are under way.  A run that is not there has no bytes, and reads as zeros.)
    auto load_codes = [&](Codes& to, int u, int page) __attribute__((always_inline)) {
        const int key0 = run_of(u);
        const bool seen = u < n && is_seen(key0), there = page >= 0 && page < p.pages;
        const int left = seen && there ? (tile_end - key0 < RUN ? tile_end - key0 : RUN) : 0;
        const bool partly = WINDOW && key0 < tile_first && key0 + RUN > p.sinks;
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const Side& side = p.side[s];
            const int64_t at = there ? page : 0;
            const auto rows = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>((s ? vh : kh) + at * side.page + (key0 & mask) * side.row), 0, left > 0 ? (int)((left - 1) * side.row) + D : 0, 0x00020000);
            const auto scales = __builtin_amdgcn_make_buffer_rsrc(side.scales + at * side.scale_page + head * side.scale_head + (key0 & mask), 0, 4 * left, 0x00020000);
#pragma unroll
            for (int i = 0; i < CODE_LOADS; ++i) {
                const bool hidden = partly && is_hidden(key0 + i * CODE_ROWS + lane / CODE_LANES);
                to.codes[s][i] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rows, hidden ? (int)0x80000000 : code_off[s][i], 0, 0));
            }
            to.scale[s] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(scales, partly && is_hidden(key0 + lane % RUN) ? (int)0x80000000 : 4 * (lane % RUN), 0, 0));
        }
        to.none = seen && !there;
    };
    auto keep_codes = [&](const Codes& of, char* kt, char* vt, float* st) __attribute__((always_inline)) {
        auto& codes = of.codes;
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int i = 0; i < CODE_LOADS; ++i) {
                const int r = RUN * wave + i * CODE_ROWS + lane / CODE_LANES, chunk = 2 * (lane % CODE_LANES);
                char* const to = (s ? vt : kt) + r * L::ROW;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    u32x4 w;
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        w[2 * j] = code_pair<T, KIND, false>(codes[s][i][2 * h + j]);
                        w[2 * j + 1] = code_pair<T, KIND, true>(codes[s][i][2 * h + j]);
                    }
                    *reinterpret_cast<u32x4*>(to + (((chunk + h) ^ L::mix(r)) << 4)) = w;
                }
            }
        if (lane < 2 * RUN) st[(lane / RUN) * kStep + RUN * wave + lane % RUN] = lane >= RUN ? of.scale[1] : of.none ? NAN : of.scale[0];
    };
    Codes even, odd;               // of steps t0, t0 + 2, ..; of the others
    int page = 0, page2 = 0;
    if constexpr (CODES) {
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int i = 0; i < CODE_LOADS; ++i) code_off[s][i] = (i * CODE_ROWS + lane / CODE_LANES) * (int)p.side[s].row + 16 * (lane % CODE_LANES);
    } else {
#pragma unroll
        for (int i = 0; i < L::LOADS; ++i) {
            k_off[i] = L::load_row(lane, 0, i) * (int)p.side[0].row + L::load_byte(lane, wave, i);
            v_off[i] = L::load_row(lane, 0, i) * (int)p.side[1].row + L::load_byte(lane, wave, i);
        }
    }
    // Q as an operand: channels 16 c + 8 half .. + 7 of this lane's row.  (On its way while pages are looked up: a step of 30 single tokens and pieces of 256 and 33, with a window, 45.9 -> 44.6 us.)
    u32x4 qw[NC];
    {
        const char* const at = p.q + (rq.start + token) * p.q_row + hq * p.q_head + 16 * half;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            qw[c] = u32x4{0, 0, 0, 0};
            if (live) qw[c] = *reinterpret_cast<const u32x4*>(at + 32 * c);
        }
    }
    if (t0 < n) {
        page = look_up(t0);
        page2 = look_up(t0 + 1);
        if constexpr (CODES) {
            load_codes(even, t0, page);
            load_codes(odd, t0 + 1, page2);
            page = look_up(t0 + 2);
            page2 = look_up(t0 + 3);
        } else {
            bring(t0, page, tile0, tile1);
            page = page2;
        }
    }

    V8 qf[NC];
#pragma unroll
    for (int c = 0; c < NC; ++c) qf[c] = __builtin_bit_cast(V8, qw[c] ^ p.flip);
    int k_at[NC], v_at[NB][2];
#pragma unroll
    for (int c = 0; c < NC; ++c) k_at[c] = L::at(lane, c);
#pragma unroll
    for (int b = 0; b < NB; ++b) { v_at[b][0] = L::at_transposed(lane, b, 0); v_at[b][1] = L::at_transposed(lane, b, 1); }

    f32x16 acc[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b) acc[b] = f32x16{};
    float m = kLowest, l = 0.f;       // (l: of this lane's half of the keys)
    float R = 0.f;                    // fp16 and codes: what weights are relative to, the largest scale of V so far that this lane's row sees, but for a factor of 64

    auto step = [&](int u, const char* kt, const char* vt, const float* st) __attribute__((always_inline)) {
        const int key0 = at_step(u) * kStep;
        if (key0 >= wave_end) return;
        if (WINDOW && key0 >= p.sinks && key0 + kStep <= wave_first) return;
        const bool behind = WINDOW && key0 < wave_from && key0 + kStep > p.sinks;      // (some row of the wavefront does not look back on all of these keys)
        f32x16 s[2] = {f32x16{}, f32x16{}};
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int h = 0; h < 2; ++h) s[h] = mfma32(read_rows<V8>(kt + 32 * h * L::ROW, k_at[c]), qf[c], s[h]);
        reads_ahead<2 * NC, 2 * NC, 8>();
        if constexpr (CODES) {
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const f32x4 by = *reinterpret_cast<const f32x4*>(st + 32 * h + 8 * i + 4 * half);
#pragma unroll
                    for (int j = 0; j < 4; ++j) s[h][4 * i + j] *= by[j];
                }
        }
        if (key0 + kStep > wave_all) {          // (some row of the wavefront does not see all of these keys)
            const int left = end - key0 - 4 * half;
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int e = 0; e < 16; ++e) s[h][e] = 32 * h + 8 * (e >> 2) + (e & 3) < left ? s[h][e] : -INFINITY;
        }
        if (behind) {
            const int out = from - key0 - 4 * half, in = p.sinks - key0 - 4 * half;
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int e = 0; e < 16; ++e) { const int j = 32 * h + 8 * (e >> 2) + (e & 3); s[h][e] = j >= out || j < in ? s[h][e] : -INFINITY; }
        }
        float top = s[0][0];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int e = 0; e < 16; ++e) top = fmaxf(top, s[h][e]);
        top = over_halves_max(top) * p.scale_log2;
        if (__any(top > m + kMaxSlack)) {
            const float to = fmaxf(m, top), by = __builtin_amdgcn_exp2f(m - to);
            m = to;
            l *= by;
#pragma unroll
            for (int b = 0; b < NB; ++b) acc[b] *= by;
        }
        float over = 1.f;
        if constexpr (CODES && __is_same(T, _Float16)) {
            // Weights p scale in fp16 would leave its range where values are small.  (A row's own keys alone say what they are relative to: those of a later token, whose values may be 2^25 times as large,
            // would make all of an earlier one's weights 0.  Steps in which no key is masked need not ask.)
            auto most_of = [&](auto masked) __attribute__((always_inline)) {
                float top = 0.f;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const f32x4 by = *reinterpret_cast<const f32x4*>(st + kStep + 8 * i + 4 * half);
#pragma unroll
                    for (int j = 0; j < 4; ++j) top = fmaxf(top, decltype(masked)::value && s[i / 4][4 * (i % 4) + j] == -INFINITY ? 0.f : by[j]);
                }
                return top;
            };
            float most = key0 + kStep > wave_all || behind ? most_of(Int<1>{}) : most_of(Int<0>{});
            if (__any(most > 64.f * R)) {
                most = fmaxf(fmaxf(R, over_halves_max(most)), 0x1p-100f);      // (far below what fp16 holds, and its reciprocal is a number)
                const float by = R / most;
#pragma unroll
                for (int b = 0; b < NB; ++b) acc[b] *= by;
                R = most;
            }
            over = R > 0.f ? 1.f / R : 1.f;
        }
        // (at head dim 64, with twice the exponentials to a product, the second half of a step goes before another wavefront's first)
        if constexpr (D == 64) __builtin_amdgcn_s_setprio(1);
        V8 pf[4];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                u32x4 w;
                f32x4 by[2];
                if constexpr (CODES) {
#pragma unroll
                    for (int i = 0; i < 2; ++i) by[i] = *reinterpret_cast<const f32x4*>(st + kStep + 32 * h + 16 * c + 8 * i + 4 * half);
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int e = 8 * c + 2 * i;
                    float a = __builtin_amdgcn_exp2f(__builtin_fmaf(s[h][e], p.scale_log2, -m)), b = __builtin_amdgcn_exp2f(__builtin_fmaf(s[h][e + 1], p.scale_log2, -m));
                    l += a;
                    l += b;
                    if constexpr (CODES) {
                        // (the factor first: a masked weight of 0 stays that beside a scale that is far above the row's own)
                        a = a * over * by[i / 2][2 * (i % 2)];
                        b = b * over * by[i / 2][2 * (i % 2) + 1];
                    }
                    w[i] = round2<T>(a, b);
                }
                pf[2 * h + c] = __builtin_bit_cast(V8, w);
            }
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int b = 0; b < NB; ++b) acc[b] = mfma32(read_channels<V8>(vt + 16 * c * L::ROW, v_at[b][0], v_at[b][1]), pf[c], acc[b]);
        if constexpr (D == 64) __builtin_amdgcn_s_setprio(0);
    };
    if constexpr (CODES) {
        // A step's codes are on their way while the two before are computed, and go to LDS during the one before.  (One step ahead two workgroups of a unit have half as many bytes under way: the pieces and
        // single tokens above, then all as tiles, 189 us, two steps ahead 160.)
        auto next = [&](Codes& codes, int& at, int u, char* kt, char* vt, float* st) __attribute__((always_inline)) {
            keep_codes(codes, kt, vt, st);
            load_codes(codes, u + 2, at);
            at = look_up(u + 4);
        };
        if (t0 < n) next(even, page, t0, tile0, tile1, scales0);
        for (int t = t0; t < n; t += 2) {
            meet_in_lds();
            if (t + 1 < n) next(odd, page2, t + 1, tile2, tile3, scales1);
            step(t, tile0, tile1, scales0);
            if (t + 1 == n) break;
            meet_in_lds();
            if (t + 2 < n) next(even, page, t + 2, tile0, tile1, scales0);
            step(t + 1, tile2, tile3, scales1);
        }
    } else {
        for (int t = t0; t < n; t += 2) {
            meet();
            if (t + 1 < n) { bring(t + 1, page, tile2, tile3); page = look_up(t + 2); }
            step(t, tile0, tile1, scales0);
            if (t + 1 == n) break;
            meet();
            if (t + 2 < n) { bring(t + 2, page, tile0, tile1); page = look_up(t + 3); }
            step(t + 1, tile2, tile3, scales0);
        }
    }
    if (!live) return;
    if constexpr (CODES && __is_same(T, _Float16)) {
#pragma unroll
        for (int b = 0; b < NB; ++b) acc[b] *= R;
    }
    l = over_halves_sum(l);
    if (f.parts > 1) {
        float* const part = p.parts + (((int64_t)block.index * p.Hkv + head) * p.most_parts + block.part) * kPartFloats<D> + (32 * wave + (lane & 31)) * (D + 2);
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int i = 0; i < 4; ++i) *reinterpret_cast<f32x2*>(part + 2 + 32 * b + 8 * i + 4 * half) = f32x2{acc[b][4 * i], acc[b][4 * i + 1]}, *reinterpret_cast<f32x2*>(part + 4 + 32 * b + 8 * i + 4 * half) = f32x2{acc[b][4 * i + 2], acc[b][4 * i + 3]};
        if (half == 0) *reinterpret_cast<f32x2*>(part) = f32x2{m, l};
        return;
    }
    float by = l > 0.f ? 1.f / l : l == 0.f ? 0.f : l;
    float lse = l > 0.f ? (m + __builtin_amdgcn_logf(l)) * 0.693147180559945309f : l == 0.f ? -INFINITY : l;
    if (f.n.lk < 0) by = lse = NAN;
    char* const at = p.o + (rq.start + token) * p.o_row + hq * p.o_head + 8 * half;
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int i = 0; i < 4; ++i)
            *reinterpret_cast<u32x2*>(at + 64 * b + 16 * i) = u32x2{round2<T>(acc[b][4 * i] * by, acc[b][4 * i + 1] * by), round2<T>(acc[b][4 * i + 2] * by, acc[b][4 * i + 3] * by)};
    if (p.lse && half == 0) p.lse[(rq.start + token) * p.lse_row + hq] = lse;
#endif
}

// ---- what was cut: the parts added up, in their order.  A workgroup for each key head and short sequence, behind these one for each key head and tile's 32 rows.  (256 threads: most workgroups find
// nothing to do, and 1024 threads each of them take two rounds of the chip; 62 tiles of 8 heads, few of them cut, 9 us instead of 20, and 10.4 with those that find nothing in between.  16 rows each: 9.8.)
constexpr int kJoinRows = 32;
template <typename T, int D, bool WINDOW>
__global__ void __launch_bounds__(kThreads) cache_chunk_join_kernel(const ChunkParams p) {
#if defined(__HIP_DEVICE_COMPILE__)
    constexpr int LANES = D / 8, AT_ONCE = kThreads / LANES, TILE_BLOCKS = kRows / kJoinRows;
    // (short sequences', then the tiles' in their order: what there is none of comes last)
    const int shorts = p.short_parts > 1 ? p.n_seq * p.Hkv : 0, lane = threadIdx.x % LANES, c = 8 * lane;
    const bool of_tile = (int)blockIdx.x >= shorts;
    const int b = of_tile ? blockIdx.x - shorts : blockIdx.x, head = b % p.Hkv, rest = b / p.Hkv, index = of_tile ? rest / TILE_BLOCKS : rest, row0 = of_tile ? rest % TILE_BLOCKS * kJoinRows : 0;
    const Found f = of_tile ? find<RowTilesOf<WINDOW, true>>(p, index) : find<ShortTiles<WINDOW>>(p, index);
    if (f.seq < 0 || f.parts <= 1) return;
    const Range rq = rows_of_sequence(p.cu_q, f.seq, f.n.lq);
    // (a part's rows lie apart: max and sum in front of a tile's D sums, behind all rows of a short one)
    const int first = of_tile ? f.tile * kRows : 0, rows = rq.length * p.group - first, size = of_tile ? kPartFloats<D> : kShortFloats<D>;
    const float* const sums = (of_tile ? p.parts + ((int64_t)index * p.Hkv + head) * p.most_parts * kPartFloats<D> + 2 : p.short_sums + ((int64_t)index * p.Hkv + head) * p.short_parts * kShortFloats<D>) + c;
    const float* const stat = of_tile ? sums - c - 2 : sums - c + kShortRows * D;
    const int row_floats = of_tile ? D + 2 : D, stat_floats = of_tile ? D + 2 : 2;
    for (int r = row0 + threadIdx.x / LANES; r < rows && r < row0 + kJoinRows; r += AT_ONCE) {
        float top = kLowest, sum = 0.f, o[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
        for (int s = 0; s < f.parts; ++s) top = fmaxf(top, stat[s * size + r * stat_floats]);
#pragma unroll 4
        for (int s = 0; s < f.parts; ++s) {
            const float* const at = sums + s * size + r * row_floats;
            const f32x2 st = *reinterpret_cast<const f32x2*>(stat + s * size + r * stat_floats);
            const float by = __builtin_amdgcn_exp2f(st[0] - top);
            sum += by * st[1];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const f32x2 x = *reinterpret_cast<const f32x2*>(at + 2 * i);
                o[2 * i] += by * x[0];
                o[2 * i + 1] += by * x[1];
            }
        }
        store_row<T>(p, rq.start, head, first + r, c, o, top, sum, false);
    }
#endif
}

// ---- C ABI
// tiles, and the parts that they may be cut into: as packed sequences of as many keys as a sequence may have; short sequences as well
constexpr int kLeastTile = 4, kLeastShort = 6;      // steps of a part
struct Cut { int64_t tiles; int parts, least, short_rows, short_parts, short_least; size_t bytes, short_bytes; };
Cut cut_of(const cosmos_attn_cache_desc* d, Window w) {
    const int64_t group = d->Hq / d->Hkv, tiles = most_tiles(d->rows * group, d->B), most = (int64_t)d->width * d->page_size;
    auto steps_of = [&](int step, int64_t tokens) {
        const int64_t all = (most + step - 1) / step, seen = ((int64_t)w.window + tokens) / step + 2 + ((int64_t)w.sinks + step - 1) / step;
        return w.window && seen < all ? seen : all;
    };
    Cut c = {};
    c.tiles = tiles;
    c.least = kLeastTile;
    // (no list of exactly the parts that there are: the search for it takes 4 us more in each workgroup)
    c.parts = group <= kShortRows && d->rows * group <= kShortRows ? 1 : most_parts(tiles * d->Hkv, steps_of(kStep, kRows / group + 1), c.least, false, 4 * kNumCUs);
    c.bytes = c.parts > 1 ? (size_t)tiles * d->Hkv * c.parts * kRows * (d->D + 2) * sizeof(float) : 0;
    if (group <= kShortRows && d->B) {
        c.short_rows = kShortRows;
        c.short_least = kLeastShort;
        c.short_parts = most_parts((int64_t)d->B * d->Hkv, steps_of(kShortStep, kShortRows), c.short_least);
        c.short_bytes = c.short_parts > 1 ? (size_t)d->B * d->Hkv * c.short_parts * kShortRows * (d->D + 2) * sizeof(float) : 0;
    }
    return c;
}
size_t workspace_of(const Cut& c) { return (c.bytes + 255) / 256 * 256 + c.short_bytes; }
int check_chunk(const cosmos_attn_cache_desc* d, int64_t window, int64_t sinks) {
    int st = check(d);
    if (st != COSMOS_ATTN_OK) return st;
    if (window < 0 || sinks < 0 || d->rows < 0 || d->Hq < 1 || !(fabsf(d->sm_scale) <= 3.0e38f)) return COSMOS_ATTN_BAD_ARG;
    if (d->Hq % d->Hkv) return COSMOS_ATTN_BAD_SHAPE;
    const int64_t group = d->Hq / d->Hkv;
    // (rows are 32-bit numbers, and so are the threads of a launch)
    if (d->rows > kMost || d->rows * group > kMost / 2 || (d->rows * group / kRows + 2 * (int64_t)d->B + 1) * d->Hkv > kMostBlocks / 2) return COSMOS_ATTN_UNSUPPORTED;
    if (!d->rows) return COSMOS_ATTN_OK;
    if (!d->cu || (d->B && !d->lens)) return COSMOS_ATTN_BAD_ARG;
    if (d->q_stride[0] * 2 > kMostRowBytes || d->o_stride[0] * 2 > kMostRowBytes) return COSMOS_ATTN_BAD_STRIDE;
    st = check_rows(d->q, d->q_stride);
    if (st == COSMOS_ATTN_OK) st = check_out(d->o, d->o_stride, d->rows, d->Hq, d->D);
    return st != COSMOS_ATTN_OK ? st : check_in_place(d, d->rows);
}

}  // namespace

extern "C" {

size_t cosmos_attn_cache_chunk_workspace_bytes(const cosmos_attn_cache_desc* desc, int64_t window, int64_t sinks) {
    return check_chunk(desc, window, sinks) == COSMOS_ATTN_OK && desc->rows ? workspace_of(cut_of(desc, window_of(desc, window, sinks))) : 0;
}

int cosmos_attn_cache_chunk(const cosmos_attn_cache_desc* desc, int64_t window, int64_t sinks, void* workspace, size_t workspace_bytes, void* stream) {
    const int st = check_chunk(desc, window, sinks);
    if (st != COSMOS_ATTN_OK || !desc->rows) return st;
    const Window w = window_of(desc, window, sinks);
    const Cut cut = cut_of(desc, w);
    const size_t wanted = workspace_of(cut);
    if (workspace_bytes < wanted || (wanted && !workspace)) return COSMOS_ATTN_WORKSPACE_TOO_SMALL;
    if (wanted && !aligned16(workspace)) return COSMOS_ATTN_BAD_STRIDE;
    if (!device_is_whole_mi355x()) return COSMOS_ATTN_WRONG_DEVICE;
    const CacheParams c = params_of(desc);
    ChunkParams p = {};
    p.q = (const char*)desc->q; p.o = (char*)desc->o; p.lse = desc->lse;
    p.cu_q = desc->cu; p.lens = desc->lens;
    p.q_row = 2 * desc->q_stride[0]; p.q_head = 2 * desc->q_stride[1]; p.o_row = 2 * desc->o_stride[0]; p.o_head = 2 * desc->o_stride[1];
    p.lse_row = desc->Hq; p.lse_head = 1;
    p.n_seq = desc->B; p.Tq = (int)desc->rows; p.Hkv = desc->Hkv; p.group = desc->Hq / desc->Hkv; p.causal = 1;
    p.fill = desc->fill == COSMOS_ATTN_FILL_LSE && !desc->lse ? 0 : desc->fill;
    p.tiles = (int)cut.tiles; p.most_parts = cut.parts; p.least = cut.least;
    p.window = w.window; p.sinks = w.sinks;
    p.most_keys = desc->width * desc->page_size;
    p.parts = (float*)workspace;
    p.short_rows = cut.short_rows; p.short_parts = cut.short_parts; p.short_least = cut.short_least;
    p.short_blocks = cut.short_rows ? desc->B * desc->Hkv * cut.short_parts : 0;
    p.short_sums = (float*)((char*)workspace + wanted - cut.short_bytes);
    p.scale = desc->sm_scale;
    p.scale_log2 = fmaxf(fabsf(desc->sm_scale) * 1.44269504088896341f, 1e-37f);      // (a masked score of -inf stays that)
    p.flip = signbit(desc->sm_scale) ? 0x80008000u : 0u;
    p.side[0] = c.side[0]; p.side[1] = c.side[1];
    p.table = desc->table; p.table_row = desc->table_stride; p.pages = (int)desc->pages; p.page_shift = c.page_shift;
    return with_type(desc, [&](auto* t, auto dim, auto kind) {
        typedef std::remove_pointer_t<decltype(t)> T;
        constexpr int D = decltype(dim)::value, K = decltype(kind)::value;
        auto run = [&](auto windowed) {
            constexpr bool WINDOW = decltype(windowed)::value;
            const int done = launch(cache_chunk_kernel<T, K, D, WINDOW>, cut.tiles * p.Hkv * cut.parts + p.short_blocks, 0, p, stream);
            const int64_t joins = (cut.parts > 1 ? cut.tiles * p.Hkv * (kRows / kJoinRows) : 0) + (cut.short_parts > 1 ? (int64_t)p.n_seq * p.Hkv : 0);
            return done != COSMOS_ATTN_OK ? done : launch(cache_chunk_join_kernel<T, D, WINDOW>, joins, 0, p, stream);
        };
        return w.window ? run(Int<1>{}) : run(Int<0>{});
    });
}

}  // extern "C"
