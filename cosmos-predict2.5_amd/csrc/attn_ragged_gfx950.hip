// Attention over packed sequences of different lengths with grouped heads, forward and backward, for gfx950: kernels and C ABI (cosmos_attn_ragged, cosmos_attn_ragged_bwd).
//
// Sequence i has the rows cu_q[i] .. cu_q[i + 1] - 1 of q and the rows cu_k[i] .. of k and v.  With c the scale, t and j counted from the sequence's start, Lq and Lk its lengths:
//     s_tj = c q_t k_j,   visible: j <= t + Lk - Lq (causal, aligned at the ends) or all,   p = exp(s - lse),   o_t = sum_j p_tj v_j,   lse_t = log sum_j exp(s_tj)
//     dp_tj = do_t v_j,   delta_t = sum_d do_t o_t,   ds = p (dp - delta),   dq_t = c sum_j ds_tj k_j,   dk_j = c sum_t ds_tj q_t,   dv_j = sum_t p_tj do_t
// A row that sees no key: o = 0, lse = -inf, no gradient.
//
// Grouped heads.  The `group` query heads of a key head are rows of one matrix: row r of sequence i and key head h is token r / group, query head h group + r % group.  A tile of
// rows then shares K and V among the heads, few tokens still fill a tile, a causal tile's diagonal is `group` times shorter, and the sums over the group that dk and dv need
// are part of the contraction over rows.
//
// Who does what.  Lengths stay on the device: the grid is what the tensors' row counts allow at most, and every workgroup finds its tile from the offsets (each wavefront for itself).  No work
// list, no copy to the host, nothing to prepare, and a captured call follows its offsets.  Where a call has few tiles, those with more than an equal share of all steps are cut along
// their keys (rows), and a second kernel adds the parts up, in their order.
//
// Offsets are not trusted: a sequence whose offsets do not ascend within the tensors, or that begins before the end of an earlier one, has no rows; one whose keys' offsets are such has rows of
// NaN (no gradients: zeros).  Rows that no sequence is left for are those of no sequence.  No two sequences then have a row or a key in common, whatever the offsets hold: each row is one workgroup's to write, and there are never more tiles than workgroups.
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

constexpr int kThreads = 256;      // four wavefronts of 32 rows (or keys) each
constexpr int kRows = 128;         // of a workgroup
constexpr int kStep = 64;          // keys (or rows) that are in LDS at a time, twice

struct RaggedParams {
    const char *q, *k, *v, *o_in, *dout;
    char *o, *dq, *dk, *dv;
    float* lse;                    // [Hq, Tq]; written by the forward (may be null), read by the backward
    char* rest;                    // [Tq, Hq, D]: what rounding o left off, 16 bits again (may be null)
    float* delta;                  // [Hq, Tq]: of the backward's first kernel for its second
    const int *cu_q, *cu_k;
    // bytes between rows and between heads
    int64_t q_row, q_head, k_row, k_head, v_row, v_head, o_row, o_head, do_row, do_head, dq_row, dq_head, dk_row, dk_head, dv_row, dv_head;
    int n_seq, Tq, Tk, Hkv, group, causal, fill;
    int tiles, most_parts, least;  // tiles that there may be, parts that one may be cut into, steps of a part
    float* parts;                  // what they leave: of part s of tile i and key head h, at (i Hkv + h) most_parts + s
    float scale, scale_log2;       // scale_log2 >= 0: `flip` says that q's signs are turned instead
    unsigned flip;
};

// ---- a tile in LDS: N rows of D 16-bit elements, as chunks of 16 bytes.  Chunk c of row r lies at c XOR mix(r): what a wavefront reads at once, 16 bytes of each of 32 rows (a fragment
// with lane = row) or, transposing, 64 bytes of each of 8 rows, then lies in different banks, and a load to LDS still takes whole rows.
template <int D, int N = kStep> struct Tile {
    static constexpr int ROW = 2 * D, BYTES = N * ROW, CHUNKS = D / 8, ROWS_PER_LOAD = 1024 / ROW, LOADS = N / 4 / ROWS_PER_LOAD;
    static __device__ __forceinline__ int mix(int r) { return D == 128 ? 4 * (r & 3) | ((r >> 2) & 3) : 4 * ((r >> 1) & 1) | ((r >> 2) & 3); }
    // where lane reads chunk 2 c + lane / 32 of row lane % 32
    static __device__ __forceinline__ int at(int lane, int c) { return (lane & 31) * ROW + ((((2 * c) | (lane >> 5)) ^ mix(lane & 31)) << 4); }
    // where lane passes the address for channels 32 db .. + 31, rows 4 (lane / 32) .. + 3 + 8 s, transposing
    static __device__ __forceinline__ int at_transposed(int lane, int db, int s) {
        const int row = 8 * s + 4 * (lane >> 5) + ((lane & 15) >> 2), chunk = 4 * db + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
        return row * ROW + ((chunk ^ mix(row)) << 4) + 8 * (lane & 1);
    }
    // the row (of the tile) and the byte in that row that this lane loads with load i of wavefront `wave`
    static __device__ __forceinline__ int load_row(int lane, int wave, int i) { return N / 4 * wave + i * ROWS_PER_LOAD + lane / CHUNKS; }
    static __device__ __forceinline__ int load_byte(int lane, int wave, int i) { return ((lane % CHUNKS) ^ mix(load_row(lane, wave, i))) << 4; }
    static __device__ __forceinline__ int load_to(int wave, int i) { return (N / 4 * wave + i * ROWS_PER_LOAD) * ROW; }
};

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
// of a tile's part: its rows' max, sum of exponentials and D sums
template <int D> constexpr int kPartFloats = kRows * (D + 2);

__device__ __forceinline__ void load_to_lds(__amdgpu_buffer_rsrc_t rsrc, char* dst, int offset) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (__attribute__((address_space(3))) void*)dst, 16, offset, 0, 0, 0);
}
template <typename V8> __device__ __forceinline__ V8 read_rows(const char* part, int at) { return *reinterpret_cast<const V8*>(part + at); }
// the 16 rows 16 c .. + 15 of 32 channels as an operand with lane = channel: slot s of a lane is row 16 c + 8 (s / 4) + 4 (lane / 32) + s % 4, the order of a product's result registers
template <typename V8> __device__ __forceinline__ V8 read_channels(const char* part, int at0, int at1) {
    typedef __attribute__((address_space(3))) s16x4* P;
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((P)(part + at0)), hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((P)(part + at1));
    return __builtin_bit_cast(V8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
}
// Two pairs of tiles, the one read while the other is loaded.  Arrays of their own: the compiler waits for loads to LDS in front of a read that may be of the same array.
#define LDS_TILES(L) __shared__ __attribute__((aligned(1024))) char tile0[L::BYTES], tile1[L::BYTES], tile2[L::BYTES], tile3[L::BYTES]
// all loads to LDS have landed and all reads have returned; then the workgroup meets.  (Through the builtin, which the compiler counts with: it then waits for nothing else in front of reads.)
constexpr int kNothingUnderWay = 0x0070;      // vmcnt 0, lgkmcnt 0
__device__ __forceinline__ void meet() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(kNothingUnderWay);
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}
// `rows_left` rows from `at` on (at most N are read), what lies behind them reads as zeros
template <int D, int N = kStep> __device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_of(const char* at, int64_t row_bytes, int rows_left) {
    const int rows = rows_left < N ? rows_left : N;
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(at), 0, rows > 0 ? (int)((rows - 1) * row_bytes) + 2 * D : 0, 0x00020000);
}
// four elements of o, and what their rounding leaves off.  The backward's delta = dout . o is taken off every dP of a row, next to which it is large where a row's weight lies on few keys:
// with o's 8 bits alone dq and dk of sharp softmaxes (scores of a deviation of 4, 1000 positions, bf16) are 3.6e-3 off, with 16 bits 2.5e-3; their own rounding is 1.7e-3.
template <typename T> __device__ __forceinline__ float element(unsigned w, int i) {
    typedef T V2 __attribute__((ext_vector_type(2)));
    return (float)__builtin_bit_cast(V2, w)[i];
}
template <typename T> __device__ __forceinline__ void store_rounded(char* to, char* rest, float a, float b, float c, float d) {
    u32x2 w = {round2<T>(a, b), round2<T>(c, d)};
    *reinterpret_cast<u32x2*>(to) = w;
#if defined(__HIP_DEVICE_COMPILE__)
    asm("" : "+v"(w));      // (what is stored: left to itself the compiler rounds a second time, a product of fp16 then in one step with the multiplication, which next to a tie goes elsewhere)
#endif
    if (rest) *reinterpret_cast<u32x2*>(rest) = u32x2{round2<T>(a - element<T>(w[0], 0), b - element<T>(w[0], 1)), round2<T>(c - element<T>(w[1], 0), d - element<T>(w[1], 1))};
}
// dS in fp16.  P is about one over the number of keys and dP as large as dout, so that dS = P (dP - delta) leaves fp16's range downwards (2^-14) where dq and dk are well within it (4096 keys,
// dout 1e-3: they would be 5e-3 off), and upwards (65504) where dout is scaled up and weights lie on few keys.  It is held as 2^up dS: `up` begins at kUp and
// goes down whenever one is above kMostDs, so that the largest so far lies between 2^8 and 2^9; what is summed up is scaled with it.  A row (dq) or a key (dk) has its own.  bf16 has the range
// of fp32.
// (Gradients in fp16 take 3 % longer at head dim 128, 5 at 64: four documents of 7678 positions, 32 heads on 8, us, without / with 789 / 814; 8192 positions, 16 heads of 64, 570 / 598.)
template <typename T> constexpr bool kNarrow = __is_same(T, _Float16);
constexpr int kUp = 48;
// P as dv's operand, which is 1 at most and below 2^-14 from some 16 000 keys on, is 2^kUpP P throughout.
constexpr int kUpP = 14;
constexpr float kMostDs = 16384.f;
__device__ __forceinline__ float largest(f32x16 s) {
    float top = fabsf(s[0]);
#pragma unroll
    for (int e = 1; e < 16; ++e) top = fmaxf(top, fabsf(s[e]));
    return top;
}
// how far down, in powers of two, for a largest one of `top`
__device__ __forceinline__ int too_many(float top) { return top > kMostDs && top < INFINITY ? __builtin_amdgcn_frexp_expf(top) - 9 : 0; }
__device__ __forceinline__ float power_of_two(int n) { return __builtin_amdgcn_ldexpf(1.f, n); }
// The order of a block's LDS reads and matrix products, READS to PRODUCTS: AHEAD reads first, then each product with its share of the others.  (Left alone the compiler reads the operands of two
// products and waits for them: 2 % of the forward, and of the dK/dV kernel, where no more registers are free for it.)
template <int READS, int PRODUCTS, int AHEAD> __device__ __forceinline__ void reads_ahead() {
#if defined(__HIP_DEVICE_COMPILE__)
    constexpr int FIRST = AHEAD < READS ? AHEAD : READS, PER = READS / PRODUCTS, WITH = (READS - FIRST) / PER;
    __builtin_amdgcn_sched_group_barrier(0x100, FIRST, 0);
#pragma unroll
    for (int i = 0; i < WITH; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, PER, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x008, PRODUCTS - WITH, 0);
#endif
}
__device__ __forceinline__ float over_halves_sum(float x) { float lo, hi; both_halves(x, lo, hi); return lo + hi; }
__device__ __forceinline__ float over_halves_max(float x) { float lo, hi; both_halves(x, lo, hi); return fmaxf(lo, hi); }

// ---- which sequence
struct Range { int start, length; };
__device__ __forceinline__ Range range_of(const int* cu, int i, int total) {
    const int a = cu[i], b = cu[i + 1];
    return a >= 0 && a <= b && b <= total ? Range{a, b - a} : Range{0, -1};
}
// the rows of sequence i, of which find() says how many there are
__device__ __forceinline__ Range rows_of_sequence(const int* cu, int i, int length) { return {length < 0 ? 0 : cu[i], length}; }
// Where offsets do not ascend throughout, a sequence may begin before the end of an earlier one.  Of the 64 from `base` on, in a lane each: the length, -1 where it has none of its own, and the
// end of the last one in front of it; `end`: of the last one so far.  Empty ones hold nothing and are passed over.  If no start lies before an end in front of it, all of them are sequences
// (500 prompts of 30 positions and 500 offsets of zero behind them, 32 heads of 128 on 8, forward and gradients 345 and 749 us, one
// after the other 3085 and 6096; the last offset again instead of zeros, which ascends, 134 and 347); if not, one after the other, as each depends on those in front.
struct Own { int start, length, before; };
template <int CTRL, int ROWS> __device__ __forceinline__ int dpp_most(int v) {
    const int moved = __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xF, false);      // (0 where no lane is)
    return v > moved ? v : moved;
}
__device__ __forceinline__ Own apart(const int* cu, int base, int n_seq, int total, int& end) {
    const int lane = threadIdx.x & 63;
    const Range r = base + lane < n_seq ? range_of(cu, base + lane, total) : Range{0, -1};
    int most = r.length > 0 ? r.start + r.length : 0;      // of the ends up to this lane
    most = dpp_most<0x111, 0xF>(most);
    most = dpp_most<0x112, 0xF>(most);
    most = dpp_most<0x114, 0xF>(most);
    most = dpp_most<0x118, 0xF>(most);
    most = dpp_most<0x142, 0xA>(most);
    most = dpp_most<0x143, 0xC>(most);
    const int front = __shfl_up(most, 1), last = __builtin_amdgcn_readlane(most, 63);
    Own own = {r.start, r.length, lane && front > end ? front : end};
    if (!__any(r.length > 0 && r.start < own.before)) {
        end = last > end ? last : end;
        return own;
    }
    for (unsigned long long left = __ballot(r.length > 0); left; left &= left - 1) {
        const int at = __builtin_ctzll(left), a = __builtin_amdgcn_readlane(r.start, at);
        if (lane == at) own = {a, a < end ? -1 : r.length, end};
        if (a >= end) end = a + __builtin_amdgcn_readlane(r.length, at);
    }
    return own;
}

// The tiles of a kernel: ROWS rows (or keys) of a sequence each, with `steps` of STEP keys (rows) that go by.  Rank 0 of a sequence's tiles is the longest one; the last rows
// see the most keys, the first keys are seen by the most rows.
struct Lengths { int lq, lk; };      // lq < 0 or lk < 0: bad offsets
template <bool KEYS, int ROWS, int STEP> struct Tiles {
    const RaggedParams& p;
    __device__ __forceinline__ Lengths lengths(int i) const { return {range_of(p.cu_q, i, p.Tq).length, range_of(p.cu_k, i, p.Tk).length}; }
    __device__ __forceinline__ int count(Lengths n) const {
        const int64_t rows = KEYS ? n.lk : (int64_t)n.lq * p.group;
        return rows > 0 ? (int)((rows + ROWS - 1) / ROWS) : 0;
    }
    static __device__ __forceinline__ int at(int rank, int tiles) { return KEYS ? rank : tiles - 1 - rank; }
    // first row that sees key j, in rows; (rounded up to steps where none does)
    __device__ __forceinline__ int first_row(Lengths n, int j) const {
        const int lq = n.lq > 0 ? n.lq : 0, t = j - (n.lk - lq);
        return !p.causal || t <= 0 ? 0 : t >= lq ? (lq * p.group + STEP - 1) / STEP * STEP : t * p.group;
    }
    // keys that row r's token sees
    __device__ __forceinline__ int keys(Lengths n, int r) const {
        const int lk = n.lk > 0 ? n.lk : 0, e = r / p.group + lk - n.lq + 1;
        return !p.causal || e > lk ? lk : e < 0 ? 0 : e;
    }
    __device__ __forceinline__ int first_step(Lengths n, int tile) const { return KEYS ? first_row(n, tile * ROWS) / STEP : 0; }
    __device__ __forceinline__ int end_step(Lengths n, int tile) const {
        if (KEYS) return n.lq > 0 ? (n.lq * p.group + STEP - 1) / STEP : 0;
        const int rows = n.lq * p.group, last = tile * ROWS + ROWS - 1;
        return (keys(n, last < rows ? last : rows - 1) + STEP - 1) / STEP;
    }
    __device__ __forceinline__ int steps(Lengths n, int tile) const { return end_step(n, tile) - first_step(n, tile); }
    static constexpr bool OF_KEYS = KEYS;
};

// Parts are written and read in fp32 and joined by a launch of its own, so they have `least` steps at least.  dk and dv, and where shares are large: parts of three fifths of a workgroup's
// share of all steps, as 512 causal tiles are dealt out evenly only if the long ones are in pieces that short ones fit beside (gradients of 16384 positions, 16 heads on 4, us, parts of a
// share / of 3/5 / of 2/5: 4558 / 3973 / 3890).  Else five quarters, which are all on the chip at once: a few more than fit take a second round (512 queries, 8 heads each, on 8192 keys: 704
// parts 72, 520 75, 455 63).  On other sizes, us, this rule / five quarters throughout, forward and gradients: 3000 + 1700 + 1040 positions, 16 heads on 4, 109 / 95 and 311 / 285; 4096 108 / 105 and
// 323 / 309; 1024 queries on 8192 keys, 16 heads on 2, 94 / 91 and 306 / 297; 512 on 32768, 8 heads on 1, 84 / 89 and 302 / 298; 8192, 8 heads on 2, 178 / 177 and 548 / 548.
constexpr int kAtOnce = 2 * kNumCUs;      // workgroups
constexpr int least_steps(int D) { return D == 128 ? 12 : 24; }
constexpr int least_rows(int D) { return D == 128 ? 512 : 2048; }       // (of dk and dv, in rows)
typedef Tiles<false, kRows, kStep> RowTiles;
// of dk and dv
constexpr int row_step(int D) { return D == 128 ? 32 : 64; }
template <int D> using KeyTiles = Tiles<true, kRows, row_step(D)>;
struct Found { int seq, tile, parts; Lengths n; bool odd; };     // seq < 0: behind the last tile, `tile` of them; odd: offsets that do not ascend were among those looked at
// Tile `index` of all sequences', in the sequences' order and the longest of each first, and how many parts it is cut into.
// (The longest of all first, by counts of the tiles longer than some length, for which the length is searched: 5 % slower on 12 prompts and on four documents.  Short tiles, which are mostly
// waiting, then run beside each other at the end instead of beside long ones.)
// Few sequences each wavefront looks through for itself, 64 at a time; more of them the workgroup's THREADS together (1000 prompts of 30 positions, 32 heads of 128 on 8, us, forward / gradients,
// together 238 / 565, each wavefront for itself 315 / 650; but 100 of them 24 / 101, and 24 / 93).
constexpr int kFew = 128;
template <typename Kind, int THREADS = kThreads> __device__ __forceinline__ Found find(const RaggedParams& p, int index) {
    constexpr bool KEYS = Kind::OF_KEYS;
    const Kind T{p};
    const int lane = threadIdx.x & 63;
    Found f = {-1, 0, 1, {0, 0}, false};
    // (a sequence's: all of its tiles times the mean of the longest and the shortest; as many of them as are added up in 32 bits are no more than those hold)
    auto share_of = [&](Lengths n, int tiles, int most) {
        const int64_t sum = tiles ? (int64_t)tiles * (T.steps(n, T.at(0, tiles)) + T.steps(n, T.at(tiles - 1, tiles))) / 2 : 0;
        return (int)(sum < most ? sum : most);
    };
    int before = 0;
    int64_t all = 0;                 // steps
    auto lengths = [&](int i) { return i < p.n_seq ? T.lengths(i) : Lengths{-1, -1}; };
    auto is_odd = [&](int i, Lengths n) { return i < p.n_seq && (n.lq < 0 || n.lk < 0); };
    // 64 sequences from `base` on; is that all there is to know?
    auto look = [&](int base, Lengths n) __attribute__((always_inline)) {
        const int tiles = T.count(n), sum = sums_up_to(tiles);
        const unsigned long long past = __ballot(before + sum > index);
        if (past && f.seq < 0) {
            const int at = __builtin_ctzll(past), of = __builtin_amdgcn_readlane(tiles, at);
            f.seq = base + at;
            f.n = {__builtin_amdgcn_readlane(n.lq, at), __builtin_amdgcn_readlane(n.lk, at)};
            f.tile = T.at(index - (before + __builtin_amdgcn_readlane(sum, at) - of), of);
            if (p.most_parts <= 1) return true;
        }
        before += __builtin_amdgcn_readlane(sum, 63);
        if (p.most_parts > 1) all += sum_of(share_of(n, tiles, (1 << 25) - 1));
        return false;
    };
    if (p.n_seq <= kFew) {
        for (int base = 0; base < p.n_seq; base += 64) {
            const Lengths n = lengths(base + lane);
            if (__any(is_odd(base + lane, n))) { f.odd = true; break; }
            if (look(base, n)) return f;
        }
    } else {
        constexpr int WAVES = THREADS / 64, ODD = 1 << 26;      // (more than there are tiles)
        __shared__ int sums[2][WAVES];
        __shared__ int64_t shares[WAVES];
        __shared__ Found found;
        const int wave = threadIdx.x >> 6;
        for (int base = 0, turn = 0; base < p.n_seq; base += THREADS, turn ^= 1) {
            const int mine = base + threadIdx.x;
            const Lengths n = lengths(mine);
            const int tiles = T.count(n), sum = sums_up_to(tiles);
            const bool odd = __any(is_odd(mine, n));
            if (lane == 63) sums[turn][wave] = odd ? ODD : sum;
            if (p.most_parts > 1) all += sum_of(share_of(n, tiles, (1 << 25) - 1));
            __syncthreads();
            int at = before + sum - tiles, past = before;
#pragma unroll
            for (int w = 0; w < WAVES; ++w) {
                at += w < wave ? sums[turn][w] : 0;
                past += sums[turn][w];
            }
            if (__builtin_amdgcn_readfirstlane(past) >= ODD) { f.odd = true; break; }
            if (f.seq < 0 && index < past) {
                if (index >= at && index < at + tiles) found = {mine, T.at(index - at, tiles), 1, n, false};
                f.seq = 0;           // (it is in `found`)
                if (p.most_parts <= 1) break;
            }
            before = past;
        }
        if (!f.odd) {
            if (lane == 0) shares[wave] = all;
            __syncthreads();
            if (f.seq >= 0) {
                f = {__builtin_amdgcn_readfirstlane(found.seq), __builtin_amdgcn_readfirstlane(found.tile), 1, {__builtin_amdgcn_readfirstlane(found.n.lq), __builtin_amdgcn_readfirstlane(found.n.lk)}, false};
                if (p.most_parts <= 1) return f;
                all = 0;
#pragma unroll
                for (int w = 0; w < WAVES; ++w) all += shares[w];
            }
        }
    }
    if (f.odd) {                     // once more from the start, each wavefront for itself
        int end_q = 0, end_k = 0;
        f.seq = -1;
        before = 0;
        all = 0;
        for (int base = 0; base < p.n_seq; base += 64)
            if (look(base, {apart(p.cu_q, base, p.n_seq, p.Tq, end_q).length, apart(p.cu_k, base, p.n_seq, p.Tk, end_k).length})) return f;
    }
    if (f.seq < 0) { f.tile = index - before; return f; }
    const int64_t share = (all * p.Hkv + kAtOnce - 1) / kAtOnce;
    const int steps = T.steps(f.n, f.tile);
    const int64_t wish = KEYS || share >= 2 * p.least ? 3 * share / 5 : 5 * share / 4;
    const int per = wish > p.least ? (int)wish : p.least, parts = (steps + per - 1) / per;
    f.parts = __builtin_amdgcn_readfirstlane(parts < 1 ? 1 : parts < p.most_parts ? parts : p.most_parts);
    return f;
}
// Of block `b`: the key head, the tile's place among all, the part.  Last parts first, which only long tiles have, and all tiles' first parts at the end, so that short tiles end the call.
// Parts of one number lie together: a die hands workgroups to its four shader engines in turn, and parts that are
// not there (their workgroups end at once) among the others leave some engines with nothing else: 37 us became 54 on 368 tiles of 25 steps.
struct Block { int head, index, part; };
__device__ __forceinline__ Block block_of(const RaggedParams& p, int b) {
    const int rest = b / p.Hkv, before = p.most_parts > 1 ? rest / p.tiles : 0;
    return {b - rest * p.Hkv, rest - before * p.tiles, p.most_parts - 1 - before};
}

// ---- rows of no sequence: zeros, lse = -inf.  They are counted through, whatever lies between them, and a workgroup behind the last tile has `rows` of them.
template <int D> __device__ __forceinline__ void clear_rows(char* out, int64_t row, int64_t head, const int* cu, int n, int total, int heads, int first_head, int rows, Found f, float* lse) {
    constexpr int CHUNKS = D / 8;
    int64_t first = (int64_t)f.tile * rows;      // the workgroup's first one, counted from the next row to be cleared
    auto clear = [&](int from, int to) {         // the tensor's rows from .. to - 1
        const int64_t count = (int64_t)(to - from) * heads, lo = first < 0 ? 0 : first, hi = first + rows < count ? first + rows : count;
        for (int i = threadIdx.x; i < (hi - lo) * CHUNKS; i += kThreads) {
            const int64_t r = lo + i / CHUNKS;
            const int t = from + (int)(r / heads), h = first_head + (int)(r % heads);
            if (out) *reinterpret_cast<u32x4*>(out + t * row + h * head + 16 * (i % CHUNKS)) = u32x4{0, 0, 0, 0};
            if (lse && i % CHUNKS == 0) lse[(int64_t)h * total + t] = -INFINITY;
        }
        first -= count;
    };
    if (!f.odd) {
        int lead = cu[0], from = cu[n];
        lead = lead < 0 ? 0 : lead > total ? total : lead;
        from = from < lead ? lead : from > total ? total : from;
        clear(0, lead);
        clear(from, total);
        return;
    }
    // (between the sequences that there are as well)
    int end = 0;
    for (int base = 0; base < n && first > -rows; base += 64) {
        const Own own = apart(cu, base, n, total, end);
        for (unsigned long long left = __ballot(own.length > 0 && own.start > own.before); left; left &= left - 1) {
            const int at = __builtin_ctzll(left);
            clear(__builtin_amdgcn_readlane(own.before, at), __builtin_amdgcn_readlane(own.start, at));
        }
    }
    if (first > -rows) clear(end, total);
}

constexpr float kLowest = -3.0e38f;      // a max that no score has moved yet: exponentials of masked scores stay 0 and those of the sums so far too

// ---- forward.  A workgroup: kRows rows of one sequence and key head; a wavefront 32 of them, one a lane and its other half: S^T = K Q^T has the keys in registers, so that the softmax
// needs one exchange between the halves, and P^T, rounded, is the next product's operand where it lies.  Two workgroups a compute unit (head dim 64: four), so that one's products and another's
// exponentials go on beside each other.  16384 causal positions, 16 heads of 128 on 4: 950 to 1000 us, 1.1 to 1.15 PFLOP/s, the matrix unit busy 63 % of the time at 1.8 GHz: every product of
// 32 x 32 x 16 has a fragment from LDS to itself, which a stream of such products alone runs at 1.09 to 1.15 PFLOP/s with.  Head dim 64: 8192 positions, 16 heads, 297 us, 0.92 PFLOP/s (causal 187,
// 0.73).  Short calls end with their longest tiles: 12 causal prompts of 1 to 2048 positions, 32 heads on 8, 125 us, 0.77 PFLOP/s, 84 % of the units busy.
template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 2) ragged_fwd_kernel(const RaggedParams p) {
#if defined(__HIP_DEVICE_COMPILE__)
    typedef typename VecOf<T>::v8 V8;
    typedef Tile<D> L;
    constexpr int NC = D / 16, NB = D / 32;
    LDS_TILES(L);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5;
    const Block block = block_of(p, blockIdx.x);
    const int head = block.head;
    const Found f = find<RowTiles>(p, block.index);
    if (f.seq < 0) {
        if (p.fill && block.part == 0) clear_rows<D>(p.fill == COSMOS_ATTN_FILL_LSE ? nullptr : p.o, p.o_row, p.o_head, p.cu_q, p.n_seq, p.Tq, p.group, head * p.group, kRows, f, p.lse);
        return;
    }
    if (block.part >= f.parts) return;
    const int tile = f.tile;
    const Range rq = rows_of_sequence(p.cu_q, f.seq, f.n.lq), rk = rows_of_sequence(p.cu_k, f.seq, f.n.lk);
    const int rows = rq.length * p.group, lk = rk.length > 0 ? rk.length : 0, shift = lk - rq.length;
    const int row = tile * kRows + 32 * wave + (lane & 31);
    const bool live = row < rows;
    const int token = row / p.group, hq = head * p.group + (row - token * p.group);
    // keys that this lane's row sees, the most of this wavefront's and of the workgroup's rows, the fewest of this wavefront's
    auto keys_of = [&](int t) { const int e = t + shift + 1; return !p.causal || e > lk ? lk : e < 0 ? 0 : e; };
    const int end = live ? keys_of(token) : 0;
    const int first = tile * kRows + 32 * wave;
    auto token_at = [&](int r) { return __builtin_amdgcn_readfirstlane((r < rows ? r : rows - 1) / p.group); };
    const int wave_end = first < rows ? keys_of(token_at(first + 31)) : 0, wave_all = keys_of(token_at(first));
    // steps of this part
    const int steps = RowTiles{p}.end_step(f.n, tile);
    const int t0 = (int)((int64_t)block.part * steps / f.parts), n = (int)((int64_t)(block.part + 1) * steps / f.parts);

    const char* const kp = p.k + rk.start * p.k_row + head * p.k_head;
    const char* const vp = p.v + rk.start * p.v_row + head * p.v_head;
    int k_off[L::LOADS], v_off[L::LOADS];
#pragma unroll
    for (int i = 0; i < L::LOADS; ++i) {
        k_off[i] = L::load_row(lane, wave, i) * (int)p.k_row + L::load_byte(lane, wave, i);
        v_off[i] = L::load_row(lane, wave, i) * (int)p.v_row + L::load_byte(lane, wave, i);
    }
    auto fill = [&](int t, char* kt, char* vt) __attribute__((always_inline)) {
        const auto kr = rows_of<D>(kp + (int64_t)t * kStep * p.k_row, p.k_row, lk - t * kStep), vr = rows_of<D>(vp + (int64_t)t * kStep * p.v_row, p.v_row, lk - t * kStep);
#pragma unroll
        for (int i = 0; i < L::LOADS; ++i) load_to_lds(kr, kt + L::load_to(wave, i), k_off[i]);
#pragma unroll
        for (int i = 0; i < L::LOADS; ++i) load_to_lds(vr, vt + L::load_to(wave, i), v_off[i]);
    };
    if (t0 < n) fill(t0, tile0, tile1);

    // Q as an operand: channels 16 c + 8 half .. + 7 of this lane's row
    V8 qf[NC];
    {
        const char* const at = p.q + (rq.start + token) * p.q_row + hq * p.q_head + 16 * half;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            u32x4 w = {0, 0, 0, 0};
            if (live) w = *reinterpret_cast<const u32x4*>(at + 32 * c);
            w ^= p.flip;
            qf[c] = __builtin_bit_cast(V8, w);
        }
    }
    int k_at[NC], v_at[NB][2];
#pragma unroll
    for (int c = 0; c < NC; ++c) k_at[c] = L::at(lane, c);
#pragma unroll
    for (int b = 0; b < NB; ++b) { v_at[b][0] = L::at_transposed(lane, b, 0); v_at[b][1] = L::at_transposed(lane, b, 1); }

    f32x16 acc[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b) acc[b] = f32x16{};
    float m = kLowest, l = 0.f;       // (l: of this lane's half of the keys)

    auto step = [&](int t, const char* kt, const char* vt) __attribute__((always_inline)) {
        const int key0 = t * kStep;
        if (key0 >= wave_end) return;
        f32x16 s[2] = {f32x16{}, f32x16{}};
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int h = 0; h < 2; ++h) s[h] = mfma32(read_rows<V8>(kt + 32 * h * L::ROW, k_at[c]), qf[c], s[h]);
        reads_ahead<2 * NC, 2 * NC, 8>();
        if (key0 + kStep > wave_all) {          // (some row of the wavefront does not see all of these keys)
            const int left = end - key0 - 4 * half;
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int e = 0; e < 16; ++e) s[h][e] = 32 * h + 8 * (e >> 2) + (e & 3) < left ? s[h][e] : -INFINITY;
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
        // (at head dim 64, with twice the exponentials to a product, the second half of a step goes before another wavefront's first: 321 us become 309 on 8192 positions, 16 heads; at 128 1 % slower)
        if constexpr (D == 64) __builtin_amdgcn_s_setprio(1);
        V8 pf[4];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                u32x4 w;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int e = 8 * c + 2 * i;
                    const float a = __builtin_amdgcn_exp2f(__builtin_fmaf(s[h][e], p.scale_log2, -m)), b = __builtin_amdgcn_exp2f(__builtin_fmaf(s[h][e + 1], p.scale_log2, -m));
                    l += a;
                    l += b;
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
    for (int t = t0; t < n; t += 2) {
        meet();
        if (t + 1 < n) fill(t + 1, tile2, tile3);
        step(t, tile0, tile1);
        if (t + 1 == n) break;
        meet();
        if (t + 2 < n) fill(t + 2, tile0, tile1);
        step(t + 1, tile2, tile3);
    }
    if (!live) return;
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
    if (rk.length < 0) by = lse = NAN;
    char* const at = p.o + (rq.start + token) * p.o_row + hq * p.o_head + 8 * half;
    char* const rest = p.rest ? p.rest + ((int64_t)(rq.start + token) * p.group * p.Hkv + hq) * (2 * D) + 8 * half : nullptr;
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int i = 0; i < 4; ++i)
            store_rounded<T>(at + 64 * b + 16 * i, rest ? rest + 64 * b + 16 * i : nullptr, acc[b][4 * i] * by, acc[b][4 * i + 1] * by, acc[b][4 * i + 2] * by, acc[b][4 * i + 3] * by);
    if (p.lse && half == 0) p.lse[(int64_t)hq * p.Tq + rq.start + token] = lse;
#endif
}

// ---- backward, first kernel: delta and dq.  The forward's rows and tiles, with P from lse, dP^T = V dO^T beside S^T, and dQ^T = K^T dS^T.  Matrix unit busy 65 % at 1.7 GHz (8192 positions, 32
// heads of 128 on 8): three products to an exponential, under the power limit.
template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 2) ragged_dq_kernel(const RaggedParams p) {
#if defined(__HIP_DEVICE_COMPILE__)
    typedef typename VecOf<T>::v8 V8;
    typedef Tile<D> L;
    constexpr int NC = D / 16, NB = D / 32;
    LDS_TILES(L);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5;
    const Block block = block_of(p, blockIdx.x);
    const int head = block.head;
    const Found f = find<RowTiles>(p, block.index);
    if (f.seq < 0) {
        if (block.part == 0) clear_rows<D>(p.dq, p.dq_row, p.dq_head, p.cu_q, p.n_seq, p.Tq, p.group, head * p.group, kRows, f, nullptr);
        return;
    }
    if (block.part >= f.parts) return;
    const int tile = f.tile;
    const Range rq = rows_of_sequence(p.cu_q, f.seq, f.n.lq), rk = rows_of_sequence(p.cu_k, f.seq, f.n.lk);
    const int rows = rq.length * p.group, lk = rk.length > 0 ? rk.length : 0, shift = lk - rq.length;
    const int row = tile * kRows + 32 * wave + (lane & 31);
    const bool live = row < rows;
    const int token = row / p.group, hq = head * p.group + (row - token * p.group);
    auto keys_of = [&](int t) { const int e = t + shift + 1; return !p.causal || e > lk ? lk : e < 0 ? 0 : e; };
    const int end = live ? keys_of(token) : 0;
    const int first = tile * kRows + 32 * wave;
    auto token_at = [&](int r) { return __builtin_amdgcn_readfirstlane((r < rows ? r : rows - 1) / p.group); };
    const int wave_end = first < rows ? keys_of(token_at(first + 31)) : 0, wave_all = keys_of(token_at(first));
    // steps of this part
    const int steps = RowTiles{p}.end_step(f.n, tile);
    const int t0 = (int)((int64_t)block.part * steps / f.parts), n = (int)((int64_t)(block.part + 1) * steps / f.parts);

    const char* const kp = p.k + rk.start * p.k_row + head * p.k_head;
    const char* const vp = p.v + rk.start * p.v_row + head * p.v_head;
    int k_off[L::LOADS], v_off[L::LOADS];
#pragma unroll
    for (int i = 0; i < L::LOADS; ++i) {
        k_off[i] = L::load_row(lane, wave, i) * (int)p.k_row + L::load_byte(lane, wave, i);
        v_off[i] = L::load_row(lane, wave, i) * (int)p.v_row + L::load_byte(lane, wave, i);
    }
    auto fill = [&](int t, char* kt, char* vt) __attribute__((always_inline)) {
        const auto kr = rows_of<D>(kp + (int64_t)t * kStep * p.k_row, p.k_row, lk - t * kStep), vr = rows_of<D>(vp + (int64_t)t * kStep * p.v_row, p.v_row, lk - t * kStep);
#pragma unroll
        for (int i = 0; i < L::LOADS; ++i) load_to_lds(kr, kt + L::load_to(wave, i), k_off[i]);
#pragma unroll
        for (int i = 0; i < L::LOADS; ++i) load_to_lds(vr, vt + L::load_to(wave, i), v_off[i]);
    };
    if (t0 < n) fill(t0, tile0, tile1);

    V8 qf[NC], gf[NC];
    float delta = 0.f;
    {
        const char* const qa = p.q + (rq.start + token) * p.q_row + hq * p.q_head + 16 * half;
        const char* const ga = p.dout + (rq.start + token) * p.do_row + hq * p.do_head + 16 * half;
        const char* const oa = p.o_in + (rq.start + token) * p.o_row + hq * p.o_head + 16 * half;
        const char* const ra = p.rest + ((int64_t)(rq.start + token) * p.group * p.Hkv + hq) * (2 * D) + 16 * half;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            u32x4 a = {0, 0, 0, 0}, b = a, o = a, r = a;
            if (live) {
                a = *reinterpret_cast<const u32x4*>(qa + 32 * c);
                b = *reinterpret_cast<const u32x4*>(ga + 32 * c);
                o = *reinterpret_cast<const u32x4*>(oa + 32 * c);
                if (p.rest) r = *reinterpret_cast<const u32x4*>(ra + 32 * c);
            }
            a ^= p.flip;
            qf[c] = __builtin_bit_cast(V8, a);
            gf[c] = __builtin_bit_cast(V8, b);
            const V8 of = __builtin_bit_cast(V8, o), rf = __builtin_bit_cast(V8, r);
#pragma unroll
            for (int i = 0; i < 8; ++i) delta = __builtin_fmaf((float)gf[c][i], (float)of[i] + (float)rf[i], delta);
        }
        delta = over_halves_sum(delta);
    }
    const int64_t stat = (int64_t)hq * p.Tq + rq.start + token;
    float lse2 = INFINITY;            // (P = 0 where there is no row, or nothing that it sees)
    if (live) {
        const float x = p.lse[stat];
        lse2 = x == -INFINITY ? INFINITY : x * 1.44269504088896341f;
        if (half == 0 && block.part == 0) p.delta[stat] = delta;
    }
    const float lse0 = lse2;
    if constexpr (kNarrow<T>) lse2 -= kUp;      // (P is not needed but for dS: 2^up is part of its exponent)
    int k_at[NC], k_tr[NB][2];
#pragma unroll
    for (int c = 0; c < NC; ++c) k_at[c] = L::at(lane, c);
#pragma unroll
    for (int b = 0; b < NB; ++b) { k_tr[b][0] = L::at_transposed(lane, b, 0); k_tr[b][1] = L::at_transposed(lane, b, 1); }
    f32x16 acc[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b) acc[b] = f32x16{};

    auto step = [&](int t, const char* kt, const char* vt) __attribute__((always_inline)) {
        const int key0 = t * kStep;
        if (key0 >= wave_end) return;
        const bool masked = key0 + kStep > wave_all;
        const int left = end - key0 - 4 * half;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            f32x16 s = f32x16{}, g = f32x16{};
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                s = mfma32(read_rows<V8>(kt + 32 * h * L::ROW, k_at[c]), qf[c], s);
                g = mfma32(read_rows<V8>(vt + 32 * h * L::ROW, k_at[c]), gf[c], g);
            }
            V8 df[2];
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const float pe = __builtin_amdgcn_exp2f(__builtin_fmaf(s[e], p.scale_log2, -lse2));
                s[e] = pe * (g[e] - delta);
            }
            if (masked)
#pragma unroll
                for (int e = 0; e < 16; ++e) s[e] = 32 * h + 8 * (e >> 2) + (e & 3) < left ? s[e] : 0.f;
            if constexpr (kNarrow<T>) {
                const float top = largest(s);
                if (__any(top > kMostDs)) {
                    const int down = too_many(over_halves_max(top));
                    lse2 += down;
                    s *= power_of_two(-down);
#pragma unroll
                    for (int b = 0; b < NB; ++b) acc[b] *= power_of_two(-down);
                }
            }
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                u32x4 w;
#pragma unroll
                for (int i = 0; i < 4; ++i) w[i] = round2<T>(s[8 * c + 2 * i], s[8 * c + 2 * i + 1]);
                df[c] = __builtin_bit_cast(V8, w);
            }
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
                for (int b = 0; b < NB; ++b) acc[b] = mfma32(read_channels<V8>(kt + (32 * h + 16 * c) * L::ROW, k_tr[b][0], k_tr[b][1]), df[c], acc[b]);
            reads_ahead<4 * NB, 2 * NB, 8>();
        }
    };
    for (int t = t0; t < n; t += 2) {
        meet();
        if (t + 1 < n) fill(t + 1, tile2, tile3);
        step(t, tile0, tile1);
        if (t + 1 == n) break;
        meet();
        if (t + 2 < n) fill(t + 2, tile0, tile1);
        step(t + 1, tile2, tile3);
    }
    if (!live) return;
    if constexpr (kNarrow<T>) {
        const float back = lse0 < INFINITY ? power_of_two((int)rintf(lse2 - lse0)) : 1.f;      // (a whole number but for its rounding)
#pragma unroll
        for (int b = 0; b < NB; ++b) acc[b] *= back;
    }
    if (f.parts > 1) {
        float* const part = p.parts + (((int64_t)block.index * p.Hkv + head) * p.most_parts + block.part) * (kRows * D) + (32 * wave + (lane & 31)) * D;
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int i = 0; i < 4; ++i) *reinterpret_cast<f32x4*>(part + 32 * b + 8 * i + 4 * half) = f32x4{acc[b][4 * i], acc[b][4 * i + 1], acc[b][4 * i + 2], acc[b][4 * i + 3]};
        return;
    }
    const float by = p.scale;
    char* const at = p.dq + (rq.start + token) * p.dq_row + hq * p.dq_head + 8 * half;
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int i = 0; i < 4; ++i)
            *reinterpret_cast<u32x2*>(at + 64 * b + 16 * i) = u32x2{round2<T>(acc[b][4 * i] * by, acc[b][4 * i + 1] * by), round2<T>(acc[b][4 * i + 2] * by, acc[b][4 * i + 3] * by)};
#endif
}

// ---- backward, second kernel: dk and dv.  A workgroup: 128 keys of one sequence and key head, a wavefront 32 of them, one a lane; the sequence's rows (of all heads of the group) go by in
// steps of STEP.  S = Q K^T has the rows in registers: P and dS, rounded, are operands of dV^T += dO^T P and dK^T += Q^T dS where they lie.  K stays in registers, V too at head dim 64 and in
// LDS at 128: with both in registers there are too many for two wavefronts on a SIMD, whose matrix products and other arithmetic go on beside each other (head dim 64, 1560 + 880 + 390 positions,
// 16 heads, us, dq with it, V in LDS / in registers: 95 / 87).  Matrix unit busy 51 % at 1.8 GHz (8192 positions, 32 heads of 128 on 8); what it waits for are reads from LDS, four to a product
// of K's and V's side, for which no more registers are free to be ahead (two wavefronts a SIMD have 256 each, all taken).  With dq 1.12 PFLOP/s of seven products.
// (64 keys and half of a step's rows to a wavefront, one on a SIMD with all 512 registers, so that every fragment of Q and dO feeds two products: as fast on 8192 positions, 10 to 20 % slower on 512 to
// 4096 and on prompts of mixed lengths, where a tile's start and end then have no other workgroup beside them.)
template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 2) ragged_dkdv_kernel(const RaggedParams p) {
#if defined(__HIP_DEVICE_COMPILE__)
    typedef typename VecOf<T>::v8 V8;
    constexpr int STEP = row_step(D), NC = D / 16, NB = D / 32;
    typedef Tile<D, STEP> L;
    typedef Tile<D, kRows> LV;
    LDS_TILES(L);
    constexpr bool V_IN_LDS = D == 128;
    __shared__ __attribute__((aligned(1024))) char values[V_IN_LDS ? LV::BYTES : 16];
    __shared__ __attribute__((aligned(16))) float stats0[2 * STEP], stats1[2 * STEP];      // lse, delta of a step's rows
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5;
    const Block block = block_of(p, blockIdx.x);
    const int head = block.head;
    const Found f = find<KeyTiles<D>>(p, block.index);
    if (f.seq < 0) {
        if (block.part) return;
        clear_rows<D>(p.dk, p.dk_row, p.dk_head, p.cu_k, p.n_seq, p.Tk, 1, head, kRows, f, nullptr);
        clear_rows<D>(p.dv, p.dv_row, p.dv_head, p.cu_k, p.n_seq, p.Tk, 1, head, kRows, f, nullptr);
        return;
    }
    if (block.part >= f.parts) return;
    const Range rq = rows_of_sequence(p.cu_q, f.seq, f.n.lq), rk = rows_of_sequence(p.cu_k, f.seq, f.n.lk);
    const int lq = rq.length > 0 ? rq.length : 0;
    const int key0 = f.tile * kRows, key = key0 + 32 * wave + (lane & 31);
    const bool live = key < rk.length;
    const KeyTiles<D> tiles{p};
    const int from = tiles.first_row(f.n, key);
    const int wave_first = __builtin_amdgcn_readfirstlane(tiles.first_row(f.n, key0 + 32 * wave)), wave_all = __builtin_amdgcn_readfirstlane(tiles.first_row(f.n, key0 + 32 * wave + 31));
    // steps of this part
    const int begin = tiles.first_step(f.n, f.tile), steps = tiles.end_step(f.n, f.tile) - begin;
    const int t0 = begin + (int)((int64_t)block.part * steps / f.parts), n = begin + (int)((int64_t)(block.part + 1) * steps / f.parts);

    if constexpr (V_IN_LDS) {
        const auto vr = rows_of<D, kRows>(p.v + (rk.start + (int64_t)key0) * p.v_row + head * p.v_head, p.v_row, rk.length - key0);
#pragma unroll
        for (int i = 0; i < LV::LOADS; ++i) load_to_lds(vr, values + LV::load_to(wave, i), LV::load_row(lane, wave, i) * (int)p.v_row + LV::load_byte(lane, wave, i));
    }
    V8 kf[NC], vf[NC];
    {
        const char* const ka = p.k + (rk.start + (live ? key : 0)) * p.k_row + head * p.k_head + 16 * half;
        const char* const va = p.v + (rk.start + (live ? key : 0)) * p.v_row + head * p.v_head + 16 * half;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            kf[c] = __builtin_bit_cast(V8, *reinterpret_cast<const u32x4*>(ka + 32 * c) ^ p.flip);
            if constexpr (!V_IN_LDS) vf[c] = __builtin_bit_cast(V8, *reinterpret_cast<const u32x4*>(va + 32 * c));
        }
    }
    // this lane's row of the first load: the token and the head; they go on by ROWS_PER_LOAD rows a load (no registers are left for each load's own) and by STEP rows a step
    const int step_tokens = STEP / p.group, step_heads = STEP - step_tokens * p.group, load_tokens = L::ROWS_PER_LOAD / p.group, load_heads = L::ROWS_PER_LOAD - load_tokens * p.group;
    int token = (t0 * STEP + L::load_row(lane, wave, 0)) / p.group, hd = t0 * STEP + L::load_row(lane, wave, 0) - token * p.group, byte[L::LOADS];
#pragma unroll
    for (int i = 0; i < L::LOADS; ++i) byte[i] = L::load_byte(lane, wave, i);
    const int stat_row = threadIdx.x & (STEP - 1);
    int stat_token = (t0 * STEP + stat_row) / p.group, stat_head = t0 * STEP + stat_row - stat_token * p.group;
    float stat = 0.f;
    const char* const qp = p.q + rq.start * p.q_row + (int64_t)head * p.group * p.q_head;
    const char* const gp = p.dout + rq.start * p.do_row + (int64_t)head * p.group * p.do_head;
    auto next = [&](int& t, int& h, int tokens, int heads) { t += tokens; h += heads; const bool over = h >= p.group; t += over; h -= over ? p.group : 0; };
    auto fill = [&](int t, char* qt, char* gt) __attribute__((always_inline)) {
        const int base = t * STEP / p.group;      // (uniform) token that offsets are counted from
        const auto qr = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(qp + base * p.q_row), 0, 0x7FFFFFFF, 0x00020000);
        const auto gr = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(gp + base * p.do_row), 0, 0x7FFFFFFF, 0x00020000);
        int at = token, h = hd;
#pragma unroll
        for (int i = 0; i < L::LOADS; ++i) {
            const bool in = at < lq;
            load_to_lds(qr, qt + L::load_to(wave, i), in ? (at - base) * (int)p.q_row + h * (int)p.q_head + byte[i] : (int)0x80000000);
            load_to_lds(gr, gt + L::load_to(wave, i), in ? (at - base) * (int)p.do_row + h * (int)p.do_head + byte[i] : (int)0x80000000);
            next(at, h, load_tokens, load_heads);
        }
        next(token, hd, step_tokens, step_heads);
        if (threadIdx.x < 2 * STEP) {             // lse (threads 0 ..) and delta (threads STEP ..) of the step's rows
            const bool in = stat_token < lq;
            const float* const of = threadIdx.x < STEP ? p.lse : p.delta;
            stat = threadIdx.x < STEP ? -INFINITY : 0.f;
            if (in) stat = of[(int64_t)(head * p.group + stat_head) * p.Tq + rq.start + stat_token];
            next(stat_token, stat_head, step_tokens, step_heads);
        }
    };
    int q_at[NC], q_tr[NB][2];
#pragma unroll
    for (int c = 0; c < NC; ++c) q_at[c] = L::at(lane, c);
#pragma unroll
    for (int b = 0; b < NB; ++b) { q_tr[b][0] = L::at_transposed(lane, b, 0); q_tr[b][1] = L::at_transposed(lane, b, 1); }
    const char* const mine = values + 32 * wave * L::ROW;
    f32x16 dk[NB], dv[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b) dk[b] = dv[b] = f32x16{};
    float up = power_of_two(kUp - kUpP);        // (of what is P here)

    auto step = [&](int t, const char* qt, const char* gt, const float* st) __attribute__((always_inline)) {
        const int row0 = t * STEP;
        if (row0 + STEP <= wave_first) return;
#pragma unroll
        for (int h = 0; h < STEP / 32; ++h) {
            if constexpr (D == 128) SCHED_FENCE();      // (both halves at once need more registers than there are)
            f32x16 s = f32x16{}, g = f32x16{};
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                s = mfma32(read_rows<V8>(qt + 32 * h * L::ROW, q_at[c]), kf[c], s);
                if constexpr (V_IN_LDS) g = mfma32(read_rows<V8>(gt + 32 * h * L::ROW, q_at[c]), read_rows<V8>(mine, q_at[c]), g);
                else g = mfma32(read_rows<V8>(gt + 32 * h * L::ROW, q_at[c]), vf[c], g);
            }
            // element e: row 8 (e / 4) + 4 half + e % 4
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const f32x4 lse = *reinterpret_cast<const f32x4*>(st + 32 * h + 8 * i + 4 * half), delta = *reinterpret_cast<const f32x4*>(st + STEP + 32 * h + 8 * i + 4 * half);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    s[4 * i + j] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[4 * i + j], p.scale_log2, -lse[j]));
                    g[4 * i + j] -= delta[j];
                }
            }
            if (row0 < wave_all) {
                const int left = from - row0 - 32 * h - 4 * half;
#pragma unroll
                for (int e = 0; e < 16; ++e) s[e] = 8 * (e >> 2) + (e & 3) >= left ? s[e] : 0.f;
            }
            V8 pf[2], df[2];
            g *= s;
            if constexpr (kNarrow<T>) {
                g *= up;
                const float top = largest(g);
                if (__any(top > kMostDs)) {
                    const float by = power_of_two(-too_many(over_halves_max(top)));
                    up *= by;
                    g *= by;
#pragma unroll
                    for (int b = 0; b < NB; ++b) dk[b] *= by;
                }
            }
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                u32x4 w, x;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int e = 8 * c + 2 * i;
                    w[i] = round2<T>(s[e], s[e + 1]);
                    x[i] = round2<T>(g[e], g[e + 1]);
                }
                pf[c] = __builtin_bit_cast(V8, w);
                df[c] = __builtin_bit_cast(V8, x);
            }
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    dv[b] = mfma32(read_channels<V8>(gt + (32 * h + 16 * c) * L::ROW, q_tr[b][0], q_tr[b][1]), pf[c], dv[b]);
                    dk[b] = mfma32(read_channels<V8>(qt + (32 * h + 16 * c) * L::ROW, q_tr[b][0], q_tr[b][1]), df[c], dk[b]);
                }
            reads_ahead<8 * NB, 4 * NB, 8>();
        }
    };
    // (P = 0 where there is no row, or nothing that it sees)
    auto keep = [&](float* st) __attribute__((always_inline)) {
        if (threadIdx.x < 2 * STEP) st[threadIdx.x] = threadIdx.x >= STEP ? stat : stat == -INFINITY ? INFINITY : stat * 1.44269504088896341f - (kNarrow<T> ? kUpP : 0);
    };
    if (t0 < n) fill(t0, tile0, tile1);
    for (int t = t0; t < n; t += 2) {
        keep(stats0);
        meet();
        if (t + 1 < n) fill(t + 1, tile2, tile3);
        step(t, tile0, tile1, stats0);
        if (t + 1 == n) break;
        keep(stats1);
        meet();
        if (t + 2 < n) fill(t + 2, tile0, tile1);
        step(t + 1, tile2, tile3, stats1);
    }
    if (!live) return;
    if constexpr (kNarrow<T>) {
        const float back = power_of_two(1 - kUpP - __builtin_amdgcn_frexp_expf(up));      // (of a power of two: the exponent and one)
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            dk[b] *= back;
            dv[b] *= power_of_two(-kUpP);
        }
    }
    if (f.parts > 1) {
        float* const part = p.parts + (((int64_t)block.index * p.Hkv + head) * p.most_parts + block.part) * (2 * kRows * D) + (32 * wave + (lane & 31)) * D;
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                *reinterpret_cast<f32x4*>(part + 32 * b + 8 * i + 4 * half) = f32x4{dk[b][4 * i], dk[b][4 * i + 1], dk[b][4 * i + 2], dk[b][4 * i + 3]};
                *reinterpret_cast<f32x4*>(part + kRows * D + 32 * b + 8 * i + 4 * half) = f32x4{dv[b][4 * i], dv[b][4 * i + 1], dv[b][4 * i + 2], dv[b][4 * i + 3]};
            }
        return;
    }
    char* const ka = p.dk + (rk.start + key) * p.dk_row + head * p.dk_head + 8 * half;
    char* const va = p.dv + (rk.start + key) * p.dv_row + head * p.dv_head + 8 * half;
    const float by = p.scale;
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            *reinterpret_cast<u32x2*>(ka + 64 * b + 16 * i) = u32x2{round2<T>(dk[b][4 * i] * by, dk[b][4 * i + 1] * by), round2<T>(dk[b][4 * i + 2] * by, dk[b][4 * i + 3] * by)};
            *reinterpret_cast<u32x2*>(va + 64 * b + 16 * i) = u32x2{round2<T>(dv[b][4 * i], dv[b][4 * i + 1]), round2<T>(dv[b][4 * i + 2], dv[b][4 * i + 3])};
        }
#endif
}

// ---- the tiles that were cut: their parts added up, D / 4 lanes to a row.  WHICH: 0 o and lse, 1 dq, 2 dk and dv.  Memory and a launch: 512 + 77
// + 1 queries of 16 heads, the long ones in some four parts each, 10 us; dk and dv of four causal documents, 7678 keys of 8 heads, 30 us.  (80 scalar registers: with 83 a unit holds one workgroup
// of 16 wavefronts instead of two, 37 us.)
constexpr int kJoinThreads = 1024;
template <int D> constexpr int kJoinBlocks = kRows * (D / 4) / kJoinThreads;      // of a tile
template <typename T, int D, int WHICH>
__global__ void __launch_bounds__(kJoinThreads) __attribute__((amdgpu_num_sgpr(80))) ragged_join_kernel(const RaggedParams p) {
#if defined(__HIP_DEVICE_COMPILE__)
    constexpr bool KEYS = WHICH == 2;
    constexpr int LANES = D / 4, AT_ONCE = kJoinThreads / LANES;
    const int head = blockIdx.x % p.Hkv, index = blockIdx.x / p.Hkv % p.tiles;
    const Found f = find<std::conditional_t<KEYS, KeyTiles<D>, RowTiles>, kJoinThreads>(p, index);
    if (f.seq < 0 || f.parts <= 1) return;
    const int c = 4 * (threadIdx.x % LANES);
    const Range r = rows_of_sequence(KEYS ? p.cu_k : p.cu_q, f.seq, KEYS ? f.n.lk : f.n.lq);
    const int rows = KEYS ? r.length : r.length * p.group;
    const float* const from = p.parts + ((int64_t)index * p.Hkv + head) * p.most_parts * (WHICH == 0 ? kPartFloats<D> : WHICH * kRows * D);
    auto store = [&](char* to, f32x4 x) { *reinterpret_cast<u32x2*>(to + 2 * c) = u32x2{round2<T>(x[0], x[1]), round2<T>(x[2], x[3])}; };
    const int i = blockIdx.x / (p.Hkv * p.tiles) * AT_ONCE + threadIdx.x / LANES;
    const int row = f.tile * kRows + i;
    if (row >= rows) return;
    const int token = KEYS ? row : row / p.group, h = KEYS ? head : head * p.group + (row - token * p.group);
    if constexpr (WHICH == 0) {
        const float* const at = from + i * (D + 2);
        float m = kLowest, l = 0.f;
        f32x4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
        for (int s = 0; s < f.parts; ++s) m = fmaxf(m, at[s * kPartFloats<D>]);
#pragma unroll 4
        for (int s = 0; s < f.parts; ++s) {
            const float* const a = at + s * kPartFloats<D>;
            const float by = __builtin_amdgcn_exp2f(a[0] - m);
            const f32x2 lo = *reinterpret_cast<const f32x2*>(a + 2 + c), hi = *reinterpret_cast<const f32x2*>(a + 4 + c);
            l += by * a[1];
            sum += by * f32x4{lo[0], lo[1], hi[0], hi[1]};
        }
        const float by = l > 0.f ? 1.f / l : l == 0.f ? 0.f : l;
        sum *= by;
        char* const rest = p.rest ? p.rest + ((int64_t)(r.start + token) * p.group * p.Hkv + h) * (2 * D) + 2 * c : nullptr;
        store_rounded<T>(p.o + (r.start + token) * p.o_row + h * p.o_head + 2 * c, rest, sum[0], sum[1], sum[2], sum[3]);
        if (p.lse && c == 0) p.lse[(int64_t)h * p.Tq + r.start + token] = l > 0.f ? (m + __builtin_amdgcn_logf(l)) * 0.693147180559945309f : l == 0.f ? -INFINITY : l;
    } else {
        f32x4 sum[WHICH];
#pragma unroll
        for (int w = 0; w < WHICH; ++w) {
            sum[w] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
            for (int s = 0; s < f.parts; ++s) sum[w] += *reinterpret_cast<const f32x4*>(from + (WHICH * s + w) * (kRows * D) + i * D + c);
        }
        if constexpr (WHICH == 1) {
            store(p.dq + (r.start + token) * p.dq_row + h * p.dq_head, sum[0] * p.scale);
        } else {
            store(p.dk + (r.start + token) * p.dk_row + h * p.dk_head, sum[0] * p.scale);
            store(p.dv + (r.start + token) * p.dv_row + h * p.dv_head, sum[1]);
        }
    }
#endif
}

// ---- C ABI
constexpr int64_t kMost = 0x7FFFFFFF, kMostBlocks = 0xFFFFFFFF / kThreads;
// rows of a step and a token's heads are addressed with 32 bits
constexpr int64_t kMostRowBytes = (int64_t)1 << 23;

int check_tensor(const void* at, const int64_t* stride, int64_t rows, int heads, int D) {
    if (!at) return COSMOS_ATTN_BAD_ARG;
    if (!aligned16(at) || stride[0] % 8 || stride[1] % 8) return COSMOS_ATTN_BAD_STRIDE;
    if (rows > 1 && stride[0] < D) return COSMOS_ATTN_BAD_STRIDE;
    if (stride[0] * 2 > kMostRowBytes || stride[1] < 0 || (heads > 1 && stride[1] * 2 * heads > ((int64_t)1 << 30))) return COSMOS_ATTN_BAD_STRIDE;
    return COSMOS_ATTN_OK;
}
// rows or heads that share memory can be read, not written
int check_output(const void* at, const int64_t* stride, int64_t rows, int heads, int D) {
    const int st = check_tensor(at, stride, rows, heads, D);
    if (st != COSMOS_ATTN_OK) return st;
    if (heads > 1 && stride[1] < D) return COSMOS_ATTN_BAD_STRIDE;
    // one of the two dims holds the other
    const bool by_row = rows <= 1 || stride[0] >= (heads - 1) * stride[1] + D, by_head = heads <= 1 || stride[1] >= (rows - 1) * stride[0] + D;
    return by_row || by_head ? COSMOS_ATTN_OK : COSMOS_ATTN_BAD_STRIDE;
}

int check(const cosmos_attn_ragged_desc* d, bool backward) {
    if (!d || d->abi_version != COSMOS_ATTN_ABI_VERSION) return COSMOS_ATTN_BAD_ARG;
    if (d->dtype != COSMOS_ATTN_BF16 && d->dtype != COSMOS_ATTN_FP16) return COSMOS_ATTN_UNSUPPORTED;
    if (d->n_seq < 0 || d->Hq < 1 || d->Hkv < 1 || d->Tq < 0 || d->Tk < 0 || !(fabsf(d->sm_scale) <= 3.0e38f)) return COSMOS_ATTN_BAD_ARG;
    if (d->Hq % d->Hkv) return COSMOS_ATTN_BAD_SHAPE;
    if (d->D != 64 && d->D != 128) return COSMOS_ATTN_UNSUPPORTED;
    const int64_t group = d->Hq / d->Hkv;
    // (rows are 32-bit numbers, and so are the threads of a launch)
    if (d->Tq > kMost || d->Tq * group > kMost / 2 || d->Tk > kMost / 2) return COSMOS_ATTN_UNSUPPORTED;
    if (((d->Tq * group + d->Tk) / kRows + d->n_seq + 1) * d->Hkv > kMostBlocks) return COSMOS_ATTN_UNSUPPORTED;
    if (!d->cu_q || !d->cu_k) return COSMOS_ATTN_BAD_ARG;
    if ((reinterpret_cast<uintptr_t>(d->cu_q) | reinterpret_cast<uintptr_t>(d->cu_k)) & 3) return COSMOS_ATTN_BAD_STRIDE;
    int st = COSMOS_ATTN_OK;
    auto in = [&](const void* at, const int64_t* stride, int64_t rows, int heads) { if (st == COSMOS_ATTN_OK && rows) st = check_tensor(at, stride, rows, heads, d->D); };
    auto out = [&](const void* at, const int64_t* stride, int64_t rows, int heads) { if (st == COSMOS_ATTN_OK && rows) st = check_output(at, stride, rows, heads, d->D); };
    in(d->q, d->q_stride, d->Tq, d->Hq);
    in(d->k, d->k_stride, d->Tk, d->Hkv);
    in(d->v, d->v_stride, d->Tk, d->Hkv);
    if (d->rest && !aligned16(d->rest)) return COSMOS_ATTN_BAD_STRIDE;
    if (!backward) {
        out(d->o, d->o_stride, d->Tq, d->Hq);
    } else {
        in(d->o, d->o_stride, d->Tq, d->Hq);
        in(d->dout, d->dout_stride, d->Tq, d->Hq);
        out(d->dq, d->dq_stride, d->Tq, d->Hq);
        out(d->dk, d->dk_stride, d->Tk, d->Hkv);
        out(d->dv, d->dv_stride, d->Tk, d->Hkv);
        if (st == COSMOS_ATTN_OK && d->Tq && !d->lse) st = COSMOS_ATTN_BAD_ARG;
    }
    return st;
}

RaggedParams params_of(const cosmos_attn_ragged_desc* d) {
    RaggedParams p = {};
    p.q = (const char*)d->q; p.k = (const char*)d->k; p.v = (const char*)d->v;
    p.o = (char*)d->o; p.o_in = (const char*)d->o; p.dout = (const char*)d->dout;
    p.dq = (char*)d->dq; p.dk = (char*)d->dk; p.dv = (char*)d->dv;
    p.lse = d->lse;
    p.rest = (char*)d->rest;
    p.cu_q = d->cu_q; p.cu_k = d->cu_k;
    p.q_row = 2 * d->q_stride[0]; p.q_head = 2 * d->q_stride[1];
    // (one row may have any stride; those behind it, which are read as zeros, lie past its end)
    p.k_row = 2 * (d->Tk > 1 ? d->k_stride[0] : d->D); p.k_head = 2 * d->k_stride[1];
    p.v_row = 2 * (d->Tk > 1 ? d->v_stride[0] : d->D); p.v_head = 2 * d->v_stride[1];
    p.o_row = 2 * d->o_stride[0]; p.o_head = 2 * d->o_stride[1];
    p.do_row = 2 * d->dout_stride[0]; p.do_head = 2 * d->dout_stride[1];
    p.dq_row = 2 * d->dq_stride[0]; p.dq_head = 2 * d->dq_stride[1];
    p.dk_row = 2 * d->dk_stride[0]; p.dk_head = 2 * d->dk_stride[1];
    p.dv_row = 2 * d->dv_stride[0]; p.dv_head = 2 * d->dv_stride[1];
    p.n_seq = d->n_seq; p.Tq = (int)d->Tq; p.Tk = (int)d->Tk; p.Hkv = d->Hkv; p.group = d->Hq / d->Hkv;
    p.causal = d->causal != 0; p.fill = d->fill == COSMOS_ATTN_FILL_LSE && !d->lse ? 0 : d->fill;
    p.scale = d->sm_scale;
    p.scale_log2 = fmaxf(fabsf(d->sm_scale) * 1.44269504088896341f, 1e-37f);      // (a masked score of -inf stays that)
    p.flip = signbit(d->sm_scale) ? 0x80008000u : 0u;
    return p;
}

int launch(void (*kernel)(RaggedParams), int64_t blocks, const RaggedParams& p, void* stream, int threads = kThreads) {
    if (blocks <= 0) return COSMOS_ATTN_OK;
    kernel<<<dim3((unsigned)blocks), dim3(threads), 0, (hipStream_t)stream>>>(p);
    return hipGetLastError() == hipSuccess ? COSMOS_ATTN_OK : COSMOS_ATTN_LAUNCH_FAILED;
}
template <typename F> int with_type(int dtype, int D, F&& f) {
    if (dtype == COSMOS_ATTN_BF16) return D == 128 ? f((__bf16*)nullptr, Int<128>{}) : f((__bf16*)nullptr, Int<64>{});
    return D == 128 ? f((_Float16*)nullptr, Int<128>{}) : f((_Float16*)nullptr, Int<64>{});
}
// at most so many tiles are there: each sequence rounds up once, and so do the rows of none
int64_t most_tiles(int64_t rows, int n_seq) { return rows / kRows + n_seq + 1; }
// Parts that a tile may be cut into.  A call with fewer tiles than some rounds of workgroups ends with its longest tiles on a few compute units; one with more is dealt out evenly as it is.
// (The workgroups of parts that a tile does not have end at once.)
constexpr int64_t kFullGrid = 6 * kNumCUs;
int most_parts(int64_t tiles, int64_t longest, int least) {
    int64_t parts = (kFullGrid + tiles - 1) / tiles;
    parts = parts < 16 ? parts : 16;
    const int64_t of_length = longest / least;
    parts = parts < of_length ? parts : of_length;
    return parts > 1 ? (int)parts : 1;
}
struct Cut { int64_t tiles; int parts, least; size_t bytes; };
Cut cut_of(const cosmos_attn_ragged_desc* d, int which) {
    const int step = row_step(d->D);
    const int64_t group = d->Hq / d->Hkv, rows = d->Tq * group, tiles = which == 2 ? most_tiles(d->Tk, d->n_seq) : most_tiles(rows, d->n_seq);
    const int64_t longest = which == 2 ? (rows + step - 1) / step : (d->Tk + kStep - 1) / kStep;
    const int least = which == 2 ? least_rows(d->D) / step : least_steps(d->D), parts = most_parts(tiles * d->Hkv, longest, least);
    return {tiles, parts, least, parts > 1 ? (size_t)tiles * d->Hkv * parts * kRows * (which == 0 ? d->D + 2 : which * d->D) * sizeof(float) : 0};
}
size_t up(size_t n) { return (n + 255) / 256 * 256; }

}  // namespace

extern "C" {

size_t cosmos_attn_ragged_workspace_bytes(const cosmos_attn_ragged_desc* desc) { return check(desc, false) == COSMOS_ATTN_OK ? cut_of(desc, 0).bytes : 0; }

int cosmos_attn_ragged(const cosmos_attn_ragged_desc* desc, void* workspace, size_t workspace_bytes, void* stream) {
    const int st = check(desc, false);
    if (st != COSMOS_ATTN_OK) return st;
    if (!desc->Tq) return COSMOS_ATTN_OK;
    const Cut cut = cut_of(desc, 0);
    if (workspace_bytes < cut.bytes || (cut.bytes && !workspace)) return COSMOS_ATTN_WORKSPACE_TOO_SMALL;
    if (cut.bytes && !aligned16(workspace)) return COSMOS_ATTN_BAD_STRIDE;
    if (!device_is_whole_mi355x()) return COSMOS_ATTN_WRONG_DEVICE;
    RaggedParams p = params_of(desc);
    p.tiles = (int)cut.tiles; p.most_parts = cut.parts; p.least = cut.least;
    p.parts = (float*)workspace;
    return with_type(desc->dtype, desc->D, [&](auto* t, auto d) {
        constexpr int D = decltype(d)::value;
        typedef std::remove_pointer_t<decltype(t)> T;
        const int done = launch(ragged_fwd_kernel<T, D>, cut.tiles * p.Hkv * cut.parts, p, stream);
        return done != COSMOS_ATTN_OK || cut.parts == 1 ? done : launch(ragged_join_kernel<T, D, 0>, cut.tiles * p.Hkv * kJoinBlocks<D>, p, stream, kJoinThreads);
    });
}

size_t cosmos_attn_ragged_bwd_workspace_bytes(const cosmos_attn_ragged_desc* desc) {
    if (check(desc, true) != COSMOS_ATTN_OK) return 0;
    const size_t a = cut_of(desc, 1).bytes, b = cut_of(desc, 2).bytes;
    return up((size_t)desc->Tq * desc->Hq * sizeof(float)) + (a > b ? a : b);
}

int cosmos_attn_ragged_bwd(const cosmos_attn_ragged_desc* desc, void* workspace, size_t workspace_bytes, void* stream) {
    const int st = check(desc, true);
    if (st != COSMOS_ATTN_OK) return st;
    const size_t wanted = cosmos_attn_ragged_bwd_workspace_bytes(desc);
    if (workspace_bytes < wanted || (wanted && !workspace)) return COSMOS_ATTN_WORKSPACE_TOO_SMALL;
    if (wanted && !aligned16(workspace)) return COSMOS_ATTN_BAD_STRIDE;
    if (!device_is_whole_mi355x()) return COSMOS_ATTN_WRONG_DEVICE;
    RaggedParams p = params_of(desc);
    p.delta = (float*)workspace;
    p.parts = (float*)((char*)workspace + up((size_t)desc->Tq * desc->Hq * sizeof(float)));      // (of dq, then of dk and dv)
    return with_type(desc->dtype, desc->D, [&](auto* t, auto d) {
        constexpr int D = decltype(d)::value;
        typedef std::remove_pointer_t<decltype(t)> T;
        int done = COSMOS_ATTN_OK;
        auto run = [&](const Cut& cut, auto kernel, auto join) {
            p.tiles = (int)cut.tiles; p.most_parts = cut.parts; p.least = cut.least;
            if (done == COSMOS_ATTN_OK) done = launch(kernel, cut.tiles * p.Hkv * cut.parts, p, stream);
            if (done == COSMOS_ATTN_OK && cut.parts > 1) done = launch(join, cut.tiles * p.Hkv * kJoinBlocks<D>, p, stream, kJoinThreads);
        };
        if (desc->Tq) run(cut_of(desc, 1), ragged_dq_kernel<T, D>, ragged_join_kernel<T, D, 1>);
        if (desc->Tk) run(cut_of(desc, 2), ragged_dkdv_kernel<T, D>, ragged_join_kernel<T, D, 2>);
        return done;
    });
}

}  // extern "C"
