// A paged key-value cache for gfx950: writing it, reading it back, and attention of one new token of each sequence over it: kernels and C ABI (cosmos_attn_cache_write,
// cosmos_attn_cache_read, cosmos_attn_cache_attention).
//
// Position j of sequence i lies in page table[i][j / page_size], place j % page_size.  Pages hold, for each head, page_size rows of D elements of the 16-bit type, or of 8 bits with one fp32
// scale for each row of a head:
//     scale = max |x| r,  r = fp32(1 / 448) (e4m3) or fp32(1 / 127) (int8),   code = round(x / scale) (nearest, ties to even),   x' = code scale
// in fp32, the quotient an IEEE division: values of 8 bits of mantissa often lie on a border between two codes, and these are then the same ones everywhere.  A row with a value that
// is not finite has the scale NaN.
//
// What the host's tables say is not trusted: a page outside of the cache or a length that the table does not hold makes the sequence's output NaN (attention, reading back) or writes nothing.
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

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));

constexpr int kThreads = 256;
enum Kind { SAME16 = COSMOS_ATTN_CACHE_SAME, E4M3 = COSMOS_ATTN_CACHE_E4M3, INT8 = COSMOS_ATTN_CACHE_INT8 };

// keys, or values
struct Side {
    char* pages;                                  // bytes between pages, heads and rows
    int64_t page, head, row;
    float* scales;                                // elements between pages and heads
    int64_t scale_page, scale_head;
    char* packed;                                 // rows outside of the cache: bytes between rows and heads
    int64_t packed_row, packed_head;
};
struct CacheParams {
    Side side[2];                                 // keys, values
    const int *table, *lens, *cu;
    int64_t table_row;
    int width, B, pages, page_shift, Hkv, fill;
    int64_t rows;                                 // packed rows
    // attention
    const char* q;
    char* o;
    float* lse;
    int64_t q_row, q_head, o_row, o_head;
    int group, row_blocks, slots, whole;          // slots: workgroups for the shares, per head and block of rows; whole: a workgroup has all of a sequence
    float scale_log2;
    unsigned flip;
    float* parts;
    int* share;                                   // behind the parts: a share, and the most that a part has
};

// ---- 16-bit pairs
template <typename T> __device__ __forceinline__ float low(unsigned w) {
    if constexpr (__is_same(T, __bf16)) return __builtin_bit_cast(float, w << 16);
    else return (float)__builtin_bit_cast(_Float16, (uint16_t)w);
}
template <typename T> __device__ __forceinline__ float high(unsigned w) {
    if constexpr (__is_same(T, __bf16)) return __builtin_bit_cast(float, w & 0xFFFF0000u);
    else return (float)__builtin_bit_cast(_Float16, (uint16_t)(w >> 16));
}
// elements 2 H and 2 H + 1 of four 8-bit codes as a pair of T (both types hold every code exactly)
template <typename T, int KIND, bool H> __device__ __forceinline__ unsigned code_pair(unsigned w) {
    if constexpr (KIND == E4M3) {
        if constexpr (__is_same(T, __bf16)) return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, H));
        else return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, H));
    } else {
        const int a = (int)(w << (H ? 8 : 24)) >> 24, b = (int)(w << (H ? 0 : 16)) >> 24;
        return round2<T>((float)a, (float)b);
    }
}

// max over the LANES (4 or 8) neighbouring lanes of a row
template <int CTRL> __device__ __forceinline__ unsigned dpp_max(unsigned v) {
    const unsigned moved = (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, false);
    return v > moved ? v : moved;
}
template <int LANES> __device__ __forceinline__ unsigned row_max(unsigned v) {
    v = dpp_max<0xB1>(v);       // quad_perm [1, 0, 3, 2]
    v = dpp_max<0x4E>(v);       // quad_perm [2, 3, 0, 1]
    return LANES == 8 ? dpp_max<0x141>(v) : v;      // row_half_mirror
}

// ---- packed rows: which sequence a row is of, and its place there
// the last offset of lo .. hi at or below the row (or lo)
__device__ __forceinline__ int last_below(const int* cu, int lo, int hi, int64_t row) {
    while (lo < hi) {
        const int mid = (int)(((unsigned)lo + (unsigned)hi + 1) >> 1);
        if (cu[mid] <= row) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}
struct Place {
    int seq, start, end, len;     // its offsets; keys in the cache (writing)
    __device__ __forceinline__ Place(const CacheParams& p, int at, bool lens) : seq(at), start(0), end(0), len(0) {
        if (!p.cu) {              // one row to a sequence
            start = at;
            end = at + 1;
        } else {
            start = p.cu[at];
            end = at < p.B ? p.cu[at + 1] : start;
        }
        if (lens && at < p.B) len = p.lens[at];
    }
    __device__ __forceinline__ bool has(const CacheParams& p, int row) const { return seq < p.B && start >= 0 && row >= start && row < end && end <= p.rows; }
};

// Both kernels: a lane has EACH elements of a row of a head, 8 where pages hold 16 bits and 16 where they hold codes: 16 bytes of the narrower side.  A workgroup has kThreads EACH / D rows,
// in the packed rows' order, of the keys or of the values (even and odd workgroups), so that their addresses are the scalar unit's to form, and so is the place of the first row's sequence,
// most often that of all.  16384 + 9999 + 1 + 4096 rows of 8 heads in e4m3: 42 us to write and 32 to read back; with all of that in each thread 54 and 34, with 8 elements of a code to a
// lane 95 and 53; two rows to a thread 44 and 33, four 48 and 35 (and 4.5 us instead of 3.4 for a few rows).  189 MB each way at the rate of a large copy are 37: a write forms 3 quotients,
// products and codes to a lane's element, the vector unit's work of about as long.
constexpr int each_of(int kind) { return kind == SAME16 ? 8 : 16; }
template <int D, int EACH> struct Rows {
    static constexpr int LANES = D / EACH, ROWS = kThreads / LANES;
    const Side& side;
    int64_t row0;                 // the workgroup's first packed row
    int row, head;                // row: counted from there
    bool in;                      // there is such a row
    __device__ __forceinline__ Rows(const CacheParams& p) : side(p.side[blockIdx.x & 1]) {
        const int64_t unit = (int64_t)(blockIdx.x >> 1) * ROWS;
        row0 = unit / p.Hkv;
        const unsigned u = (unsigned)(unit - row0 * p.Hkv) + threadIdx.x / LANES, r = u / (unsigned)p.Hkv;
        row = (int)r;
        head = (int)(u - r * p.Hkv);
        in = row0 + r < p.rows;
    }
    // where the row is (if there is one)
    __device__ __forceinline__ Place place(const CacheParams& p, bool lens) const {
        Place w(p, p.cu ? last_below(p.cu, 0, p.B, row0) : (int)row0, lens);
        if (in && this->at() >= w.end && w.seq < p.B) w = Place(p, p.cu ? last_below(p.cu, w.seq + 1, p.B, this->at()) : this->at(), lens);
        return w;
    }
    __device__ __forceinline__ int at() const { return (int)row0 + row; }       // of all
    __device__ __forceinline__ char* packed() const { return side.packed + row0 * side.packed_row + row * side.packed_row + head * side.packed_head + 2 * EACH * (threadIdx.x % LANES); }
    __device__ __forceinline__ char* cached(int page, int key) const { return side.pages + page * side.page + head * side.head + key * side.row + 16 * (threadIdx.x % LANES); }
    __device__ __forceinline__ float* scale(int page, int key) const { return side.scales + page * side.scale_page + head * side.scale_head + key; }
};

// x / s as IEEE division rounds it, for |x / s| up to some hundreds: x r corrected by the remainder, which fma gives exactly (Markstein's division), with r = 1 / s good to an ulp.  (That one
// correction is enough has been seen for all there is: a 16-bit x has 2^7 or 2^10 significands and s, which follows from another one, as many.)  Rows whose scale would leave the range
// in which all of that is exact are multiplied with a power of two first, as their scale is.
struct Divide {
    float s, r, by;
    __device__ __forceinline__ explicit Divide(float scale) {
        by = scale < 0x1p-60f ? 0x1p64f : 1.f;
        s = scale * by;
        r = __builtin_amdgcn_rcpf(s);
        r = __builtin_fmaf(__builtin_fmaf(-s, r, 1.f), r, r);
    }
    __device__ __forceinline__ float operator()(float x) const {
        const float q = x * r;
        return __builtin_fmaf(__builtin_fmaf(-s, q, x), r, q);
    }
};

// ---- writing
template <typename T, int KIND, int D>
__global__ void __launch_bounds__(kThreads) cache_write_kernel(const CacheParams p) {
#if defined(__HIP_DEVICE_COMPILE__)
    constexpr int EACH = each_of(KIND);
    typedef Rows<D, EACH> R;
    const R rows(p);
    u32x4 x[EACH / 8];
#pragma unroll
    for (int j = 0; j < EACH / 8; ++j) {
        x[j] = u32x4{0, 0, 0, 0};
        if (rows.in) x[j] = *reinterpret_cast<const u32x4*>(rows.packed() + 16 * j);
    }
    const Place w = rows.place(p, true);
    const int to = w.len - (w.end - rows.at()), key = to & ((1 << p.page_shift) - 1);
    int page = -1;
    if (rows.in && w.has(p, rows.at()) && w.len >= w.end - w.start && (to >> p.page_shift) < p.width) page = p.table[w.seq * p.table_row + (to >> p.page_shift)];
    const bool in = page >= 0 && page < p.pages;
    if constexpr (KIND == SAME16) {
        if (in) *reinterpret_cast<u32x4*>(rows.cached(page, key)) = x[0];
    } else {
        // the largest magnitude: of 16-bit floats without their signs as whole numbers, in whose order NaN comes behind infinity and that behind all others
        typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
        u16x2 most = {0, 0};
#pragma unroll
        for (int j = 0; j < 8; ++j) most = __builtin_elementwise_max(most, __builtin_bit_cast(u16x2, x[j / 4][j % 4] & 0x7FFF7FFFu));
        const unsigned top = row_max<R::LANES>(most[0] > most[1] ? most[0] : most[1]);
        // (a row of zeros: divided by 1; one that is not finite: codes of no meaning)
        const float scale = top < (__is_same(T, __bf16) ? 0x7F80u : 0x7C00u) ? low<T>(top) * (KIND == E4M3 ? 1.f / 448.f : 1.f / 127.f) : NAN;
        const Divide over(scale > 0.f ? scale : 1.f);
        float f[16];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            f[2 * j] = low<T>(x[j / 4][j % 4]);
            f[2 * j + 1] = high<T>(x[j / 4][j % 4]);
        }
        if (__any(over.by != 1.f)) {
#pragma unroll
            for (int j = 0; j < 16; ++j) f[j] *= over.by;
        }
#pragma unroll
        for (int j = 0; j < 16; ++j) f[j] = over(f[j]);
        u32x4 codes = {0, 0, 0, 0};
        if constexpr (KIND == E4M3) {
            // (scale's own rounding may leave a quotient just above 448; the conversion's largest code takes those below 464)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int w = __builtin_amdgcn_cvt_pk_fp8_f32(f[4 * j], f[4 * j + 1], 0, false);
                codes[j] = (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(f[4 * j + 2], f[4 * j + 3], w, true);
            }
        } else {
            // 2^23 + 2^22 + f: f rounded to a whole number, ties to even, in the low bits
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                unsigned w[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) w[k] = __builtin_bit_cast(unsigned, f[4 * j + k] + 12582912.f);
                const unsigned lo = __builtin_amdgcn_perm(w[1], w[0], 0x0C0C0400u), hi = __builtin_amdgcn_perm(w[3], w[2], 0x04000C0Cu);
                codes[j] = lo | hi;
            }
        }
        if (in) {
            *reinterpret_cast<u32x4*>(rows.cached(page, key)) = codes;
            if (threadIdx.x % R::LANES == 0) *rows.scale(page, key) = scale;
        }
    }
#endif
}

// ---- reading back
template <typename T, int KIND, int D>
__global__ void __launch_bounds__(kThreads) cache_read_kernel(const CacheParams p) {
#if defined(__HIP_DEVICE_COMPILE__)
    const Rows<D, each_of(KIND)> rows(p);
    const Place w = rows.place(p, false);
    const int from = rows.at() - w.start, key = from & ((1 << p.page_shift) - 1);
    const bool of = rows.in && w.has(p, rows.at());      // a row of some sequence
    if (!rows.in || !(of || p.fill)) return;
    int page = -1;
    if (of && (from >> p.page_shift) < p.width) page = p.table[w.seq * p.table_row + (from >> p.page_shift)];
    const bool there = page >= 0 && page < p.pages;
    const unsigned other = of ? round2<T>(NAN, NAN) : 0u;      // (of no sequence: zeros; of a page that is not there: NaN)
    float scale = 1.f;
    u32x4 codes = {0, 0, 0, 0};
    if (there) {
        codes = *reinterpret_cast<const u32x4*>(rows.cached(page, key));
        if constexpr (KIND != SAME16) scale = *rows.scale(page, key);
    }
    u32x4* const to = reinterpret_cast<u32x4*>(rows.packed());
    if constexpr (KIND == SAME16) {
        *to = there ? codes : u32x4{other, other, other, other};
    } else {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            u32x4 x;
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const unsigned a = code_pair<T, KIND, false>(codes[2 * j + k]), b = code_pair<T, KIND, true>(codes[2 * j + k]);
                x[2 * k] = round2<T>(low<T>(a) * scale, high<T>(a) * scale);
                x[2 * k + 1] = round2<T>(low<T>(b) * scale, high<T>(b) * scale);
            }
            to[j] = there ? x : u32x4{other, other, other, other};
        }
    }
#endif
}

// ---- attention of one token over the pages
// A workgroup's share is an equal part of all sequences' keys, in tiles of kTile.  A sequence of more is cut into parts, of which each has a workgroup for each key head; one in one part
// has its rows written at once, the others' parts leave sums, which cache_join_kernel adds up.  (Equal runs of one list of all sequences' tiles: a workgroup then waits for the first keys of each
// of many short sequences in turn, 32 sequences of 1 to 2817 keys in int8 25 us instead of 19, though 48 of 1 to 7817 97 instead of 100.)
// Memory: the live pages are read once, at the rate of a large copy where there are enough of them (131072 + 70001 + 99 keys of 8 heads in e4m3, 425 MB, 77 us, 5.5 TB/s; 48 sequences in bf16,
// 504 MB, 95 us, 5.3 TB/s); 57 MB 16.6 us, 3.4 TB/s, of which the first loads, behind the lengths, the table and the pages, are some 5.
constexpr int kTile = 128;           // keys: 32 of each wavefront
constexpr float kLowest = -3.0e38f;

// tiles of a length
__device__ __forceinline__ int tiles_of(const CacheParams& p, int n) {
    return n > 0 && n <= (int64_t)p.width << p.page_shift ? (n + kTile - 1) / kTile : 0;
}
// A sequence's parts have a share at most; three quarters of one where shares are large and most sequences have only a few parts, which rounding up leaves far from equal (48 sequences of 1 to
// 7817 keys, us, a share / three quarters: 106 / 100; but 131072 + 70001 + 99 keys in e4m3 84 / 88, 32 of 1 to 2817 in int8 18.9 / 20.5).  On eleven other sizes, 8 to 100 sequences of up to 3000 to 60000 keys, the rule is within 2 % of the better one
// (us, a share / three quarters / the rule: 20 of up to 30000 in int8 99 / 91 / 89, 100 of up to 12000, 16 heads on 4, 140 / 134 / 134, 20 of up to 8000 37 / 42 / 37, 30 of up to 16000, 16 heads on 2,
// 24 / 27 / 23).
struct Share {
    int per, most;
    __device__ __forceinline__ int parts(int tiles) const { return tiles > per ? (tiles + most - 1) / most : 1; }
    __device__ __forceinline__ bool is_long(int tiles) const { return 2 * tiles > per; }
};
__device__ __forceinline__ Share share_of(const CacheParams& p, int tiles) {
    int per = (tiles + p.slots - 1) / p.slots;
    per = per > 1 ? per : 1;
    return {per, per >= 8 && 4 * (int64_t)p.B > p.slots ? (3 * per + 3) / 4 : per};
}
// Every workgroup looks through all sequences: up to 64 each wavefront for itself, more of them kOwn in order to a thread, so that the lengths of kBatch are one wait (1000 sequences of 1 to 1500
// keys in tables of 4096, which are not taken whole, 32 heads of 128 on 8, int8, 306 us, 5.2 TB/s, each wavefront 64 at a time 443; but 32 sequences 20.2 instead of 19.4).
constexpr int kOwn = 4, kBatch = kOwn * kThreads, kWaves = kThreads / 64;
struct Batch {
    int tiles[kOwn];
    __device__ __forceinline__ Batch(const CacheParams& p, int base) {
        int n[kOwn];
#pragma unroll
        for (int c = 0; c < kOwn; ++c) { const int i = base + kOwn * threadIdx.x + c; n[c] = p.lens[i < p.B ? i : 0]; }
#pragma unroll
        for (int c = 0; c < kOwn; ++c) tiles[c] = base + kOwn * (int)threadIdx.x + c < p.B ? tiles_of(p, n[c]) : 0;
    }
};
// The part `slot`: first come the parts of sequences of more than half a share, in order, then the shorter ones, which end the call on what those leave (without keys: one part too).
// seq < 0: behind the last.
struct Part { int seq, part, parts, tiles; };
__device__ __forceinline__ Part part_of(const CacheParams& p, int slot) {
    if (p.B <= 64) {
        const int lane = threadIdx.x & 63, n = p.lens[lane < p.B ? lane : 0], tiles = lane < p.B ? tiles_of(p, n) : 0;
        const Share share = share_of(p, sum_of(tiles));
        if (blockIdx.x == 0 && threadIdx.x == 0) { p.share[0] = share.per; p.share[1] = share.most; }
        int before = 0;
#pragma unroll
        for (int shorter = 0; shorter < 2; ++shorter) {
            const int parts = lane < p.B && share.is_long(tiles) != (bool)shorter ? share.parts(tiles) : 0, sum = sums_up_to(parts);
            const unsigned long long past = __ballot(before + sum > slot);
            if (past) {
                const int at = __builtin_ctzll(past), of = __builtin_amdgcn_readlane(parts, at);
                return {at, slot - (before + __builtin_amdgcn_readlane(sum, at) - of), of, __builtin_amdgcn_readlane(tiles, at)};
            }
            before += __builtin_amdgcn_readlane(sum, 63);
        }
        return {-1, 0, 0, 0};
    }
    __shared__ int totals[kWaves], sums[2][kWaves];
    __shared__ Part found;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const Batch first(p, 0);
    int mine = 0;
    for (int base = 0; base < p.B; base += kBatch) {
        const Batch b = base ? Batch(p, base) : first;
#pragma unroll
        for (int c = 0; c < kOwn; ++c) mine += b.tiles[c];
    }
    mine = sum_of(mine);
    if (lane == 0) totals[wave] = mine;
    __syncthreads();
    int all = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) all += totals[w];
    const Share share = share_of(p, all);
    if (blockIdx.x == 0 && threadIdx.x == 0) { p.share[0] = share.per; p.share[1] = share.most; }
    int before = 0, turn = 0;
    for (int shorter = 0; shorter < 2; ++shorter)
        for (int base = 0; base < p.B; base += kBatch, turn ^= 1) {
            const Batch b = base ? Batch(p, base) : first;
            int parts[kOwn], own = 0;
#pragma unroll
            for (int c = 0; c < kOwn; ++c) {
                parts[c] = base + kOwn * (int)threadIdx.x + c < p.B && share.is_long(b.tiles[c]) != (bool)shorter ? share.parts(b.tiles[c]) : 0;
                own += parts[c];
            }
            const int sum = sums_up_to(own);
            if (lane == 63) sums[turn][wave] = sum;
            __syncthreads();
            int at = before + sum - own, past = before;       // parts before this thread's, up to the batch's end
#pragma unroll
            for (int w = 0; w < kWaves; ++w) {
                at += w < wave ? sums[turn][w] : 0;
                past += sums[turn][w];
            }
            if (slot < past) {
                if (slot >= at && slot < at + own) {
#pragma unroll
                    for (int c = 0; c < kOwn; ++c) {
                        if (slot >= at && slot < at + parts[c]) found = {base + kOwn * (int)threadIdx.x + c, slot - at, parts[c], b.tiles[c]};
                        at += parts[c];
                    }
                }
                __syncthreads();
                return {__builtin_amdgcn_readfirstlane(found.seq), __builtin_amdgcn_readfirstlane(found.part), __builtin_amdgcn_readfirstlane(found.parts), __builtin_amdgcn_readfirstlane(found.tiles)};
            }
            before = past;
        }
    return {-1, 0, 0, 0};
}
// floats of a part: D sums, the max they refer to, the sum of the exponentials, for each of 16 NR rows
template <int D, int NR> constexpr int kPartFloats = 16 * NR * (D + 2);

__device__ __forceinline__ float over_quarters_max(float x) {
    float lo, hi;
    both_halves(x, lo, hi);
    x = fmaxf(lo, hi);
    return fmaxf(x, __shfl_xor(x, 16));
}

template <typename T, int KIND, int D, int NR>
__global__ void __launch_bounds__(kThreads, 2) cache_attention_kernel(const CacheParams p) {
#if defined(__HIP_DEVICE_COMPILE__)
    typedef typename VecOf<T>::v8 V8;
    constexpr bool CODES = KIND != SAME16;
    constexpr int BYTES = CODES ? 1 : 2, NC = D / 32;      // NC: products of 32 channels
    constexpr int NB = D / 16;                             // and of 16 channels of the output; channels of a lane of V
    extern __shared__ __attribute__((aligned(16))) float smem[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n16 = lane & 15, g = lane >> 4;
    const int head = blockIdx.x % p.Hkv, block = blockIdx.x / p.Hkv % p.row_blocks, slot = blockIdx.x / (p.Hkv * p.row_blocks);
    const int row0 = block * 16 * NR;

    // rows of a sequence without keys: zeros, or NaN where its length is none
    auto write_empty = [&](int i) {
        const bool bad = p.lens[i] != 0;
        const unsigned w = bad ? round2<T>(NAN, NAN) : 0u;
        for (int r = 0; r < 16 * NR && row0 + r < p.group; ++r) {
            const int hq = head * p.group + row0 + r;
            if (lane < D / 8) *reinterpret_cast<u32x4*>(p.o + i * p.o_row + hq * p.o_head + 16 * lane) = u32x4{w, w, w, w};
            if (p.lse && lane == 0) p.lse[(int64_t)i * p.group * p.Hkv + hq] = bad ? NAN : -INFINITY;
        }
    };
    Part mine = {slot, 0, 1, 0};
    if (p.whole) mine.tiles = __builtin_amdgcn_readfirstlane(tiles_of(p, p.lens[slot]));
    else mine = part_of(p, slot);
    if (mine.seq < 0) return;
    const int seq = mine.seq;
    if (!mine.tiles) {
        if (wave == 0) write_empty(seq);
        return;
    }
    const int len = __builtin_amdgcn_readfirstlane(p.lens[seq]), from = (int)((int64_t)mine.part * mine.tiles / mine.parts), to = (int)((int64_t)(mine.part + 1) * mine.tiles / mine.parts);
    const int* const table = p.table + seq * p.table_row;
    const char* const kh = p.side[0].pages + head * p.side[0].head;
    const char* const vh = p.side[1].pages + head * p.side[1].head;
    const int mask = (1 << p.page_shift) - 1;
    // Q: row n16 of each block of 16, the channels that this lane's K holds
    V8 qf[NR][NC];
#pragma unroll
    for (int r = 0; r < NR; ++r) {
        const int row = row0 + 16 * r + n16;
        const char* const at = p.q + (int64_t)seq * p.q_row + (int64_t)(head * p.group + (row < p.group ? row : 0)) * p.q_head;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const int channel = CODES ? 64 * (c / 2) + 16 * g + 8 * (c % 2) : 32 * c + 8 * g;
            u32x4 w = *reinterpret_cast<const u32x4*>(at + 2 * channel);
            w ^= p.flip;
            qf[r][c] = __builtin_bit_cast(V8, row < p.group ? w : u32x4{0, 0, 0, 0});
        }
    }
    f32x4 acc[NR][NB];
    float m[NR], l[NR], R = 0.f;
    bool bad = false;
#pragma unroll
    for (int r = 0; r < NR; ++r) {
        m[r] = kLowest;
        l[r] = 0.f;
#pragma unroll
        for (int b = 0; b < NB; ++b) acc[r][b] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    // Steps of 32 keys.  A step's K is loaded behind the products of the one before, its V behind that one's, and its pages are looked up a step earlier still: nothing waits for
    // addresses, and little for what they point at.  Keys past the end are the last one's, with weights of 0: whatever else the page holds is not looked at.
    constexpr int KLOADS = CODES ? NC / 2 : NC, VWORDS = NB * BYTES / 4;
    const int most = len - 1, first_key = 32 * wave;
    int end = (len - first_key + kTile - 1) / kTile;                  // this wavefront's steps
    end = to < end ? to : end;
    u32x4 kw[2][KLOADS];
    unsigned vw[8][VWORDS];
    float ks[8], vs[8];
    // K: row n16 of key half u is key 8 (n16 / 4) + 4 u + n16 % 4, so that a lane's results of the two halves are those of 8 keys in order, 8 g .. 8 g + 7
    auto k_key = [&](int t, int u) { const int key = t * kTile + first_key + 8 * (n16 >> 2) + 4 * u + (n16 & 3); return key < most ? key : most; };
    // V: keys 8 g .. 8 g + 7, channels NB n16 .. NB n16 + NB - 1; 8 keys in order share a page
    auto v_key = [&](int t) { const int key = t * kTile + first_key + 8 * g; return key < (most & ~7) ? key : (most & ~7); };
    int kp[2], vp;
    auto look_up = [&](int t) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < 2; ++u) kp[u] = table[k_key(t, u) >> p.page_shift];
        vp = table[v_key(t) >> p.page_shift];
    };
    auto checked = [&](int page) { const bool in = page >= 0 && page < p.pages; bad |= !in; return in ? page : 0; };
    auto load_k = [&](int t) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const char* const at = kh + checked(kp[u]) * p.side[0].page + (k_key(t, u) & mask) * p.side[0].row + 16 * g;
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
        load_v(from, checked(vp));
        look_up(from + 1);
    }
    // (the last step loads nothing: a condition around the loads would have the compiler wait for all of them at the next use of any)
    auto step = [&](int t, auto more) __attribute__((always_inline)) {
        f32x4 s[NR][2];
#pragma unroll
        for (int r = 0; r < NR; ++r) s[r][0] = s[r][1] = f32x4{0.f, 0.f, 0.f, 0.f};
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
#pragma unroll
                for (int r = 0; r < NR; ++r) s[r][u] = mfma16(__builtin_bit_cast(V8, w), qf[r][c], s[r][u]);
            }
        int vnext = 0;
        if constexpr (decltype(more)::value) {
            load_k(t + 1);
            vnext = checked(vp);
            look_up(t + 2);
        }
        const int left = len - t * kTile - first_key - 8 * g;
        float by[8];                            // what V's weights are multiplied with
        if constexpr (CODES) {
#pragma unroll
            for (int i = 0; i < 8; ++i) by[i] = i < left ? vs[i] : 0.f;
            if constexpr (__is_same(T, _Float16)) {
                // Weights p scale in fp16 would leave its range where values are small.  They are held relative to the largest scale so far, but for a factor of up to 64.
                float top = by[0];
#pragma unroll
                for (int i = 1; i < 8; ++i) top = fmaxf(top, by[i]);
                if (__any(top > 64.f * R)) {
                    top = fmaxf(fmaxf(R, over_quarters_max(top)), 0x1p-100f);      // (far below what fp16 holds, and its reciprocal is a number)
                    const float f = R / top;
#pragma unroll
                    for (int r = 0; r < NR; ++r)
#pragma unroll
                        for (int b = 0; b < NB; ++b) acc[r][b] *= f;
                    R = top;
                }
                const float over = R > 0.f ? 1.f / R : 1.f;
#pragma unroll
                for (int i = 0; i < 8; ++i) by[i] *= over;
            }
        }
        V8 pf[NR];
#pragma unroll
        for (int r = 0; r < NR; ++r) {
            float x[8], top = -INFINITY;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                x[i] = s[r][i / 4][i % 4] * p.scale_log2;
                if constexpr (CODES) x[i] *= ks[i];
                x[i] = i < left ? x[i] : -INFINITY;
                top = fmaxf(top, x[i]);
            }
            if (__any(top > m[r] + kMaxSlack)) {
                top = fmaxf(m[r], over_quarters_max(top));
                const float f = __builtin_amdgcn_exp2f(m[r] - top);
                m[r] = top;
                l[r] *= f;
#pragma unroll
                for (int b = 0; b < NB; ++b) acc[r][b] *= f;
            }
            u32x4 w;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                x[i] = __builtin_amdgcn_exp2f(x[i] - m[r]);
                l[r] += x[i];
                if constexpr (CODES) x[i] *= by[i];
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = round2<T>(x[2 * i], x[2 * i + 1]);
            pf[r] = __builtin_bit_cast(V8, w);
        }
        // Past the end lie the last rows once more, whose infinite values with a weight of 0 would be NaN.  (The last step alone reaches there; a code's scale is what is infinite, or NaN, and is
        // not taken there.)
        if constexpr (!CODES && !decltype(more)::value) {
#pragma unroll
            for (int i = 0; i < 8; ++i)
#pragma unroll
                for (int j = 0; j < VWORDS; ++j) vw[i][j] = i < left ? vw[i][j] : 0u;
        }
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
#pragma unroll
            for (int r = 0; r < NR; ++r) acc[r][b] = mfma16(__builtin_bit_cast(V8, vt), pf[r], acc[r][b]);
        }
        if constexpr (decltype(more)::value) load_v(t + 1, vnext);
    };
    if (from < end) {
        for (int t = from; t + 1 < end; ++t) step(t, Int<1>{});
        step(end - 1, Int<0>{});
    }
    // ---- join the wavefronts: [wave][row][channel], then [wave][row] of max, sum
    float* const sums = smem;
    float* const stat = smem + 4 * 16 * NR * D;
    const float back = CODES && __is_same(T, _Float16) ? R : 1.f;
    const bool any_bad = __any(bad);
#pragma unroll
    for (int r = 0; r < NR; ++r) {
        float lr = l[r];
        lr += __shfl_xor(lr, 16);
        lr += __shfl_xor(lr, 32);
        if (any_bad) lr = NAN;
        if (g == 0) {
            stat[2 * (wave * 16 * NR + 16 * r + n16)] = m[r];
            stat[2 * (wave * 16 * NR + 16 * r + n16) + 1] = lr;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int b = 0; b < NB; b += 4)
                *reinterpret_cast<f32x4*>(sums + (wave * 16 * NR + 16 * r + n16) * D + NB * (4 * g + e) + b) = f32x4{acc[r][b][e], acc[r][b + 1][e], acc[r][b + 2][e], acc[r][b + 3][e]} * back;
    }
    __syncthreads();
    constexpr int LANES = D / 8, AT_ONCE = kThreads / LANES;
    for (int r = threadIdx.x / LANES; r < 16 * NR && row0 + r < p.group; r += AT_ONCE) {
        const int c = 8 * (threadIdx.x % LANES);
        float top = kLowest, sum = 0.f, f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < 4; ++w) top = fmaxf(top, stat[2 * (w * 16 * NR + r)]);
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float by = __builtin_amdgcn_exp2f(stat[2 * (w * 16 * NR + r)] - top);
            sum += by * stat[2 * (w * 16 * NR + r) + 1];
#pragma unroll
            for (int i = 0; i < 8; ++i) f[i] += by * sums[(w * 16 * NR + r) * D + c + i];
        }
        const int hq = head * p.group + row0 + r;
        if (mine.parts == 1) {
            const float by = sum > 0.f ? 1.f / sum : sum == 0.f ? 0.f : sum;
            *reinterpret_cast<u32x4*>(p.o + (int64_t)seq * p.o_row + hq * p.o_head + 2 * c) = u32x4{round2<T>(f[0] * by, f[1] * by), round2<T>(f[2] * by, f[3] * by), round2<T>(f[4] * by, f[5] * by), round2<T>(f[6] * by, f[7] * by)};
            if (p.lse && c == 0) p.lse[(int64_t)seq * p.group * p.Hkv + hq] = sum > 0.f ? (top + __builtin_amdgcn_logf(sum)) * 0.693147180559945309f : sum == 0.f ? -INFINITY : sum;
        } else {
            float* const part = p.parts + (((int64_t)slot * p.row_blocks + block) * p.Hkv + head) * kPartFloats<D, NR>;
            *reinterpret_cast<f32x4*>(part + r * D + c) = f32x4{f[0], f[1], f[2], f[3]};
            *reinterpret_cast<f32x4*>(part + r * D + c + 4) = f32x4{f[4], f[5], f[6], f[7]};
            if (c == 0) { part[16 * NR * D + 2 * r] = top; part[16 * NR * D + 2 * r + 1] = sum; }
        }
    }
#endif
}

// ---- the sequences that several workgroups have parts of: a workgroup for each sequence and query head, D / 4 lanes to a part, kThreads / (D / 4) parts at a time
// (4 to 6 us, a launch and two trips to memory)
template <typename T, int D, int NR>
__global__ void __launch_bounds__(kThreads) cache_join_kernel(const CacheParams p) {
#if defined(__HIP_DEVICE_COMPILE__)
    constexpr int LANES = D / 4, AT_ONCE = kThreads / LANES;
    __shared__ __attribute__((aligned(16))) float smem[AT_ONCE][D + 4];
    const int heads = p.group * p.Hkv, seq = blockIdx.x / heads, hq = blockIdx.x - seq * heads, head = hq / p.group, row = hq - head * p.group, block = row / (16 * NR), r = row % (16 * NR);
    const int lane = threadIdx.x & 63;
    const Share share = {p.share[0], p.share[1]};
    const int parts = share.parts(__builtin_amdgcn_readfirstlane(tiles_of(p, p.lens[seq])));
    if (parts == 1) return;
    __shared__ int sums[kWaves];
    int before = 0;
    for (int i = threadIdx.x; i < seq; i += kThreads) {
        const int n = tiles_of(p, p.lens[i]);
        before += share.is_long(n) ? share.parts(n) : 0;
    }
    before = sum_of(before);
    if (lane == 0) sums[threadIdx.x >> 6] = before;
    __syncthreads();
    int w0 = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) w0 += sums[w];
    const int w1 = w0 + parts - 1;
    const int c = 4 * (threadIdx.x % LANES), slice = threadIdx.x / LANES;
    float top = kLowest, sum = 0.f;
    f32x4 f = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 2
    for (int w = w0 + slice; w <= w1; w += AT_ONCE) {
        const float* const a = p.parts + (((int64_t)w * p.row_blocks + block) * p.Hkv + head) * kPartFloats<D, NR>;
        const float m = a[16 * NR * D + 2 * r], l = a[16 * NR * D + 2 * r + 1];
        const f32x4 x = *reinterpret_cast<const f32x4*>(a + r * D + c);
        const float to = fmaxf(top, m), was = __builtin_amdgcn_exp2f(top - to), is = __builtin_amdgcn_exp2f(m - to);
        top = to;
        sum = sum * was + l * is;
        f = f * was + x * is;
    }
    *reinterpret_cast<f32x4*>(&smem[slice][c]) = f;
    if (c == 0) { smem[slice][D] = top; smem[slice][D + 1] = sum; }
    __syncthreads();
    if (slice) return;
    for (int i = 0; i < AT_ONCE; ++i) top = fmaxf(top, smem[i][D]);
    sum = 0.f;
    f = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < AT_ONCE; ++i) {
        const float is = __builtin_amdgcn_exp2f(smem[i][D] - top);
        sum += smem[i][D + 1] * is;
        f += *reinterpret_cast<const f32x4*>(&smem[i][c]) * is;
    }
    const float by = sum > 0.f ? 1.f / sum : sum == 0.f ? 0.f : sum;
    *reinterpret_cast<u32x2*>(p.o + (int64_t)seq * p.o_row + hq * p.o_head + 2 * c) = u32x2{round2<T>(f[0] * by, f[1] * by), round2<T>(f[2] * by, f[3] * by)};
    if (p.lse && c == 0) p.lse[(int64_t)seq * heads + hq] = sum > 0.f ? (top + __builtin_amdgcn_logf(sum)) * 0.693147180559945309f : sum == 0.f ? -INFINITY : sum;
#endif
}

// ---- C ABI
constexpr int64_t kMost = 0x7FFFFFFF, kMostBlocks = 0xFFFFFFFF / kThreads;      // (the threads of a launch are a 32-bit number)
constexpr int64_t kMostKeys = (int64_t)1 << 30;       // of a sequence: positions some steps behind its last are 32-bit numbers too
constexpr int64_t kMostRowBytes = (int64_t)1 << 23;

int check_half(const void* at, const int64_t* stride, int bytes, int D) {
    if (!at) return COSMOS_ATTN_BAD_ARG;
    const int64_t unit = 16 / bytes;
    if (!aligned16(at) || stride[0] % unit || stride[1] % unit || stride[2] % unit) return COSMOS_ATTN_BAD_STRIDE;
    if (stride[0] < 0 || stride[1] < 0 || stride[2] < D || stride[2] * bytes > kMostRowBytes) return COSMOS_ATTN_BAD_STRIDE;
    return COSMOS_ATTN_OK;
}
int check_rows(const void* at, const int64_t* stride) {
    if (!at) return COSMOS_ATTN_BAD_ARG;
    return aligned16(at) && stride[0] % 8 == 0 && stride[1] % 8 == 0 && stride[0] >= 0 && stride[1] >= 0 ? COSMOS_ATTN_OK : COSMOS_ATTN_BAD_STRIDE;
}
// outputs: rows and heads that do not share memory
int check_out(const void* at, const int64_t* stride, int64_t rows, int heads, int D) {
    const int st = check_rows(at, stride);
    if (st != COSMOS_ATTN_OK) return st;
    if ((rows > 1 && stride[0] < D) || (heads > 1 && stride[1] < D)) return COSMOS_ATTN_BAD_STRIDE;
    const bool by_row = rows <= 1 || stride[0] >= (heads - 1) * stride[1] + D, by_head = heads <= 1 || stride[1] >= (rows - 1) * stride[0] + D;
    return by_row || by_head ? COSMOS_ATTN_OK : COSMOS_ATTN_BAD_STRIDE;
}
int check_scale(const float* at, const int64_t* stride) {
    if (!at) return COSMOS_ATTN_BAD_ARG;
    return aligned16(at) && stride[0] % 4 == 0 && stride[1] % 4 == 0 && stride[0] >= 0 && stride[1] >= 0 ? COSMOS_ATTN_OK : COSMOS_ATTN_BAD_STRIDE;
}
// pages to be written: of three dims of `size` elements each holds those of smaller strides, down to runs of `run` elements
bool apart(const int64_t (&stride)[3], const int64_t (&size)[3], int64_t run) {
    int order[3] = {0, 1, 2};
    for (int i = 0; i < 3; ++i)
        for (int j = i + 1; j < 3; ++j)
            if (stride[order[j]] < stride[order[i]]) std::swap(order[i], order[j]);
    __int128 extent = run;
    for (int i : order) {
        if (size[i] <= 1) continue;
        if (stride[i] < extent) return false;
        extent += (__int128)(size[i] - 1) * stride[i];
    }
    return true;
}
int check_written(const cosmos_attn_cache_desc* d) {
    const int64_t size[3] = {d->pages, d->Hkv, d->page_size}, ks[3] = {d->k_stride[0], d->k_stride[1], d->k_stride[2]}, vs[3] = {d->v_stride[0], d->v_stride[1], d->v_stride[2]};
    if (d->k == d->v) return COSMOS_ATTN_BAD_ARG;
    if (!apart(ks, size, d->D) || !apart(vs, size, d->D)) return COSMOS_ATTN_BAD_STRIDE;
    if (d->kind == COSMOS_ATTN_CACHE_SAME) return COSMOS_ATTN_OK;
    const int64_t kss[3] = {d->k_scale_stride[0], d->k_scale_stride[1], 1}, vss[3] = {d->v_scale_stride[0], d->v_scale_stride[1], 1};
    if (d->k_scale == d->v_scale) return COSMOS_ATTN_BAD_ARG;
    return apart(kss, size, 1) && apart(vss, size, 1) ? COSMOS_ATTN_OK : COSMOS_ATTN_BAD_STRIDE;
}
int check(const cosmos_attn_cache_desc* d) {
    if (!d || d->abi_version != COSMOS_ATTN_ABI_VERSION) return COSMOS_ATTN_BAD_ARG;
    if (d->dtype != COSMOS_ATTN_BF16 && d->dtype != COSMOS_ATTN_FP16) return COSMOS_ATTN_UNSUPPORTED;
    if (d->kind < COSMOS_ATTN_CACHE_SAME || d->kind > COSMOS_ATTN_CACHE_INT8) return COSMOS_ATTN_UNSUPPORTED;
    if (d->D != 64 && d->D != 128) return COSMOS_ATTN_UNSUPPORTED;
    if (d->Hkv < 1 || d->B < 0 || d->width < 0 || d->pages < 1 || d->pages > kMost) return COSMOS_ATTN_BAD_ARG;
    if (d->page_size < 16 || d->page_size > 1024 || (d->page_size & (d->page_size - 1))) return COSMOS_ATTN_BAD_SHAPE;
    if ((int64_t)d->width * d->page_size > kMostKeys) return COSMOS_ATTN_UNSUPPORTED;
    const int bytes = d->kind == COSMOS_ATTN_CACHE_SAME ? 2 : 1;
    int st = check_half(d->k, d->k_stride, bytes, d->D);
    if (st == COSMOS_ATTN_OK) st = check_half(d->v, d->v_stride, bytes, d->D);
    if (st == COSMOS_ATTN_OK && bytes == 1) st = check_scale(d->k_scale, d->k_scale_stride);
    if (st == COSMOS_ATTN_OK && bytes == 1) st = check_scale(d->v_scale, d->v_scale_stride);
    if (st != COSMOS_ATTN_OK || !d->B) return st;
    if (!d->table && d->width) return COSMOS_ATTN_BAD_ARG;
    if (d->table_stride < 0 || (reinterpret_cast<uintptr_t>(d->table) | reinterpret_cast<uintptr_t>(d->lens) | reinterpret_cast<uintptr_t>(d->cu)) & 3) return COSMOS_ATTN_BAD_STRIDE;
    return COSMOS_ATTN_OK;
}

CacheParams params_of(const cosmos_attn_cache_desc* d) {
    CacheParams p = {};
    const int bytes = d->kind == COSMOS_ATTN_CACHE_SAME ? 2 : 1;
    auto side = [&](void* pages, const int64_t* stride, float* scales, const int64_t* scale_stride, void* packed, const int64_t* packed_stride) {
        return Side{(char*)pages, bytes * stride[0], bytes * stride[1], bytes * stride[2], scales, scale_stride[0], scale_stride[1], (char*)packed, 2 * packed_stride[0], 2 * packed_stride[1]};
    };
    p.side[0] = side(d->k, d->k_stride, d->k_scale, d->k_scale_stride, d->k_rows, d->k_rows_stride);
    p.side[1] = side(d->v, d->v_stride, d->v_scale, d->v_scale_stride, d->v_rows, d->v_rows_stride);
    p.table = d->table; p.lens = d->lens; p.cu = d->cu; p.table_row = d->table_stride;
    p.width = d->width; p.B = d->B; p.pages = (int)d->pages; p.page_shift = __builtin_ctz(d->page_size); p.Hkv = d->Hkv; p.fill = d->fill != 0;
    p.rows = d->rows;
    return p;
}

template <typename F> int with_type(const cosmos_attn_cache_desc* d, F&& f) {
    auto kind = [&](auto* t, auto dim) {
        return d->kind == COSMOS_ATTN_CACHE_SAME ? f(t, dim, Int<SAME16>{}) : d->kind == COSMOS_ATTN_CACHE_E4M3 ? f(t, dim, Int<E4M3>{}) : f(t, dim, Int<INT8>{});
    };
    if (d->dtype == COSMOS_ATTN_BF16) return d->D == 128 ? kind((__bf16*)nullptr, Int<128>{}) : kind((__bf16*)nullptr, Int<64>{});
    return d->D == 128 ? kind((_Float16*)nullptr, Int<128>{}) : kind((_Float16*)nullptr, Int<64>{});
}
int launch(void (*kernel)(CacheParams), int64_t blocks, size_t lds, const CacheParams& p, void* stream) {
    if (blocks <= 0) return COSMOS_ATTN_OK;
    if (blocks > kMostBlocks) return COSMOS_ATTN_UNSUPPORTED;
    if (lds && !allow_lds((const void*)kernel, lds)) return COSMOS_ATTN_LAUNCH_FAILED;
    kernel<<<dim3((unsigned)blocks), dim3(kThreads), lds, (hipStream_t)stream>>>(p);
    return hipGetLastError() == hipSuccess ? COSMOS_ATTN_OK : COSMOS_ATTN_LAUNCH_FAILED;
}

int64_t packed_blocks(const cosmos_attn_cache_desc* d) {
    const int64_t per = kThreads / (d->D / each_of(d->kind));
    return 2 * ((d->rows * d->Hkv + per - 1) / per);
}
int check_packed(const cosmos_attn_cache_desc* d, bool out) {
    int st = check(d);
    if (st != COSMOS_ATTN_OK) return st;
    if (d->rows < 0 || d->rows > kMost) return COSMOS_ATTN_BAD_ARG;
    if (!d->rows) return COSMOS_ATTN_OK;
    if (d->B && !(out ? (const void*)d->cu : (const void*)d->lens)) return COSMOS_ATTN_BAD_ARG;
    if (!out && !d->cu && d->rows != d->B) return COSMOS_ATTN_BAD_SHAPE;
    if (packed_blocks(d) > kMostBlocks) return COSMOS_ATTN_UNSUPPORTED;
    if (!out) st = check_written(d);
    if (st != COSMOS_ATTN_OK) return st;
    if (!d->B && out && !d->cu) return COSMOS_ATTN_BAD_ARG;
    for (int i = 0; st == COSMOS_ATTN_OK && i < 2; ++i) {
        const void* const at = i ? d->v_rows : d->k_rows;
        const int64_t* const stride = i ? d->v_rows_stride : d->k_rows_stride;
        st = out ? check_out(at, stride, d->rows, d->Hkv, d->D) : check_rows(at, stride);
    }
    return st;
}

int check_attention(const cosmos_attn_cache_desc* d) {
    int st = check(d);
    if (st != COSMOS_ATTN_OK) return st;
    if (d->Hq < 1 || !(fabsf(d->sm_scale) <= 3.0e38f)) return COSMOS_ATTN_BAD_ARG;
    if (d->Hq % d->Hkv) return COSMOS_ATTN_BAD_SHAPE;
    if (!d->B) return COSMOS_ATTN_OK;
    if (!d->lens) return COSMOS_ATTN_BAD_ARG;
    // (tiles of all sequences are counted in 32 bits)
    if ((int64_t)d->B * (((int64_t)d->width * d->page_size + kTile - 1) / kTile) > kMost / 2 || (int64_t)d->B * d->Hq > kMostBlocks / 2) return COSMOS_ATTN_UNSUPPORTED;
    st = check_rows(d->q, d->q_stride);
    return st != COSMOS_ATTN_OK ? st : check_out(d->o, d->o_stride, d->B, d->Hq, d->D);
}
// Tables of few tiles: a workgroup for each sequence and head, and nothing to join, which a second launch would be for (333 keys of 4 heads: 6.3 us, as parts 5.8 and 3.8 for the join).  Of
// some more tiles too where there are many workgroups (us, whole / as parts: 32 sequences of 1000 keys, 64 heads of 64 on 8, 13.9 / 20.2; 300 of them in int8 78 / 90; 128 of 2000 keys, 32 heads of 128 on
// 8, 101 / 106; but 40 of them 70 / 68), up to lengths at which the longest alone takes some 20 us.
constexpr int kWholeTiles = 4, kWholeManyTiles = 16, kMany = 32;       // kMany: workgroups to a tile of the table's
struct Shape { int row_blocks, rows16, slots; bool whole; };
Shape shape_of(const cosmos_attn_cache_desc* d) {
    const int group = d->Hq / d->Hkv, rows16 = group <= 16 ? 1 : 2, row_blocks = (group + 16 * rows16 - 1) / (16 * rows16);
    const int64_t capacity = ((int64_t)d->width * d->page_size + kTile - 1) / kTile, most = (int64_t)d->B * capacity;
    if (capacity <= kWholeTiles || (capacity <= kWholeManyTiles && (int64_t)d->B * d->Hkv * row_blocks >= kMany * capacity)) return {row_blocks, rows16, 1, true};
    // two workgroups a compute unit, if the tables hold that many tiles
    int64_t slots = 2 * kNumCUs / ((int64_t)d->Hkv * row_blocks);
    slots = slots < 1 ? 1 : slots;
    return {row_blocks, rows16, (int)(slots > most ? most : slots), false};
}

constexpr size_t kShareBytes = 16;
// parts of all sequences, for a head: each rounds up once (parts are three quarters of a share, rounded up, at least)
int64_t most_parts(int64_t B, int64_t slots) { return 4 * slots / 3 + 1 + B; }

}  // namespace

extern "C" {

int cosmos_attn_cache_write(const cosmos_attn_cache_desc* desc, void* stream) {
    const int st = check_packed(desc, false);
    if (st != COSMOS_ATTN_OK || !desc->rows || !desc->B) return st;
    if (!device_is_whole_mi355x()) return COSMOS_ATTN_WRONG_DEVICE;
    const CacheParams p = params_of(desc);
    return with_type(desc, [&](auto* t, auto dim, auto kind) {
        return launch(cache_write_kernel<std::remove_pointer_t<decltype(t)>, decltype(kind)::value, decltype(dim)::value>, packed_blocks(desc), 0, p, stream);
    });
}

int cosmos_attn_cache_read(const cosmos_attn_cache_desc* desc, void* stream) {
    const int st = check_packed(desc, true);
    if (st != COSMOS_ATTN_OK || !desc->rows) return st;
    if (!device_is_whole_mi355x()) return COSMOS_ATTN_WRONG_DEVICE;
    const CacheParams p = params_of(desc);
    return with_type(desc, [&](auto* t, auto dim, auto kind) {
        return launch(cache_read_kernel<std::remove_pointer_t<decltype(t)>, decltype(kind)::value, decltype(dim)::value>, packed_blocks(desc), 0, p, stream);
    });
}

size_t cosmos_attn_cache_attention_workspace_bytes(const cosmos_attn_cache_desc* desc) {
    if (check_attention(desc) != COSMOS_ATTN_OK || !desc->B) return 0;
    const Shape s = shape_of(desc);
    return s.whole ? 0 : (size_t)most_parts(desc->B, s.slots) * s.row_blocks * desc->Hkv * 16 * s.rows16 * (desc->D + 2) * sizeof(float) + kShareBytes;
}

int cosmos_attn_cache_attention(const cosmos_attn_cache_desc* desc, void* workspace, size_t workspace_bytes, void* stream) {
    const int st = check_attention(desc);
    if (st != COSMOS_ATTN_OK || !desc->B) return st;
    const size_t wanted = cosmos_attn_cache_attention_workspace_bytes(desc);
    if (workspace_bytes < wanted || (wanted && !workspace)) return COSMOS_ATTN_WORKSPACE_TOO_SMALL;
    if (wanted && !aligned16(workspace)) return COSMOS_ATTN_BAD_STRIDE;
    if (!device_is_whole_mi355x()) return COSMOS_ATTN_WRONG_DEVICE;
    const Shape s = shape_of(desc);
    CacheParams p = params_of(desc);
    p.q = (const char*)desc->q; p.o = (char*)desc->o; p.lse = desc->lse;
    p.q_row = 2 * desc->q_stride[0]; p.q_head = 2 * desc->q_stride[1]; p.o_row = 2 * desc->o_stride[0]; p.o_head = 2 * desc->o_stride[1];
    p.group = desc->Hq / desc->Hkv; p.row_blocks = s.row_blocks; p.slots = s.slots; p.whole = s.whole;
    p.scale_log2 = fmaxf(fabsf(desc->sm_scale) * 1.44269504088896341f, 1e-37f);
    p.flip = signbit(desc->sm_scale) ? 0x80008000u : 0u;
    p.parts = (float*)workspace;
    p.share = wanted ? (int*)((char*)workspace + wanted - kShareBytes) : nullptr;
    return with_type(desc, [&](auto* t, auto dim, auto kind) {
        typedef std::remove_pointer_t<decltype(t)> T;
        constexpr int D = decltype(dim)::value, K = decltype(kind)::value;
        auto run = [&](auto blocks16) {
            constexpr int NR = decltype(blocks16)::value;
            const int done = launch(cache_attention_kernel<T, K, D, NR>, (int64_t)p.Hkv * p.row_blocks * (s.whole ? p.B : most_parts(p.B, p.slots)), 4 * 16 * NR * (D + 2) * sizeof(float), p, stream);
            return done != COSMOS_ATTN_OK || s.whole ? done : launch(cache_join_kernel<T, D, NR>, (int64_t)desc->Hq * p.B, 0, p, stream);
        };
        return s.rows16 == 1 ? run(Int<1>{}) : run(Int<2>{});
    });
}

}  // extern "C"
