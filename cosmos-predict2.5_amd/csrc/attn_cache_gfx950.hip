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

struct CacheParams {
    char *k, *v;                                  // bytes between pages, heads and rows
    int64_t k_page, k_head, v_page, v_head;
    int k_row, v_row;
    float *k_scale, *v_scale;                     // elements between pages and heads
    int64_t ks_page, ks_head, vs_page, vs_head;
    const int *table, *lens, *cu;
    int64_t table_row;
    int width, B, pages, page_shift, Hkv, fill;
    int64_t rows;                                 // packed rows
    char *k_rows, *v_rows;                        // bytes between rows and heads
    int64_t kr_row, kr_head, vr_row, vr_head;
    // attention
    const char* q;
    char* o;
    float* lse;
    int64_t q_row, q_head, o_row, o_head;
    int group, row_blocks, slots;                 // slots: workgroups per head and block of rows
    float scale_log2;
    unsigned flip;
    float* parts;
};

// ---- 16-bit pairs
template <typename T> __device__ __forceinline__ unsigned round2(float a, float b) {
    typedef T V2 __attribute__((ext_vector_type(2)));
    const V2 two = {(T)a, (T)b};
    return __builtin_bit_cast(unsigned, two);
}
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

// max over the LANES (8 or 16) neighbouring lanes of a row
template <int CTRL> __device__ __forceinline__ float dpp_max(float v) {
    return fmaxf(v, __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xF, 0xF, false)));
}
template <int LANES> __device__ __forceinline__ float row_max(float v) {
    v = dpp_max<0xB1>(v);       // quad_perm [1, 0, 3, 2]
    v = dpp_max<0x4E>(v);       // quad_perm [2, 3, 0, 1]
    v = dpp_max<0x141>(v);      // row_half_mirror
    return LANES == 16 ? dpp_max<0x140>(v) : v;      // row_mirror
}

// ---- packed rows: which sequence a row is of, and its place there; false: of none
__device__ __forceinline__ bool place_of(const int* cu, int n, int64_t row, int64_t rows, int& seq, int& place, int& length) {
    int lo = 0, hi = n;                           // the last offset at or below the row
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (cu[mid] <= row) lo = mid;
        else hi = mid - 1;
    }
    const int64_t a = cu[lo], b = lo < n ? cu[lo + 1] : a;
    seq = lo;
    place = (int)(row - a);
    length = (int)(b - a);
    return lo < n && a >= 0 && row >= a && row < b && b <= rows;
}

constexpr int kRowsPerThread = 4;      // rows that a thread has under way

// ---- writing: D / 8 lanes to a row, its max by exchanges among them
template <typename T, int KIND, int D>
__global__ void __launch_bounds__(kThreads) cache_write_kernel(const CacheParams p) {
#if defined(__HIP_DEVICE_COMPILE__)
    constexpr int LANES = D / 8, ROWS = kThreads / LANES;
    const int part = threadIdx.x % LANES;
    const int64_t units = p.rows * 2 * p.Hkv;
#pragma unroll
    for (int i = 0; i < kRowsPerThread; ++i) {
        const int64_t u = ((int64_t)blockIdx.x * kRowsPerThread + i) * ROWS + threadIdx.x / LANES;
        if (u >= units) return;
        const int64_t row = u / (2 * p.Hkv);
        const int which = (int)(u - row * 2 * p.Hkv), value = which >= p.Hkv, h = value ? which - p.Hkv : which;
        int seq = (int)row, place = 0, fresh = 1;
        if (p.cu && !place_of(p.cu, p.B, row, p.rows, seq, place, fresh)) continue;
        const int at = p.lens[seq] - fresh + place;
        if (at < 0 || p.lens[seq] < fresh || (at >> p.page_shift) >= p.width) continue;
        const int page = p.table[seq * p.table_row + (at >> p.page_shift)];
        if (page < 0 || page >= p.pages) continue;
        const int in_page = at & ((1 << p.page_shift) - 1);
        const u32x4 x = *reinterpret_cast<const u32x4*>((value ? p.v_rows + row * p.vr_row + h * p.vr_head : p.k_rows + row * p.kr_row + h * p.kr_head) + 16 * part);
        char* const to = value ? p.v + page * p.v_page + h * p.v_head + (int64_t)in_page * p.v_row : p.k + page * p.k_page + h * p.k_head + (int64_t)in_page * p.k_row;
        if constexpr (KIND == SAME16) {
            *reinterpret_cast<u32x4*>(to + 16 * part) = x;
        } else {
            float f[8], top = 0.f, nan = 0.f;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                f[2 * j] = low<T>(x[j]);
                f[2 * j + 1] = high<T>(x[j]);
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                top = fmaxf(top, fabsf(f[j]));
                nan = f[j] == f[j] ? nan : INFINITY;           // (a max passes over NaN)
            }
            top = row_max<LANES>(fmaxf(top, nan));
            const bool finite = top < INFINITY;
            const float scale = finite ? top * (KIND == E4M3 ? 1.f / 448.f : 1.f / 127.f) : NAN;
            const bool some = finite && scale > 0.f;
            u32x2 codes = {0, 0};
#pragma unroll
            for (int j = 0; j < 8; ++j) f[j] = some ? f[j] / scale : 0.f;
            if constexpr (KIND == E4M3) {
                // (scale's own rounding may leave a quotient just above 448; the conversion's largest code takes those below 464)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    int w = __builtin_amdgcn_cvt_pk_fp8_f32(f[4 * j], f[4 * j + 1], 0, false);
                    codes[j] = (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(f[4 * j + 2], f[4 * j + 3], w, true);
                }
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) codes[j / 4] |= ((unsigned)(int)__builtin_rintf(fminf(fmaxf(f[j], -127.f), 127.f)) & 0xFFu) << 8 * (j % 4);
            }
            *reinterpret_cast<u32x2*>(to + 8 * part) = codes;
            if (part == 0) (value ? p.v_scale + page * p.vs_page + h * p.vs_head : p.k_scale + page * p.ks_page + h * p.ks_head)[in_page] = scale;
        }
    }
#endif
}

// ---- reading back
template <typename T, int KIND, int D>
__global__ void __launch_bounds__(kThreads) cache_read_kernel(const CacheParams p) {
#if defined(__HIP_DEVICE_COMPILE__)
    constexpr int LANES = D / 8, ROWS = kThreads / LANES;
    const int part = threadIdx.x % LANES;
    const int64_t units = p.rows * 2 * p.Hkv;
#pragma unroll
    for (int i = 0; i < kRowsPerThread; ++i) {
        const int64_t u = ((int64_t)blockIdx.x * kRowsPerThread + i) * ROWS + threadIdx.x / LANES;
        if (u >= units) return;
        const int64_t row = u / (2 * p.Hkv);
        const int which = (int)(u - row * 2 * p.Hkv), value = which >= p.Hkv, h = value ? which - p.Hkv : which;
        u32x4* const to = reinterpret_cast<u32x4*>((value ? p.v_rows + row * p.vr_row + h * p.vr_head : p.k_rows + row * p.kr_row + h * p.kr_head) + 16 * part);
        int seq, at, length;
        if (!place_of(p.cu, p.B, row, p.rows, seq, at, length)) {
            if (p.fill) *to = u32x4{0, 0, 0, 0};
            continue;
        }
        int page = -1;
        if ((at >> p.page_shift) < p.width) page = p.table[seq * p.table_row + (at >> p.page_shift)];
        if (page < 0 || page >= p.pages) {
            const unsigned nan = round2<T>(NAN, NAN);
            *to = u32x4{nan, nan, nan, nan};
            continue;
        }
        const int in_page = at & ((1 << p.page_shift) - 1);
        const char* const from = value ? p.v + page * p.v_page + h * p.v_head + (int64_t)in_page * p.v_row : p.k + page * p.k_page + h * p.k_head + (int64_t)in_page * p.k_row;
        if constexpr (KIND == SAME16) {
            *to = *reinterpret_cast<const u32x4*>(from + 16 * part);
        } else {
            const u32x2 codes = *reinterpret_cast<const u32x2*>(from + 8 * part);
            const float scale = (value ? p.v_scale + page * p.vs_page + h * p.vs_head : p.k_scale + page * p.ks_page + h * p.ks_head)[in_page];
            u32x4 w;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const unsigned a = code_pair<T, KIND, false>(codes[j]), b = code_pair<T, KIND, true>(codes[j]);
                w[2 * j] = round2<T>(low<T>(a) * scale, high<T>(a) * scale);
                w[2 * j + 1] = round2<T>(low<T>(b) * scale, high<T>(b) * scale);
            }
            *to = w;
        }
    }
#endif
}

// ---- attention of one token over the pages
// The keys of all sequences, in tiles of kTile (each sequence rounded up), are one list per key head, dealt out to `slots` workgroups in equal runs.  A workgroup writes the sequences
// that lie in its run whole; of one that its neighbours share it leaves sums of its part, which cache_join_kernel adds up.
constexpr int kTile = 128;           // keys: 32 of each wavefront
constexpr int kLeast = 1;            // tiles of a workgroup
constexpr float kLowest = -3.0e38f;

__device__ __forceinline__ int tiles_of(const CacheParams& p, int i) {
    const int n = p.lens[i];
    return n > 0 && n <= (int64_t)p.width << p.page_shift ? (n + kTile - 1) / kTile : 0;
}
// the tiles in front of sequence i (or all of them, i = B) and those of sequences up to 64 on: sums over 64 sequences a step
struct Scan { int before, sum, tiles; };
__device__ __forceinline__ int scan64(int tiles) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) { const int up = __shfl_up(tiles, d); tiles += lane >= d ? up : 0; }
    return tiles;
}
__device__ __forceinline__ int total_tiles(const CacheParams& p) {
    const int lane = threadIdx.x & 63;
    int mine = 0;
    for (int base = 0; base < p.B; base += 64) mine += base + lane < p.B ? tiles_of(p, base + lane) : 0;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) mine += __shfl_xor(mine, d);
    return __builtin_amdgcn_readfirstlane(mine);
}
__device__ __forceinline__ int run_length(int total, int slots) {
    const int per = (total + slots - 1) / slots;
    return per > kLeast ? per : kLeast;
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

    const int total = total_tiles(p), per = run_length(total, p.slots);
    const int first = slot * per, last = first + per < total ? first + per : total;
    // (sequences of nothing are whole wherever they lie: the first workgroup's)
    if (slot == 0) {
        for (int i = wave; i < p.B; i += kThreads / 64) {
            if (tiles_of(p, i)) continue;
            const bool bad = p.lens[i] != 0;
            for (int r = 0; r < 16 * NR && row0 + r < p.group; ++r) {
                const int hq = head * p.group + row0 + r;
                const unsigned w = bad ? round2<T>(NAN, NAN) : 0u;
                if (lane < D / 8) *reinterpret_cast<u32x4*>(p.o + i * p.o_row + hq * p.o_head + 16 * lane) = u32x4{w, w, w, w};
                if (p.lse && lane == 0) p.lse[(int64_t)i * p.group * p.Hkv + hq] = bad ? NAN : -INFINITY;
            }
        }
    }
    if (first >= last) return;

    // the first sequence of the run
    int seq = 0, begin = 0;                       // (begin: of its tiles in the list)
    for (int base = 0, before = 0; base < p.B; base += 64) {
        const int sum = scan64(base + lane < p.B ? tiles_of(p, base + lane) : 0);
        const unsigned long long past = __ballot(before + sum > first);
        if (past) {
            const int at = __builtin_ctzll(past);
            seq = base + at;
            begin = before + __builtin_amdgcn_readlane(sum, at) - __builtin_amdgcn_readfirstlane(tiles_of(p, seq));
            break;
        }
        before += __builtin_amdgcn_readlane(sum, 63);
    }

    const char* const kh = p.k + head * p.k_head;
    const char* const vh = p.v + head * p.v_head;
    const int mask = (1 << p.page_shift) - 1;
    for (int tile = first; tile < last;) {
        const int len = __builtin_amdgcn_readfirstlane(p.lens[seq]), tiles = __builtin_amdgcn_readfirstlane(tiles_of(p, seq));
        if (!tiles) { ++seq; continue; }
        const int from = tile - begin, to = last - begin < tiles ? last - begin : tiles;      // of this sequence's tiles
        const int* const table = p.table + seq * p.table_row;

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
        for (int t = from; t < to; ++t) {
            const int key0 = t * kTile + 32 * wave;
            if (key0 >= len) break;
            // Keys past the end are the last one's, with weights of 0: whatever else the page holds is not looked at.
            const int most = len - 1;
            auto page_at = [&](int key) {
                const int page = table[key >> p.page_shift];
                const bool in = page >= 0 && page < p.pages;
                bad |= !in;
                return in ? page : 0;
            };
            // K: row n16 of key half u is key 8 (n16 / 4) + 4 u + n16 % 4, so that a lane's results of the two halves are those of 8 keys in order, 8 g .. 8 g + 7
            unsigned kw[2][CODES ? NC / 2 : NC][4];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                int key = key0 + 8 * (n16 >> 2) + 4 * u + (n16 & 3);
                key = key < most ? key : most;
                const char* const at = kh + page_at(key) * p.k_page + (int64_t)(key & mask) * p.k_row;
#pragma unroll
                for (int c = 0; c < (CODES ? NC / 2 : NC); ++c) {
                    const u32x4 w = *reinterpret_cast<const u32x4*>(at + 64 * c + 16 * g);
#pragma unroll
                    for (int i = 0; i < 4; ++i) kw[u][c][i] = w[i];
                }
            }
            // V: keys 8 g .. 8 g + 7, channels NB n16 .. NB n16 + NB - 1
            unsigned vw[8][NB / 2];
            float ks[8], vs[8];
            const int key8 = key0 + 8 * g < (most & ~7) ? key0 + 8 * g : (most & ~7);
            const int page8 = page_at(key8), in8 = key8 & mask;
            {
                const char* const at = vh + page8 * p.v_page + (int64_t)in8 * p.v_row + NB * BYTES * n16;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const char* const a = at + (int64_t)(key8 + i < most ? i : most - key8) * p.v_row;
                    constexpr int WORDS = NB * BYTES / 4;
                    unsigned w[WORDS];
                    __builtin_memcpy(w, __builtin_assume_aligned(a, 4 * WORDS), 4 * WORDS);
                    if constexpr (CODES) {
#pragma unroll
                        for (int j = 0; j < WORDS; ++j) {
                            vw[i][2 * j] = code_pair<T, KIND, false>(w[j]);
                            vw[i][2 * j + 1] = code_pair<T, KIND, true>(w[j]);
                        }
                    } else {
#pragma unroll
                        for (int j = 0; j < WORDS; ++j) vw[i][j] = w[j];
                    }
                }
            }
            if constexpr (CODES) {
                const float* const a = p.k_scale + page8 * p.ks_page + head * p.ks_head + in8;
                const float* const b = p.v_scale + page8 * p.vs_page + head * p.vs_head + in8;
                __builtin_memcpy(ks, __builtin_assume_aligned(a, 16), 32);
                __builtin_memcpy(vs, __builtin_assume_aligned(b, 16), 32);
            }
            const int left = len - key0 - 8 * g;
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
                        top = fmaxf(R, over_quarters_max(top));
                        const float f = R / top;
#pragma unroll
                        for (int r = 0; r < NR; ++r)
#pragma unroll
                            for (int b = 0; b < NB; ++b) acc[r][b] *= f;
                        R = top;
                    }
#pragma unroll
                    for (int i = 0; i < 8; ++i) by[i] = R > 0.f ? by[i] / R : by[i];
                }
            }
#pragma unroll
            for (int r = 0; r < NR; ++r) {
                f32x4 s[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
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
#pragma unroll
                            for (int i = 0; i < 4; ++i) w[i] = kw[u][c][i];
                        }
                        s[u] = mfma16(__builtin_bit_cast(V8, w), qf[r][c], s[u]);
                    }
                float x[8], top = -INFINITY;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    x[i] = s[i / 4][i % 4] * p.scale_log2;
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
                const V8 pf = __builtin_bit_cast(V8, w);
                // output rows NB n + b, n = 0 .. 15: what lane n16 holds of V, transposed in its registers
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    u32x4 vt;
#pragma unroll
                    for (int i = 0; i < 4; ++i) vt[i] = __builtin_amdgcn_perm(vw[2 * i + 1][b / 2], vw[2 * i][b / 2], b % 2 ? 0x07060302u : 0x05040100u);
                    acc[r][b] = mfma16(__builtin_bit_cast(V8, vt), pf, acc[r][b]);
                }
            }
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
        const bool whole = from == 0 && to == tiles;
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
            if (whole) {
                const float by = sum > 0.f ? 1.f / sum : sum == 0.f ? 0.f : sum;
                *reinterpret_cast<u32x4*>(p.o + (int64_t)seq * p.o_row + hq * p.o_head + 2 * c) = u32x4{round2<T>(f[0] * by, f[1] * by), round2<T>(f[2] * by, f[3] * by), round2<T>(f[4] * by, f[5] * by), round2<T>(f[6] * by, f[7] * by)};
                if (p.lse && c == 0) p.lse[(int64_t)seq * p.group * p.Hkv + hq] = sum > 0.f ? (top + __builtin_amdgcn_logf(sum)) * 0.693147180559945309f : sum == 0.f ? -INFINITY : sum;
            } else {
                // a run's first sequence may be its predecessors' too (part 0), its last one its successors' (part 1, unless it is the first as well)
                float* const part = p.parts + ((((int64_t)slot * p.row_blocks + block) * p.Hkv + head) * 2 + (from == 0)) * kPartFloats<D, NR>;
                *reinterpret_cast<f32x4*>(part + r * D + c) = f32x4{f[0], f[1], f[2], f[3]};
                *reinterpret_cast<f32x4*>(part + r * D + c + 4) = f32x4{f[4], f[5], f[6], f[7]};
                if (c == 0) { part[16 * NR * D + 2 * r] = top; part[16 * NR * D + 2 * r + 1] = sum; }
            }
        }
        __syncthreads();
        tile = begin + to;
        begin += tiles;
        ++seq;
    }
#endif
}

// ---- the sequences that several workgroups have parts of: one workgroup for each sequence, key head and block of rows
template <typename T, int D, int NR>
__global__ void __launch_bounds__(kThreads) cache_join_kernel(const CacheParams p) {
#if defined(__HIP_DEVICE_COMPILE__)
    const int head = blockIdx.x % p.Hkv, block = blockIdx.x / p.Hkv % p.row_blocks, seq = blockIdx.x / (p.Hkv * p.row_blocks), lane = threadIdx.x & 63;
    const int tiles = tiles_of(p, seq);
    if (!tiles) return;
    int all = 0, before = 0;
    for (int base = 0; base < p.B; base += 64) {
        const int n = base + lane < p.B ? tiles_of(p, base + lane) : 0;
        all += n;
        before += base + lane < seq ? n : 0;
    }
#pragma unroll
    for (int d = 1; d < 64; d *= 2) { all += __shfl_xor(all, d); before += __shfl_xor(before, d); }
    const int per = run_length(all, p.slots), w0 = before / per, w1 = (before + tiles - 1) / per;
    if (w0 == w1) return;
    constexpr int LANES = D / 4, AT_ONCE = kThreads / LANES;
    const int row0 = block * 16 * NR;
    auto part = [&](int w) { return p.parts + ((((int64_t)w * p.row_blocks + block) * p.Hkv + head) * 2 + (w == w0)) * kPartFloats<D, NR>; };
    for (int r = threadIdx.x / LANES; r < 16 * NR && row0 + r < p.group; r += AT_ONCE) {
        const int c = 4 * (threadIdx.x % LANES);
        float top = kLowest, sum = 0.f;
        f32x4 f = {0.f, 0.f, 0.f, 0.f};
        for (int w = w0; w <= w1; ++w) top = fmaxf(top, part(w)[16 * NR * D + 2 * r]);
        for (int w = w0; w <= w1; ++w) {
            const float* const a = part(w);
            const float by = __builtin_amdgcn_exp2f(a[16 * NR * D + 2 * r] - top);
            sum += by * a[16 * NR * D + 2 * r + 1];
            f += by * *reinterpret_cast<const f32x4*>(a + r * D + c);
        }
        const float by = sum > 0.f ? 1.f / sum : sum == 0.f ? 0.f : sum;
        const int hq = head * p.group + row0 + r;
        *reinterpret_cast<u32x2*>(p.o + (int64_t)seq * p.o_row + hq * p.o_head + 2 * c) = u32x2{round2<T>(f[0] * by, f[1] * by), round2<T>(f[2] * by, f[3] * by)};
        if (p.lse && c == 0) p.lse[(int64_t)seq * p.group * p.Hkv + hq] = sum > 0.f ? (top + __builtin_amdgcn_logf(sum)) * 0.693147180559945309f : sum == 0.f ? -INFINITY : sum;
    }
#endif
}

// ---- C ABI
constexpr int64_t kMost = 0x7FFFFFFF;
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
int check(const cosmos_attn_cache_desc* d) {
    if (!d || d->abi_version != COSMOS_ATTN_ABI_VERSION) return COSMOS_ATTN_BAD_ARG;
    if (d->dtype != COSMOS_ATTN_BF16 && d->dtype != COSMOS_ATTN_FP16) return COSMOS_ATTN_UNSUPPORTED;
    if (d->kind < COSMOS_ATTN_CACHE_SAME || d->kind > COSMOS_ATTN_CACHE_INT8) return COSMOS_ATTN_UNSUPPORTED;
    if (d->D != 64 && d->D != 128) return COSMOS_ATTN_UNSUPPORTED;
    if (d->Hkv < 1 || d->B < 0 || d->width < 0 || d->pages < 1 || d->pages > kMost) return COSMOS_ATTN_BAD_ARG;
    if (d->page_size < 16 || d->page_size > 1024 || (d->page_size & (d->page_size - 1))) return COSMOS_ATTN_BAD_SHAPE;
    if ((int64_t)d->width * d->page_size > kMost) return COSMOS_ATTN_UNSUPPORTED;
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
    p.k = (char*)d->k; p.v = (char*)d->v;
    p.k_page = bytes * d->k_stride[0]; p.k_head = bytes * d->k_stride[1]; p.k_row = (int)(bytes * d->k_stride[2]);
    p.v_page = bytes * d->v_stride[0]; p.v_head = bytes * d->v_stride[1]; p.v_row = (int)(bytes * d->v_stride[2]);
    p.k_scale = d->k_scale; p.v_scale = d->v_scale;
    p.ks_page = d->k_scale_stride[0]; p.ks_head = d->k_scale_stride[1]; p.vs_page = d->v_scale_stride[0]; p.vs_head = d->v_scale_stride[1];
    p.table = d->table; p.lens = d->lens; p.cu = d->cu; p.table_row = d->table_stride;
    p.width = d->width; p.B = d->B; p.pages = (int)d->pages; p.page_shift = __builtin_ctz(d->page_size); p.Hkv = d->Hkv; p.fill = d->fill != 0;
    p.rows = d->rows;
    p.k_rows = (char*)d->k_rows; p.v_rows = (char*)d->v_rows;
    p.kr_row = 2 * d->k_rows_stride[0]; p.kr_head = 2 * d->k_rows_stride[1]; p.vr_row = 2 * d->v_rows_stride[0]; p.vr_head = 2 * d->v_rows_stride[1];
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
    if (blocks > kMost) return COSMOS_ATTN_UNSUPPORTED;
    if (lds && !allow_lds((const void*)kernel, lds)) return COSMOS_ATTN_LAUNCH_FAILED;
    kernel<<<dim3((unsigned)blocks), dim3(kThreads), lds, (hipStream_t)stream>>>(p);
    return hipGetLastError() == hipSuccess ? COSMOS_ATTN_OK : COSMOS_ATTN_LAUNCH_FAILED;
}

int check_packed(const cosmos_attn_cache_desc* d, bool out) {
    int st = check(d);
    if (st != COSMOS_ATTN_OK) return st;
    if (d->rows < 0 || d->rows > kMost) return COSMOS_ATTN_BAD_ARG;
    if (!d->rows) return COSMOS_ATTN_OK;
    if (d->B && !(out ? (const void*)d->cu : (const void*)d->lens)) return COSMOS_ATTN_BAD_ARG;
    if (!out && !d->cu && d->rows != d->B) return COSMOS_ATTN_BAD_SHAPE;
    if (!d->B && out && !d->cu) return COSMOS_ATTN_BAD_ARG;
    for (int i = 0; st == COSMOS_ATTN_OK && i < 2; ++i) {
        const void* const at = i ? d->v_rows : d->k_rows;
        const int64_t* const stride = i ? d->v_rows_stride : d->k_rows_stride;
        st = out ? check_out(at, stride, d->rows, d->Hkv, d->D) : check_rows(at, stride);
    }
    return st;
}
int64_t packed_blocks(const cosmos_attn_cache_desc* d) {
    const int64_t per = (int64_t)kRowsPerThread * (kThreads / (d->D / 8));
    return (d->rows * 2 * d->Hkv + per - 1) / per;
}

int check_attention(const cosmos_attn_cache_desc* d) {
    int st = check(d);
    if (st != COSMOS_ATTN_OK) return st;
    if (d->Hq < 1 || !(fabsf(d->sm_scale) <= 3.0e38f)) return COSMOS_ATTN_BAD_ARG;
    if (d->Hq % d->Hkv) return COSMOS_ATTN_BAD_SHAPE;
    if (!d->B) return COSMOS_ATTN_OK;
    if (!d->lens) return COSMOS_ATTN_BAD_ARG;
    // (tiles of all sequences are counted in 32 bits)
    if ((int64_t)d->B * (((int64_t)d->width * d->page_size + kTile - 1) / kTile) > kMost / 2) return COSMOS_ATTN_UNSUPPORTED;
    st = check_rows(d->q, d->q_stride);
    return st != COSMOS_ATTN_OK ? st : check_out(d->o, d->o_stride, d->B, d->Hq, d->D);
}
struct Shape { int row_blocks, rows16, slots; bool whole; };
Shape shape_of(const cosmos_attn_cache_desc* d) {
    const int group = d->Hq / d->Hkv, rows16 = group <= 16 ? 1 : 2, row_blocks = (group + 16 * rows16 - 1) / (16 * rows16);
    const int64_t capacity = ((int64_t)d->width * d->page_size + kTile - 1) / kTile, most = (int64_t)d->B * capacity;
    // as many workgroups as fit on the chip at once, if the tables hold that many tiles
    int64_t slots = 2 * kNumCUs / ((int64_t)d->Hkv * row_blocks);
    slots = slots < 1 ? 1 : slots;
    slots = slots > most ? most : slots;
    return {row_blocks, rows16, (int)(slots < 1 ? 1 : slots), capacity <= 1};
}

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
    return s.whole ? 0 : (size_t)s.slots * s.row_blocks * desc->Hkv * 2 * 16 * s.rows16 * (desc->D + 2) * sizeof(float);
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
    p.group = desc->Hq / desc->Hkv; p.row_blocks = s.row_blocks; p.slots = s.slots;
    p.scale_log2 = fmaxf(fabsf(desc->sm_scale) * 1.44269504088896341f, 1e-37f);
    p.flip = signbit(desc->sm_scale) ? 0x80008000u : 0u;
    p.parts = (float*)workspace;
    return with_type(desc, [&](auto* t, auto dim, auto kind) {
        typedef std::remove_pointer_t<decltype(t)> T;
        constexpr int D = decltype(dim)::value, K = decltype(kind)::value;
        auto run = [&](auto blocks16) {
            constexpr int NR = decltype(blocks16)::value;
            const int done = launch(cache_attention_kernel<T, K, D, NR>, (int64_t)p.Hkv * p.row_blocks * p.slots, 4 * 16 * NR * (D + 2) * sizeof(float), p, stream);
            return done != COSMOS_ATTN_OK || s.whole ? done : launch(cache_join_kernel<T, D, NR>, (int64_t)p.Hkv * p.row_blocks * p.B, 0, p, stream);
        };
        return s.rows16 == 1 ? run(Int<1>{}) : run(Int<2>{});
    });
}

}  // extern "C"
