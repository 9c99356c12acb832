// Pieces shared by the kernels of the paged key-value cache: where its rows lie, codes of 8 bits, which sequence a packed row is of, checks of descriptors.  Included inside each translation
// unit's anonymous namespace, behind attn_common_gfx950.h and a definition of kThreads.
//
// Position j of sequence i lies in page table[i][j / page_size], place j % page_size.  Pages hold, for each head, page_size rows of D elements of the 16-bit type, or of 8 bits with one fp32
// scale for each row of a head:
//     scale = max |x| r,  r = fp32(1 / 448) (e4m3) or fp32(1 / 127) (int8),   code = round(x / scale) (nearest, ties to even),   x' = code scale
// in fp32, the quotient an IEEE division: values of 8 bits of mantissa often lie on a border between two codes, and these are then the same ones everywhere.  A row with a value that
// is not finite has the scale NaN.
//
// What the host's tables say is not trusted: a page outside of the cache or a length that the table does not hold makes the sequence's output NaN (attention, reading back) or writes nothing.
#ifndef COSMOS_ATTN_CACHE_GFX950_H
#define COSMOS_ATTN_CACHE_GFX950_H

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));

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
    int window, sinks;                            // keys that a token looks back on, its own among them; first keys that every one sees
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

// the codes of four quotients
template <int KIND> __device__ __forceinline__ unsigned code_word(float a, float b, float c, float d) {
#if defined(__HIP_DEVICE_COMPILE__)
    if constexpr (KIND == E4M3) {
        // (a scale's own rounding may leave a quotient just above 448; the conversion's largest code takes those below 464)
        return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false), true);
    } else {
        // 2^23 + 2^22 + f: f rounded to a whole number, ties to even, in the low bits
        const unsigned w[4] = {__builtin_bit_cast(unsigned, a + 12582912.f), __builtin_bit_cast(unsigned, b + 12582912.f), __builtin_bit_cast(unsigned, c + 12582912.f),
                               __builtin_bit_cast(unsigned, d + 12582912.f)};
        return __builtin_amdgcn_perm(w[1], w[0], 0x0C0C0400u) | __builtin_amdgcn_perm(w[3], w[2], 0x04000C0Cu);
    }
#else
    return 0;
#endif
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

// x / s as IEEE division rounds it, for fp32 numbers with |x / s| up to some hundreds: x r corrected by the remainder (Markstein's division), with r = 1 / s corrected by its own.  With the nearest r, which this
// is for each of the 2^23 significands of s (the instruction is good to one unit), that is 3 units times 2^-24 off at most before its rounding; of quotients that close to the middle of two numbers there are
// 29 million, and all of them come out right.  (tests/test_host_division.py has the bound and how to find them.)  Rows whose scale would leave the range in which all of that is exact are multiplied
// with a power of two first, as their scale is.
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
// Rows of D 16-bit elements, [rows, heads]: do two such tensors have an element in common?  Of different row strides they are taken to where their extents meet.
struct Packed { const void* at; const int64_t* stride; int heads; };
bool meet_in_memory(Packed a, Packed b, int64_t rows, int D) {
    const bool one_row = rows <= 1;
    auto extent = [&](Packed x) { return (__int128)(one_row ? 0 : rows - 1) * x.stride[0] + (__int128)(x.heads - 1) * x.stride[1] + D; };
    const __int128 between = ((__int128)reinterpret_cast<uintptr_t>(b.at) - (__int128)reinterpret_cast<uintptr_t>(a.at)) / 2;      // elements from a's first row to b's (of 16-byte steps)
    if (between >= extent(a) || -between >= extent(b)) return false;
    if (extent(a) >> 62 || extent(b) >> 62 || (!one_row && a.stride[0] != b.stride[0])) return true;
    const int64_t step = one_row ? 0 : a.stride[0], d0 = (int64_t)between, ea = (a.heads - 1) * a.stride[1] + D, eb = (b.heads - 1) * b.stride[1] + D;
    // parts of wider rows, the most frequent case: b's lies between a's and the next row's
    if (step > 0) {
        const int64_t in = (d0 % step + step) % step;
        if (in >= ea && in + eb <= step) return false;
    }
    for (int i = 0; i < a.heads; ++i)
        for (int j = 0; j < b.heads; ++j) {
            const int64_t d = d0 + j * b.stride[1] - i * a.stride[1], n = step ? -d / step : 0;
            // some row of b, `k` rows behind one of a, is less than a row's D elements from it
            for (int64_t k = n - 1; k <= n + 1; ++k)
                if (k < rows && -k < rows && d + k * step < D && -(d + k * step) < D) return true;
        }
    return false;
}
// Queries and the output of as many rows and heads: apart, or the same rows, which a lane (a workgroup) has read before it writes them.
int check_in_place(const cosmos_attn_cache_desc* d, int64_t rows) {
    const bool same = d->o == d->q && (rows <= 1 || d->o_stride[0] == d->q_stride[0]) && (d->Hq <= 1 || d->o_stride[1] == d->q_stride[1]);
    return same || !meet_in_memory({d->o, d->o_stride, d->Hq}, {d->q, d->q_stride, d->Hq}, rows, d->D) ? COSMOS_ATTN_OK : COSMOS_ATTN_BAD_ARG;
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

// The window of a call, 0 keys where it hides none of as many as the table holds.
struct Window { int window = 0, sinks = 0; };
Window window_of(const cosmos_attn_cache_desc* d, int64_t window, int64_t sinks) {
    const int64_t most = (int64_t)d->width * d->page_size;
    return window && window < most && sinks < most ? Window{(int)window, (int)sinks} : Window{};
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

template <typename P> int launch(void (*kernel)(P), int64_t blocks, size_t lds, const P& p, void* stream, int threads = kThreads) {
    if (blocks <= 0) return COSMOS_ATTN_OK;
    if (blocks > kMostBlocks) return COSMOS_ATTN_UNSUPPORTED;
    if (lds && !allow_lds((const void*)kernel, lds)) return COSMOS_ATTN_LAUNCH_FAILED;
    kernel<<<dim3((unsigned)blocks), dim3(threads), lds, (hipStream_t)stream>>>(p);
    return hipGetLastError() == hipSuccess ? COSMOS_ATTN_OK : COSMOS_ATTN_LAUNCH_FAILED;
}
template <typename F> int with_type(const cosmos_attn_cache_desc* d, F&& f) {
    auto kind = [&](auto* t, auto dim) {
        return d->kind == COSMOS_ATTN_CACHE_SAME ? f(t, dim, Int<SAME16>{}) : d->kind == COSMOS_ATTN_CACHE_E4M3 ? f(t, dim, Int<E4M3>{}) : f(t, dim, Int<INT8>{});
    };
    if (d->dtype == COSMOS_ATTN_BF16) return d->D == 128 ? kind((__bf16*)nullptr, Int<128>{}) : kind((__bf16*)nullptr, Int<64>{});
    return d->D == 128 ? kind((_Float16*)nullptr, Int<128>{}) : kind((_Float16*)nullptr, Int<64>{});
}
#endif
