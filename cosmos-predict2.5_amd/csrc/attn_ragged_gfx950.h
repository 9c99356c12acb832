// Pieces shared by the kernels whose rows are packed sequences' (their keys packed too, or in pages): tiles in LDS, which sequence and tile a workgroup has, rows of no sequence, the parts of tiles
// that were cut.  Included inside each translation unit's anonymous namespace, behind attn_common_gfx950.h.
#ifndef COSMOS_ATTN_RAGGED_GFX950_H
#define COSMOS_ATTN_RAGGED_GFX950_H

constexpr int kThreads = 256;      // four wavefronts of 32 rows (or keys) each
constexpr int kRows = 128;         // of a workgroup
constexpr int kStep = 64;          // keys (or rows) that are in LDS at a time, twice

struct RaggedParams {
    const char *q, *k, *v, *o_in, *dout;
    char *o, *dq, *dk, *dv;
    float* lse;                    // [Hq, Tq] (keys in pages: [Tq, Hq]); written by the forward (may be null), read by the backward
    char* rest;                    // [Tq, Hq, D]: what rounding o left off, 16 bits again (may be null)
    float* delta;                  // [Hq, Tq]: of the backward's first kernel for its second
    const int *cu_q, *cu_k;
    // bytes between rows and between heads
    int64_t q_row, q_head, k_row, k_head, v_row, v_head, o_row, o_head, do_row, do_head, dq_row, dq_head, dk_row, dk_head, dv_row, dv_head;
    int n_seq, Tq, Tk, Hkv, group, causal, fill;
    int tiles, most_parts, least;  // tiles that there may be, parts that one may be cut into, steps of a part
    int window, sinks;             // keys that a row looks back on, its own among them; first keys that every row sees
    const int* lens;               // keys in pages: a sequence's number of them, which `most_keys` is the most of
    int most_keys;
    int short_rows;                // sequences of so many rows and fewer are not cut into tiles (others have them)
    int short_parts, short_least;  // parts that one of these may be cut into, steps of a part
    int64_t lse_row, lse_head;     // elements
    int piece, slots, sink_tiles;  // the first keys' tiles, dk and dv: steps of a piece, pieces that there may be, tiles of a sequence
    float* pieces;                 // of slot s, tile j and key head h, at (s sink_tiles + j) Hkv + h
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
// WINDOW: the row of position p (of the keys) sees key j if j <= p and (j > p - window or j < sinks).  A tile of rows passes over the steps between the first keys and those that its first row
// looks back on: its step u is step u, or from the last one of the first keys on u + gap.  A tile of keys ends with the last row that looks back on one of them, or that of all rows where it
// has one of the first keys.
// PAGED: how many keys there are says `lens`.
struct Lengths { int lq, lk; };      // lq < 0 or lk < 0: bad offsets (or a bad length)
template <bool KEYS, int ROWS, int STEP, bool WINDOW = false, bool PAGED = false> struct Tiles {
    const RaggedParams& p;
    __device__ __forceinline__ int keys_of(int i) const {
        if constexpr (PAGED) { const int n = p.lens[i]; return n >= 0 && n <= p.most_keys ? n : -1; }
        else return range_of(p.cu_k, i, p.Tk).length;
    }
    __device__ __forceinline__ Lengths lengths(int i) const { return {range_of(p.cu_q, i, p.Tq).length, keys_of(i)}; }
    __device__ __forceinline__ int count(Lengths n) const {
        const int64_t rows = KEYS ? n.lk : (int64_t)n.lq * p.group;
        return rows > (PAGED ? p.short_rows : 0) ? (int)((rows + ROWS - 1) / ROWS) : 0;
    }
    __device__ __forceinline__ int most_parts() const { return p.most_parts; }
    __device__ __forceinline__ int least() const { return p.least; }
    static __device__ __forceinline__ int at(int rank, int tiles) { return KEYS ? rank : tiles - 1 - rank; }
    // first row that sees key j, in rows; (rounded up to steps where none does)
    __device__ __forceinline__ int first_row(Lengths n, int j) const {
        const int lq = n.lq > 0 ? n.lq : 0, t = j - (n.lk - lq);
        return (!WINDOW && !p.causal) || t <= 0 ? 0 : t >= lq ? (lq * p.group + STEP - 1) / STEP * STEP : t * p.group;
    }
    // one behind the last row that sees key j, in rows
    __device__ __forceinline__ int end_row(Lengths n, int j) const {
        const int lq = n.lq > 0 ? n.lq : 0;
        if (!WINDOW || j < p.sinks) return lq * p.group;
        const int64_t t = (int64_t)j + p.window - (n.lk - lq);
        return t <= 0 ? 0 : t >= lq ? lq * p.group : (int)t * p.group;
    }
    // keys that row r's token sees
    __device__ __forceinline__ int keys(Lengths n, int r) const {
        const int lk = n.lk > 0 ? n.lk : 0, e = r / p.group + lk - n.lq + 1;
        return (!WINDOW && !p.causal) || e > lk ? lk : e < 0 ? 0 : e;
    }
    // first key that row r's token looks back on
    __device__ __forceinline__ int first_key(Lengths n, int r) const {
        const int lk = n.lk > 0 ? n.lk : 0, from = r / p.group + lk - n.lq + 1 - p.window;
        return WINDOW && from > 0 ? from : 0;
    }
    __device__ __forceinline__ int sink_steps() const { return WINDOW ? (p.sinks + STEP - 1) / STEP : 0; }
    __device__ __forceinline__ int gap(Lengths n, int tile) const {
        if (!WINDOW || KEYS) return 0;
        const int past = first_key(n, tile * ROWS) / STEP - sink_steps();
        return past > 0 ? past : 0;
    }
    __device__ __forceinline__ int first_step(Lengths n, int tile) const { return KEYS ? first_row(n, tile * ROWS) / STEP : 0; }
    __device__ __forceinline__ int end_step(Lengths n, int tile) const {
        if (KEYS && WINDOW) {
            const int last = tile * ROWS + ROWS - 1, first = first_step(n, tile), end = (end_row(n, tile * ROWS < p.sinks ? 0 : last < n.lk ? last : n.lk - 1) + STEP - 1) / STEP;
            return end > first ? end : first;
        }
        if (KEYS) return n.lq > 0 ? (n.lq * p.group + STEP - 1) / STEP : 0;
        const int rows = n.lq * p.group, last = tile * ROWS + ROWS - 1;
        return (keys(n, last < rows ? last : rows - 1) + STEP - 1) / STEP - gap(n, tile);
    }
    __device__ __forceinline__ int steps(Lengths n, int tile) const { return end_step(n, tile) - first_step(n, tile); }
    // pieces that a tile with some of the first keys is cut into, 0 or 2 and more
    __device__ __forceinline__ int pieces(Lengths n, int tile) const {
        if (!WINDOW || !KEYS || tile >= p.sink_tiles || n.lq <= 0) return 0;
        const int count = (n.lq * p.group / STEP - first_step(n, tile)) / p.piece;
        return count > 1 ? count : 0;
    }
    // of all of its tiles: all of them times the mean of the longest and the shortest; of a window's, which are of one length but for the first rows' and the first keys', the middle one
    __device__ __forceinline__ int64_t all_steps(Lengths n, int tiles) const {
        if (WINDOW) return (int64_t)tiles * steps(n, tiles / 2) + (KEYS && tiles > 1 ? steps(n, 0) : 0);
        return (int64_t)tiles * (steps(n, at(0, tiles)) + steps(n, at(tiles - 1, tiles))) / 2;
    }
    static constexpr bool OF_KEYS = KEYS, IN_PAGES = PAGED;
};

// Parts are written and read in fp32 and joined by a launch of its own, so they have `least` steps at least.  dk and dv, and where shares are large: parts of three fifths of a workgroup's
// share of all steps, as 512 causal tiles are dealt out evenly only if the long ones are in pieces that short ones fit beside (gradients of 16384 positions, 16 heads on 4, us, parts of a
// share / of 3/5 / of 2/5: 4558 / 3973 / 3890).  Else five quarters, which are all on the chip at once: a few more than fit take a second round (512 queries, 8 heads each, on 8192 keys: 704
// parts 72, 520 75, 455 63).  On other sizes, us, this rule / five quarters throughout, forward and gradients: 3000 + 1700 + 1040 positions, 16 heads on 4, 109 / 95 and 311 / 285; 4096 108 / 105 and
// 323 / 309; 1024 queries on 8192 keys, 16 heads on 2, 94 / 91 and 306 / 297; 512 on 32768, 8 heads on 1, 84 / 89 and 302 / 298; 8192, 8 heads on 2, 178 / 177 and 548 / 548.
// Keys in pages: five quarters throughout, and nothing of up to two parts' least steps is cut (512 tokens on 9001 positions, 32 heads on 8, 92 us, by three fifths 106).
constexpr int kAtOnce = 2 * kNumCUs;      // workgroups
constexpr int least_steps(int D) { return D == 128 ? 12 : 24; }
constexpr int least_rows(int D) { return D == 128 ? 512 : 2048; }       // (of dk and dv, in rows)
template <bool WINDOW, bool PAGED = false> using RowTilesOf = Tiles<false, kRows, kStep, WINDOW, PAGED>;
// of dk and dv
constexpr int row_step(int D) { return D == 128 ? 32 : 64; }
template <int D, bool WINDOW = false> using KeyTiles = Tiles<true, kRows, row_step(D), WINDOW>;
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
    // (a sequence's: as many of them as are added up in 32 bits are no more than those hold)
    auto share_of = [&](Lengths n, int tiles, int most) {
        const int64_t sum = tiles ? T.all_steps(n, tiles) : 0;
        return (int)(sum < most ? sum : most);
    };
    int before = 0;
    int64_t all = 0;                 // steps
    auto lengths = [&](int i) { return i < p.n_seq ? T.lengths(i) : Lengths{-1, -1}; };
    auto is_odd = [&](int i, Lengths n) { return i < p.n_seq && (n.lq < 0 || (!Kind::IN_PAGES && n.lk < 0)); };
    // 64 sequences from `base` on; is that all there is to know?
    auto look = [&](int base, Lengths n) __attribute__((always_inline)) {
        const int tiles = T.count(n), sum = sums_up_to(tiles);
        const unsigned long long past = __ballot(before + sum > index);
        if (past && f.seq < 0) {
            const int at = __builtin_ctzll(past), of = __builtin_amdgcn_readlane(tiles, at);
            f.seq = base + at;
            f.n = {__builtin_amdgcn_readlane(n.lq, at), __builtin_amdgcn_readlane(n.lk, at)};
            f.tile = T.at(index - (before + __builtin_amdgcn_readlane(sum, at) - of), of);
            if (T.most_parts() <= 1) return true;
        }
        before += __builtin_amdgcn_readlane(sum, 63);
        if (T.most_parts() > 1) all += sum_of(share_of(n, tiles, (1 << 25) - 1));
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
            if (T.most_parts() > 1) all += sum_of(share_of(n, tiles, (1 << 25) - 1));
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
                if (T.most_parts() <= 1) break;
            }
            before = past;
        }
        if (!f.odd) {
            if (lane == 0) shares[wave] = all;
            __syncthreads();
            if (f.seq >= 0) {
                f = {__builtin_amdgcn_readfirstlane(found.seq), __builtin_amdgcn_readfirstlane(found.tile), 1, {__builtin_amdgcn_readfirstlane(found.n.lq), __builtin_amdgcn_readfirstlane(found.n.lk)}, false};
                if (T.most_parts() <= 1) return f;
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
        for (int base = 0; base < p.n_seq; base += 64) {
            Lengths n = {apart(p.cu_q, base, p.n_seq, p.Tq, end_q).length, -1};
            if constexpr (!Kind::IN_PAGES) n.lk = apart(p.cu_k, base, p.n_seq, p.Tk, end_k).length;
            else if (base + lane < p.n_seq) n.lk = T.keys_of(base + lane);
            if (look(base, n)) return f;
        }
    }
    if (f.seq < 0) { f.tile = index - before; return f; }
    const int64_t share = (all * p.Hkv + kAtOnce - 1) / kAtOnce;
    const int steps = T.steps(f.n, f.tile);
    const int64_t wish = !Kind::IN_PAGES && (KEYS || share >= 2 * T.least()) ? 3 * share / 5 : 5 * share / 4;
    const int per = wish > T.least() ? (int)wish : T.least(), parts = Kind::IN_PAGES && steps <= 2 * T.least() ? 1 : (steps + per - 1) / per;
    f.parts = __builtin_amdgcn_readfirstlane(parts < 1 ? 1 : parts < T.most_parts() ? parts : T.most_parts());
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

// ---- WINDOW, dk and dv: the first keys are seen by all rows, so that their tiles have all of a sequence's steps where the others have a window's.  From two pieces of `piece` steps on such a tile is
// cut into these (the last one has what is left over), in workgroups of their own, which go first.  How many there are follows from the rows, and which slot a piece has from its place
// among all of them: pieces are `piece` STEP rows and more, disjoint, so that no two begin in one slot of as many rows.
template <int STEP> __device__ __forceinline__ int slot_of(const RaggedParams& p, int row0, int step) { return (int)(((int64_t)row0 + (int64_t)step * STEP) / ((int64_t)p.piece * STEP)); }
struct Piece { int seq, index, count; Lengths n; };      // seq < 0: no piece begins there
template <typename Kind, int STEP> __device__ __forceinline__ Piece find_piece(const RaggedParams& p, int tile, int slot) {
    const Kind T{p};
    const int lane = threadIdx.x & 63;
    const int64_t size = (int64_t)p.piece * STEP;
    int end_q = 0, end_k = 0;
    for (int base = 0; base < p.n_seq; base += 64) {
        const Own q = apart(p.cu_q, base, p.n_seq, p.Tq, end_q), k = apart(p.cu_k, base, p.n_seq, p.Tk, end_k);
        const Lengths n = {q.length, k.length};
        const int count = tile < T.count(n) ? T.pieces(n, tile) : 0;
        const int64_t first = (int64_t)q.start * p.group + (int64_t)T.first_step(n, tile) * STEP, past = slot * size - first;
        const int64_t index = past <= 0 ? 0 : (past + size - 1) / size;
        const bool mine = index < count && first + index * size < (slot + 1) * size;
        const unsigned long long found = __ballot(mine);
        if (found) {
            const int at = __builtin_ctzll(found);
            return {base + at, __builtin_amdgcn_readlane((int)index, at), __builtin_amdgcn_readlane(count, at), {__builtin_amdgcn_readlane(n.lq, at), __builtin_amdgcn_readlane(n.lk, at)}};
        }
    }
    return {-1, 0, 0, {0, 0}};
}

// ---- rows of no sequence: zeros, lse = -inf.  They are counted through, whatever lies between them, and a workgroup behind the last tile has `rows` of them.
template <int D> __device__ __forceinline__ void clear_rows(char* out, int64_t row, int64_t head, const int* cu, int n, int total, int heads, int first_head, int rows, Found f, float* lse, int64_t lse_row = 0, int64_t lse_head = 0) {
    constexpr int CHUNKS = D / 8;
    int64_t first = (int64_t)f.tile * rows;      // the workgroup's first one, counted from the next row to be cleared
    auto clear = [&](int from, int to) {         // the tensor's rows from .. to - 1
        const int64_t count = (int64_t)(to - from) * heads, lo = first < 0 ? 0 : first, hi = first + rows < count ? first + rows : count;
        for (int i = threadIdx.x; i < (hi - lo) * CHUNKS; i += kThreads) {
            const int64_t r = lo + i / CHUNKS;
            const int t = from + (int)(r / heads), h = first_head + (int)(r % heads);
            if (out) *reinterpret_cast<u32x4*>(out + t * row + h * head + 16 * (i % CHUNKS)) = u32x4{0, 0, 0, 0};
            if (lse && i % CHUNKS == 0) lse[h * lse_head + t * lse_row] = -INFINITY;
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

// ---- the tiles that were cut: their parts added up, D / 4 lanes to a row.  WHICH: 0 o and lse, 1 dq, 2 dk and dv.  Memory and a launch: 512 + 77
// + 1 queries of 16 heads, the long ones in some four parts each, 10 us; dk and dv of four causal documents, 7678 keys of 8 heads, 30 us.  (80 scalar registers: with 83 a unit holds one workgroup
// of 16 wavefronts instead of two, 37 us.)
constexpr int kJoinThreads = 1024;
template <int D> constexpr int kJoinBlocks = kRows * (D / 4) / kJoinThreads;      // of a tile
template <typename T, int D, int WHICH, bool WINDOW = false>
__global__ void __launch_bounds__(kJoinThreads) __attribute__((amdgpu_num_sgpr(80))) ragged_join_kernel(const RaggedParams p) {
#if defined(__HIP_DEVICE_COMPILE__)
    constexpr bool KEYS = WHICH == 2;
    constexpr int LANES = D / 4, AT_ONCE = kJoinThreads / LANES;
    const int head = blockIdx.x % p.Hkv, index = blockIdx.x / p.Hkv % p.tiles;
    const Found f = find<std::conditional_t<KEYS, KeyTiles<D, WINDOW>, RowTilesOf<WINDOW>>, kJoinThreads>(p, index);
    if (f.seq < 0 || f.parts <= 1) return;
    if constexpr (KEYS && WINDOW) {
        if (KeyTiles<D, WINDOW>{p}.pieces(f.n, f.tile)) return;
    }
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
        if (p.lse && c == 0) p.lse[h * p.lse_head + (r.start + token) * p.lse_row] = l > 0.f ? (m + __builtin_amdgcn_logf(l)) * 0.693147180559945309f : l == 0.f ? -INFINITY : l;
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

// WINDOW: the pieces of a tile with some of the first keys, at the workgroup whose slot is the first one's.  A key's sums are in the pieces with a row that sees it: a first key's in all.
template <typename T, int D>
__global__ void __launch_bounds__(kJoinThreads) ragged_pieces_kernel(const RaggedParams p) {
#if defined(__HIP_DEVICE_COMPILE__)
    constexpr int LANES = D / 4, AT_ONCE = kJoinThreads / LANES, STEP = row_step(D);
    typedef KeyTiles<D, true> Tiles;
    const int head = blockIdx.x % p.Hkv, rest = blockIdx.x / p.Hkv, tile = rest % p.sink_tiles, slot = rest / p.sink_tiles % p.slots;
    const Piece f = find_piece<Tiles, STEP>(p, tile, slot);
    if (f.seq < 0 || f.index) return;
    const Range q = rows_of_sequence(p.cu_q, f.seq, f.n.lq), k = rows_of_sequence(p.cu_k, f.seq, f.n.lk);
    const int c = 4 * (threadIdx.x % LANES), i = rest / p.sink_tiles / p.slots * AT_ONCE + threadIdx.x / LANES, key = tile * kRows + i;
    if (key >= k.length) return;
    const Tiles tiles{p};
    const int begin = tiles.first_step(f.n, tile), until = tiles.end_row(f.n, key);
    f32x4 dk = {0.f, 0.f, 0.f, 0.f}, dv = dk;
#pragma unroll 4
    for (int s = 0; s < f.count; ++s) {
        const int step = begin + s * p.piece;
        if (step * STEP >= until) break;
        const float* const at = p.pieces + (((int64_t)slot_of<STEP>(p, q.start * p.group, step) * p.sink_tiles + tile) * p.Hkv + head) * (2 * kRows * D) + i * D + c;
        dk += *reinterpret_cast<const f32x4*>(at);
        dv += *reinterpret_cast<const f32x4*>(at + kRows * D);
    }
    dk *= p.scale;
    *reinterpret_cast<u32x2*>(p.dk + (k.start + key) * p.dk_row + head * p.dk_head + 2 * c) = u32x2{round2<T>(dk[0], dk[1]), round2<T>(dk[2], dk[3])};
    *reinterpret_cast<u32x2*>(p.dv + (k.start + key) * p.dv_row + head * p.dv_head + 2 * c) = u32x2{round2<T>(dv[0], dv[1]), round2<T>(dv[2], dv[3])};
#endif
}

// at most so many tiles are there: each sequence rounds up once, and so do the rows of none
inline int64_t most_tiles(int64_t rows, int n_seq) { return rows / kRows + n_seq + 1; }
// Parts that a tile may be cut into.  A call with fewer tiles than some rounds of workgroups ends with its longest tiles on a few compute units; one with more is dealt out evenly as it is.
// (The workgroups of parts that a tile does not have end at once.)
constexpr int64_t kFullGrid = 6 * kNumCUs;
// (WINDOW: tiles are of one length, so that there is nothing to deal out, and those that fill the chip once are left as they are: forward and gradients of 12728 positions, window 1024, 32 heads on 8,
// 1110 us, cut by the rule of the others 1210, both before dS had a second operand in dq.)
inline int most_parts(int64_t tiles, int64_t longest, int least, bool window = false, int64_t grid = kFullGrid) {
    int64_t parts = window ? kAtOnce / tiles : (grid + tiles - 1) / tiles;
    parts = parts < 16 ? parts : 16;
    const int64_t of_length = longest / least;
    parts = parts < of_length ? parts : of_length;
    return parts > 1 ? (int)parts : 1;
}
#endif
