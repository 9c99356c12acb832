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
};

// what was written to LDS is there and all reads have returned; then the workgroup meets, with loads to registers under way
__device__ __forceinline__ void meet_in_lds() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0xC07F);           // lgkmcnt 0 alone
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// ---- A workgroup: as ragged_fwd_kernel, with K and V out of pages.
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

    // (of constant memory, so that the scalar unit looks up: a vector load's result in scalar registers is waited for at once, with all loads in front of it)
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
    float R = 0.f;                    // fp16 and codes: what weights are relative to, the largest scale of V so far but for a factor of 64

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
            // weights p scale in fp16 would leave its range where values are small
            float most = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const f32x4 by = *reinterpret_cast<const f32x4*>(st + kStep + 8 * i + 4 * half);
#pragma unroll
                for (int j = 0; j < 4; ++j) most = fmaxf(most, by[j]);
            }
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
                    for (int i = 0; i < 2; ++i) by[i] = *reinterpret_cast<const f32x4*>(st + kStep + 32 * h + 16 * c + 8 * i + 4 * half) * over;
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int e = 8 * c + 2 * i;
                    float a = __builtin_amdgcn_exp2f(__builtin_fmaf(s[h][e], p.scale_log2, -m)), b = __builtin_amdgcn_exp2f(__builtin_fmaf(s[h][e + 1], p.scale_log2, -m));
                    l += a;
                    l += b;
                    if constexpr (CODES) {
                        a *= by[i / 2][2 * (i % 2)];
                        b *= by[i / 2][2 * (i % 2) + 1];
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
        // A step's codes are on their way while the two before are computed, and go to LDS during the one before.  (One step ahead: two workgroups of a unit have half as many bytes under way, 46 single
        // tokens of up to 8000 keys beside two pieces in e4m3 ... us instead of ...)
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

// ---- C ABI
// tiles, and the parts that they may be cut into: as packed sequences of as many keys as a sequence may have
struct Cut { int64_t tiles; int parts, least; size_t bytes; };
Cut cut_of(const cosmos_attn_cache_desc* d, Window w) {
    const int64_t group = d->Hq / d->Hkv, tiles = most_tiles(d->rows * group, d->B), most = (int64_t)d->width * d->page_size;
    int64_t longest = (most + kStep - 1) / kStep;
    if (w.window) {
        const int64_t seen = ((int64_t)w.window + kRows / group + 1) / kStep + 2 + ((int64_t)w.sinks + kStep - 1) / kStep;
        longest = seen < longest ? seen : longest;
    }
    const int least = least_steps(d->D), parts = most_parts(tiles * d->Hkv, longest, least);
    return {tiles, parts, least, parts > 1 ? (size_t)tiles * d->Hkv * parts * kRows * (d->D + 2) * sizeof(float) : 0};
}
int check_chunk(const cosmos_attn_cache_desc* d, int64_t window, int64_t sinks) {
    int st = check(d);
    if (st != COSMOS_ATTN_OK) return st;
    if (window < 0 || sinks < 0 || d->rows < 0 || d->Hq < 1 || !(fabsf(d->sm_scale) <= 3.0e38f)) return COSMOS_ATTN_BAD_ARG;
    if (d->Hq % d->Hkv) return COSMOS_ATTN_BAD_SHAPE;
    const int64_t group = d->Hq / d->Hkv;
    // (rows are 32-bit numbers, and so are the threads of a launch)
    if (d->rows > kMost || d->rows * group > kMost / 2 || (d->rows * group / kRows + d->B + 1) * d->Hkv > kMostBlocks) return COSMOS_ATTN_UNSUPPORTED;
    if (!d->rows) return COSMOS_ATTN_OK;
    if (!d->cu || (d->B && !d->lens)) return COSMOS_ATTN_BAD_ARG;
    if (d->q_stride[0] * 2 > kMostRowBytes || d->o_stride[0] * 2 > kMostRowBytes) return COSMOS_ATTN_BAD_STRIDE;
    st = check_rows(d->q, d->q_stride);
    return st != COSMOS_ATTN_OK ? st : check_out(d->o, d->o_stride, d->rows, d->Hq, d->D);
}

}  // namespace

extern "C" {

size_t cosmos_attn_cache_chunk_workspace_bytes(const cosmos_attn_cache_desc* desc, int64_t window, int64_t sinks) {
    return check_chunk(desc, window, sinks) == COSMOS_ATTN_OK && desc->rows ? cut_of(desc, window_of(desc, window, sinks)).bytes : 0;
}

int cosmos_attn_cache_chunk(const cosmos_attn_cache_desc* desc, int64_t window, int64_t sinks, void* workspace, size_t workspace_bytes, void* stream) {
    const int st = check_chunk(desc, window, sinks);
    if (st != COSMOS_ATTN_OK || !desc->rows) return st;
    const Window w = window_of(desc, window, sinks);
    const Cut cut = cut_of(desc, w);
    if (workspace_bytes < cut.bytes || (cut.bytes && !workspace)) return COSMOS_ATTN_WORKSPACE_TOO_SMALL;
    if (cut.bytes && !aligned16(workspace)) return COSMOS_ATTN_BAD_STRIDE;
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
            const int done = launch(cache_chunk_kernel<T, K, D, WINDOW>, cut.tiles * p.Hkv * cut.parts, 0, p, stream);
            if (done != COSMOS_ATTN_OK || cut.parts == 1) return done;
            return launch(ragged_join_kernel<T, D, 0, WINDOW, true>, cut.tiles * p.Hkv * kJoinBlocks<D>, 0, (const RaggedParams&)p, stream, kJoinThreads);
        };
        return w.window ? run(Int<1>{}) : run(Int<0>{});
    });
}

}  // extern "C"
