// Attention over packed sequences of different lengths with grouped heads, forward and backward, for gfx950: kernels and C ABI (cosmos_attn_ragged, cosmos_attn_ragged_bwd).
//
// Sequence i has the rows cu_q[i] .. cu_q[i + 1] - 1 of q and the rows cu_k[i] .. of k and v.  With c the scale, t and j counted from the sequence's start, Lq and Lk its lengths:
//     s_tj = c q_t k_j,   visible: j <= t + Lk - Lq (causal, aligned at the ends) or all,   p = exp(s - lse),   o_t = sum_j p_tj v_j,   lse_t = log sum_j exp(s_tj)
//     dp_tj = do_t v_j,   delta_t = sum_d do_t o_t,   ds = p (dp - delta),   dq_t = c sum_j ds_tj k_j,   dk_j = c sum_t ds_tj q_t,   dv_j = sum_t p_tj do_t
// A row that sees no key: o = 0, lse = -inf, no gradient.  A row that sees one: ds = 0.
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

#include "attn_ragged_gfx950.h"

// ---- forward.  A workgroup: kRows rows of one sequence and key head; a wavefront 32 of them, one a lane and its other half: S^T = K Q^T has the keys in registers, so that the softmax
// needs one exchange between the halves, and P^T, rounded, is the next product's operand where it lies.  Two workgroups a compute unit (head dim 64: four), so that one's products and another's
// exponentials go on beside each other.  16384 causal positions, 16 heads of 128 on 4: 950 to 1000 us, 1.1 to 1.15 PFLOP/s, the matrix unit busy 63 % of the time at 1.8 GHz.  (Not
// all that a fragment from LDS to each product of 32 x 32 x 16 allows: the forward of sequences of one length, attn_fwd_jvp_gfx950.hip, has come to 1.3 that way, with three wavefronts on a SIMD, no max in front
// of the exponentials and the softmax between the products.  Here are two, and 32 maxima and an exchange between the halves in every step.)  Head dim 64: 8192 positions, 16 heads, 297 us, 0.92 PFLOP/s (causal 187,
// 0.73).  Short calls end with their longest tiles: 12 causal prompts of 1 to 2048 positions, 32 heads on 8, 125 us, 0.77 PFLOP/s, 84 % of the units busy.
// WINDOW: 16384 + 5000 + 1777 + 1 positions, 1024 keys and the first 4, 16 heads on 4, 232 us, 0.79 PFLOP/s of what is seen (all of it 1.1): a tile of 32 tokens has 18.5 steps of 64 keys for 16 that each row
// sees, of which one holds the 4 first keys.
template <typename T, int D, bool WINDOW>
__global__ void __launch_bounds__(kThreads, 2) ragged_fwd_kernel(const RaggedParams p) {
#if defined(__HIP_DEVICE_COMPILE__)
    typedef typename VecOf<T>::v8 V8;
    typedef Tile<D> L;
    constexpr int NC = D / 16, NB = D / 32;
    LDS_TILES(L);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5;
    const Block block = block_of(p, blockIdx.x);
    const int head = block.head;
    typedef RowTilesOf<WINDOW> Rows;
    const Found f = find<Rows>(p, block.index);
    if (f.seq < 0) {
        if (p.fill && block.part == 0) clear_rows<D>(p.fill == COSMOS_ATTN_FILL_LSE ? nullptr : p.o, p.o_row, p.o_head, p.cu_q, p.n_seq, p.Tq, p.group, head * p.group, kRows, f, p.lse, p.lse_row, p.lse_head);
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
    auto keys_of = [&](int t) { const int e = t + shift + 1; return (!WINDOW && !p.causal) || e > lk ? lk : e < 0 ? 0 : e; };
    const int end = live ? keys_of(token) : 0;
    const int first = tile * kRows + 32 * wave;
    auto token_at = [&](int r) { return __builtin_amdgcn_readfirstlane((r < rows ? r : rows - 1) / p.group); };
    const int wave_end = first < rows ? keys_of(token_at(first + 31)) : 0, wave_all = keys_of(token_at(first));
    // (WINDOW: the first key that this lane's row looks back on, the last and the first of those of this wavefront's)
    const int from = WINDOW ? Rows{p}.first_key(f.n, row) : 0, wave_from = WINDOW ? __builtin_amdgcn_readfirstlane(Rows{p}.first_key(f.n, first + 31)) : 0,
              wave_first = WINDOW ? __builtin_amdgcn_readfirstlane(Rows{p}.first_key(f.n, first)) : 0;
    // steps of this part; of step u, where its keys begin
    const int steps = Rows{p}.end_step(f.n, tile), sink_steps = Rows{p}.sink_steps(), gap = Rows{p}.gap(f.n, tile);
    auto at_step = [&](int u) { return WINDOW && u >= sink_steps ? u + gap : u; };
    const int t0 = (int)((int64_t)block.part * steps / f.parts), n = (int)((int64_t)(block.part + 1) * steps / f.parts);

    const char* const kp = p.k + rk.start * p.k_row + head * p.k_head;
    const char* const vp = p.v + rk.start * p.v_row + head * p.v_head;
    int k_off[L::LOADS], v_off[L::LOADS];
#pragma unroll
    for (int i = 0; i < L::LOADS; ++i) {
        k_off[i] = L::load_row(lane, wave, i) * (int)p.k_row + L::load_byte(lane, wave, i);
        v_off[i] = L::load_row(lane, wave, i) * (int)p.v_row + L::load_byte(lane, wave, i);
    }
    auto fill = [&](int u, char* kt, char* vt) __attribute__((always_inline)) {
        const int t = at_step(u);
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

    auto step = [&](int u, const char* kt, const char* vt) __attribute__((always_inline)) {
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
// WINDOW: what rounding dS leaves off is a second operand of the last product, whose other one is there already.  dq's error is then 1.03 of its own rounding instead of 1.46 (dS sums to zero over a row, so
// that its errors are larger next to dq than next to dS), for 12 to 16 % of this kernel.  (Its reads are left to the compiler: in the order of the others a pass takes as long.)
template <typename T, int D, bool WINDOW>
__global__ void __launch_bounds__(kThreads, 2) ragged_dq_kernel(const RaggedParams p) {
#if defined(__HIP_DEVICE_COMPILE__)
    typedef typename VecOf<T>::v8 V8;
    typedef Tile<D> L;
    constexpr int NC = D / 16, NB = D / 32;
    LDS_TILES(L);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5;
    const Block block = block_of(p, blockIdx.x);
    const int head = block.head;
    typedef RowTilesOf<WINDOW> Rows;
    const Found f = find<Rows>(p, block.index);
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
    auto keys_of = [&](int t) { const int e = t + shift + 1; return (!WINDOW && !p.causal) || e > lk ? lk : e < 0 ? 0 : e; };
    const int end = live ? keys_of(token) : 0;
    const int first = tile * kRows + 32 * wave;
    auto token_at = [&](int r) { return __builtin_amdgcn_readfirstlane((r < rows ? r : rows - 1) / p.group); };
    const int wave_end = first < rows ? keys_of(token_at(first + 31)) : 0, wave_all = keys_of(token_at(first));
    // (WINDOW: the first key that this lane's row looks back on, the last and the first of those of this wavefront's)
    const int from = WINDOW ? Rows{p}.first_key(f.n, row) : 0, wave_from = WINDOW ? __builtin_amdgcn_readfirstlane(Rows{p}.first_key(f.n, first + 31)) : 0,
              wave_first = WINDOW ? __builtin_amdgcn_readfirstlane(Rows{p}.first_key(f.n, first)) : 0;
    // steps of this part; of step u, where its keys begin
    const int steps = Rows{p}.end_step(f.n, tile), sink_steps = Rows{p}.sink_steps(), gap = Rows{p}.gap(f.n, tile);
    auto at_step = [&](int u) { return WINDOW && u >= sink_steps ? u + gap : u; };
    const int t0 = (int)((int64_t)block.part * steps / f.parts), n = (int)((int64_t)(block.part + 1) * steps / f.parts);

    const char* const kp = p.k + rk.start * p.k_row + head * p.k_head;
    const char* const vp = p.v + rk.start * p.v_row + head * p.v_head;
    int k_off[L::LOADS], v_off[L::LOADS];
#pragma unroll
    for (int i = 0; i < L::LOADS; ++i) {
        k_off[i] = L::load_row(lane, wave, i) * (int)p.k_row + L::load_byte(lane, wave, i);
        v_off[i] = L::load_row(lane, wave, i) * (int)p.v_row + L::load_byte(lane, wave, i);
    }
    auto fill = [&](int u, char* kt, char* vt) __attribute__((always_inline)) {
        const int t = at_step(u);
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
    // A row that sees one key has the weight 1 on it whatever its score, and dS = 0, not what the roundings of dP and delta leave.  Here it has no P; its delta for the second kernel is its
    // dP, the same products of 16 channels in the same order as there, so that their difference is 0.  (In front of the loop: in either kernel's loop a few registers more cost 2 to 9 %.)
    const bool one = end - (WINDOW && from > p.sinks ? from - p.sinks : 0) == 1;
    const unsigned long long ones = __ballot(one);
    if (ones && block.part == 0) {
        // (the last key that it sees; the wavefront's lie behind each other, from the first such row's on)
        const int base = __builtin_amdgcn_readlane(end, __builtin_ctzll(ones)) - 1, at = base + (lane & 31), own = end - 1 - base - 4 * half;
        const char* const va = vp + (int64_t)(at < lk ? at : lk - 1) * p.v_row + 16 * half;
        f32x16 g = f32x16{};
#pragma unroll
        for (int c = 0; c < NC; ++c) g = mfma32(__builtin_bit_cast(V8, *reinterpret_cast<const u32x4*>(va + 32 * c)), gf[c], g);
        float dp = 0.f;
#pragma unroll
        for (int e = 0; e < 16; ++e) dp = 8 * (e >> 2) + (e & 3) == own ? g[e] : dp;
        if (one && own >= 0 && !(own & 4)) p.delta[(int64_t)hq * p.Tq + rq.start + token] = dp;
    }
    const int64_t stat = (int64_t)hq * p.Tq + rq.start + token;
    float lse2 = INFINITY;            // (P = 0 where there is no row, or nothing that it sees)
    if (live) {
        const float x = p.lse[stat];
        lse2 = x == -INFINITY || one ? INFINITY : x * 1.44269504088896341f;
        if (half == 0 && block.part == 0 && !one) p.delta[stat] = delta;
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

    auto step = [&](int u, const char* kt, const char* vt) __attribute__((always_inline)) {
        const int key0 = at_step(u) * kStep;
        if (key0 >= wave_end) return;
        if (WINDOW && key0 >= p.sinks && key0 + kStep <= wave_first) return;
        const bool behind = WINDOW && key0 < wave_from && key0 + kStep > p.sinks;      // (some row of the wavefront does not look back on all of these keys)
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
            V8 df[2], dr[2];
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const float pe = __builtin_amdgcn_exp2f(__builtin_fmaf(s[e], p.scale_log2, -lse2));
                s[e] = pe * (g[e] - delta);
            }
            if (masked)
#pragma unroll
                for (int e = 0; e < 16; ++e) s[e] = 32 * h + 8 * (e >> 2) + (e & 3) < left ? s[e] : 0.f;
            if (behind) {
                const int out = from - key0 - 4 * half, in = p.sinks - key0 - 4 * half;
#pragma unroll
                for (int e = 0; e < 16; ++e) { const int j = 32 * h + 8 * (e >> 2) + (e & 3); s[e] = j >= out || j < in ? s[e] : 0.f; }
            }
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
                if constexpr (WINDOW) {
                    u32x4 x;
                    asm("" : "+v"(w));          // (what the product takes)
#pragma unroll
                    for (int i = 0; i < 4; ++i) x[i] = round2<T>(s[8 * c + 2 * i] - element<T>(w[i], 0), s[8 * c + 2 * i + 1] - element<T>(w[i], 1));
                    dr[c] = __builtin_bit_cast(V8, x);
                }
                df[c] = __builtin_bit_cast(V8, w);
            }
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    const V8 kt8 = read_channels<V8>(kt + (32 * h + 16 * c) * L::ROW, k_tr[b][0], k_tr[b][1]);
                    acc[b] = mfma32(kt8, df[c], acc[b]);
                    if constexpr (WINDOW) acc[b] = mfma32(kt8, dr[c], acc[b]);
                }
            if constexpr (!WINDOW) reads_ahead<4 * NB, 2 * NB, 8>();
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
// WINDOW: 12728 positions, 1024 keys and the first 4, 32 heads on 8, 481 us (least 464); before the first keys' tiles were cut into pieces 1146.
// (64 keys and half of a step's rows to a wavefront, one on a SIMD with all 512 registers, so that every fragment of Q and dO feeds two products: as fast on 8192 positions, 10 to 20 % slower on 512 to
// 4096 and on prompts of mixed lengths, where a tile's start and end then have no other workgroup beside them.)
template <typename T, int D, bool WINDOW>
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
    // (WINDOW: the pieces of the first keys' tiles go first)
    const int pieces = WINDOW ? p.slots * p.sink_tiles * p.Hkv : 0;
    const bool of_piece = WINDOW && (int)blockIdx.x < pieces;
    const Block block = of_piece ? Block{(int)blockIdx.x % p.Hkv, 0, 0} : block_of(p, blockIdx.x - pieces);
    const int head = block.head;
    Found f = {-1, 0, 1, {0, 0}, false};
    Piece piece = {0, 0, 0, {0, 0}};
    if (of_piece) {
        const int slot = blockIdx.x / (p.Hkv * p.sink_tiles);
        f.tile = blockIdx.x / p.Hkv % p.sink_tiles;
        piece = find_piece<KeyTiles<D, WINDOW>, STEP>(p, f.tile, slot);
        if (piece.seq < 0) return;
        f.seq = piece.seq;
        f.n = piece.n;
    } else {
        f = find<KeyTiles<D, WINDOW>>(p, block.index);
    }
    if (f.seq < 0) {
        if (block.part) return;
        clear_rows<D>(p.dk, p.dk_row, p.dk_head, p.cu_k, p.n_seq, p.Tk, 1, head, kRows, f, nullptr);
        clear_rows<D>(p.dv, p.dv_row, p.dv_head, p.cu_k, p.n_seq, p.Tk, 1, head, kRows, f, nullptr);
        return;
    }
    if (block.part >= f.parts || (WINDOW && !of_piece && KeyTiles<D, WINDOW>{p}.pieces(f.n, f.tile))) return;
    const Range rq = rows_of_sequence(p.cu_q, f.seq, f.n.lq), rk = rows_of_sequence(p.cu_k, f.seq, f.n.lk);
    const int lq = rq.length > 0 ? rq.length : 0;
    const int key0 = f.tile * kRows, key = key0 + 32 * wave + (lane & 31);
    const bool live = key < rk.length;
    const KeyTiles<D, WINDOW> tiles{p};
    const int from = tiles.first_row(f.n, key);
    // (WINDOW: one behind the last row that sees this lane's key; the most and the fewest of the wavefront's)
    const int wave_key = key0 + 32 * wave, until = WINDOW ? tiles.end_row(f.n, key) : 0;
    const int wave_until = WINDOW ? __builtin_amdgcn_readfirstlane(tiles.end_row(f.n, wave_key < p.sinks ? 0 : wave_key + 31)) : 0,
              wave_least = WINDOW ? __builtin_amdgcn_readfirstlane(tiles.end_row(f.n, wave_key < p.sinks && p.sinks < wave_key + 32 ? p.sinks : wave_key)) : 0;
    const int wave_first = __builtin_amdgcn_readfirstlane(tiles.first_row(f.n, key0 + 32 * wave)), wave_all = __builtin_amdgcn_readfirstlane(tiles.first_row(f.n, key0 + 32 * wave + 31));
    // steps of this part
    const int begin = tiles.first_step(f.n, f.tile), steps = tiles.end_step(f.n, f.tile) - begin;
    int t0 = begin + (int)((int64_t)block.part * steps / f.parts), n = begin + (int)((int64_t)(block.part + 1) * steps / f.parts);
    if (of_piece) {
        t0 = begin + piece.index * p.piece;
        if (piece.index + 1 < piece.count) n = t0 + p.piece;
    }

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
        if (row0 + STEP <= wave_first || (WINDOW && row0 >= wave_until)) return;
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
            if (WINDOW && row0 + STEP > wave_least) {
                const int left = until - row0 - 32 * h - 4 * half;
#pragma unroll
                for (int e = 0; e < 16; ++e) s[e] = 8 * (e >> 2) + (e & 3) < left ? s[e] : 0.f;
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
    if (of_piece && until <= t0 * STEP) return;          // (no row of the piece sees the key, and none is added up for it)
    if (f.parts > 1 || of_piece) {
        float* const part = (of_piece ? p.pieces + (int64_t)blockIdx.x * (2 * kRows * D) : p.parts + (((int64_t)block.index * p.Hkv + head) * p.most_parts + block.part) * (2 * kRows * D)) +
                            (32 * wave + (lane & 31)) * D;
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
    p.lse_row = 1; p.lse_head = d->Tq;
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
struct Cut { int64_t tiles; int parts, least; size_t bytes; };
// The window of a call, 0 keys where it hides none (sizes say so: a row's position is below Tk).
struct Window { int window = 0, sinks = 0; };
int check_window(const cosmos_attn_ragged_desc* d, int64_t window, int64_t sinks) {
    if (window < 0 || sinks < 0) return COSMOS_ATTN_BAD_ARG;
    // (a few thousand workgroups more than without)
    if (window && ((d->Tq * (d->Hq / d->Hkv) + d->Tk) / kRows + d->n_seq + 1) * d->Hkv > kMostBlocks - 4096) return COSMOS_ATTN_UNSUPPORTED;
    return window && !d->causal ? COSMOS_ATTN_UNSUPPORTED : COSMOS_ATTN_OK;
}
Window window_of(const cosmos_attn_ragged_desc* d, int64_t window, int64_t sinks) {
    return window && window < d->Tk && sinks < d->Tk ? Window{(int)window, (int)sinks} : Window{};
}
// The first keys' tiles of dk and dv: pieces of three quarters of a window's steps, 1024 rows at least, and about as many pieces at most as twice the workgroups that run at once (each tile may have one more:
// 1536, and what they leave is 192 MiB, at most).
struct Pieces { int piece, slots, tiles; size_t bytes; };
Pieces pieces_of(const cosmos_attn_ragged_desc* d, Window w) {
    if (!w.window || !w.sinks || !d->Tq) return {};
    const int step = row_step(d->D);
    const int64_t group = d->Hq / d->Hkv, rows = d->Tq * group, tiles = (w.sinks + kRows - 1) / kRows, most = 4 * kNumCUs / (tiles * d->Hkv) + 1;
    if (tiles * d->Hkv > 2 * kNumCUs) return {};         // (so many fill the chip as they are)
    int64_t piece = 3 * ((int64_t)w.window + kRows) * group / (4 * step);
    piece = piece > 1024 / step ? piece : 1024 / step;
    piece = piece > rows / (step * most) ? piece : rows / (step * most) + 1;
    if (piece > rows / (2 * step)) return {};            // (no sequence has two)
    const int64_t slots = rows / (piece * step) + 1;
    return {(int)piece, (int)slots, (int)tiles, (size_t)(slots * tiles * d->Hkv) * 2 * kRows * d->D * sizeof(float)};
}
Cut cut_of(const cosmos_attn_ragged_desc* d, int which, Window w) {
    const int step = row_step(d->D);
    const int64_t group = d->Hq / d->Hkv, rows = d->Tq * group, tiles = which == 2 ? most_tiles(d->Tk, d->n_seq) : most_tiles(rows, d->n_seq);
    int64_t longest = which == 2 ? (rows + step - 1) / step : (d->Tk + kStep - 1) / kStep;
    if (w.window) {
        int64_t seen = which == 2 ? ((int64_t)w.window + kRows) * group / step + 2 : ((int64_t)w.window + kRows / group + 1) / kStep + 2 + (w.sinks + kStep - 1) / kStep;
        if (which == 2 && w.sinks) {                  // (the first keys' tiles that are not cut into pieces)
            const Pieces cut = pieces_of(d, w);
            seen = !cut.piece ? longest : seen > 2 * cut.piece + 1 ? seen : 2 * cut.piece + 1;
        }
        longest = seen < longest ? seen : longest;
    }
    const int least = which == 2 ? least_rows(d->D) / step : least_steps(d->D), parts = most_parts(tiles * d->Hkv, longest, least, w.window != 0);
    return {tiles, parts, least, parts > 1 ? (size_t)tiles * d->Hkv * parts * kRows * (which == 0 ? d->D + 2 : which * d->D) * sizeof(float) : 0};
}
size_t up(size_t n) { return (n + 255) / 256 * 256; }

size_t forward_bytes(const cosmos_attn_ragged_desc* desc, int64_t window, int64_t sinks) {
    return check(desc, false) == COSMOS_ATTN_OK && check_window(desc, window, sinks) == COSMOS_ATTN_OK ? cut_of(desc, 0, window_of(desc, window, sinks)).bytes : 0;
}
int forward(const cosmos_attn_ragged_desc* desc, int64_t window, int64_t sinks, void* workspace, size_t workspace_bytes, void* stream) {
    int st = check(desc, false);
    if (st == COSMOS_ATTN_OK) st = check_window(desc, window, sinks);
    if (st != COSMOS_ATTN_OK) return st;
    if (!desc->Tq) return COSMOS_ATTN_OK;
    const Window w = window_of(desc, window, sinks);
    const Cut cut = cut_of(desc, 0, w);
    if (workspace_bytes < cut.bytes || (cut.bytes && !workspace)) return COSMOS_ATTN_WORKSPACE_TOO_SMALL;
    if (cut.bytes && !aligned16(workspace)) return COSMOS_ATTN_BAD_STRIDE;
    if (!device_is_whole_mi355x()) return COSMOS_ATTN_WRONG_DEVICE;
    RaggedParams p = params_of(desc);
    p.tiles = (int)cut.tiles; p.most_parts = cut.parts; p.least = cut.least;
    p.window = w.window; p.sinks = w.sinks;
    p.parts = (float*)workspace;
    return with_type(desc->dtype, desc->D, [&](auto* t, auto d) {
        constexpr int D = decltype(d)::value;
        typedef std::remove_pointer_t<decltype(t)> T;
        auto run = [&](auto windowed) {
            constexpr bool WINDOW = decltype(windowed)::value;
            const int done = launch(ragged_fwd_kernel<T, D, WINDOW>, cut.tiles * p.Hkv * cut.parts, p, stream);
            return done != COSMOS_ATTN_OK || cut.parts == 1 ? done : launch(ragged_join_kernel<T, D, 0, WINDOW>, cut.tiles * p.Hkv * kJoinBlocks<D>, p, stream, kJoinThreads);
        };
        return w.window ? run(Int<1>{}) : run(Int<0>{});
    });
}

size_t backward_bytes(const cosmos_attn_ragged_desc* desc, int64_t window, int64_t sinks) {
    if (check(desc, true) != COSMOS_ATTN_OK || check_window(desc, window, sinks) != COSMOS_ATTN_OK) return 0;
    const Window w = window_of(desc, window, sinks);
    const size_t a = cut_of(desc, 1, w).bytes, b = cut_of(desc, 2, w).bytes;
    return up((size_t)desc->Tq * desc->Hq * sizeof(float)) + up(a > b ? a : b) + pieces_of(desc, w).bytes;
}
int backward(const cosmos_attn_ragged_desc* desc, int64_t window, int64_t sinks, void* workspace, size_t workspace_bytes, void* stream) {
    int st = check(desc, true);
    if (st == COSMOS_ATTN_OK) st = check_window(desc, window, sinks);
    if (st != COSMOS_ATTN_OK) return st;
    const size_t wanted = backward_bytes(desc, window, sinks);
    if (workspace_bytes < wanted || (wanted && !workspace)) return COSMOS_ATTN_WORKSPACE_TOO_SMALL;
    if (wanted && !aligned16(workspace)) return COSMOS_ATTN_BAD_STRIDE;
    if (!device_is_whole_mi355x()) return COSMOS_ATTN_WRONG_DEVICE;
    const Window w = window_of(desc, window, sinks);
    RaggedParams p = params_of(desc);
    p.window = w.window; p.sinks = w.sinks;
    p.delta = (float*)workspace;
    p.parts = (float*)((char*)workspace + up((size_t)desc->Tq * desc->Hq * sizeof(float)));      // (of dq, then of dk and dv)
    const Pieces pieces = pieces_of(desc, w);
    p.piece = pieces.piece; p.slots = pieces.slots; p.sink_tiles = pieces.tiles;
    p.pieces = (float*)((char*)workspace + wanted - pieces.bytes);
    return with_type(desc->dtype, desc->D, [&](auto* t, auto d) {
        constexpr int D = decltype(d)::value;
        typedef std::remove_pointer_t<decltype(t)> T;
        int done = COSMOS_ATTN_OK;
        auto one = [&](const Cut& cut, auto kernel, auto join, int64_t before = 0) {
            p.tiles = (int)cut.tiles; p.most_parts = cut.parts; p.least = cut.least;
            if (done == COSMOS_ATTN_OK) done = launch(kernel, before + cut.tiles * p.Hkv * cut.parts, p, stream);
            if (done == COSMOS_ATTN_OK && cut.parts > 1) done = launch(join, cut.tiles * p.Hkv * kJoinBlocks<D>, p, stream, kJoinThreads);
        };
        auto run = [&](auto windowed) {
            constexpr bool WINDOW = decltype(windowed)::value;
            if (desc->Tq) one(cut_of(desc, 1, w), ragged_dq_kernel<T, D, WINDOW>, ragged_join_kernel<T, D, 1, WINDOW>);
            if (!desc->Tk) return done;
            const int64_t blocks = (int64_t)p.slots * p.sink_tiles * p.Hkv;
            one(cut_of(desc, 2, w), ragged_dkdv_kernel<T, D, WINDOW>, ragged_join_kernel<T, D, 2, WINDOW>, blocks);
            if constexpr (WINDOW) {
                if (done == COSMOS_ATTN_OK && blocks) done = launch(ragged_pieces_kernel<T, D>, blocks * kJoinBlocks<D>, p, stream, kJoinThreads);
            }
            return done;
        };
        return w.window ? run(Int<1>{}) : run(Int<0>{});
    });
}

}  // namespace

extern "C" {

size_t cosmos_attn_ragged_workspace_bytes(const cosmos_attn_ragged_desc* desc) { return forward_bytes(desc, 0, 0); }
int cosmos_attn_ragged(const cosmos_attn_ragged_desc* desc, void* workspace, size_t workspace_bytes, void* stream) { return forward(desc, 0, 0, workspace, workspace_bytes, stream); }
size_t cosmos_attn_ragged_bwd_workspace_bytes(const cosmos_attn_ragged_desc* desc) { return backward_bytes(desc, 0, 0); }
int cosmos_attn_ragged_bwd(const cosmos_attn_ragged_desc* desc, void* workspace, size_t workspace_bytes, void* stream) { return backward(desc, 0, 0, workspace, workspace_bytes, stream); }

size_t cosmos_attn_ragged_window_workspace_bytes(const cosmos_attn_ragged_desc* desc, int64_t window, int64_t sinks) { return forward_bytes(desc, window, sinks); }
int cosmos_attn_ragged_window(const cosmos_attn_ragged_desc* desc, int64_t window, int64_t sinks, void* workspace, size_t workspace_bytes, void* stream) {
    return forward(desc, window, sinks, workspace, workspace_bytes, stream);
}
size_t cosmos_attn_ragged_window_bwd_workspace_bytes(const cosmos_attn_ragged_desc* desc, int64_t window, int64_t sinks) { return backward_bytes(desc, window, sinks); }
int cosmos_attn_ragged_window_bwd(const cosmos_attn_ragged_desc* desc, int64_t window, int64_t sinks, void* workspace, size_t workspace_bytes, void* stream) {
    return backward(desc, window, sinks, workspace, workspace_bytes, stream);
}

}  // extern "C"
