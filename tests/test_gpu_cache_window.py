"""Attention over the paged cache of several new tokens of each sequence, and with a window, against the definitions in 64 bits (bounds: oracle/ragged_oracle.py)."""
import math

import pytest
import torch

from test_gpu_cache import BF16, E4M3, FP16, INT8, TYPES, empty, filled
from test_gpu_ragged import cu, near, offsets, rows

pytestmark = pytest.mark.gpu


def want(oracle, q, new, K, V, scale, dtype, window, sinks):
    """Packed rows over their sequences' rows of the cache: (o, lse, bounds); lse [rows, Hq]."""
    parts = []
    for a, b, k, v in zip(cu(new)[:-1], cu(new)[1:], K, V):
        O, L, OT, LT = oracle.ragged_fwd(q[a:b], k, v, [0, b - a], [0, len(k)], True, scale, dtype, window=window, sinks=sinks)
        # (weights in fp16 are relative to the largest scale of a row of V as well: their subnormals are worth up to the largest element; weights times scales are rounded once in fp32)
        OT = OT + (2.0 ** -25 * len(k) * v.abs().max() if dtype == FP16 and len(k) else 0.0) + 4 * oracle.F32 * O.abs()
        # Weights are powers of two in fp32, relative to a row's largest but for a factor of 2^6 upwards, so that their sum is 1 at least.  What of a weight, of its product with a scale, or of its
        # 16-bit rounding is below the smallest normal number, 2^-126, counts as 0: three times 2^-126 for each row of V, times its elements (or, scale included, its codes up to 448), at most.
        OT = OT + 3 * 2.0 ** -126 * (v.abs().sum(0).amax() + 448 * len(k) if len(k) else 0)
        parts.append((O, L.t(), OT, LT.t()))
    return [torch.cat(x) for x in zip(*parts)]


def check(pkg, oracle, gpu, lens, new, page, Hq, Hkv, D, dtype, kind, window=None, sinks=0, scale=None, size=1.0, single=False):
    cache, table, K, V = filled(pkg, oracle, gpu, lens, page, Hkv, D, dtype, kind, size=size)
    q = rows(sum(new), Hq, D, dtype, gpu, 5, size)
    o, lse = pkg.cache_attention(q, cache, table, offsets(lens, gpu), sm_scale=scale, need_lse=True, cu=None if single else offsets(cu(new), gpu), window=window, sinks=sinks)
    O, L, o_tol, l_tol = want(oracle, q, new, K, V, D ** -0.5 if scale is None else scale, dtype, window, sinks)
    near(o, O, o_tol, "o")
    near(lse, L, l_tol, "lse")


@pytest.mark.parametrize("dtype, kind", TYPES)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("window, sinks", [(None, 0), (30, 3), (100, 70)])
@pytest.mark.parametrize("lens, new, page", [([1], [1], 16), ([33, 0, 128, 129, 5], [33, 0, 60, 1, 2], 16), ([300, 1, 257], [150, 1, 64], 64), ([700], [100], 1024)])
def test_pieces(pkg, ragged_oracle, gpu, lens, new, page, window, sinks, D, dtype, kind):
    check(pkg, ragged_oracle, gpu, lens, new, page, 4, 2, D, dtype, kind, window, sinks)


@pytest.mark.parametrize("Hq, Hkv", [(1, 1), (3, 3), (7, 1), (16, 1), (33, 1), (70, 2), (40, 8)])
@pytest.mark.parametrize("window, sinks", [(None, 0), (50, 4)])
def test_heads(pkg, ragged_oracle, gpu, Hq, Hkv, window, sinks):
    check(pkg, ragged_oracle, gpu, [140, 20, 300], [9, 20, 35], 16, Hq, Hkv, 128, BF16, INT8, window, sinks)


@pytest.mark.parametrize("kind", [BF16, E4M3, INT8])
@pytest.mark.parametrize("scale, size", [(-0.3, 1.0), (0.0, 1.0), (None, 6.0)])
def test_scales(pkg, ragged_oracle, gpu, scale, size, kind):
    check(pkg, ragged_oracle, gpu, [300, 31], [70, 31], 32, 8, 2, 64, BF16, kind, scale=scale, size=size)


@pytest.mark.parametrize("kind", [BF16, INT8])
@pytest.mark.parametrize("window, sinks", [(None, 0), (3000, 130)])
def test_long_and_short_ones_together(pkg, ragged_oracle, gpu, window, sinks, kind):
    """Single tokens of long sequences, whose tiles are cut and joined, beside pieces and sequences without tokens."""
    lens = [9000, 1, 0, 5, 128, 4000, 700] + [(37 * i) % 190 for i in range(70)]
    new = [1, 1, 0, 5, 100, 130, 0] + [min(n, 1 + i % 2) for i, n in enumerate(lens[7:])]
    check(pkg, ragged_oracle, gpu, lens, new, 16, 4, 2, 64, BF16, kind, window, sinks)


@pytest.mark.parametrize("n", [150, 1100])
def test_many_sequences(pkg, ragged_oracle, gpu, n):
    g = torch.Generator().manual_seed(n)
    lens = torch.randint(0, 40, (n,), generator=g).tolist()
    lens[n // 3] = 900
    check(pkg, ragged_oracle, gpu, lens, [min(m, 1 + i % 5) for i, m in enumerate(lens)], 16, 2, 1, 64, BF16, INT8)


@pytest.mark.parametrize("dtype, kind", TYPES)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("window, sinks", [(1, 0), (1, 1), (100, 0), (128, 4), (129, 130), (300, 17)])
@pytest.mark.parametrize("lens, page", [([1, 130, 0, 128, 700], 16), ([1000, 1, 257], 64), ([1500], 1024)])
def test_one_token_with_a_window(pkg, ragged_oracle, gpu, lens, page, window, sinks, D, dtype, kind):
    check(pkg, ragged_oracle, gpu, [n for n in lens if n], [1] * len([n for n in lens if n]), page, 4, 2, D, dtype, kind, window, sinks, single=True)


@pytest.mark.parametrize("window, sinks", [(2000, 4), (700, 1000), (4000, 0)])
def test_one_token_of_long_and_short_ones_with_a_window(pkg, ragged_oracle, gpu, window, sinks):
    lens = [20000, 1, 5, 128, 9000, 2100] + [1 + (37 * i) % 190 for i in range(140)]
    check(pkg, ragged_oracle, gpu, lens, [1] * len(lens), 16, 4, 2, 64, BF16, INT8, window, sinks, single=True)


@pytest.mark.parametrize("single", [True, False])
@pytest.mark.parametrize("dtype, kind", TYPES)
def test_pages_behind_the_window_are_not_looked_at(pkg, ragged_oracle, gpu, dtype, kind, single):
    """Their entries may be anything, and so may the rows that the token no longer sees in pages that are still there."""
    lens, page, window, sinks = [700, 333], 16, 100, 5
    cache, table, K, V = filled(pkg, ragged_oracle, gpu, lens, page, 2, 64, dtype, kind)
    new = [1, 1] if single else [9, 30]
    q, on = rows(sum(new), 4, 64, dtype, gpu, 5), None if single else offsets(cu(new), gpu)
    good = pkg.cache_attention(q, cache, table, offsets(lens, gpu), need_lse=True, cu=on, window=window, sinks=sinks)
    O, _, tol, _ = want(ragged_oracle, q, new, K, V, 0.125, dtype, window, sinks)
    near(good[0], O, tol, "o")
    gone = table.clone()
    for i, (n, m) in enumerate(zip(lens, new)):
        first = n - m + 1 - window                    # of the first token's window
        gone[i, 1:first // page] = torch.tensor([-1, 1 << 30, cache.pages], dtype=torch.int32, device=gpu).repeat(100)[:first // page - 1]
        for j in list(range(sinks, page)) + list(range(first // page * page, first)):
            for x, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
                x.view(torch.uint8 if kind in (E4M3, INT8) else dtype)[table[i, j // page], :, j % page] = 127 if kind in (E4M3, INT8) else math.nan
                if s is not None:
                    s[table[i, j // page], :, j % page] = math.nan
    got = pkg.cache_attention(q, cache, gone, offsets(lens, gpu), need_lse=True, cu=on, window=window, sinks=sinks)
    assert torch.equal(got[0], good[0]) and torch.equal(got[1], good[1])


@pytest.mark.parametrize("kind", [BF16, E4M3, INT8])
def test_what_cannot_be_looked_up_is_nan(pkg, ragged_oracle, gpu, kind):
    lens, new = [100, 40, 60, 0], [30, 40, 1, 0]
    cache, table, K, V = filled(pkg, ragged_oracle, gpu, lens, 16, 2, 64, BF16, kind)
    q, on = rows(71, 4, 64, BF16, gpu, 5), offsets(cu(new), gpu)
    good = pkg.cache_attention(q, cache, table, offsets(lens, gpu), cu=on)[0]
    bad = table.clone()
    bad[0, 5], bad[1, 1] = cache.pages, -7              # positions 80 .. 95 and 16 .. 31
    o, lse = pkg.cache_attention(q, cache, bad, offsets(lens, gpu), need_lse=True, cu=on)
    assert torch.equal(o[:10], good[:10]) and o[10:30].isnan().all() and lse[10:30].isnan().all()
    assert torch.equal(o[30:46], good[30:46]) and o[46:70].isnan().all() and torch.equal(o[70:], good[70:])
    o, lse = pkg.cache_attention(q, cache, table, offsets([100, -1, 16 * table.shape[1] + 1, 0], gpu), need_lse=True, cu=on)
    assert torch.equal(o[:30], good[:30]) and o[30:].isnan().all() and lse[30:].isnan().all()
    # fewer positions than rows: the first rows have none
    o, lse = pkg.cache_attention(q, cache, table, offsets([7, 40, 60, 0], gpu), need_lse=True, cu=on)
    assert (o[:23] == 0).all() and (lse[:23] == -math.inf).all() and o[23:30].isfinite().all() and lse[23:30].isfinite().all() and torch.equal(o[30:], good[30:])


def test_rows_of_no_sequence_and_offsets_that_go_back(pkg, ragged_oracle, gpu):
    lens = [100, 40]
    cache, table, K, V = filled(pkg, ragged_oracle, gpu, lens, 16, 2, 64, BF16, BF16)
    q = rows(60, 4, 64, BF16, gpu, 5)
    out = torch.full_like(q, 3.0)
    o, lse = pkg.cache_attention(q, cache, table, offsets(lens, gpu), need_lse=True, cu=offsets([5, 25, 45], gpu))
    pkg.cache_attention(q, cache, table, offsets(lens, gpu), cu=offsets([5, 25, 45], gpu), out=out)
    for x, filler in ((o, 0), (out, 3)):
        assert (x[:5] == filler).all() and (x[45:] == filler).all() and torch.equal(x[5:45], o[5:45])
    assert (lse[:5] == -math.inf).all() and (lse[45:] == -math.inf).all()
    assert torch.equal(o[5:45], pkg.cache_attention(q[5:45], cache, table, offsets(lens, gpu), cu=offsets([0, 20, 40], gpu))[0])
    o = pkg.cache_attention(q, cache, table, offsets(lens, gpu), cu=offsets([0, 30, 20], gpu))[0]
    assert torch.equal(o[:30], pkg.cache_attention(q[:30], cache, table[:1], offsets(lens[:1], gpu), cu=offsets([0, 30], gpu))[0]) and (o[30:] == 0).all()
    none = pkg.cache_attention(q[:0], cache, table, offsets(lens, gpu), need_lse=True, cu=offsets([0, 0, 0], gpu))
    assert none[0].shape == (0, 4, 64) and none[1].shape == (0, 4)
    o = pkg.cache_attention(q, cache, table[:0], offsets([], gpu), cu=offsets([0], gpu))[0]
    assert (o == 0).all()


@pytest.mark.parametrize("kind", [BF16, INT8])
def test_layouts(pkg, ragged_oracle, gpu, kind):
    """Keys and values in one pool, rows of all heads side by side, queries and outputs that are parts of larger tensors, a table that is part of a wider one."""
    lens, new, page, heads, D = [90, 200], [50, 7], 32, 2, 64
    cache, table, K, V = filled(pkg, ragged_oracle, gpu, lens, page, heads, D, BF16, kind)
    q, on = rows(57, 8, D, BF16, gpu, 5), offsets(cu(new), gpu)
    want_ = pkg.cache_attention(q, cache, table, offsets(lens, gpu), need_lse=True, cu=on, window=60, sinks=2)
    pool = torch.empty((cache.pages, 2, page, heads, D), dtype=kind, device=gpu)
    scales = torch.empty((2, heads, cache.pages, page), dtype=torch.float32, device=gpu)
    k, v = pool[:, 0].transpose(1, 2), pool[:, 1].transpose(1, 2)
    k.copy_(cache.k), v.copy_(cache.v)
    ks, vs = (None, None) if kind == BF16 else (scales[0].transpose(0, 1), scales[1].transpose(0, 1))
    if ks is not None:
        ks.copy_(cache.k_scale), vs.copy_(cache.v_scale)
    other = pkg.KVCache(k, v, ks, vs)
    wide = torch.full((57, 12, D), 7.0, dtype=BF16, device=gpu)
    wide[:, 2:10] = q
    out = torch.full((57, 20, D), 5.0, dtype=BF16, device=gpu)
    wide_table = torch.cat([table, torch.full_like(table, -1)], 1)[:, :table.shape[1]]
    got = pkg.cache_attention(wide[:, 2:10], other, wide_table, offsets(lens, gpu), need_lse=True, out=out[:, 4:12], cu=on, window=60, sinks=2)
    assert torch.equal(out[:, 4:12], want_[0]) and torch.equal(got[1], want_[1]) and (out[:, :4] == 5).all() and (out[:, 12:] == 5).all()


def test_pages_behind_32_bits(pkg, ragged_oracle, gpu):
    page, heads, D = 16, 1, 64
    step = 1 << 21                                   # elements between pages
    pages = (1 << 32) // (2 * step) + 8
    pool = torch.empty(pages * step, dtype=BF16, device=gpu)
    view = lambda at: pool.as_strided((pages, heads, page, D), (step, page * D, D, 1), at)
    cache = pkg.KVCache(view(0), view(page * D))
    lens, new = [40, 70], [20, 70]
    table = torch.tensor([[pages - 1, 2, pages - 3, -1, -1], [0, pages - 2, 1, pages - 5, pages - 6]], dtype=torch.int32, device=gpu)
    k, v = rows(110, heads, D, BF16, gpu, 0), rows(110, heads, D, BF16, gpu, 1)
    pkg.cache_write(cache, k, v, table, offsets(lens, gpu), offsets(cu(lens), gpu))
    q = rows(90, 2, D, BF16, gpu, 2)
    o, _ = pkg.cache_attention(q, cache, table, offsets(lens, gpu), cu=offsets(cu(new), gpu))
    c = lambda x: [x[:40].double().cpu(), x[40:].double().cpu()]
    O, _, tol, _ = want(ragged_oracle, q, new, c(k), c(v), 0.125, BF16, None, 0)
    near(o, O, tol, "o")


def test_small_values_in_fp16(pkg, ragged_oracle, gpu):
    """Scales far below the range of fp16: weights are held relative to the largest so far, which grows on the way."""
    lens, page = [400], 16
    cache, table, _, _ = filled(pkg, ragged_oracle, gpu, lens, page, 2, 64, FP16, INT8)
    k, v = rows(400, 2, 64, FP16, gpu, 0), rows(400, 2, 64, FP16, gpu, 1) * 2.0 ** -9
    v[300:] *= 256
    pkg.cache_write(cache, k, v, table, offsets(lens, gpu), offsets([0, 400], gpu))
    q = rows(150, 4, 64, FP16, gpu, 2)
    o, _ = pkg.cache_attention(q, cache, table, offsets(lens, gpu), cu=offsets([0, 150], gpu))
    held = [[ragged_oracle.dequantise(*ragged_oracle.quantise(x.cpu(), INT8))] for x in (k, v)]
    O, _, tol, _ = want(ragged_oracle, q, [150], *held, 0.125, FP16, None, 0)
    near(o, O, tol, "o")


@pytest.mark.parametrize("kind", [BF16, E4M3])
def test_a_piece_of_one_token_is_one_token(pkg, ragged_oracle, gpu, kind):
    """Both forms of the call say the same but for the order of sums."""
    lens = [700, 33, 1, 128]
    cache, table, K, V = filled(pkg, ragged_oracle, gpu, lens, 16, 2, 128, BF16, kind)
    q = rows(4, 8, 128, BF16, gpu, 5)
    for window, sinks in ((None, 0), (90, 3)):
        a, la = pkg.cache_attention(q, cache, table, offsets(lens, gpu), need_lse=True, window=window, sinks=sinks)
        b, lb = pkg.cache_attention(q, cache, table, offsets(lens, gpu), need_lse=True, cu=offsets([0, 1, 2, 3, 4], gpu), window=window, sinks=sinks)
        O, L, tol, l_tol = want(ragged_oracle, q, [1] * 4, K, V, 128 ** -0.5, BF16, window, sinks)
        for x, l in ((a, la), (b, lb)):
            near(x, O, tol, "o")
            near(l, L, l_tol, "lse")


def test_a_window_that_hides_nothing(pkg, ragged_oracle, gpu):
    lens = [700, 33]
    cache, table, _, _ = filled(pkg, ragged_oracle, gpu, lens, 16, 2, 64, BF16, INT8)
    q, held = rows(2, 4, 64, BF16, gpu, 5), 16 * table.shape[1]
    for on in (None, offsets([0, 1, 2], gpu)):
        a = pkg.cache_attention(q, cache, table, offsets(lens, gpu), need_lse=True, cu=on)
        for window, sinks in ((held, 0), (1 << 40, 5), (3, 1 << 40)):
            b = pkg.cache_attention(q, cache, table, offsets(lens, gpu), need_lse=True, cu=on, window=window, sinks=sinks)
            assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_captured_calls_follow_their_lengths_and_tables(pkg, ragged_oracle, gpu):
    lens, new = [300, 90], [40, 7]
    cache, table, _, _ = filled(pkg, ragged_oracle, gpu, lens, 16, 2, 64, BF16, E4M3)
    q, n, on = rows(47, 4, 64, BF16, gpu, 5), offsets(lens, gpu), offsets(cu(new), gpu)

    def step():
        return (*pkg.cache_attention(q, cache, table, n, need_lse=True, cu=on), *pkg.cache_attention(q, cache, table, n, need_lse=True, cu=on, window=33, sinks=2),
                *pkg.cache_attention(q[:2], cache, table, n, need_lse=True, window=33, sinks=2))

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        made = step()
    for values, at in (([300, 90], [0, 40, 47]), ([200, 90], [0, 7, 47]), ([1, 60], [0, 0, 20]), ([300, 90], [0, 40, 47])):
        n.copy_(offsets(values, gpu)), on.copy_(offsets(at, gpu))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(made, step()))
