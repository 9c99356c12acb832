"""New tokens normalised, turned by their positions and written into the paged cache, against the definitions in 64 bits; and the cache's operators together, as a layer uses them."""
import math

import pytest
import torch

from test_gpu_cache import BF16, E4M3, FP16, INT8, TYPES, empty, stands_for, tables
from test_gpu_cache_window import want as attended
from test_gpu_ragged import cu, near, offsets, rows

pytestmark = pytest.mark.gpu


def freqs_of(pairs, axes=1, base=10000.0):
    f = base ** (-torch.arange(pairs, dtype=torch.float64) / max(1, pairs))
    of = torch.arange(pairs) * axes // max(1, pairs)
    return torch.stack([torch.where(of == a, f, 0.0) for a in range(axes)]).float()


def places(lens, new):
    return torch.cat([torch.arange(n - m, n) for n, m in zip(lens, new)])[:, None]


def held(oracle, y, far, kind, dtype):
    """What the cache may read back as, in 64 bits: (values, bounds).  8 bits: within half a step of the code's scale, which is itself off as the largest value is."""
    u = torch.finfo(dtype).eps / 2
    tiny = 2.0 ** -25 if dtype == FP16 else 2.0 ** -134
    if kind not in (E4M3, INT8):
        return y, far + u * (y.abs() + far) + tiny
    top = y.abs().amax(-1, keepdim=True)
    scale = (top + far.amax(-1, keepdim=True)) / (448 if kind == E4M3 else 127) * (1 + 4 * oracle.F32)
    # int8: half a step.  e4m3: a relative 2^-4, half of the smallest step, 2^-10, below.  A quotient and a product in fp32; the result read back in 16 bits.
    step = scale / 2 if kind == INT8 else torch.maximum(2.0 ** -4 * y.abs(), 2.0 ** -10 * scale)
    off = 1.1 * far + step * (1 + 2.0 ** -20) + 8 * oracle.F32 * top
    return y, off + u * (y.abs() + off) + tiny


def check(pkg, oracle, gpu, lens, new, page, Hq, Hkv, D, dtype, kind, R, axes=0, interleaved=False, norm=None, single=False, size=1.0, base=10000.0):
    table, pages = tables(lens, page, gpu)
    cache = empty(pkg, pages, Hkv, page, D, kind, gpu)
    n = sum(new)
    q, k, v = (rows(n, h, D, dtype, gpu, i, size) for i, h in enumerate((Hq, Hkv, Hkv)))
    freqs = freqs_of(R, max(1, axes), base) if R else None
    positions = torch.randint(-50, 5000, (n, axes), generator=torch.Generator().manual_seed(3)) if axes else None
    weights = [None, None] if norm is None else [(1 + 0.3 * torch.randn(D, generator=torch.Generator().manual_seed(8 + i))).to(norm) for i in range(2)]
    on = None if single else offsets(cu(new), gpu)
    before = [x.clone() for x in (cache.k, cache.v)]
    got = pkg.cache_append(cache, q, k, v, table, offsets(lens, gpu), on, freqs=None if freqs is None else freqs.to(gpu), positions=None if positions is None else positions.to(gpu),
                           interleaved=interleaved, q_weight=None if norm is None else weights[0].to(gpu), k_weight=None if norm is None else weights[1].to(gpu), eps=1e-5)
    at = positions if axes else places(lens, new)
    u = torch.finfo(dtype).eps / 2
    y, far = oracle.turned(q, weights[0], 1e-5, at, freqs, interleaved)
    near(got, y, far + u * (y.abs() + far) + (2.0 ** -25 if dtype == FP16 else 2.0 ** -134), "q")
    K, V = pkg.cache_read(cache, table, offsets(cu(lens), gpu), sum(lens), dtype=dtype)
    fresh = torch.cat([torch.arange(b - m, b) for b, m in zip(cu(lens)[1:], new)])
    near(K[fresh.to(gpu)], *held(oracle, *oracle.turned(k, weights[1], 1e-5, at, freqs, interleaved), kind, dtype), "k")
    # values, and everything that was not to be written: as cache_write leaves them
    other = empty(pkg, pages, Hkv, page, D, kind, gpu)
    pkg.cache_write(other, k, v, table, offsets(lens, gpu), on)
    bits = lambda x: x.view(torch.uint8 if kind in (E4M3, INT8) else torch.int16)
    assert torch.equal(bits(cache.v), bits(other.v)) and (cache.v_scale is None or torch.equal(cache.v_scale.nan_to_num(-1.0), other.v_scale.nan_to_num(-1.0)))
    same = (bits(cache.k) == bits(before[0])).cpu().transpose(1, 2)
    touched = torch.zeros(pages, page, dtype=torch.bool)
    for i, (m, w) in enumerate(zip(lens, new)):
        for j in range(m - w, m):
            touched[table[i, j // page], j % page] = True
    assert same[~touched].all()


@pytest.mark.parametrize("dtype, kind", TYPES)
@pytest.mark.parametrize("D, R", [(64, 32), (64, 8), (128, 64), (128, 32), (128, 0)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("norm", [None, torch.float32, "rows"])
def test_types_and_layouts(pkg, ragged_oracle, gpu, norm, interleaved, D, R, dtype, kind):
    check(pkg, ragged_oracle, gpu, [17, 0, 1, 200], [17, 0, 1, 63], 16, 6, 2, D, dtype, kind, R, interleaved=interleaved, norm=dtype if norm == "rows" else norm)


@pytest.mark.parametrize("Hq, Hkv", [(1, 1), (3, 3), (7, 1), (16, 5), (33, 1), (40, 8)])
@pytest.mark.parametrize("new", [[1, 1], [130, 1], [3000, 1500]])
def test_heads_and_rows(pkg, ragged_oracle, gpu, Hq, Hkv, new):
    """One head to a group of lanes and several, numbers of them that do not divide."""
    check(pkg, ragged_oracle, gpu, [3100, 1501], new, 64, Hq, Hkv, 64, BF16, INT8 if Hkv == 5 else BF16, 32, norm=torch.float32)


@pytest.mark.parametrize("axes", [1, 2, 3, 8])
def test_positions(pkg, ragged_oracle, gpu, axes):
    check(pkg, ragged_oracle, gpu, [40, 33], [40, 9], 16, 4, 2, 128, FP16, FP16, 64, axes=axes)


@pytest.mark.parametrize("kind", [BF16, INT8])
def test_one_token_of_each(pkg, ragged_oracle, gpu, kind):
    check(pkg, ragged_oracle, gpu, [(37 * i) % 190 + 1 for i in range(70)], [1] * 70, 16, 8, 2, 64, BF16, kind, 32, single=True)


@pytest.mark.parametrize("dtype, kind", [(BF16, BF16), (FP16, INT8), (BF16, E4M3)])
@pytest.mark.parametrize("size", [1e-4, 30.0])
def test_sizes(pkg, ragged_oracle, gpu, size, dtype, kind):
    check(pkg, ragged_oracle, gpu, [90], [90], 16, 4, 2, 128, dtype, kind, 64, size=size)


def test_far_positions(pkg, ragged_oracle, gpu):
    """Angles of a million radians and more."""
    D, R, n = 128, 64, 200
    table, pages = tables([n], 16, gpu)
    cache = empty(pkg, pages, 2, 16, D, FP16, gpu)
    q, k = rows(n, 4, D, FP16, gpu, 0), rows(n, 2, D, FP16, gpu, 1)
    at = torch.randint(1 << 20, 1 << 24, (n, 1), generator=torch.Generator().manual_seed(3))
    freqs = freqs_of(R)
    got = pkg.cache_append(cache, q, k, k, table, offsets([n], gpu), offsets([0, n], gpu), freqs=freqs.to(gpu), positions=at.to(gpu))
    y, far = ragged_oracle.turned(q, None, 0, at, freqs, False)
    near(got, y, far + 2.0 ** -11 * (y.abs() + far) + 2.0 ** -25, "q")


def test_every_eighth_of_a_turn(pkg, ragged_oracle, gpu):
    """Angles on and beside the borders at which they are reduced."""
    D, R, n = 64, 32, 129
    table, pages = tables([n], 16, gpu)
    cache = empty(pkg, pages, 1, 16, D, FP16, gpu)
    freqs = torch.full((R,), math.pi / 64) * (1 + (torch.arange(R) - 16) * 2.0 ** -20)
    q = torch.full((n, 1, D), 1.0, dtype=FP16, device=gpu)
    q[..., R:] = 0.5
    at = torch.arange(n)[:, None] - 64
    got = pkg.cache_append(cache, q, q, q, table, offsets([n], gpu), offsets([0, n], gpu), freqs=freqs.to(gpu), positions=at.to(gpu))
    y, far = ragged_oracle.turned(q, None, 0, at, freqs[None], False)
    near(got, y, far + 2.0 ** -11 * (y.abs() + far) + 2.0 ** -25, "q")


def test_strides_and_in_place(pkg, gpu):
    """Queries, keys and values as the projection's output has them; the queries turned where they lie; positions and weights that are views."""
    lens, Hq, Hkv, D = [50, 130], 6, 2, 64
    table, pages = tables(lens, 16, gpu)
    make = lambda: empty(pkg, pages, Hkv, 16, D, INT8, gpu)
    qkv = rows(180, Hq + 2 * Hkv, D, BF16, gpu, 5)
    q, k, v = qkv[:, :Hq], qkv[:, Hq:Hq + Hkv], qkv[:, Hq + Hkv:]
    at, on, n = torch.arange(360, dtype=torch.int64, device=gpu).reshape(180, 2) % 77, offsets(cu(lens), gpu), offsets(lens, gpu)
    freqs, w = freqs_of(16, 2).to(gpu), torch.rand(D, 2, device=gpu)[:, 0] + 0.5
    a, b = make(), make()
    want = pkg.cache_append(a, q.clone(), k.clone(), v.clone(), table, n, on, freqs=freqs, positions=at.int().contiguous(), q_weight=w.clone(), k_weight=w.clone())
    got = pkg.cache_append(b, q, k, v, table, n, on, freqs=freqs.double(), positions=torch.stack([at[:, 1], at[:, 0]], 1).flip(1), q_weight=w, k_weight=w, out=q)
    assert got is q and torch.equal(q, want) and all(torch.equal(x, y) for x, y in ((a.k, b.k), (a.v, b.v), (a.k_scale.nan_to_num(-1), b.k_scale.nan_to_num(-1))))
    assert pkg.cache_append(b, None, k, v, table, n, on, freqs=freqs, positions=at, k_weight=w) is None and torch.equal(a.k, b.k)
    heads_first = q.transpose(0, 1).contiguous().transpose(0, 1)
    out = torch.full((180, 20, D), 5.0, dtype=BF16, device=gpu)
    pkg.cache_append(b, heads_first, k, v, table, n, on, out=out[:, 4:10])
    assert torch.equal(out[:, 4:10], q) and (out[:, :4] == 5).all() and (out[:, 10:] == 5).all()       # neither norm nor freqs: as they are


def test_rows_of_no_sequence_and_places_that_are_not_there(pkg, gpu):
    cache = empty(pkg, 4, 2, 16, 64, BF16, gpu)
    cache.k.fill_(0), cache.v.fill_(0)
    table = torch.tensor([[0, 4], [1, -1], [2, 1 << 30], [3, 3]], dtype=torch.int32, device=gpu)
    q, k, freqs = rows(90, 4, 64, BF16, gpu, 0), rows(90, 2, 64, BF16, gpu, 1), freqs_of(32).to(gpu)
    on = offsets([3, 23, 43, 63, 83], gpu)
    out = torch.full_like(q, 3.0)
    a = pkg.cache_append(cache, q, k, k, table, offsets([20, 20, 20, 40], gpu), on, freqs=freqs)
    pkg.cache_append(cache, q, k, k, table, offsets([20, 20, 20, 40], gpu), on, freqs=freqs, out=out)
    assert (a[:3] == 0).all() and (a[83:] == 0).all() and (out[:3] == 3).all() and (out[83:] == 3).all() and torch.equal(a[3:83], out[3:83]) and (a[3:83] != 0).any(-1).all()
    for i in range(3):
        assert torch.equal(cache.v[i].transpose(0, 1), k[3 + 20 * i:19 + 20 * i])
    assert torch.equal(cache.v[3].transpose(0, 1)[4:], k[63:75])
    assert torch.equal(a[3:4], q[3:4]) and torch.equal(cache.k[0, :, 0], k[3])          # position 0
    before = cache.k.clone()
    b = pkg.cache_append(cache, q[:8], k[:8], k[:8], table, offsets([1, 0, -3, 1 << 30], gpu), offsets([0, 2, 4, 6, 8], gpu), freqs=freqs)
    assert torch.equal(cache.k, before) and (b[:6] == 0).all() and (b[6:] != 0).any()
    # a padded batch: one token of each, the second is none
    b = pkg.cache_append(cache, q[:4], k[:4], k[:4], table, offsets([1, 0, 1, 1], gpu), freqs=freqs)
    assert (b[1] == 0).all() and torch.equal(b[[0, 2, 3]], q[[0, 2, 3]]) and torch.equal(cache.k[1], before[1])
    assert pkg.cache_append(cache, q[:0], k[:0], k[:0], table, offsets([0] * 4, gpu), offsets([0] * 5, gpu), freqs=freqs).shape == (0, 4, 64)


@pytest.mark.parametrize("kind", [BF16, E4M3, INT8])
def test_values_that_are_not_finite_stay_in_their_rows(pkg, gpu, kind):
    table, pages = tables([40], 16, gpu)
    q, k, freqs, w = rows(40, 2, 64, BF16, gpu, 0), rows(40, 2, 64, BF16, gpu, 1), freqs_of(32).to(gpu), torch.ones(64, device=gpu)
    clean = empty(pkg, pages, 2, 16, 64, kind, gpu)
    good = pkg.cache_append(clean, q, k, k, table, offsets([40], gpu), offsets([0, 40], gpu), freqs=freqs, q_weight=w, k_weight=w)
    q[5, 0, 3], k[7, 1, 60], k[8, 0, 0], k[9] = math.nan, math.inf, math.nan, 0
    cache = empty(pkg, pages, 2, 16, 64, kind, gpu)
    got = pkg.cache_append(cache, q, k, k, table, offsets([40], gpu), offsets([0, 40], gpu), freqs=freqs, q_weight=w, k_weight=w)
    assert got[5, 0].isnan().all() and torch.equal(got[5, 1], good[5, 1]) and torch.equal(got[6:], good[6:])
    K, V = pkg.cache_read(cache, table, offsets([0, 40], gpu), 40, dtype=BF16)
    K0, V0 = pkg.cache_read(clean, table, offsets([0, 40], gpu), 40, dtype=BF16)
    # an infinite value: its row's norm divides the others by infinity and itself into NaN, which goes to both channels of its pair; in 8 bits the scale is the row's
    pair = torch.tensor([i in (28, 60) or kind != BF16 for i in range(64)], device=gpu)
    assert K[7, 1, pair].isnan().all() and (K[7, 1, ~pair] == 0).all() and K[8, 0].isnan().all() and torch.equal(K[7, 0], K0[7, 0]) and torch.equal(K[8, 1], K0[8, 1]) and (K[9] == 0).all() and (V[9] == 0).all()
    assert torch.equal(K[10:], K0[10:]) and torch.equal(V[10:], V0[10:]) and torch.equal(K[:7], K0[:7])


def test_pages_behind_32_bits(pkg, gpu):
    page, D, step = 16, 64, 1 << 21
    pages = (1 << 32) // (2 * step) + 8
    pool = torch.empty(pages * step, dtype=BF16, device=gpu)
    view = lambda at: pool.as_strided((pages, 1, page, D), (step, page * D, D, 1), at)
    cache = pkg.KVCache(view(0), view(page * D))
    table = torch.tensor([[pages - 1, 2, pages - 3]], dtype=torch.int32, device=gpu)
    k, v = rows(40, 1, D, BF16, gpu, 0), rows(40, 1, D, BF16, gpu, 1)
    pkg.cache_append(cache, None, k, v, table, offsets([40], gpu), offsets([0, 40], gpu))
    K, V = pkg.cache_read(cache, table, offsets([0, 40], gpu), 40)
    assert torch.equal(K, k) and torch.equal(V, v)


def test_captured_calls_follow_their_lengths(pkg, gpu):
    table, pages = tables([100, 100], 16, gpu)
    cache = empty(pkg, pages, 2, 16, 64, BF16, gpu)
    q, k, v, freqs = rows(9, 4, 64, BF16, gpu, 0), rows(9, 2, 64, BF16, gpu, 1), rows(9, 2, 64, BF16, gpu, 2), freqs_of(32).to(gpu)
    n, on = offsets([4, 5], gpu), offsets([0, 4, 9], gpu)
    step = lambda: pkg.cache_append(cache, q, k, v, table, n, on, freqs=freqs)
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        made = step()
    for lens, at in (([4, 5], [0, 4, 9]), ([90, 20], [0, 4, 9]), ([100, 1], [0, 8, 9]), ([4, 5], [0, 4, 9])):
        n.copy_(offsets(lens, gpu)), on.copy_(offsets(at, gpu))
        cache.k.zero_(), cache.v.zero_()
        graph.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in (made, cache.k, cache.v)]
        cache.k.zero_(), cache.v.zero_()
        assert all(torch.equal(a, b) for a, b in zip(got, (step(), cache.k, cache.v)))


@pytest.mark.parametrize("window, sinks", [(None, 0), (40, 3)])
@pytest.mark.parametrize("dtype, kind", [(BF16, BF16), (FP16, FP16), (BF16, E4M3), (FP16, INT8)])
def test_a_layer_piece_by_piece_and_token_by_token(pkg, ragged_oracle, gpu, dtype, kind, window, sinks):
    """The operators as they are used together: pieces of prompts and single tokens appended and attended to, against the oracle's attention over what the cache holds by then."""
    page, Hq, Hkv, D = 16, 6, 2, 64
    total = [90, 41]
    table, pages = tables(total, page, gpu)
    cache = empty(pkg, pages, Hkv, page, D, kind, gpu)
    q, k, v = ([rows(n, h, D, dtype, gpu, s + i) for i, n in enumerate(total)] for s, h in ((20, Hq), (30, Hkv), (40, Hkv)))
    freqs, w = freqs_of(16).to(gpu), [(0.5 + torch.rand(D, generator=torch.Generator().manual_seed(i))).to(gpu) for i in range(2)]
    done = [0, 0]
    for piece in ([50, 1], [30, 30], [1, 0], [1, 1], [1, 1], [7, 8]):
        end = [a + b for a, b in zip(done, piece)]
        single = piece == [1, 1]
        take = lambda x: torch.cat([y[a:b] for y, a, b in zip(x, done, end)])
        on = None if single else offsets(cu(piece), gpu)
        Q = pkg.cache_append(cache, take(q), take(k), take(v), table, offsets(end, gpu), on, freqs=freqs, q_weight=w[0], k_weight=w[1])
        o, lse = pkg.cache_attention(Q, cache, table, offsets(end, gpu), need_lse=True, cu=on, window=window, sinks=sinks)
        K, V = pkg.cache_read(cache, table, offsets(cu(end), gpu), sum(end), dtype=dtype)
        if kind not in (E4M3, INT8):
            K, V = ([x[a:b].double().cpu() for a, b in zip(cu(end)[:-1], cu(end)[1:])] for x in (K, V))
        else:           # (what 16 bits round off is not the attention's)
            at = [(table[i].long()[torch.arange(n, device=gpu) // page], torch.arange(n, device=gpu) % page) for i, n in enumerate(end)]
            by = lambda x, s: [ragged_oracle.dequantise(x.view(torch.uint8)[p, :, j].view(kind).cpu(), s[p, :, j].cpu()) for p, j in at]
            K, V = by(cache.k, cache.k_scale), by(cache.v, cache.v_scale)
        O, L, tol, l_tol = attended(ragged_oracle, Q, piece, K, V, D ** -0.5, dtype, window, sinks)
        near(o, O, tol, "o")
        near(lse, L, l_tol, "lse")
        done = end
    # what is there by now: keys of all positions
    at = places(total, done)
    for i in range(2):
        got = pkg.cache_read(cache, table[i:i + 1], offsets([0, done[i]], gpu), done[i], dtype=dtype)[0]
        y = ragged_oracle.turned(k[i][:done[i]], w[1], 1e-6, torch.arange(done[i])[:, None], freqs[:].cpu().reshape(1, -1), False)
        near(got, *held(ragged_oracle, *y, kind, dtype), "k")


@pytest.mark.parametrize("kind", [BF16, INT8])
def test_two_streams_at_once(pkg, gpu, kind):
    """Two layers' steps, each on its own cache, together what they are one after the other: nothing is shared between calls."""
    page, Hq, Hkv, D, lens, new = 16, 8, 2, 128, [900, 700, 40], [300, 1, 16]
    table, pages = tables(lens, page, gpu)
    freqs, on, at = freqs_of(64).to(gpu), offsets(cu(new), gpu), offsets(lens, gpu)
    w = torch.ones(D, device=gpu)

    def layer(seed):
        cache = empty(pkg, pages, Hkv, page, D, kind, gpu)
        k, v = (rows(sum(lens), Hkv, D, BF16, gpu, seed + i) for i in range(2))
        pkg.cache_write(cache, k, v, table, at, offsets(cu(lens), gpu))
        return cache, rows(sum(new), Hq, D, BF16, gpu, seed + 2), k[:sum(new)] * 2, v[:sum(new)] * 2

    def step(cache, q, k, v):
        q = pkg.cache_append(cache, q, k, v, table, at, on, freqs=freqs, q_weight=w, k_weight=w)
        return q, *pkg.cache_attention(q, cache, table, at, need_lse=True, cu=on), *pkg.cache_attention(q, cache, table, at, need_lse=True, cu=on, window=200, sinks=4)

    layers = [layer(10), layer(20)]
    want = [step(*x) for x in layers]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in layers]
    for _ in range(5):
        got = []
        for stream, x in zip(streams, layers):
            with torch.cuda.stream(stream):
                got.append(step(*x))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for x, y in zip(got, want) for a, b in zip(x, y))
