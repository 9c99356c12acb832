"""The paged key-value cache: writing, reading back and attention of one token, against the definitions; and a prompt that goes through all of it in pieces."""
import copy
import math

import pytest
import torch

from test_gpu_ragged import BF16, FP16, cu, near, offsets, rows

pytestmark = pytest.mark.gpu

E4M3, INT8 = torch.float8_e4m3fn, torch.int8
TYPES = [(BF16, BF16), (FP16, FP16), (BF16, E4M3), (FP16, E4M3), (BF16, INT8), (FP16, INT8)]


def empty(pkg, pages, heads, page, D, kind, gpu):
    """A cache whose every byte is NaN or the largest code, scales NaN."""
    cache = pkg.KVCache.empty(pages, heads, page, D, dtype=kind, device=gpu)
    for x in (cache.k, cache.v):
        x.view(torch.uint8 if kind in (E4M3, INT8) else kind).fill_(127 if kind in (E4M3, INT8) else math.nan)
    for x in (cache.k_scale, cache.v_scale):
        if x is not None:
            x.fill_(math.nan)
    return cache


def tables(lens, page, gpu, spare=2, seed=0, behind=-1):
    """Pages in no order; entries behind a sequence's last page are no pages."""
    held = [-(-n // page) for n in lens]
    width = max(held + [1]) + 1
    order = torch.randperm(sum(held) + spare, generator=torch.Generator().manual_seed(seed)).tolist()
    table = [[order.pop() for _ in range(h)] + [behind] * (width - h) for h in held]
    return torch.tensor(table, dtype=torch.int32, device=gpu).reshape(len(lens), width), sum(held) + spare


def stands_for(oracle, x, kind):
    """What rows are once they were written, in 64 bits."""
    if kind in (BF16, FP16):
        return x.double().cpu()
    return oracle.dequantise(*oracle.quantise(x.cpu(), kind))


@pytest.mark.parametrize("dtype, kind", TYPES)
@pytest.mark.parametrize("D, page, heads", [(64, 16, 1), (128, 64, 3), (128, 16, 8), (64, 1024, 2)])
def test_write_and_read_back(pkg, ragged_oracle, gpu, D, page, heads, dtype, kind):
    lens = [17, 0, 1, 64, 130]
    table, pages = tables(lens, page, gpu)
    cache = empty(pkg, pages, heads, page, D, kind, gpu)
    k, v = rows(sum(lens), heads, D, dtype, gpu, 0, 3.0), rows(sum(lens), heads, D, dtype, gpu, 1)
    k[5] = 0
    on = offsets(cu(lens), gpu)
    before = [x.clone() for x in (cache.k, cache.v)]
    pkg.cache_write(cache, k, v, table, offsets(lens, gpu), on)
    got = pkg.cache_read(cache, table, on, sum(lens), dtype=dtype)
    for x, y in zip((k, v), got):
        if kind in (BF16, FP16):
            assert torch.equal(x, y)
        else:
            codes, scale = ragged_oracle.quantise(x.cpu(), kind)
            assert torch.equal(y.cpu(), (codes.float() * scale[..., None]).to(dtype))
    # nothing but the sequences' places was written
    for x, b in zip((cache.k, cache.v), before):
        touched = torch.zeros(cache.k.shape[0], page, dtype=torch.bool)
        for i, n in enumerate(lens):
            for j in range(n):
                touched[table[i, j // page], j % page] = True
        same = (x.view(torch.int8 if kind in (E4M3, INT8) else torch.int16) == b.view(torch.int8 if kind in (E4M3, INT8) else torch.int16)).cpu()
        assert same.transpose(1, 2)[~touched].all()


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("kind", [E4M3, INT8])
def test_codes_of_all_sizes(pkg, ragged_oracle, gpu, kind, dtype):
    """From the type's smallest to its largest, ties, zeros, and values that are not finite."""
    x = torch.randn(600, 2, 64, generator=torch.Generator().manual_seed(1))
    x *= 2.0 ** torch.linspace(-20 if dtype == FP16 else -130, 14 if dtype == FP16 else 120, 600)[:, None, None]
    x[7, 0] = torch.arange(64) - 31.5
    x[7, 0, 63] = 127.0 if kind == INT8 else 448.0
    x[8, 1, 3], x[9, 0, 60], x[10] = math.inf, math.nan, 0
    x = x.to(dtype)
    table, pages = tables([600], 32, gpu)
    cache = empty(pkg, pages, 2, 32, 64, kind, gpu)
    on = offsets([0, 600], gpu)
    pkg.cache_write(cache, x.to(gpu), x.to(gpu).flip(0), table, offsets([600], gpu), on)
    for y, z in zip(pkg.cache_read(cache, table, on, 600, dtype=dtype), (x, x.flip(0))):
        codes, scale = ragged_oracle.quantise(z, kind)
        want = (codes.float() * scale[..., None]).to(dtype)
        y = y.cpu()
        assert torch.equal(y.isnan(), want.isnan()) and torch.equal(y.nan_to_num(), want.nan_to_num())


@pytest.mark.parametrize("dtype, bits", [(BF16, 7), (FP16, 10)])
@pytest.mark.parametrize("kind", [E4M3, INT8])
def test_every_quotient(pkg, ragged_oracle, gpu, kind, dtype, bits):
    """All significands of a value, over two binades, over all significands of its row's largest: codes next to a border are those of IEEE division."""
    n = 1 << bits
    tops = 1 + torch.arange(n) / n
    values = torch.cat([1 + torch.arange(n) / n, (1 + torch.arange(n) / n) / 2])
    values = torch.cat([values, values.new_zeros(-len(values) % 127)]).reshape(-1, 127)
    x = torch.empty(n, len(values), 128)
    x[:, :, :127] = torch.minimum(values[None], tops[:, None, None])
    x[:, :, 1:127:2] *= -1
    x[:, :, 127] = tops[:, None]
    x = x.reshape(1, -1, 128).transpose(0, 1).to(dtype)
    table, pages = tables([len(x)], 64, gpu)
    cache = empty(pkg, pages, 1, 64, 128, kind, gpu)
    on = offsets([0, len(x)], gpu)
    pkg.cache_write(cache, x.to(gpu), (x * 2.0 ** 3).to(gpu), table, offsets([len(x)], gpu), on)
    codes, scale = ragged_oracle.quantise(x, kind)
    at = torch.arange(len(x), device=gpu)
    for got, got_scale, by in ((cache.k, cache.k_scale, 1.0), (cache.v, cache.v_scale, 8.0)):
        assert torch.equal(got_scale[table[0, at // 64].long(), 0, at % 64].cpu(), scale[:, 0] * by)
        assert torch.equal(got.view(torch.uint8)[table[0, at // 64].long(), 0, at % 64].cpu().view(kind).float(), codes[:, 0].float())      # (zeros of either sign)


def test_only_new_tokens_are_written(pkg, gpu):
    lens, new = [20, 5, 1], [3, 5, 0]
    table, pages = tables(lens, 16, gpu)
    cache = empty(pkg, pages, 2, 16, 64, BF16, gpu)
    k, v = rows(26, 2, 64, BF16, gpu, 0), rows(26, 2, 64, BF16, gpu, 1)
    pkg.cache_write(cache, k, v, table, offsets(lens, gpu), offsets(cu(lens), gpu))
    k1, v1 = rows(8, 2, 64, BF16, gpu, 2), rows(8, 2, 64, BF16, gpu, 3)
    pkg.cache_write(cache, k1, v1, table, offsets(lens, gpu), offsets(cu(new), gpu))
    K, V = pkg.cache_read(cache, table, offsets(cu(lens), gpu), 26)
    assert torch.equal(K, torch.cat([k[:17], k1, k[25:]])) and torch.equal(V, torch.cat([v[:17], v1, v[25:]]))
    k2 = rows(3, 2, 64, BF16, gpu, 4)
    pkg.cache_write(cache, k2, k2, table, offsets([20, 0, 1], gpu))       # one of each; a padded sequence writes nothing
    K2, _ = pkg.cache_read(cache, table, offsets(cu(lens), gpu), 26)
    assert torch.equal(K2, torch.cat([K[:19], k2[:1], K[20:25], k2[2:]]))


def test_places_that_are_not_there(pkg, gpu):
    """Pages outside of the cache, lengths the table does not hold or that are below the rows: nothing is written; reading back gives NaN."""
    cache = empty(pkg, 4, 2, 16, 64, BF16, gpu)
    cache.k.fill_(0), cache.v.fill_(0)
    table = torch.tensor([[0, 4], [1, -1], [2, 1 << 30], [3, 3]], dtype=torch.int32, device=gpu)
    k = rows(80, 2, 64, BF16, gpu, 0)
    pkg.cache_write(cache, k, k, table, offsets([20, 20, 20, 40], gpu), offsets([0, 20, 40, 60, 80], gpu))
    for i in range(3):
        assert torch.equal(cache.k[i].transpose(0, 1), k[20 * i:20 * i + 16])
    assert torch.equal(cache.k[3].transpose(0, 1)[4:], k[60:72])
    K, V = pkg.cache_read(cache, table, offsets([0, 20, 40, 60, 100], gpu), 100)
    for i in range(3):
        assert torch.equal(K[20 * i:20 * i + 16], k[20 * i:20 * i + 16]) and K[20 * i + 16:20 * i + 20].isnan().all() and V[20 * i + 16:20 * i + 20].isnan().all()
    assert K[92:].isnan().all() and K[60:92].isfinite().all()
    before = cache.k.clone()
    pkg.cache_write(cache, k[:8], k[:8], table, offsets([1, 0, -3, 1 << 30], gpu), offsets([0, 2, 4, 6, 8], gpu))
    assert torch.equal(cache.k, before)


def test_copies_have_pages_of_their_own(pkg, gpu):
    cache, table = empty(pkg, 2, 2, 16, 64, torch.int8, gpu), torch.tensor([[1]], dtype=torch.int32, device=gpu)
    for x in (cache.k, cache.v, cache.k_scale, cache.v_scale):
        x.zero_()
    other, same = copy.deepcopy(cache), copy.copy(cache)
    k = rows(3, 2, 64, BF16, gpu, 0)
    pkg.cache_write(other, k, k, table, offsets([3], gpu), offsets([0, 3], gpu))
    assert (other.k_scale[1, :, :3] > 0).all() and (cache.k == 0).all() and (cache.k_scale == 0).all()
    pkg.cache_write(same, k, k, table, offsets([3], gpu), offsets([0, 3], gpu))
    assert torch.equal(cache.k, other.k) and torch.equal(cache.v_scale, other.v_scale)
    with pytest.raises(AttributeError):
        cache.k = other.k


def test_rows_of_no_sequence_are_neither_written_nor_read(pkg, gpu):
    table, pages = tables([10, 20], 16, gpu)
    cache = empty(pkg, pages, 1, 16, 64, BF16, gpu)
    k = rows(40, 1, 64, BF16, gpu, 0)
    on = offsets([3, 13, 33], gpu)
    pkg.cache_write(cache, k, k, table, offsets([10, 20], gpu), on)
    K, V = pkg.cache_read(cache, table, on, 40)
    assert torch.equal(K[3:33], k[3:33]) and torch.equal(V[3:33], k[3:33])
    assert all((x[:3] == 0).all() and (x[33:] == 0).all() for x in (K, V))


def filled(pkg, oracle, gpu, lens, page, heads, D, dtype, kind, seed=0, size=1.0):
    table, pages = tables(lens, page, gpu, seed=seed)
    cache = empty(pkg, pages, heads, page, D, kind, gpu)
    k, v = rows(sum(lens), heads, D, dtype, gpu, seed, size), rows(sum(lens), heads, D, dtype, gpu, seed + 1)
    pkg.cache_write(cache, k, v, table, offsets(lens, gpu), offsets(cu(lens), gpu))
    at = cu(lens)
    K, V = ([stands_for(oracle, x[a:b], kind) for a, b in zip(at[:-1], at[1:])] for x in (k, v))
    return cache, table, K, V


def check_decode(pkg, oracle, gpu, lens, page, Hq, Hkv, D, dtype, kind, scale=None, size=1.0):
    cache, table, K, V = filled(pkg, oracle, gpu, lens, page, Hkv, D, dtype, kind, size=size)
    q = rows(len(lens), Hq, D, dtype, gpu, 5, size)
    o, lse = pkg.cache_attention(q, cache, table, offsets(lens, gpu), sm_scale=scale, need_lse=True)
    O, L, o_tol, l_tol = oracle.decode(q, K, V, D ** -0.5 if scale is None else scale, dtype)
    near(o, O, o_tol, "o")
    near(lse, L, l_tol, "lse")


@pytest.mark.parametrize("dtype, kind", TYPES)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("lens, page", [([1], 16), ([33, 0, 128, 129, 5], 16), ([495, 0, 384], 16), ([1000, 1, 257], 64), ([700], 1024), ([0, 600, 1], 16)])
def test_one_token(pkg, ragged_oracle, gpu, lens, page, D, dtype, kind):
    check_decode(pkg, ragged_oracle, gpu, lens, page, 4, 2, D, dtype, kind)


@pytest.mark.parametrize("Hq, Hkv", [(1, 1), (3, 3), (7, 1), (16, 1), (17, 1), (32, 1), (33, 1), (70, 2), (40, 8), (96, 1)])
def test_heads_of_one_token(pkg, ragged_oracle, gpu, Hq, Hkv):
    check_decode(pkg, ragged_oracle, gpu, [140, 20, 300], 16, Hq, Hkv, 128, BF16, BF16)


@pytest.mark.parametrize("kind", [BF16, E4M3, INT8])
@pytest.mark.parametrize("scale, size", [(-0.3, 1.0), (0.0, 1.0), (None, 6.0)])
def test_scales_of_one_token(pkg, ragged_oracle, gpu, scale, size, kind):
    check_decode(pkg, ragged_oracle, gpu, [300, 31], 32, 8, 2, 64, BF16, kind, scale, size)


def test_long_and_short_ones_together(pkg, ragged_oracle, gpu):
    """Runs of the list that begin and end inside of sequences, and hold many."""
    lens = [20000, 1, 0, 5, 128, 9000] + [(37 * i) % 190 for i in range(140)]
    check_decode(pkg, ragged_oracle, gpu, lens, 16, 4, 2, 64, BF16, INT8)


@pytest.mark.parametrize("B, longest, of", [(100, 1500, 99), (65, 700, 0), (300, 900, 150), (1100, 2176, 1050), (1024, 2200, 1023)])
def test_many_sequences(pkg, ragged_oracle, gpu, B, longest, of):
    """More sequences than one look at their lengths takes, cut and whole, the longest anywhere, empty ones between."""
    g = torch.Generator().manual_seed(B)
    lens = torch.randint(0, 40, (B,), generator=g).tolist()
    lens[of], lens[B // 3], lens[2 * B // 3] = longest, longest // 2, 300
    check_decode(pkg, ragged_oracle, gpu, lens, 16, 2, 1, 64, BF16, INT8)


def test_small_values_in_fp16(pkg, ragged_oracle, gpu):
    """Scales far below the range of fp16: weights are held relative to the largest."""
    lens = [400]
    table, pages = tables(lens, 16, gpu)
    cache = empty(pkg, pages, 2, 16, 64, INT8, gpu)
    k, v = rows(400, 2, 64, FP16, gpu, 0), rows(400, 2, 64, FP16, gpu, 1) * 2.0 ** -9
    v[300:] *= 256
    on = offsets([0, 400], gpu)
    pkg.cache_write(cache, k, v, table, offsets(lens, gpu), on)
    q = rows(1, 4, 64, FP16, gpu, 2)
    o, _ = pkg.cache_attention(q, cache, table, offsets(lens, gpu))
    O, _, tol, _ = ragged_oracle.decode(q, [stands_for(ragged_oracle, k, INT8)], [stands_for(ragged_oracle, v, INT8)], 0.125, FP16)
    near(o, O, tol, "o")


def test_what_cannot_be_looked_up_is_nan(pkg, ragged_oracle, gpu):
    lens = [100, 40, 60, 0]
    cache, table, K, V = filled(pkg, ragged_oracle, gpu, lens, 16, 2, 64, BF16, BF16)
    q = rows(4, 4, 64, BF16, gpu, 5)
    good = pkg.cache_attention(q, cache, table, offsets(lens, gpu))[0]
    bad = table.clone()
    bad[0, 2], bad[2, 0] = cache.pages, -7
    o, lse = pkg.cache_attention(q, cache, bad, offsets(lens, gpu), need_lse=True)
    assert o[0].isnan().all() and o[2].isnan().all() and lse[0].isnan().all() and torch.equal(o[1], good[1]) and (o[3] == 0).all()
    o, lse = pkg.cache_attention(q, cache, table, offsets([100, -1, 16 * table.shape[1] + 1, 0], gpu), need_lse=True)
    assert torch.equal(o[0], good[0]) and o[1:3].isnan().all() and lse[1:3].isnan().all() and (lse[3] == -math.inf).all()


def test_a_table_of_one_page_takes_one_kernel(pkg, ragged_oracle, gpu):
    """No workspace, nothing to join."""
    assert pkg.kv_cache._workspace_bytes(2, 64, 128, 3, 1, 4) == 0 == pkg.kv_cache._workspace_bytes(2, 64, 128, 3, 4, 4) < pkg.kv_cache._workspace_bytes(2, 64, 128, 3, 5, 4)
    cache = empty(pkg, 3, 2, 128, 64, BF16, gpu)
    k, v = rows(200, 2, 64, BF16, gpu, 0), rows(200, 2, 64, BF16, gpu, 1)
    table, lens = offsets([2, 0, 1], gpu)[:, None], [128, 0, 72]
    pkg.cache_write(cache, k, v, table, offsets(lens, gpu), offsets(cu(lens), gpu))
    q = rows(3, 4, 64, BF16, gpu, 2)
    o, lse = pkg.cache_attention(q, cache, table, offsets(lens, gpu), need_lse=True)
    O, L, tol, l_tol = ragged_oracle.decode(q, [k[:128].double().cpu(), k[:0].double().cpu(), k[128:].double().cpu()], [v[:128].double().cpu(), v[:0].double().cpu(), v[128:].double().cpu()], 0.125, BF16)
    near(o, O, tol, "o")
    near(lse, L, l_tol, "lse")


@pytest.mark.parametrize("kind", [BF16, INT8])
def test_layouts(pkg, ragged_oracle, gpu, kind):
    """Keys and values in one pool, rows of all heads side by side, queries and outputs that are parts of larger tensors."""
    lens, page, heads, D = [90, 200], 32, 2, 64
    cache, table, K, V = filled(pkg, ragged_oracle, gpu, lens, page, heads, D, BF16, kind)
    q = rows(2, 8, D, BF16, gpu, 5)
    want = pkg.cache_attention(q, cache, table, offsets(lens, gpu), need_lse=True)
    pool = torch.empty((cache.pages, 2, page, heads, D), dtype=kind, device=gpu)
    scales = torch.empty((2, heads, cache.pages, page), dtype=torch.float32, device=gpu)
    k, v = pool[:, 0].transpose(1, 2), pool[:, 1].transpose(1, 2)
    k.copy_(cache.k), v.copy_(cache.v)
    ks, vs = (None, None) if kind == BF16 else (scales[0].transpose(0, 1), scales[1].transpose(0, 1))
    if ks is not None:
        ks.copy_(cache.k_scale), vs.copy_(cache.v_scale)
    other = pkg.KVCache(k, v, ks, vs)
    wide = torch.full((2, 12, D), 7.0, dtype=BF16, device=gpu)
    wide[:, 2:10] = q
    out = torch.full((2, 20, D), 5.0, dtype=BF16, device=gpu)
    wide_table = torch.cat([table, torch.full_like(table, -1)], 1)[:, :table.shape[1]]
    got = pkg.cache_attention(wide[:, 2:10], other, wide_table, offsets(lens, gpu), need_lse=True, out=out[:, 4:12])
    assert torch.equal(out[:, 4:12], want[0]) and torch.equal(got[1], want[1]) and (out[:, :4] == 5).all() and (out[:, 12:] == 5).all()
    on = offsets(cu(lens), gpu)
    assert all(torch.equal(a, b) for a, b in zip(pkg.cache_read(other, wide_table, on, 290), pkg.cache_read(cache, table, on, 290)))
    rows_in = rows(290, 3 * heads, D, BF16, gpu, 11)
    pkg.cache_write(other, rows_in[:, heads:2 * heads], rows_in[:, 2 * heads:], wide_table, offsets(lens, gpu), on)
    pkg.cache_write(cache, rows_in[:, heads:2 * heads].contiguous(), rows_in[:, 2 * heads:].contiguous(), table, offsets(lens, gpu), on)
    assert all(torch.equal(a, b) for a, b in zip(pkg.cache_read(other, wide_table, on, 290), pkg.cache_read(cache, table, on, 290)))


def test_pages_behind_32_bits(pkg, ragged_oracle, gpu):
    """A pool of more than 2^32 bytes, of which the last pages are used."""
    page, heads, D = 16, 1, 64
    step = 1 << 21                                   # elements between pages
    pages = (1 << 32) // (2 * step) + 8
    pool = torch.empty(pages * step, dtype=BF16, device=gpu)
    view = lambda at: pool.as_strided((pages, heads, page, D), (step, page * D, D, 1), at)
    cache = pkg.KVCache(view(0), view(page * D))
    lens = [40, 70]
    table = torch.tensor([[pages - 1, 2, pages - 3, -1, -1], [0, pages - 2, 1, pages - 5, pages - 6]], dtype=torch.int32, device=gpu)
    k, v = rows(110, heads, D, BF16, gpu, 0), rows(110, heads, D, BF16, gpu, 1)
    on = offsets(cu(lens), gpu)
    pkg.cache_write(cache, k, v, table, offsets(lens, gpu), on)
    K, V = pkg.cache_read(cache, table, on, 110)
    assert torch.equal(K, k) and torch.equal(V, v)
    assert torch.equal(cache.k[pages - 1, 0], k[:16, 0])
    q = rows(2, 2, D, BF16, gpu, 2)
    o, _ = pkg.cache_attention(q, cache, table, offsets(lens, gpu))
    c = lambda x: [x[:40].double().cpu(), x[40:].double().cpu()]
    O, _, tol, _ = ragged_oracle.decode(q, c(k), c(v), 0.125, BF16)
    near(o, O, tol, "o")


@pytest.mark.parametrize("dtype, kind", [(BF16, BF16), (FP16, E4M3), (BF16, INT8)])
def test_a_prompt_in_pieces_and_then_token_by_token(pkg, ragged_oracle, gpu, dtype, kind):
    """The operators as they are used together: each piece is written, read back with all before it and attended to causally; then single tokens.  Against the whole at once."""
    page, Hq, Hkv, D = 16, 6, 2, 64
    total = [90, 41]
    table, pages = tables(total, page, gpu)
    cache = empty(pkg, pages, Hkv, page, D, kind, gpu)
    q = [rows(n, Hq, D, dtype, gpu, 20 + i) for i, n in enumerate(total)]
    k = [rows(n, Hkv, D, dtype, gpu, 30 + i) for i, n in enumerate(total)]
    v = [rows(n, Hkv, D, dtype, gpu, 40 + i) for i, n in enumerate(total)]
    got = [torch.zeros_like(x) for x in q]
    known = [0, 0]
    for piece in ([50, 1], [33, 35]):
        upto = [a + b for a, b in zip(known, piece)]
        take = lambda xs: torch.cat([x[a:b] for x, a, b in zip(xs, known, upto)])
        pkg.cache_write(cache, take(k), take(v), table, offsets(upto, gpu), offsets(cu(piece), gpu))
        K, V = pkg.cache_read(cache, table, offsets(cu(upto), gpu), sum(upto), dtype=dtype)
        o = pkg.attention_ragged(take(q), K, V, offsets(cu(piece), gpu), offsets(cu(upto), gpu), causal=True)
        for i, (a, b) in enumerate(zip(known, upto)):
            got[i][a:b] = o[cu(piece)[i]:cu(piece)[i + 1]]
        known = upto
    while known[0] < total[0]:
        lens = [min(a + 1, n) for a, n in zip(known, total)]
        last = lambda xs: torch.stack([x[n - 1] for x, n in zip(xs, lens)])
        pkg.cache_write(cache, last(k), last(v), table, offsets(lens, gpu))
        o, _ = pkg.cache_attention(last(q), cache, table, offsets(lens, gpu))
        for i, n in enumerate(lens):
            got[i][n - 1] = o[i]
        known = lens
    for i, n in enumerate(total):
        K, V = stands_for(ragged_oracle, k[i], kind), stands_for(ragged_oracle, v[i], kind)
        O, _, tol, _ = ragged_oracle.ragged_fwd(q[i], K, V, [0, n], [0, n], True, D ** -0.5, dtype)
        if kind not in (BF16, FP16):
            # (pieces are attended to as read back in 16 bits: K and V rounded once more, u of each; a score moves by u c sum |q k|, o by twice that of sum p |v|)
            u = torch.finfo(dtype).eps / 2
            for h in range(Hq):
                c = D ** -0.5 * (q[i][:, h].double().cpu().abs() @ K[:, h // 3].abs().t())
                mask = ragged_oracle.visible(n, n, True)
                P = ragged_oracle.attend(q[i][:, h].double().cpu(), K[:, h // 3], V[:, h // 3], mask, D ** -0.5)[2]
                tol[:, h] += u * (2 * (c * mask).amax(-1, keepdim=True) + 1) * (P @ V[:, h // 3].abs()) * 1.1
        near(got[i], O, tol, f"sequence {i}")


def test_captured_steps_follow_their_tables(pkg, ragged_oracle, gpu):
    """One token of each sequence, written and attended to in a captured graph; lengths and tables change between replays."""
    page, heads, D = 16, 2, 64
    cache = empty(pkg, 40, heads, page, D, INT8, gpu)
    eager = empty(pkg, 40, heads, page, D, INT8, gpu)
    table, lens = torch.zeros((2, 20), dtype=torch.int32, device=gpu), offsets([1, 1], gpu)
    table.copy_(torch.randperm(40, generator=torch.Generator().manual_seed(3)).reshape(2, 20))
    q, k, v = (rows(2, h, D, BF16, gpu, i) for i, h in enumerate((4, heads, heads)))

    def step(cache):
        pkg.cache_write(cache, k, v, table, lens)
        return pkg.cache_attention(q, cache, table, lens, need_lse=True)

    step(cache), step(eager)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        made = step(cache)
    for i, at in enumerate(([1, 1], [2, 1], [3, 0], [4, 1], [5, 2])):
        lens.copy_(offsets(at, gpu))
        for x, h in ((q, 4), (k, heads), (v, heads)):
            x.copy_(rows(2, h, D, BF16, gpu, 100 * i + h))
        if i == 3:
            table[1] = table[1].flip(0).clone()
        graph.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in made]
        want = step(eager)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_two_streams_at_once(pkg, ragged_oracle, gpu):
    lens = [3000, 50]
    cache, table, K, V = filled(pkg, ragged_oracle, gpu, lens, 16, 2, 64, BF16, BF16)
    q = [rows(2, 4, 64, BF16, gpu, 50 + i) for i in range(2)]
    on = offsets(lens, gpu)
    want = [pkg.cache_attention(x, cache, table, on)[0] for x in q]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in q], [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(pkg.cache_attention(q[i], cache, table, on)[0])
    torch.cuda.synchronize()
    assert all(torch.equal(x, w) for g, w in zip(got, want) for x in g)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("lens, page", [([1, 5, 8, 13, 0, 33, 100], 16), ([129, 700, 6], 64), ([2500, 3, 1030], 16)])
def test_infinite_values(pkg, ragged_oracle, gpu, lens, page, D, dtype):
    """In the last row, and in any of a sequence: infinite in their channels, and nothing elsewhere."""
    table, pages = tables(lens, page, gpu)
    cache = empty(pkg, pages, 2, page, D, dtype, gpu)
    k, v, q = rows(sum(lens), 2, D, dtype, gpu, 0), rows(sum(lens), 2, D, dtype, gpu, 1), rows(len(lens), 4, D, dtype, gpu, 2, 0.5)
    on = cu(lens)
    plain = v.clone()
    want = {}
    for i, (a, b) in enumerate(zip(on[:-1], on[1:])):
        for channel, row, sign in ((3, b - 1, 1), (D - 1, max(a, b - 6), -1), (20, a + (b - a) // 2, 1)):
            if a < b:
                v[row, :, channel], plain[a:b, :, channel] = sign * math.inf, 0
                want[i, channel] = sign * math.inf
    pkg.cache_write(cache, k, v, table, offsets(lens, gpu), offsets(on, gpu))
    o, lse = pkg.cache_attention(q, cache, table, offsets(lens, gpu), need_lse=True)
    for (i, channel), w in want.items():
        assert (o[i, :, channel] == w).all(), (i, channel)
        o[i, :, channel] = 0
    c = lambda x: [x[a:b].double().cpu() for a, b in zip(on[:-1], on[1:])]
    O, L, tol, l_tol = ragged_oracle.decode(q, c(k), c(plain), D ** -0.5, dtype)
    near(o, O, tol, "o")
    near(lse, L, l_tol, "lse")


@pytest.mark.parametrize("kind", [E4M3, INT8])
@pytest.mark.parametrize("power", [-132, -126, -120, -60])
def test_values_that_fp16_does_not_reach(pkg, ragged_oracle, gpu, kind, power):
    """Written as bf16 with scales below fp32's normal numbers, attended to in fp16: zeros, and beside larger values nothing.  (2^132 is infinite in fp32: the third sequence has rows that are
    not finite then, and NaN by definition.)"""
    lens = [200, 40, 300]
    table, pages = tables(lens, 16, gpu)
    cache = empty(pkg, pages, 2, 16, 64, kind, gpu)
    k, v = rows(540, 2, 64, BF16, gpu, 0), rows(540, 2, 64, BF16, gpu, 1) * 2.0 ** power
    v[500:] *= 2.0 ** -power
    on = cu(lens)
    pkg.cache_write(cache, k, v, table, offsets(lens, gpu), offsets(on, gpu))
    q = rows(3, 4, 64, FP16, gpu, 2)
    o, lse = pkg.cache_attention(q, cache, table, offsets(lens, gpu), need_lse=True)
    K, V = ([stands_for(ragged_oracle, x[a:b], kind) for a, b in zip(on[:-1], on[1:])] for x in (k, v))
    O, L, tol, l_tol = ragged_oracle.decode(q, K, V, 0.125, FP16)
    near(o, O, tol.nan_to_num(0), "o")
    near(lse, L, l_tol, "lse")
    assert (o[:2] == 0).all() and (o[2].isnan().all() if power == -132 else o[2].abs().max() > 0.01)
