"""Pages outside of the cache that some rows see: among the first keys, inside the window, beside keys that are hidden, in sequences that are cut.  NaN goes to the rows that see one, and to no other."""
import pytest
import torch

from test_gpu_cache import BF16, E4M3, FP16, INT8, filled
from test_gpu_cache_window import want
from test_gpu_ragged import cu, near, offsets, rows

pytestmark = pytest.mark.gpu


def check(pkg, oracle, gpu, lens, new, page, Hq, Hkv, D, dtype, kind, window, sinks, gone, single=False):
    """`gone`: (sequence, key whose page is not there)."""
    cache, table, K, V = filled(pkg, oracle, gpu, lens, page, Hkv, D, dtype, kind)
    q = rows(sum(new), Hq, D, dtype, gpu, 5)
    bad, hit = table.clone(), torch.zeros(sum(new), dtype=torch.bool)
    for n, (i, key) in enumerate(gone):
        bad[i, key // page] = (cache.pages, -1, 1 << 30, -(1 << 31))[n % 4]
        at = torch.arange(key // page * page, min(lens[i], (key // page + 1) * page))
        for t in range(new[i]):
            p = lens[i] - new[i] + t
            seen = at <= p if window is None else (at <= p) & ((at > p - window) | (at < sinks))
            hit[cu(new)[i] + t] |= bool(seen.any())
    o, lse = pkg.cache_attention(q, cache, bad, offsets(lens, gpu), need_lse=True, cu=None if single else offsets(cu(new), gpu), window=window, sinks=sinks)
    O, L, tol, l_tol = want(oracle, q, new, K, V, D ** -0.5, dtype, window, sinks)
    assert hit.any() and not hit.all(), "some rows and not all"
    assert o[hit].isnan().all() and lse[hit].isnan().all()
    near(o[~hit], O[~hit], tol[~hit], "o")
    near(lse[~hit], L[~hit], l_tol[~hit], "lse")


KINDS = [(BF16, BF16), (BF16, INT8), (FP16, E4M3)]
PIECES = [
    ([3000, 700], [200, 130], 16, 4, 2, 64, 300, 40, [(0, 2600)]),                    # some rows have passed it
    ([3000, 700], [200, 130], 16, 4, 2, 64, 300, 40, [(1, 0)]),                       # among the first keys: all rows of the one sequence
    ([3000, 700], [200, 130], 16, 4, 2, 128, 300, 20, [(0, 19), (1, 300)]),           # the last first key, whose neighbours are hidden
    ([700, 3000], [130, 200], 16, 4, 2, 128, 300, 20, [(0, 271), (1, 2990)]),         # where the first token's window begins; the last page
    ([9000, 40], [200, 40], 16, 2, 1, 64, None, 0, [(0, 8900)]),                      # cut along the keys
    ([9000, 40], [200, 40], 64, 2, 1, 64, 4000, 130, [(0, 4820), (1, 10)]),           # and with a window
    ([5000, 300], [8, 8], 16, 2, 1, 64, 6, 3, [(0, 4990)]),                           # few rows
    ([5000, 300], [8, 8], 16, 2, 1, 128, 3000, 3, [(0, 1999)]),                       # few rows, cut: all but the last one see it
    ([5000, 300], [8, 8], 32, 2, 1, 64, 3000, 40, [(0, 39)]),
    ([4996, 300], [8, 8], 16, 2, 1, 64, None, 0, [(0, 4992)]),
    ([5000, 300, 2000], [1, 90, 16], 16, 4, 4, 64, 1000, 20, [(0, 4500), (1, 250), (2, 1987)]),
]


@pytest.mark.parametrize("dtype, kind", KINDS)
@pytest.mark.parametrize("lens, new, page, Hq, Hkv, D, window, sinks, gone", PIECES)
def test_pieces(pkg, ragged_oracle, gpu, lens, new, page, Hq, Hkv, D, window, sinks, gone, dtype, kind):
    check(pkg, ragged_oracle, gpu, lens, new, page, Hq, Hkv, D, dtype, kind, window, sinks, gone)


@pytest.mark.parametrize("dtype, kind", KINDS)
@pytest.mark.parametrize("window, sinks, gone", [(3000, 4, [(0, 2500)]), (3000, 4, [(0, 3)]), (100, 4, [(1, 620)]), (100, 20, [(0, 19), (2, 0)]), (3000, 0, [(0, 1999), (3, 128)])])
def test_one_token(pkg, ragged_oracle, gpu, window, sinks, gone, dtype, kind):
    check(pkg, ragged_oracle, gpu, [5000, 700, 1, 129], [1] * 4, 16, 4, 2, 64, dtype, kind, window, sinks, gone, single=True)


@pytest.mark.parametrize("dtype, kind", KINDS)
def test_one_token_of_many_and_long_sequences(pkg, ragged_oracle, gpu, dtype, kind):
    """More sequences than a wavefront looks through, long ones cut: parts without a number are joined."""
    lens = [9000, 1, 5, 128, 4000] + [1 + (37 * i) % 190 for i in range(80)]
    check(pkg, ragged_oracle, gpu, lens, [1] * len(lens), 16, 4, 2, 64, dtype, kind, 3500, 4, [(0, 7000), (4, 2), (17, 0)], single=True)
