"""Pieces over the cache whose offsets go back, leave rows out or leave the tensors, among more sequences than one look takes: the sequences that there are, and zeros beside them."""
import math

import pytest
import torch

from test_gpu_cache import BF16, FP16, INT8, filled
from test_gpu_cache_window import want
from test_gpu_ragged import near, offsets, rows

pytestmark = pytest.mark.gpu


def owned(cu, total):
    """(rows' start, length) of each sequence, None where it has none: offsets out of range or descending, or a start before the end of an earlier one that has rows."""
    end, got = 0, []
    for a, b in zip(cu[:-1], cu[1:]):
        ok = 0 <= a <= b <= total and (a == b or a >= end)
        got.append((a, b - a) if ok and b > a else None)
        end = max(end, b) if ok and b > a else end
    return got


def check(pkg, oracle, gpu, lens, cu, total, Hq, Hkv, D, dtype, kind, window=None, sinks=0):
    cache, table, K, V = filled(pkg, oracle, gpu, lens, 16, Hkv, D, dtype, kind)
    q, on = rows(total, Hq, D, dtype, gpu, 5), offsets(cu, gpu)
    o, lse = pkg.cache_attention(q, cache, table, offsets(lens, gpu), need_lse=True, cu=on, window=window, sinks=sinks)
    out = torch.full_like(q, 7.0)
    pkg.cache_attention(q, cache, table, offsets(lens, gpu), cu=on, window=window, sinks=sinks, out=out)
    of_none = torch.ones(total, dtype=torch.bool)
    for i, own in enumerate(owned(cu, total)):
        if own is None:
            continue
        at = slice(own[0], own[0] + own[1])
        of_none[at] = False
        O, L, tol, l_tol = want(oracle, q[at], [own[1]], [K[i]], [V[i]], D ** -0.5, dtype, window, sinks)
        near(o[at], O, tol, f"o of sequence {i}")
        near(lse[at], L, l_tol, f"lse of sequence {i}")
        assert torch.equal(out[at], o[at])
    assert of_none.any() and (o[of_none] == 0).all() and (lse[of_none] == -math.inf).all() and (out[of_none] == 7).all()


@pytest.mark.parametrize("window, sinks", [(None, 0), (20, 3)])
@pytest.mark.parametrize("n, Hq, Hkv, dtype, kind", [(40, 4, 2, BF16, BF16), (300, 2, 1, FP16, INT8), (700, 8, 1, BF16, INT8), (300, 20, 1, BF16, BF16)])
def test_offsets_at_random(pkg, ragged_oracle, gpu, n, Hq, Hkv, dtype, kind, window, sinks):
    g = torch.Generator().manual_seed(n)
    new = torch.randint(0, 5, (n,), generator=g).tolist()
    for i in range(7, n, 61):
        new[i] = 90
    cu = [3]
    for m in new:
        cu.append(cu[-1] + m)
    total = cu[-1] + 9
    lens = [m + int(torch.randint(0, 60, (1,), generator=g)) for m in new]
    for i in range(5, n, 13):          # back, ahead, out of range on either side
        cu[i] = (cu[i] - 30, cu[i] + 4, -1, total + 1)[i // 13 % 4]
    check(pkg, ragged_oracle, gpu, lens, cu, total, Hq, Hkv, 64, dtype, kind, window, sinks)


def test_rows_left_out(pkg, ragged_oracle, gpu):
    """In front of the first sequence and behind the last; where one goes back, and the next begins inside of an earlier one."""
    check(pkg, ragged_oracle, gpu, [40, 300, 70], [2, 22, 150, 150], 170, 4, 2, 128, BF16, BF16)
    check(pkg, ragged_oracle, gpu, [40, 300, 70], [0, 20, 10, 30], 40, 4, 2, 128, BF16, BF16)
