"""Pieces over a cache of 8 bits whose tokens' values differ by powers of ten: what a row does not see does not enter its result, nor its bound.

A row's weights as operands in fp16 are off by half a step: a relative u (in the oracle's bound) or, as subnormals, 2^-25 of the scale that they are relative to, which is one of the row's own keys'.  A code
has at most 448 (127), and that times the largest scale is the largest value that the row sees: 2^-25 of it for each of the row's keys, next to a sum of weights of 1 at least.  Products of a weight
with its scale and with the factor are rounded in fp32, once each, and so is the factor: 4 F32 of the values' weighted sum."""
import pytest
import torch

from test_gpu_cache import BF16, E4M3, FP16, INT8, empty, tables
from test_gpu_ragged import cu, near, offsets, rows

pytestmark = pytest.mark.gpu


def own(oracle, q, k, v, first, scale, dtype, window, sinks):
    """(o, bound) of the rows of one sequence, position `first` on, each from the keys that it sees alone."""
    got = []
    for t in range(q.shape[0]):
        j, p = torch.arange(first + t + 1), first + t
        seen = j if window is None else j[(j > p - window) | (j < sinks)]
        O, _, tol, _ = oracle.ragged_fwd(q[t:t + 1], k[seen], v[seen], [0, 1], [0, len(seen)], False, scale, dtype)
        size, _, _, _ = oracle.ragged_fwd(q[t:t + 1], k[seen], v[seen].abs(), [0, 1], [0, len(seen)], False, scale, dtype)
        got.append((O, tol + 4 * oracle.F32 * size + (2.0 ** -25 * len(seen) * v[seen].abs().max() if dtype == FP16 else 0.0)))
    return [torch.cat(x) for x in zip(*got)]


def check(pkg, oracle, gpu, lens, new, Hq, Hkv, D, dtype, kind, window, sinks, sizes, page=16):
    table, pages = tables(lens, page, gpu)
    cache = empty(pkg, pages, Hkv, page, D, kind, gpu)
    k = rows(sum(lens), Hkv, D, dtype, gpu, 0)
    v = torch.cat([rows(n, Hkv, D, torch.float32, gpu, 1 + i) * sizes(n)[:, None, None].to(gpu) for i, n in enumerate(lens)]).clamp(-6e4, 6e4).to(dtype)
    pkg.cache_write(cache, k, v, table, offsets(lens, gpu), offsets(cu(lens), gpu))
    q = rows(sum(new), Hq, D, dtype, gpu, 50)
    o, _ = pkg.cache_attention(q, cache, table, offsets(lens, gpu), cu=offsets(cu(new), gpu), window=window, sinks=sinks)
    held = [oracle.dequantise(*oracle.quantise(x.cpu(), kind)) for x in (k, v)]
    for i, (n, m) in enumerate(zip(lens, new)):
        of, at = slice(cu(lens)[i], cu(lens)[i + 1]), slice(cu(new)[i], cu(new)[i + 1])
        O, tol = own(oracle, q[at], held[0][of], held[1][of], n - m, D ** -0.5, dtype, window, sinks)
        near(o[at], O, tol, f"o of sequence {i}")


growing = lambda n: 10.0 ** torch.linspace(-4, 4, n)
mixed = lambda n: 10.0 ** (8 * torch.rand(n, generator=torch.Generator().manual_seed(n)) - 4)


@pytest.mark.parametrize("dtype, kind", [(FP16, E4M3), (FP16, INT8), (BF16, INT8)])
@pytest.mark.parametrize("window, sinks", [(None, 0), (20, 2)])
@pytest.mark.parametrize("sizes", [growing, mixed], ids=["growing", "mixed"])
@pytest.mark.parametrize("lens, new, Hq, Hkv, D", [([2, 8, 150], [2, 8, 4], 4, 2, 64), ([300, 16], [16, 16], 1, 1, 128), ([64, 90], [64, 70], 4, 2, 64), ([300, 33], [140, 33], 8, 2, 128)])
def test_values_of_all_sizes(pkg, ragged_oracle, gpu, lens, new, Hq, Hkv, D, sizes, window, sinks, kind, dtype):
    check(pkg, ragged_oracle, gpu, lens, new, Hq, Hkv, D, dtype, kind, window, sinks, sizes)


@pytest.mark.parametrize("kind", [E4M3, INT8])
@pytest.mark.parametrize("lens, new", [([4000], [16]), ([4000], [60])])
def test_values_of_all_sizes_in_parts(pkg, ragged_oracle, gpu, lens, new, kind):
    """Long ones, which are cut: parts of small values and of large ones are joined."""
    for sizes in (growing, mixed):
        check(pkg, ragged_oracle, gpu, lens, new, 1, 1, 64, FP16, kind, None, 0, sizes)


@pytest.mark.parametrize("kind", [E4M3, INT8])
@pytest.mark.parametrize("n, group", [(2, 1), (2, 8), (16, 1), (64, 1), (64, 4), (200, 2)])
def test_a_later_token_does_not_change_an_earlier_one(pkg, gpu, kind, n, group):
    """Values of 1e-4 beside ones of 3e4, of which the earlier tokens see none: 1e-4, to within its code's step and a rounding."""
    cache = pkg.KVCache.empty(8, 1, 64, 64, dtype=kind)
    v = torch.full((n, 1, 64), 3e4, dtype=FP16, device=gpu)
    v[:n // 2] = 1e-4
    table, lens, on = offsets([list(range(8))], gpu), offsets([n], gpu), offsets([0, n], gpu)
    pkg.cache_write(cache, torch.zeros_like(v), v, table, lens, on)
    o, _ = pkg.cache_attention(rows(n, group, 64, FP16, gpu, 0), cache, table, lens, cu=on)
    small, early = float(v[0, 0, 0]), o[:n // 2].double()
    assert ((early - small).abs() <= 2.0 ** -24 + 2.0 ** -11 * small + 2.0 ** -25 * n * small + 2.0 ** -20 * small).all()      # (fp16's subnormal step, the weights', fp32's sums)
