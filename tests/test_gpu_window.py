"""Attention over packed sequences where a query looks back on a window of keys and on the first ones, forward and gradients, against the oracle in 64 bits (bounds: oracle/ragged_oracle.py)."""
import math

import pytest
import torch

from test_gpu_ragged import BF16, FP16, cu, near, offsets, rows

pytestmark = pytest.mark.gpu


def both(pkg, oracle, gpu, ql, kl, Hq, Hkv, D, dtype, window, sinks, scale=None, size=1.0, seed=0, backward=True):
    q, k, v = rows(sum(ql), Hq, D, dtype, gpu, seed, size), rows(sum(kl), Hkv, D, dtype, gpu, seed + 1, size), rows(sum(kl), Hkv, D, dtype, gpu, seed + 2)
    c = D ** -0.5 if scale is None else scale
    at = (cu(ql), cu(kl))
    on, rest = [offsets(x, gpu) for x in at], torch.full_like(q, math.nan)
    o, lse = pkg.ragged_fwd(q, k, v, *on, causal=True, sm_scale=scale, rest=rest, window=window, sinks=sinks)
    O, L, o_tol, l_tol = oracle.ragged_fwd(q, k, v, *at, True, c, dtype, window=window, sinks=sinks)
    near(o, O, o_tol, "o")
    near(lse, L, l_tol, "lse")
    if not backward:
        return
    g = rows(sum(ql), Hq, D, dtype, gpu, seed + 3)
    got = pkg.ragged_bwd(q, k, v, o, lse, g, *on, causal=True, sm_scale=scale, rest=rest, window=window, sinks=sinks)
    want, tols = oracle.ragged_bwd(q, k, v, g, *at, True, c, dtype, rest=True, window=window, sinks=sinks)
    for name, a, b, t in zip(("dq", "dk", "dv"), got, want, tols):
        near(a, b, t, name)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("window, sinks", [(1, 0), (1, 1), (17, 0), (64, 4), (65, 64), (100, 65), (128, 130), (200, 1)])
@pytest.mark.parametrize("lens", [[1], [65], [129, 0, 64], [300, 1, 470]])
def test_windows(pkg, ragged_oracle, gpu, lens, window, sinks, D, dtype):
    both(pkg, ragged_oracle, gpu, lens, lens, 4, 2, D, dtype, window, sinks)


@pytest.mark.parametrize("Hq, Hkv", [(1, 1), (3, 1), (14, 2), (16, 1), (40, 8), (67, 1)])
def test_heads(pkg, ragged_oracle, gpu, Hq, Hkv):
    both(pkg, ragged_oracle, gpu, [70, 1, 250], [70, 1, 250], Hq, Hkv, 64, BF16, 90, 3)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("window, sinks", [(1, 0), (50, 4), (130, 70), (1000, 2)])
@pytest.mark.parametrize("ql, kl", [([5], [300]), ([1, 1, 1], [1, 64, 129]), ([70, 3, 9], [10, 3, 200]), ([4, 0, 6], [0, 7, 5]), ([200], [131]), ([130, 40], [700, 0])])
def test_queries_and_keys_of_different_numbers(pkg, ragged_oracle, gpu, ql, kl, window, sinks, D):
    both(pkg, ragged_oracle, gpu, ql, kl, 6, 2, D, BF16, window, sinks)


@pytest.mark.parametrize("ql, kl, window, sinks", [([1], [9000], 4000, 4), ([3, 1, 0, 40], [700, 5000, 300, 1100], 900, 100), ([1500], [1500], 1200, 1), ([2600], [2600], 130, 4), ([2600, 300], [2600, 300], 30, 140),
                                                   ([600] + [1] * 70, [2000] + [3] * 70, 1000, 0), ([1200, 64], [500, 1100], 700, 5)])
def test_tiles_that_are_cut(pkg, ragged_oracle, gpu, ql, kl, window, sinks):
    """Few tiles, and those of the first keys, which all rows see: cut along their keys, or rows, and joined."""
    both(pkg, ragged_oracle, gpu, ql, kl, 2, 1, 64, BF16, window, sinks)


@pytest.mark.parametrize("D, dtype", [(64, BF16), (64, FP16), (128, BF16), (128, FP16)])
@pytest.mark.parametrize("ql, kl, window, sinks", [([2200], [2200], 10, 1), ([1100, 60, 2500], [1100, 60, 2500], 40, 4), ([2300, 1200], [2600, 900], 150, 129), ([3000], [2000], 30, 260), ([4100], [4100], 1500, 128)])
def test_first_keys_in_pieces(pkg, ragged_oracle, gpu, ql, kl, window, sinks, D, dtype):
    """Tiles of first keys that all rows see, cut into pieces of 1024 rows and more."""
    both(pkg, ragged_oracle, gpu, ql, kl, 2, 1, D, dtype, window, sinks)


def test_first_keys_in_pieces_of_many_sequences(pkg, ragged_oracle, gpu):
    """Pieces that begin close to each other's ends, sequences of one piece and of none between, offsets that go back."""
    lens = [1030, 1, 0, 2050, 511, 512, 1024, 513, 3] + [7] * 70 + [1500]
    both(pkg, ragged_oracle, gpu, lens, lens, 2, 1, 64, BF16, 5, 2)
    n = sum(lens)
    q, k, v, g = (rows(n, h, 64, BF16, gpu, i) for i, h in enumerate((2, 1, 1, 2)))
    at = cu(lens)
    odd = at[:4] + [at[3] - 700, at[4]] + at[4:]           # one that begins inside of the one before, and the next one from there
    on, once = offsets(odd, gpu), offsets(at, gpu)
    o, lse = pkg.ragged_fwd(q, k, v, once, causal=True, window=5, sinks=2)
    a = pkg.ragged_bwd(q, k, v, o, lse, g, once, causal=True, window=5, sinks=2)
    b = pkg.ragged_bwd(q, k, v, o, lse, g, on, causal=True, window=5, sinks=2)
    keep = torch.ones(n, dtype=torch.bool, device=gpu)
    keep[at[3]:at[4]] = False
    for x, y in zip(a, b):
        assert torch.equal(x[keep], y[keep]) and y.isfinite().all()

@pytest.mark.parametrize("n", [150, 300, 1100])
def test_many_sequences(pkg, ragged_oracle, gpu, n):
    lens = [(7 * i * i) % 23 for i in range(n)]
    lens[n // 2] = 700
    both(pkg, ragged_oracle, gpu, lens, lens, 2, 1, 64, FP16, 9, 2)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("scale, size", [(-0.2, 1.0), (0.0, 1.0), (None, 6.0)])
def test_scales(pkg, ragged_oracle, gpu, scale, size, dtype):
    both(pkg, ragged_oracle, gpu, [90, 300], [90, 300], 4, 2, 128, dtype, 100, 4, scale=scale, size=size, backward=size == 1.0)


def test_hidden_scores_that_are_large(pkg, ragged_oracle, gpu):
    """Keys that have left the window score far above those in it: their exponentials, relative to what a row sees, have no number."""
    q, k, v, g = (rows(400, h, 64, BF16, gpu, i) for i, h in enumerate((4, 2, 2, 4)))
    k[10:60] *= 300
    at, on = [0, 400], offsets([0, 400], gpu)
    rest = torch.empty_like(q)
    o, lse = pkg.ragged_fwd(q, k, v, on, causal=True, rest=rest, window=80, sinks=3)
    keep = slice(60 + 80, 400)               # rows that see none of them
    O, L, tol, l_tol = ragged_oracle.ragged_fwd(q, k, v, at, at, True, 0.125, BF16, window=80, sinks=3)
    near(o[keep], O[keep], tol[keep], "o")
    near(lse[:, keep], L[:, keep], l_tol[:, keep], "lse")
    dq, dk, dv = pkg.ragged_bwd(q, k, v, o, lse, g, on, causal=True, rest=rest, window=80, sinks=3)
    want, tols = ragged_oracle.ragged_bwd(q, k, v, g, at, at, True, 0.125, BF16, rest=True, window=80, sinks=3)
    near(dq[keep], want[0][keep], tols[0][keep], "dq")
    near(dk[200:], want[1][200:], tols[1][200:], "dk")
    near(dv[200:], want[2][200:], tols[2][200:], "dv")
    assert all(x.isfinite().all() for x in (dq, dk, dv))


@pytest.mark.parametrize("D, dtype", [(64, FP16), (128, BF16)])
def test_one_key_to_a_row(pkg, gpu, D, dtype):
    """Its weight is 1: o is its value, dv its rows' gradients, and nothing depends on scores."""
    q, k, v, g = (rows(300, h, D, dtype, gpu, i) for i, h in enumerate((4, 2, 2, 4)))
    on = offsets([0, 100, 101, 300], gpu)
    rest = torch.empty_like(q)
    o, lse = pkg.ragged_fwd(q, k, v, on, causal=True, rest=rest, window=1)
    # (a weight of 1 to within fp32's exponential, 1e-5: the score, some 10, is rounded once more where the row's largest is taken off it)
    of = v.repeat_interleave(2, 1)
    assert torch.equal(o, of) and (rest.double().abs() <= 1e-5 * of.double().abs() + 2.0 ** -24).all()
    dq, dk, dv = pkg.ragged_bwd(q, k, v, o, lse, g, on, causal=True, rest=rest, window=1)
    want = g.double().reshape(300, 2, 2, D).sum(2)
    assert (dq == 0).all() and (dk == 0).all()
    # (such a weight as an operand and the result are rounded once each)
    u, size = torch.finfo(dtype).eps / 2, g.double().abs().reshape(300, 2, 2, D).sum(2)
    assert ((dv.double() - want).abs() <= u * want.abs() + (u + 1e-5) * size + 2.0 ** -24).all()


def test_a_window_that_hides_nothing(pkg, gpu):
    """As long as there are keys: the results of the call without it."""
    q, k, v, g = (rows(300, h, 128, BF16, gpu, i) for i, h in enumerate((4, 2, 2, 4)))
    on = offsets([0, 100, 300], gpu)
    o, lse = pkg.ragged_fwd(q, k, v, on, causal=True)
    grads = pkg.ragged_bwd(q, k, v, o, lse, g, on, causal=True)
    for window, sinks in ((300, 0), (1 << 40, 7), (5, 300), (5, 1 << 50)):
        O, L = pkg.ragged_fwd(q, k, v, on, causal=True, window=window, sinks=sinks)
        assert torch.equal(o, O) and torch.equal(lse, L)
        assert all(torch.equal(a, b) for a, b in zip(grads, pkg.ragged_bwd(q, k, v, o, lse, g, on, causal=True, window=window, sinks=sinks)))
    # longer than every sequence, though not than all keys together
    O, L = pkg.ragged_fwd(q, k, v, on, causal=True, window=200)
    assert (o.float() - O.float()).abs().max() <= 2.0 ** -7 * o.float().abs().max() and (lse - L).abs().max() <= 1e-5


def test_rows_of_no_sequence_and_offsets_that_go_back(pkg, gpu):
    q, k, v, g = (rows(200, h, 64, BF16, gpu, i) for i, h in enumerate((4, 2, 2, 4)))
    on = offsets([7, 100, 150], gpu)
    out = torch.full_like(q, 3.0)
    o, lse = pkg.ragged_fwd(q, k, v, on, causal=True, window=20, sinks=2)
    pkg.ragged_fwd(q, k, v, on, causal=True, window=20, sinks=2, out=out)
    inside = torch.zeros(200, dtype=torch.bool, device=gpu)
    inside[7:150] = True
    assert torch.equal(out[inside], o[inside]) and (out[~inside] == 3).all() and (o[~inside] == 0).all() and (lse[:, ~inside] == -math.inf).all()
    for x in pkg.ragged_bwd(q, k, v, o, lse, g, on, causal=True, window=20, sinks=2):
        assert (x[~inside] == 0).all() and x.isfinite().all()
    odd = offsets([0, 100, 50, 200, 201], gpu)       # the second is none, the third begins before the first one's end, the last leaves the tensors
    a, la = pkg.ragged_fwd(q, k, v, odd, causal=True, window=20, sinks=2)
    b, lb = pkg.ragged_fwd(q, k, v, offsets([0, 100], gpu), causal=True, window=20, sinks=2)
    assert torch.equal(a[:100], b[:100]) and torch.equal(la[:, :100], lb[:, :100]) and (a[100:] == 0).all()
    for x, y in zip(pkg.ragged_bwd(q, k, v, a, la, g, odd, causal=True, window=20, sinks=2), pkg.ragged_bwd(q, k, v, b, lb, g, offsets([0, 100], gpu), causal=True, window=20, sinks=2)):
        assert torch.equal(x, y)


def test_gradients_through_autograd(pkg, ragged_oracle, gpu):
    at = cu([37, 190])
    leaves = [rows(227, h, 64, FP16, gpu, i).requires_grad_() for i, h in enumerate((6, 2, 2))]
    g = rows(227, 6, 64, FP16, gpu, 9)
    o = pkg.attention_ragged(*leaves, offsets(at, gpu), causal=True, softmax_scale=0.2, window=40, sinks=2)
    o.backward(g)
    want, tols = ragged_oracle.ragged_bwd(*(x.detach() for x in leaves), g, at, at, True, 0.2, FP16, rest=True, window=40, sinks=2)
    for x, w, t in zip(leaves, want, tols):
        near(x.grad, w, t, "a gradient")
    assert torch.equal(o, pkg.attention_ragged(*(x.detach() for x in leaves), offsets(at, gpu), causal=True, softmax_scale=0.2, window=40, sinks=2))


def test_gradients_against_differences(pkg, ragged_oracle, gpu):
    """The oracle's formula, of which the kernels' gradients are tested above, against differences of its forward in 64 bits."""
    at = cu([9, 30])
    x = [torch.randn(39, h, 64, generator=torch.Generator().manual_seed(i), dtype=torch.float64) for i, h in enumerate((4, 2, 2))]
    g = torch.randn(39, 4, 64, generator=torch.Generator().manual_seed(9), dtype=torch.float64)
    of = lambda *y: float((ragged_oracle.ragged_fwd(*y, at, at, True, 0.125, BF16, window=6, sinks=2)[0] * g).sum())
    grads, _ = ragged_oracle.ragged_bwd(*x, g, at, at, True, 0.125, BF16, window=6, sinks=2)
    for i in range(3):
        d = torch.randn(x[i].shape, generator=torch.Generator().manual_seed(20 + i), dtype=torch.float64)
        up, down = ([y + (s * 1e-4 * d if j == i else 0) for j, y in enumerate(x)] for s in (1, -1))
        assert abs((of(*up) - of(*down)) / 2e-4 - float((grads[i] * d).sum())) <= 1e-5 * float((grads[i] * d).abs().sum())


def test_captured_calls_follow_their_offsets(pkg, gpu):
    q, k, v, g = (rows(400, h, 64, BF16, gpu, i) for i, h in enumerate((4, 2, 2, 4)))
    on = offsets([0, 100, 400], gpu)

    def step():
        o, lse = pkg.ragged_fwd(q, k, v, on, causal=True, window=50, sinks=4)
        return (o, lse, *pkg.ragged_bwd(q, k, v, o, lse, g, on, causal=True, window=50, sinks=4))

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        made = step()
    for values in ([0, 100, 400], [0, 399, 400], [0, 0, 250], [0, 200, 400]):
        on.copy_(offsets(values, gpu))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(made, step()))


def test_same_results_every_time(pkg, gpu):
    q, k, v, g = (rows(1500, h, 128, BF16, gpu, i) for i, h in enumerate((8, 2, 2, 8)))
    on = offsets([0, 300, 301, 1500], gpu)
    o, lse = pkg.ragged_fwd(q, k, v, on, causal=True, window=200, sinks=4)
    first = pkg.ragged_bwd(q, k, v, o, lse, g, on, causal=True, window=200, sinks=4)
    for _ in range(3):
        again = pkg.ragged_fwd(q, k, v, on, causal=True, window=200, sinks=4)
        assert torch.equal(again[0], o) and torch.equal(again[1], lse)
        assert all(torch.equal(a, b) for a, b in zip(pkg.ragged_bwd(q, k, v, o, lse, g, on, causal=True, window=200, sinks=4), first))
