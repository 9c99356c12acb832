"""Attention over packed sequences, forward and gradients, against the oracle in 64 bits; bounds count roundings (oracle/ragged_oracle.py)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16


def cu(lens, first=0):
    return [first + sum(lens[:i]) for i in range(len(lens) + 1)]


def offsets(values, gpu):
    return torch.tensor(values, dtype=torch.int32, device=gpu)


def rows(n, heads, D, dtype, gpu, seed, size=1.0):
    g = torch.Generator().manual_seed(seed)
    return (size * torch.randn(n, heads, D, generator=g)).to(dtype).to(gpu)


def near(got, want, tol, what):
    got = got.double().cpu()
    same = (got == want) | (got.isnan() & want.isnan())
    off = torch.where(same, torch.zeros_like(want), (got - want).abs())
    bad = ~(off <= tol)
    at = tuple(int(i) for i in bad.nonzero()[0]) if bad.any() else ()
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, at {at}: {float(got[at])} for {float(want[at])}, bound {float(tol[at])}"


def both(pkg, oracle, gpu, ql, kl, Hq, Hkv, D, dtype, causal, scale=None, size=1.0, seed=0, backward=True):
    q, k, v = rows(sum(ql), Hq, D, dtype, gpu, seed, size), rows(sum(kl), Hkv, D, dtype, gpu, seed + 1, size), rows(sum(kl), Hkv, D, dtype, gpu, seed + 2)
    c = D ** -0.5 if scale is None else scale
    at = (cu(ql), cu(kl))
    on = [offsets(x, gpu) for x in at]
    o, lse = pkg.ragged_fwd(q, k, v, *on, causal=causal, sm_scale=scale)
    O, L, o_tol, l_tol = oracle.ragged_fwd(q, k, v, *at, causal, c, dtype)
    near(o, O, o_tol, "o")
    near(lse, L, l_tol, "lse")
    if not backward:
        return
    g = rows(sum(ql), Hq, D, dtype, gpu, seed + 3)
    got = pkg.ragged_bwd(q, k, v, o, lse, g, *on, causal=causal, sm_scale=scale)
    want, tols = oracle.ragged_bwd(q, k, v, g, *at, causal, c, dtype)
    for name, a, b, t in zip(("dq", "dk", "dv"), got, want, tols):
        near(a, b, t, name)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("lens", [[1], [33], [64], [65], [128], [129], [300], [1, 0, 63, 2, 200, 0, 127]])
def test_lengths(pkg, ragged_oracle, gpu, lens, causal, D, dtype):
    both(pkg, ragged_oracle, gpu, lens, lens, 4, 2, D, dtype, causal)


@pytest.mark.parametrize("Hq, Hkv", [(1, 1), (3, 3), (3, 1), (5, 1), (14, 2), (16, 1), (8, 4), (40, 8), (67, 1)])
def test_heads(pkg, ragged_oracle, gpu, Hq, Hkv):
    both(pkg, ragged_oracle, gpu, [70, 1, 150], [70, 1, 150], Hq, Hkv, 64, BF16, True)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("ql, kl", [([5], [300]), ([1, 1, 1], [1, 64, 129]), ([70, 3, 9], [10, 3, 200]), ([4, 0, 6], [0, 7, 5]), ([200], [131]), ([130, 40], [1, 0])])
@pytest.mark.parametrize("causal", [False, True])
def test_queries_and_keys_of_different_numbers(pkg, ragged_oracle, gpu, ql, kl, causal, D):
    both(pkg, ragged_oracle, gpu, ql, kl, 6, 2, D, BF16, causal)


def test_many_sequences(pkg, ragged_oracle, gpu):
    lens = [(7 * i * i) % 23 for i in range(150)]
    both(pkg, ragged_oracle, gpu, lens, lens, 2, 1, 64, FP16, True)


@pytest.mark.parametrize("n, D, longest", [(65, 128, (40, 3500)), (100, 64, (900, 5000)), (300, 128, (1500, 1500)), (1100, 64, (300, 300)), (1030, 128, (1, 2500))])
def test_many_sequences_and_a_long_one(pkg, ragged_oracle, gpu, n, D, longest):
    """More sequences than a wavefront, or the workgroup's first look, takes; the long one's tiles are cut where they are few."""
    g = torch.Generator().manual_seed(n)
    ql = torch.randint(0, 12, (n,), generator=g).tolist()
    kl = [x + i % 3 for i, x in enumerate(ql)]
    ql[n - 2], kl[n - 2] = longest
    both(pkg, ragged_oracle, gpu, ql, kl, 2, 1, D, BF16, n % 2 == 0)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("ql, kl", [([1], [9000]), ([3, 1, 0, 40], [700, 5000, 300, 1100]), ([1500], [1500]), ([900, 1300, 17], [900, 1300, 17]), ([600] + [1] * 70, [2000] + [3] * 70), ([1200, 64], [500, 1100])])
def test_few_tiles_that_are_cut(pkg, ragged_oracle, gpu, ql, kl, causal):
    """Fewer tiles than workgroups fit on the chip: long ones are cut along their keys, or rows, and joined."""
    both(pkg, ragged_oracle, gpu, ql, kl, 2, 1, 64, BF16, causal)


def test_lengths_that_are_nearly_one(pkg, ragged_oracle, gpu):
    """The longest tiles first: as many of one length as sequences, lengths that differ by a step."""
    for lens in ([65, 64, 63, 129, 128, 127, 1, 193], [128] * 5, [300, 1, 300, 1, 299], [0, 0, 500, 0]):
        both(pkg, ragged_oracle, gpu, lens, lens, 3, 1, 64, BF16, True)
        both(pkg, ragged_oracle, gpu, lens, [n + 70 * (i % 3) for i, n in enumerate(lens)], 3, 1, 64, BF16, True)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("scale", [-0.2, 0.0, 1.0])
def test_scales(pkg, ragged_oracle, gpu, scale, dtype):
    both(pkg, ragged_oracle, gpu, [90, 200], [90, 200], 4, 2, 64, dtype, True, scale=scale)


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_scores_that_spread(pkg, ragged_oracle, gpu, dtype):
    """The running max moves late and often."""
    both(pkg, ragged_oracle, gpu, [257, 90], [257, 90], 4, 2, 128, dtype, True, size=6.0, backward=False)


def test_max_that_moves_in_the_last_tile(pkg, ragged_oracle, gpu):
    q, k, v = (rows(500, 2, 64, BF16, gpu, i) for i in range(3))
    k[450:] *= 20
    at = [0, 500]
    o, lse = pkg.ragged_fwd(q, k, v, offsets(at, gpu))
    O, L, o_tol, l_tol = ragged_oracle.ragged_fwd(q, k, v, at, at, False, 0.125, BF16)
    near(o, O, o_tol, "o")
    near(lse, L, l_tol, "lse")


def test_strides(pkg, ragged_oracle, gpu):
    """q, k and v as the projection's output has them, shared heads without a copy, a gradient that is broadcast, rows that are taken apart."""
    lens, Hq, Hkv, D = [50, 130], 6, 2, 64
    at = cu(lens)
    qkv = rows(180, Hq + 2 * Hkv, D, BF16, gpu, 5)
    q, k, v = qkv[:, :Hq], qkv[:, Hq:Hq + Hkv], qkv[:, Hq + Hkv:]
    on = offsets(at, gpu)
    want = pkg.ragged_fwd(q.clone(), k.clone(), v.clone(), on, causal=True)
    got = pkg.ragged_fwd(q, k, v, on, causal=True)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    shared = pkg.ragged_fwd(q, k[:, :1].expand(-1, 2, -1), v[:, :1].expand(-1, 2, -1), on, causal=True)
    assert torch.equal(shared[0], pkg.ragged_fwd(q, k[:, :1], v[:, :1], on, causal=True)[0])
    heads_first = q.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(pkg.ragged_fwd(heads_first, k, v, on, causal=True)[0], want[0])
    apart = torch.randn(180, Hkv, D, 2, device=gpu).to(BF16)[..., 0]
    assert torch.equal(pkg.ragged_fwd(q, apart, v, on)[0], pkg.ragged_fwd(q, apart.contiguous(), v, on)[0])
    g = torch.ones(1, 1, 1, dtype=BF16, device=gpu).expand(180, Hq, D)
    a = pkg.ragged_bwd(q, k, v, *want, g, on, causal=True)
    b = pkg.ragged_bwd(q.clone(), k.clone(), v.clone(), *want, g.contiguous(), on, causal=True)
    assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_rows_of_no_sequence(pkg, ragged_oracle, gpu):
    """In front of the first sequence and behind the last one: not read, whatever they hold; left alone in a given output, zeros in a new one."""
    lens, first = [40, 100], 7
    at, n = cu(lens, first), 7 + 140 + 9
    q, k, v, g = (rows(n, h, 128, BF16, gpu, i) for i, h in enumerate((4, 2, 2, 4)))
    outside = torch.ones(n, dtype=torch.bool, device=gpu)
    outside[7:147] = False
    for x in (q, k, v, g):
        x[outside] = math.nan
    on = offsets(at, gpu)
    o, lse = pkg.ragged_fwd(q, k, v, on, causal=True)
    assert (o[outside] == 0).all() and (lse[:, outside] == -math.inf).all()
    inside = [x[~outside] for x in (q, k, v, g)]
    O, L, o_tol, l_tol = ragged_oracle.ragged_fwd(*inside[:3], cu(lens), cu(lens), True, 128 ** -0.5, BF16)
    near(o[~outside], O, o_tol, "o")
    given = torch.full_like(q, 3.0)
    assert pkg.ragged_fwd(q, k, v, on, causal=True, out=given)[0] is given
    assert (given[outside] == 3).all() and torch.equal(given[~outside], o[~outside])
    grads = pkg.ragged_bwd(q, k, v, o, lse, g, on, causal=True)
    want, tols = ragged_oracle.ragged_bwd(*inside, cu(lens), cu(lens), True, 128 ** -0.5, BF16)
    for x, w, t in zip(grads, want, tols):
        assert (x[outside] == 0).all()
        near(x[~outside], w, t, "a gradient")


def test_no_sequences_and_no_rows(pkg, gpu):
    q, k = rows(5, 4, 64, BF16, gpu, 0), rows(3, 2, 64, BF16, gpu, 1)
    o, lse = pkg.ragged_fwd(q, k, k, offsets([0], gpu), offsets([0], gpu))
    assert (o == 0).all() and (lse == -math.inf).all()
    o, lse = pkg.ragged_fwd(q[:0], k, k, offsets([0, 0], gpu), offsets([0, 3], gpu))
    assert o.shape == (0, 4, 64)
    grads = pkg.ragged_bwd(q[:0], k, k, o, lse, q[:0], offsets([0, 0], gpu), offsets([0, 3], gpu))
    assert (grads[1] == 0).all() and (grads[2] == 0).all()
    o, lse = pkg.ragged_fwd(q, k[:0], k[:0], offsets([0, 5], gpu), offsets([0, 0], gpu))
    assert (o == 0).all() and (lse == -math.inf).all()
    grads = pkg.ragged_bwd(q, k[:0], k[:0], o, lse, q, offsets([0, 5], gpu), offsets([0, 0], gpu))
    assert (grads[0] == 0).all()


def test_offsets_that_do_not_ascend_within_the_tensors(pkg, gpu):
    """The kernels' own checks: such rows are not there, such keys make NaN; the other sequences are as ever."""
    q, k = rows(100, 4, 64, BF16, gpu, 0), rows(100, 2, 64, BF16, gpu, 1)
    good = pkg.ragged_fwd(q, k, k, offsets([0, 30, 100], gpu), causal=True)[0]
    out = torch.full_like(q, 3.0)
    pkg.ragged_fwd(q, k, k, offsets([0, 30, 101], gpu), offsets([0, 30, 100], gpu), causal=True, out=out)
    assert torch.equal(out[:30], good[:30]) and (out[30:] == 3).all()
    o, lse = pkg.ragged_fwd(q, k, k, offsets([0, 30, 100], gpu), offsets([0, 30, 1 << 30], gpu), causal=True)
    assert torch.equal(o[:30], good[:30]) and o[30:].isnan().all() and lse[:, 30:].isnan().all()
    o, _ = pkg.ragged_fwd(q, k, k, offsets([0, 30, 100], gpu), offsets([-5, 30, 20], gpu))
    assert o.isnan().all()
    grads = pkg.ragged_bwd(q, k, k, good, lse, q, offsets([0, 30, 100], gpu), offsets([-5, 30, 20], gpu))
    assert (grads[0] == 0).all()


@pytest.mark.parametrize("n", [40, 200, 1200])
def test_offsets_that_go_back(pkg, gpu, n):
    """0, 300, 0, 300, ...: every second sequence is the same one, the others are none; there are more tiles than the rows allow for."""
    q, k, g = rows(300, 4, 64, BF16, gpu, 0), rows(300, 2, 64, BF16, gpu, 1), rows(300, 4, 64, BF16, gpu, 2)
    on, once = offsets([300 * (i % 2) for i in range(n)], gpu), offsets([0, 300], gpu)
    o, lse = pkg.ragged_fwd(q, k, k, on)
    O, L = pkg.ragged_fwd(q, k, k, once)
    assert (o.float() - O.float()).abs().max() <= 2.0 ** -7 * O.float().abs().max() and (lse - L).abs().max() <= 1e-4      # (tiles cut in other parts: sums in another order)
    for x in pkg.ragged_bwd(q, k, k, O, L, g, on):
        assert x.isfinite().all()


def test_values_that_are_not_finite_stay_in_their_rows(pkg, gpu):
    """NaN in one sequence says nothing in another, and a masked score nothing at all."""
    q, k, v = (rows(200, 2, 64, BF16, gpu, i) for i in range(3))
    on = offsets([0, 100, 200], gpu)
    clean = pkg.ragged_fwd(q, k, v, on, causal=True)[0]
    k2, v2 = k.clone(), v.clone()
    k2[100:] = math.nan
    v2[100:] = math.inf
    o = pkg.ragged_fwd(q, k2, v2, on, causal=True)[0]
    assert torch.equal(o[:100], clean[:100]) and o[100:].isnan().all()
    k2 = k.clone()
    k2[60] = math.nan                # keys that a query does not see yet
    o = pkg.ragged_fwd(q, k2, v, on, causal=True)[0]
    assert torch.equal(o[:60], clean[:60]) and o[60:100].isnan().all() and torch.equal(o[100:], clean[100:])


def test_gradients_through_autograd(pkg, ragged_oracle, gpu):
    lens = [37, 90]
    at = cu(lens)
    leaves = [rows(127, h, 64, FP16, gpu, i).requires_grad_() for i, h in enumerate((6, 2, 2))]
    g = rows(127, 6, 64, FP16, gpu, 9)
    o = pkg.attention_ragged(*leaves, offsets(at, gpu), causal=True, softmax_scale=0.2)
    o.backward(g)
    want, tols = ragged_oracle.ragged_bwd(*(x.detach() for x in leaves), g, at, at, True, 0.2, FP16)
    for x, w, t in zip(leaves, want, tols):
        near(x.grad, w, t, "a gradient")
    plain = pkg.attention_ragged(*(x.detach() for x in leaves), offsets(at, gpu), causal=True, softmax_scale=0.2)
    assert torch.equal(o, plain) and not plain.requires_grad
    with pytest.raises(RuntimeError):
        a = torch.autograd.grad(pkg.attention_ragged(*leaves, offsets(at, gpu)), leaves[0], g.clone().requires_grad_(), create_graph=True)[0]
        torch.autograd.grad(a.sum(), leaves[1])


def test_gradients_of_a_sum_and_of_views(pkg, gpu):
    """A gradient without memory of its own (expanded from one element), and one that lies heads first."""
    on, x = offsets([0, 37, 90], gpu), [rows(90, h, 128, BF16, gpu, i) for i, h in enumerate((4, 2, 2))]
    grads = []
    for make in (lambda o: o.sum(), lambda o: (o * torch.ones_like(o)).sum(), lambda o: (o.transpose(0, 1) * torch.ones_like(o.transpose(0, 1).contiguous())).sum()):
        leaves = [t.clone().requires_grad_() for t in x]
        make(pkg.attention_ragged(*leaves, on, causal=True)).backward()
        grads.append([t.grad for t in leaves])
    assert all(torch.equal(a, b) for other in grads[1:] for a, b in zip(grads[0], other))
    assert all(t.abs().max() > 0 for t in grads[0][2:])


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("ql, kl, causal, size", [([5, 3, 20, 1, 130], [5, 3, 20, 1, 130], True, 1.0), ([300, 7], [300, 70], True, 4.0), ([40, 3], [4000, 2], False, 2.0)])
def test_what_rounding_left_off_o(pkg, ragged_oracle, gpu, ql, kl, causal, size, D, dtype):
    """o and the rest together are o in twice the bits, and gradients from both have that much of it; the last case's tiles are cut."""
    q, k, v, g = (rows(sum(n), h, D, dtype, gpu, i, s) for i, (n, h, s) in enumerate(((ql, 4, size), (kl, 2, 1.0), (kl, 2, 1.0), (ql, 4, 1.0))))
    at = (cu(ql), cu(kl))
    on, rest = [offsets(x, gpu) for x in at], torch.full_like(q, math.nan)
    o, lse = pkg.ragged_fwd(q, k, v, *on, causal=causal, rest=rest)
    same, _ = pkg.ragged_fwd(q, k, v, *on, causal=causal)
    assert torch.equal(o, same)
    O, _, tol, _ = ragged_oracle.ragged_fwd(q, k, v, *at, causal, D ** -0.5, dtype, rest=True)
    near(o.double() + rest.double(), O, tol, "o and the rest")
    got = pkg.ragged_bwd(q, k, v, o, lse, g, *on, causal=causal, rest=rest)
    want, tols = ragged_oracle.ragged_bwd(q, k, v, g, *at, causal, D ** -0.5, dtype, rest=True)
    for name, a, b, t in zip(("dq", "dk", "dv"), got, want, tols):
        near(a, b, t, name)
    leaves = [x.clone().requires_grad_() for x in (q, k, v)]
    pkg.attention_ragged(*leaves, *on, causal=causal).backward(g)
    assert all(torch.equal(x.grad, a) for x, a in zip(leaves, got))


def test_gradients_of_shared_and_of_frozen_tensors(pkg, gpu):
    """One tensor as key and value gets both gradients; heads shared by expansion their sum; a frozen one none."""
    q, k = rows(90, 4, 64, BF16, gpu, 0), rows(90, 1, 64, BF16, gpu, 1).requires_grad_()
    on, g = offsets([0, 90], gpu), rows(90, 4, 64, BF16, gpu, 2)
    pkg.attention_ragged(q, k, k, on, causal=True).backward(g)
    rest = torch.empty_like(q)
    o, lse = pkg.ragged_fwd(q, k.detach(), k.detach(), on, causal=True, rest=rest)
    _, dk, dv = pkg.ragged_bwd(q, k.detach(), k.detach(), o, lse, g, on, causal=True, rest=rest)
    assert torch.equal(k.grad, dk + dv) and q.grad is None
    k2 = k.detach().clone().requires_grad_()
    pkg.attention_ragged(q, k2.expand(-1, 2, -1), k.detach().expand(-1, 2, -1), on, causal=True).backward(g)
    # Two key heads of two query heads each: their gradients are rounded (half a step, 2^-8, of each: they may be far larger than their sum), their sum is, and the shared head's is.
    two = pkg.ragged_bwd(q, k.detach().expand(-1, 2, -1), k.detach().expand(-1, 2, -1), o, lse, g, on, causal=True, rest=rest)[1].double()
    assert ((k2.grad.double() - dk.double()).abs() <= 2.0 ** -8 * (1 + 2.0 ** -7) * (two.abs().sum(1, keepdim=True) + k2.grad.double().abs() + dk.double().abs()) + 1e-5).all()


def test_tangents_are_refused(pkg, gpu):
    q, at = rows(4, 2, 64, torch.bfloat16, gpu, 0), offsets([0, 4], gpu)
    with torch.autograd.forward_ad.dual_level():
        for i in range(3):
            x = [torch.autograd.forward_ad.make_dual(q, q) if i == j else q for j in range(3)]
            with pytest.raises((RuntimeError, NotImplementedError)):
                pkg.attention_ragged(*x, at)
        plain = pkg.attention_ragged(q, q, q, at)
    assert torch.equal(plain, pkg.attention_ragged(q, q, q, at))
    with pytest.raises((RuntimeError, NotImplementedError)):
        torch.func.jvp(lambda x: pkg.attention_ragged(x, q, q, at), (q,), (q,))


def test_same_results_every_time(pkg, gpu):
    q, k, v, g = (rows(1000, h, 128, BF16, gpu, i) for i, h in enumerate((8, 2, 2, 8)))
    on = offsets([0, 300, 301, 1000], gpu)
    o, lse = pkg.ragged_fwd(q, k, v, on, causal=True)
    first = pkg.ragged_bwd(q, k, v, o, lse, g, on, causal=True)
    for _ in range(5):
        again = pkg.ragged_fwd(q, k, v, on, causal=True)
        assert torch.equal(again[0], o) and torch.equal(again[1], lse)
        assert all(torch.equal(a, b) for a, b in zip(pkg.ragged_bwd(q, k, v, o, lse, g, on, causal=True), first))


def test_captured_calls_follow_their_offsets(pkg, gpu):
    q, k, v, g = (rows(400, h, 64, BF16, gpu, i) for i, h in enumerate((4, 2, 2, 4)))
    on = offsets([0, 100, 400], gpu)

    def step():
        o, lse = pkg.ragged_fwd(q, k, v, on, causal=True)
        return (o, lse, *pkg.ragged_bwd(q, k, v, o, lse, g, on, causal=True))

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        made = step()
    for at in ([0, 100, 400], [0, 399, 400], [0, 0, 250], [0, 100, 400]):
        on.copy_(offsets(at, gpu))
        graph.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in made]
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_another_stream(pkg, gpu):
    q, k, v = (rows(300, 4, 128, BF16, gpu, i) for i in range(3))
    on = offsets([0, 300], gpu)
    want = pkg.ragged_fwd(q, k, v, on, causal=True)[0]
    torch.cuda.synchronize()
    other = torch.cuda.Stream()
    with torch.cuda.stream(other):
        got = pkg.ragged_fwd(q, k, v, on, causal=True)[0]
    other.synchronize()
    assert torch.equal(got, want)


def test_rows_behind_32_bits(pkg, ragged_oracle, gpu):
    """Rows 4 MiB apart: 700 of them span more than 2^31 bytes (and elements)."""
    n, step = 1100, 1 << 21
    pool = torch.zeros(n * step, dtype=BF16, device=gpu)
    views = []
    for i, h in enumerate((4, 2, 2)):
        view = pool.as_strided((n, h, 64), (step, 64, 1), i * 1024)
        view.copy_(rows(n, h, 64, BF16, gpu, i))
        views.append(view)
    lens = [300, 800]
    on, at = offsets(cu(lens), gpu), cu(lens)
    want = pkg.ragged_fwd(*(x.contiguous() for x in views), on, causal=True)
    out = pool.as_strided((n, 4, 64), (step, 64, 1), 8192)
    got = pkg.ragged_fwd(*views, on, causal=True, out=out)
    assert torch.equal(out, want[0]) and torch.equal(got[1], want[1])
    g = rows(n, 4, 64, BF16, gpu, 7)
    a = pkg.ragged_bwd(*views, out, got[1], g, on, causal=True)
    b = pkg.ragged_bwd(*(x.contiguous() for x in views), want[0], want[1], g, on, causal=True)
    assert all(torch.equal(x, y) for x, y in zip(a, b))


def sequences(cu_q, cu_k, Tq, Tk):
    """What offsets of any kind stand for: (rows, keys) of each sequence that has rows, keys None where its offsets say none."""
    def apart(at, total):
        end, kept = 0, []
        for a, b in zip(at[:-1], at[1:]):
            good = 0 <= a <= b <= total and (a == b or a >= end)
            end = b if good and a < b else end
            kept.append((a, b) if good else None)
        return kept
    return [(r, c) for r, c in zip(apart(cu_q, Tq), apart(cu_k, Tk)) if r and r[0] < r[1]], apart(cu_k, Tk)


ODD_OFFSETS = [
    ([0, 100, 300, 0, 0], None), ([0, 30, 20], None), ([200, 30, 100], None), ([0, 100, 300, 50, 120, 300], None), ([-5, 30, 20, 40, 100], None), ([5] * 70 + [3, 60, 10, 90, 300], None),
    ([0, 300, 0, 300, 250, 290], None), ([0, 1 << 30, 50, 90, -(1 << 31), 200, 300], None), ([0, 100, 200, 300], [0, 250, 200, 300]), ([0, 100, 60, 200, 300], [0, 80, 80, 230, 300]),
    ([0, 10, 10, 20], [0, 300, 100, 300]), ([0, 299, 0, 1], [300, 0, 300, 0]),
]


@pytest.mark.parametrize("behind", [0, 150, 1200])
@pytest.mark.parametrize("cu_q, cu_k", ODD_OFFSETS)
def test_sequences_before_and_beside_odd_offsets(pkg, ragged_oracle, gpu, cu_q, cu_k, behind):
    """Whatever the other offsets are, no two sequences share a row or a key, and those that are apart have their values; `behind` more offsets of zero."""
    cu_q = cu_q + [0] * behind
    cu_k = cu_q if cu_k is None else cu_k + [0] * behind
    q, k, v, g = (rows(300, h, 64, BF16, gpu, i) for i, h in enumerate((4, 2, 2, 4)))
    held, keys = sequences(cu_q, cu_k, 300, 300)
    on = (offsets(cu_q, gpu), offsets(cu_k, gpu))
    o, lse = pkg.ragged_fwd(q, k, v, *on, causal=True)
    grads = pkg.ragged_bwd(q, k, v, o, lse, g, *on, causal=True)
    for _ in range(3):
        again = pkg.ragged_fwd(q, k, v, *on, causal=True)
        more = pkg.ragged_bwd(q, k, v, o, lse, g, *on, causal=True)
        for (a, b), c in held:
            assert torch.equal(again[0][a:b].nan_to_num(7), o[a:b].nan_to_num(7)) and torch.equal(again[1][:, a:b].nan_to_num(7), lse[:, a:b].nan_to_num(7)) and torch.equal(more[0][a:b], grads[0][a:b])
        for c in keys:
            if c:
                assert all(torch.equal(x[slice(*c)], y[slice(*c)]) for x, y in zip(more[1:], grads[1:]))
    for (a, b), c in held:
        if c is None:
            assert o[a:b].isnan().all() and lse[:, a:b].isnan().all() and (grads[0][a:b] == 0).all()
            continue
        part = (q[a:b], k[slice(*c)], v[slice(*c)])
        at = ([0, b - a], [0, c[1] - c[0]])
        O, L, o_tol, l_tol = ragged_oracle.ragged_fwd(*part, *at, True, 0.125, BF16)
        near(o[a:b], O, o_tol, f"o of {a} .. {b}")
        near(lse[:, a:b], L, l_tol, f"lse of {a} .. {b}")
        want, tols = ragged_oracle.ragged_bwd(*part, g[a:b], *at, True, 0.125, BF16)
        for x, (i, j), w, t in zip(grads, ((a, b), c, c), want, tols):
            near(x[i:j], w, t, f"a gradient of {i} .. {j}")


@pytest.mark.parametrize("n", [40, 200, 1200])
def test_gradients_of_offsets_that_go_back(pkg, ragged_oracle, gpu, n):
    """0, 300, 0, 300, ...: the sequence's gradients are those it has by itself."""
    q, k, g = rows(300, 4, 64, BF16, gpu, 0), rows(300, 2, 64, BF16, gpu, 1), rows(300, 4, 64, BF16, gpu, 2)
    o, lse = pkg.ragged_fwd(q, k, k, offsets([0, 300], gpu))
    got = pkg.ragged_bwd(q, k, k, o, lse, g, offsets([300 * (i % 2) for i in range(n)], gpu))
    want, tols = ragged_oracle.ragged_bwd(q, k, k, g, [0, 300], [0, 300], False, 0.125, BF16)
    for name, x, w, t in zip(("dq", "dk", "dv"), got, want, tols):
        near(x, w, t, name)


def fill_free_memory(*like):
    """The memory that the next tensors of these sizes get holds NaN."""
    torch.cuda.synchronize()
    kept = [torch.full_like(x, math.nan) for x in like for _ in range(4)]
    torch.cuda.synchronize()
    del kept


@pytest.mark.parametrize("behind", [0, 150])
@pytest.mark.parametrize("cu_q, cu_k", ODD_OFFSETS + [([0, 30, 100], [-5, 30, 20]), ([7, 40, 1000, 60, 61], [0, 0, 1, -1, 5])])
@pytest.mark.parametrize("group", [1, 3])
def test_rows_that_no_sequence_is_left_for(pkg, gpu, cu_q, cu_k, behind, group):
    """Between the sequences that there are, too: zeros, lse -inf, and gradients of zero, never what the memory held."""
    cu_q = cu_q + [0] * behind
    cu_k = cu_q if cu_k is None else cu_k + [0] * behind
    q, k, v, g = (rows(300, h, 128, BF16, gpu, i) for i, h in enumerate((2 * group, 2, 2, 2 * group)))
    held, keys = sequences(cu_q, cu_k, 300, 300)
    on = (offsets(cu_q, gpu), offsets(cu_k, gpu))
    none_q, none_k = torch.ones(300, dtype=torch.bool, device=gpu), torch.ones(300, dtype=torch.bool, device=gpu)
    for (a, b), _ in held:
        none_q[a:b] = False
    for c in keys:
        if c:
            none_k[slice(*c)] = False
    lse_like = torch.empty(2 * group, 300, device=gpu)
    fill_free_memory(q, lse_like)
    o, lse = pkg.ragged_fwd(q, k, v, *on)
    assert (o[none_q] == 0).all() and (lse[:, none_q] == -math.inf).all()
    fill_free_memory(q, k, v, lse_like)
    dq, dk, dv = pkg.ragged_bwd(q, k, v, o, lse, g, *on)
    assert (dq[none_q] == 0).all() and (dk[none_k] == 0).all() and (dv[none_k] == 0).all()
    assert all(x.isfinite().all() for x in (dq, dk, dv))
    out = torch.full_like(q, 3.0)
    pkg.ragged_fwd(q, k, v, *on, out=out)
    assert (out[none_q] == 3).all() and torch.equal(out[~none_q].nan_to_num(7), o[~none_q].nan_to_num(7))


@pytest.mark.parametrize("at", [[7, 47, 147], [0, 147, 100, 140], [0], [0, 156]])
def test_lse_beside_a_given_output(pkg, gpu, at):
    """lse is a new tensor, also where o is the caller's: -inf where there is no sequence."""
    q, k, v = (rows(156, h, 64, BF16, gpu, i) for i, h in enumerate((4, 2, 2)))
    on = offsets(at, gpu)
    want_o, want = pkg.ragged_fwd(q, k, v, on, causal=True)
    out = torch.full_like(q, 3.0)
    fill_free_memory(want)
    o, lse = pkg.ragged_fwd(q, k, v, on, causal=True, out=out)
    none = torch.ones(156, dtype=torch.bool, device=gpu)
    for (a, b), _ in sequences(at, at, 156, 156)[0]:
        none[a:b] = False
    assert o is out and torch.equal(lse, want) and (lse[:, none] == -math.inf).all()
    assert (out[none] == 3).all() and torch.equal(out[~none], want_o[~none])
    assert pkg.ragged_fwd(q, k, v, on, causal=True, out=out, need_lse=False)[1] is None and (out[none] == 3).all()


@pytest.mark.parametrize("ql, kl, Hq, Hkv, D, causal", [([5, 3, 20, 1, 130], [5, 3, 20, 1, 130], 4, 2, 64, True), ([700, 90], [700, 300], 2, 1, 128, True), ([40, 9], [5000, 12], 4, 1, 64, False),
                                                         ([3000], [3000], 1, 1, 128, True), ([200], [4096], 2, 2, 128, False)])
@pytest.mark.parametrize("power", [-12, -8, 10])
def test_gradients_scale_with_dout_in_fp16(pkg, gpu, ql, kl, Hq, Hkv, D, causal, power):
    """2^power times dout has 2^power times the gradients, to their own rounding (u = 2^-11, half of fp16's smallest step 2^-25) on both sides: dS has the range it needs wherever dout lies.
    Products and sums in fp32 scale exactly; an element of dS far below the largest of its row or key is rounded to 2^-33 of that one at most.  For dq the power of two is part of P's exponent,
    c s - lse + up in fp32, whose rounding goes by its size: dS moves by some 2^-20 of itself, so that where it lies next to a tie of fp16 the two sides round to neighbours, 2 u apart."""
    q, k, v = rows(sum(ql), Hq, D, FP16, gpu, 0), rows(sum(kl), Hkv, D, FP16, gpu, 1), rows(sum(kl), Hkv, D, FP16, gpu, 2)
    r = torch.Generator().manual_seed(3)
    g = ((1 + torch.randint(0, 4, q.shape, generator=r) / 4) * 2.0 ** torch.randint(-1, 1, q.shape, generator=r) * (2 * torch.randint(0, 2, q.shape, generator=r) - 1)).to(FP16).to(gpu)
    on, rest = [offsets(cu(x), gpu) for x in (ql, kl)], torch.empty_like(q)
    o, lse = pkg.ragged_fwd(q, k, v, *on, causal=causal, rest=rest)
    one = pkg.ragged_bwd(q, k, v, o, lse, g, *on, causal=causal, rest=rest)
    scaled = g * 2.0 ** power
    assert torch.equal(scaled.double(), g.double() * 2.0 ** power)
    other = pkg.ragged_bwd(q, k, v, o, lse, scaled, *on, causal=causal, rest=rest)
    flips = torch.zeros(q.shape, dtype=torch.float64, device=gpu)         # sum of |c dS K|
    for (a, b), (x, y) in zip(zip(cu(ql), cu(ql)[1:]), zip(cu(kl), cu(kl)[1:])):
        mask = torch.arange(y - x, device=gpu) <= torch.arange(b - a, device=gpu)[:, None] + (y - x - b + a) if causal else torch.ones(b - a, y - x, dtype=torch.bool, device=gpu)
        for h in range(Hq):
            Q, G, K, V = q[a:b, h].double(), g[a:b, h].double(), k[x:y, h * Hkv // Hq].double(), v[x:y, h * Hkv // Hq].double()
            P = torch.exp(D ** -0.5 * Q @ K.t().contiguous() - lse[h, a:b, None]) * mask
            flips[a:b, h] = D ** -0.5 * (P * (G @ V.t().contiguous() - (G * (P @ V)).sum(-1, keepdim=True))).abs() @ K.abs()
    most = 2 * float(g.double().norm(dim=2).max() * v.double().norm(dim=2).max()) * D ** -0.5      # of c dS
    for name, x, y, by, n in zip(("dq", "dk", "dv"), one, other, (k, q, g), (max(kl), max(ql) * Hq // Hkv, 0)):
        x, y = x.double(), y.double() * 2.0 ** -power
        assert y.isfinite().all(), name
        size = torch.maximum(x.abs(), y.abs()) * (1 + 2.0 ** -10)
        tol = 2 * 2.0 ** -11 * (size + (flips if name == "dq" else 0)) * (1 + 2.0 ** -8) + 2.0 ** -25 * (1 + 2.0 ** -power) + n * 2.0 ** -33 * most * float(by.abs().max())
        near(y, x.cpu(), tol.cpu(), name)


def gradients_and_their_roundings(q, k, v, g, c):
    """dq, dk, dv of one key head's sequence in 64 bits (rows of all its query heads together), and how far from them roundings of fp16 are: P and dS once each as operands of the last products
    and the result once, each by u = 2^-11 at most (the result by 2^-25 besides), independent of each other, so that their squares add up."""
    u = 2.0 ** -11
    s = c * q @ k.t()
    P = torch.exp(s - torch.logsumexp(s, -1, keepdim=True))
    dS = c * P * (g @ v.t() - (g * (P @ v)).sum(-1, keepdim=True))
    grads = dS @ k, dS.t() @ q, P.t() @ g
    far = (u * dS) ** 2 @ k ** 2, ((u * dS) ** 2).t() @ q ** 2, ((u * P) ** 2).t() @ g ** 2
    return grads, [f + (u * x) ** 2 + 2.0 ** -50 for f, x in zip(far, grads)]


def check_norms(pkg, gpu, Lq, Lk, D, size):
    """The errors' norm is their roundings', whose expectation is below that of `far`; three hundredths more than 1 are what sums in fp32 and the spread of a norm of thousands are."""
    q, k, v, g = rows(Lq, 2, D, FP16, gpu, 0), rows(Lk, 1, D, FP16, gpu, 1), rows(Lk, 1, D, FP16, gpu, 2), rows(Lq, 2, D, FP16, gpu, 3, size)
    leaves = [x.clone().requires_grad_() for x in (q, k, v)]
    pkg.attention_ragged(*leaves, offsets([0, Lq], gpu), offsets([0, Lk], gpu)).backward(g)
    one = lambda x: x.transpose(0, 1).reshape(-1, D).double()
    grads, far = gradients_and_their_roundings(one(q), one(k), one(v), one(g), D ** -0.5)
    for name, x, w, f in zip(("dq", "dk", "dv"), leaves, grads, far):
        off = float((one(x.grad) - w).norm())
        assert off <= 1.03 * float(f.sum().sqrt()), f"{name}: {off / float(w.norm())} of it, roundings {float(f.sum().sqrt()) / float(w.norm())}"


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("size", [2.0 ** 8, 1.0, 2.0 ** -10, 2.0 ** -13])
def test_fp16_gradients_over_many_keys(pkg, gpu, D, size):
    """P is about 2^-12, dout of any size."""
    check_norms(pkg, gpu, 300, 4096, D, size)


def test_fp16_gradients_of_weights_on_few_keys(pkg, gpu):
    """dS of more than fp16 holds, of which dq and dk are well within it: weights of about one half and dout of some thousands."""
    q, k, v = rows(6, 1, 64, FP16, gpu, 0), rows(2, 1, 64, FP16, gpu, 1, 2.0 ** -6), rows(2, 1, 64, FP16, gpu, 2, 8.0)
    q *= 2.0 ** -6
    g = rows(6, 1, 64, FP16, gpu, 3, 2.0 ** 12)
    on = [offsets([0, 6], gpu), offsets([0, 2], gpu)]
    leaves = [x.clone().requires_grad_() for x in (q, k, v)]
    pkg.attention_ragged(*leaves, *on).backward(g)
    one = lambda x: x[:, 0].double()
    grads, far = gradients_and_their_roundings(one(q), one(k), one(v), one(g), 0.125)
    c = (one(g) @ one(v).t()).abs().max()
    assert c > 65504 and grads[0].abs().max() < 65504
    for name, x, w, f in zip(("dq", "dk", "dv"), leaves, grads, far):
        assert x.grad.isfinite().all() and (one(x.grad) - w).norm() <= 2 * f.sum().sqrt(), name


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("keys", [30000, 262144])
def test_fp16_gradients_over_very_many_keys(pkg, gpu, keys, D):
    """P itself is below fp16's normal numbers."""
    check_norms(pkg, gpu, 32, keys, D, 2.0 ** 8)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_one_key_of_an_expanded_tensor(pkg, gpu, dtype, D):
    """A row without a stride of its own, whose infinite values are infinite: the rows of a step behind it are zeros, not the same row again."""
    q = rows(5, 4, D, dtype, gpu, 0)
    v = torch.ones(1, 2, D, dtype=dtype, device=gpu)
    v[:, :, 3] = math.inf
    one = lambda x: x[0].as_strided((1, 2, D), (0, D, 1))
    assert pkg.ragged.packed_ready(one(v)) and one(v).stride(0) == 0
    k = rows(1, 2, D, dtype, gpu, 1)
    on = (offsets([0, 5], gpu), offsets([0, 1], gpu))
    o, _ = pkg.ragged_fwd(q, one(k), one(v), *on)
    want, _ = pkg.ragged_fwd(q, k, v, *on)
    assert torch.equal(o, want) and (o[:, :, 3] == math.inf).all() and (o[:, :, 4:] == 1).all()


@pytest.mark.parametrize("seed", range(12))
def test_offsets_at_random(pkg, ragged_oracle, gpu, seed):
    """Any numbers as offsets, ascending for a while or not at all."""
    r = torch.Generator().manual_seed(seed)
    number = lambda lo, hi: int(torch.randint(lo, hi, (1,), generator=r))
    n = (3, 9, 70, 140, 300)[seed % 5]

    def some():
        at, x = [], number(-3, 20)
        for _ in range(n + 1):
            x = number(-20, 330) if number(0, 8) == 0 else x + number(0, 400 // n + 2)
            at.append(x)
        return at
    cu_q, cu_k = some(), some()
    q, k, v, g = (rows(300, h, 64, BF16, gpu, i) for i, h in enumerate((4, 2, 2, 4)))
    on = (offsets(cu_q, gpu), offsets(cu_k, gpu))
    fill_free_memory(q, k, torch.empty(4, 300, device=gpu))
    o, lse = pkg.ragged_fwd(q, k, v, *on, causal=True)
    grads = pkg.ragged_bwd(q, k, v, o, lse, g, *on, causal=True)
    O, O_tol, L, L_tol = torch.zeros(300, 4, 64, dtype=torch.float64), torch.zeros(300, 4, 64, dtype=torch.float64), torch.full((4, 300), -math.inf, dtype=torch.float64), torch.zeros(4, 300, dtype=torch.float64)
    want, tols = [[torch.zeros(x.shape, dtype=torch.float64) for x in (q, k, v)] for _ in range(2)]
    for (a, b), c in sequences(cu_q, cu_k, 300, 300)[0]:
        if c is None:
            O[a:b], L[:, a:b] = math.nan, math.nan
            continue
        part, at = (q[a:b], k[slice(*c)], v[slice(*c)]), ([0, b - a], [0, c[1] - c[0]])
        O[a:b], L[:, a:b], O_tol[a:b], L_tol[:, a:b] = ragged_oracle.ragged_fwd(*part, *at, True, 0.125, BF16)
        for i, (w, t) in enumerate(zip(*ragged_oracle.ragged_bwd(*part, g[a:b], *at, True, 0.125, BF16))):
            x = slice(*((a, b) if i == 0 else c))
            want[i][x], tols[i][x] = w, t
    near(o, O, O_tol, "o")
    near(lse, L, L_tol, "lse")
    for name, x, w, t in zip(("dq", "dk", "dv"), grads, want, tols):
        near(x, w, t, name)


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_a_captured_training_step(pkg, gpu, dtype):
    """Forward and gradients through autograd in a graph: inputs, gradients and offsets change between replays."""
    leaves = [rows(400, h, 64, dtype, gpu, i).requires_grad_() for i, h in enumerate((4, 2, 2))]
    g, on = rows(400, 4, 64, dtype, gpu, 9), offsets([0, 100, 400], gpu)

    def step():
        o = pkg.attention_ragged(*leaves, on, causal=True)
        return (o.detach(), *torch.autograd.grad(o, leaves, g))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        made = step()
    for i, at in enumerate(([0, 100, 400], [0, 399, 400], [0, 250, 0], [5, 100, 390])):
        on.copy_(offsets(at, gpu))
        g.copy_(rows(400, 4, 64, dtype, gpu, 20 + i, 2.0 ** (-4 * i)))
        with torch.no_grad():
            for x, h in zip(leaves, (4, 2, 2)):
                x.copy_(rows(400, h, 64, dtype, gpu, 30 + 3 * i + h))
        graph.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in made]
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        del want
