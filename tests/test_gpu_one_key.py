"""Gradients of rows that see one key: its weight is 1 whatever the score, so that dq is 0, and dk has nothing of the row.  (dv = dout, dP - delta = dout v - dout o = 0 in the formula.)"""
import pytest
import torch

from test_gpu_ragged import BF16, FP16, cu, near, offsets, rows
from test_gpu_window import both

pytestmark = pytest.mark.gpu


def seen(ql, kl, causal, window, sinks):
    """Keys that each packed row sees."""
    got = []
    for a, b in zip(ql, kl):
        for t in range(a):
            p = t + b - a
            got.append(b if not causal else 0 if p < 0 else p + 1 if window is None else p + 1 - max(0, p + 1 - window - sinks))
    return torch.tensor(got)


CASES = [([100, 1, 199], [100, 1, 199], True, None, 0), ([100, 1, 199], [100, 1, 199], True, 1, 0), ([100, 1, 199], [100, 1, 199], True, 1, 1), ([100, 1, 199], [100, 1, 199], True, 2, 0),
         ([100, 1, 199], [100, 1, 199], True, 50, 4), ([70, 40, 9], [50, 1, 200], True, None, 0), ([70, 40, 9], [50, 1, 200], True, 30, 2), ([70, 40, 9], [50, 1, 200], True, 1, 0),
         ([150, 3], [1, 7], False, None, 0), ([2300, 1200, 1300], [2300, 900, 1], True, 150, 2), ([1500], [1500], True, None, 0), ([300], [1], True, None, 0), ([1] * 150, [1] * 150, True, 3, 0)]


@pytest.mark.parametrize("D, dtype", [(64, BF16), (64, FP16), (128, BF16), (128, FP16)])
@pytest.mark.parametrize("Hq, Hkv", [(2, 1), (3, 3)])
@pytest.mark.parametrize("ql, kl, causal, window, sinks", CASES)
def test_rows_of_one_key_have_no_part_in_dq_and_dk(pkg, gpu, ql, kl, causal, window, sinks, Hq, Hkv, D, dtype):
    n, m = sum(ql), sum(kl)
    q, k, v, g = (rows(r, h, D, dtype, gpu, i) for i, (r, h) in enumerate(((n, Hq), (m, Hkv), (m, Hkv), (n, Hq))))
    on, rest = (offsets(cu(ql), gpu), offsets(cu(kl), gpu)), torch.zeros_like(q)
    o, lse = pkg.ragged_fwd(q, k, v, *on, causal=causal, rest=rest, window=window, sinks=sinks)
    grads = lambda dout: pkg.ragged_bwd(q, k, v, o, lse, dout, *on, causal=causal, rest=rest, window=window, sinks=sinks)
    dq, dk, dv = grads(g)
    count = seen(ql, kl, causal, window, sinks).to(gpu)
    one = count == 1
    assert one.any() and (dq[one] == 0).all() and (dq[count > 1].float().abs().amax((1, 2)) > 0).all()
    # whatever comes back to these rows: the others' dq, and dk, are the same bits
    other = g.clone()
    other[one] *= -300
    eq, ek, ev = grads(other)
    assert torch.equal(dq, eq) and torch.equal(dk, ek) and not torch.equal(dv, ev) and dk.isfinite().all()
    for i, (a, b) in enumerate(zip(ql, kl)):
        if b == 1 or (window == 1 and not sinks):
            assert (dk[cu(kl)[i]:cu(kl)[i + 1]] == 0).all()


def test_values_and_gradients_that_are_no_numbers_stay_that(pkg, gpu):
    """dS = P (dP - delta) of a row whose dout is NaN is NaN, one key or many."""
    q, k, v, g = (rows(40, h, 64, BF16, gpu, i) for i, h in enumerate((2, 1, 1, 2)))
    on = offsets([0, 40], gpu)
    o, lse = pkg.ragged_fwd(q, k, v, on, causal=True)
    g[0, 1] = float("nan")
    dq, dk, dv = pkg.ragged_bwd(q, k, v, o, lse, g, on, causal=True)
    assert dq[0, 1].isnan().all() and dk[0].isnan().all() and dv[0].isnan().all() and dq[0, 0].isfinite().all() and dq[1:].isfinite().all()


@pytest.mark.parametrize("D, dtype", [(64, FP16), (128, BF16)])
def test_against_the_formula(pkg, ragged_oracle, gpu, D, dtype):
    for ql, kl, causal, window, sinks in CASES:
        if causal and window and sum(ql) < 1000:
            both(pkg, ragged_oracle, gpu, ql, kl, 2, 1, D, dtype, window, sinks)
