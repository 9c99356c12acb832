"""The CPU oracle of attention over packed sequences and a paged cache against torch's own attention, its autograd and differences."""
import math

import pytest
import torch

CASES = [([3, 1, 0, 5], [3, 1, 0, 5], True), ([3, 2, 4], [7, 2, 6], True), ([2, 5], [4, 1], False), ([4, 3], [2, 0], True)]


def _cu(lens):
    return [sum(lens[:i]) for i in range(len(lens) + 1)]


def _inputs(ql, kl, Hq=4, Hkv=2, D=8, seed=0):
    g = torch.Generator().manual_seed(seed)
    new = lambda n, h: torch.randn(n, h, D, generator=g, dtype=torch.float64)
    return new(sum(ql), Hq), new(sum(kl), Hkv), new(sum(kl), Hkv), new(sum(ql), Hq)


@pytest.mark.parametrize("ql, kl, causal", CASES)
def test_forward_is_softmax_attention(ragged_oracle, ql, kl, causal):
    q, k, v, _ = _inputs(ql, kl)
    o, lse, _, _ = ragged_oracle.ragged_fwd(q, k, v, _cu(ql), _cu(kl), causal, 0.3, torch.bfloat16)
    for a, b, c, d in zip(_cu(ql)[:-1], _cu(ql)[1:], _cu(kl)[:-1], _cu(kl)[1:]):
        for t in range(b - a):
            seen = (d - c) if not causal else max(0, min(d - c, t + 1 + (d - c) - (b - a)))
            for h in range(4):
                s = k[c:c + seen, h // 2] @ q[a + t, h] * 0.3
                if not seen:
                    assert (o[a + t, h] == 0).all() and lse[h, a + t] == -math.inf
                    continue
                torch.testing.assert_close(o[a + t, h], torch.softmax(s, 0) @ v[c:c + seen, h // 2])
                torch.testing.assert_close(lse[h, a + t], torch.logsumexp(s, 0))


@pytest.mark.parametrize("ql, kl, causal", CASES)
def test_gradients_are_those_of_differences(ragged_oracle, ql, kl, causal):
    q, k, v, g = _inputs(ql, kl, seed=1)
    loss = lambda q, k, v: (ragged_oracle.ragged_fwd(q, k, v, _cu(ql), _cu(kl), causal, 0.3, torch.bfloat16)[0] * g).sum()
    grads, _ = ragged_oracle.ragged_bwd(q, k, v, g, _cu(ql), _cu(kl), causal, 0.3, torch.bfloat16)
    xs = [q, k, v]
    for i in range(3):
        direction = torch.randn(xs[i].shape, generator=torch.Generator().manual_seed(i), dtype=torch.float64)
        step = lambda by: [x + by * direction if j == i else x for j, x in enumerate(xs)]
        by = 1e-5
        torch.testing.assert_close((grads[i] * direction).sum(), (loss(*step(by)) - loss(*step(-by))) / (2 * by), rtol=1e-7, atol=1e-8)


@pytest.mark.parametrize("kind", [torch.float8_e4m3fn, torch.int8])
def test_codes_stand_for_what_was_written(ragged_oracle, kind):
    x = torch.randn(50, 3, 16, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16)
    x[3] = 0
    x[5, 1, 2] = math.inf
    codes, scale = ragged_oracle.quantise(x, kind)
    y, x = ragged_oracle.dequantise(codes, scale), x.double()
    assert (y[3] == 0).all() and y[5, 1].isnan().all() and y[5, 0].isfinite().all()
    off, top = (y - x).abs(), x.abs().amax(-1, keepdim=True)
    # int8: half a step of top / 127; e4m3: half a step of a value, 2^-4 of it, or of the smallest, 2^-10 of top / 448; and the quotient's rounding
    far = top / 254 * (1 + 1e-4) if kind == torch.int8 else x.abs() * 2.0 ** -4 * (1 + 1e-5) + top / 448 * 2.0 ** -10
    good = x.isfinite().all(-1)
    assert (off <= far)[good].all()


def test_one_token_is_the_last_row_of_a_prompt(ragged_oracle):
    q, k, v, _ = _inputs([6], [6], seed=3)
    o, lse, _, _ = ragged_oracle.ragged_fwd(q, k, v, [0, 6], [0, 6], True, 0.3, torch.bfloat16)
    o1, lse1, _, _ = ragged_oracle.decode(q[5:], [k], [v], 0.3, torch.bfloat16)
    torch.testing.assert_close(o1[0], o[5])
    torch.testing.assert_close(lse1[0], lse[:, 5])
