"""Pins of the oracle's windows and turns (no GPU): brute force over single keys, differences, complex numbers."""
import math

import pytest
import torch

BF16 = torch.bfloat16


def seen(t, j, lq, lk, window, sinks):
    p = t + lk - lq
    return j <= p and (j > p - window or j < sinks)


@pytest.mark.parametrize("lq, lk", [(1, 1), (7, 7), (3, 9), (9, 3)])
@pytest.mark.parametrize("window, sinks", [(1, 0), (2, 1), (3, 0), (5, 4), (100, 0), (1, 100)])
def test_windows_key_by_key(ragged_oracle, lq, lk, window, sinks):
    g = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn(n, 1, 8, generator=g, dtype=torch.float64) for n in (lq, lk, lk))
    o, lse, _, _ = ragged_oracle.ragged_fwd(q, k, v, [0, lq], [0, lk], True, 0.3, BF16, window=window, sinks=sinks)
    for t in range(lq):
        w = {j: math.exp(0.3 * float(q[t, 0] @ k[j, 0])) for j in range(lk) if seen(t, j, lq, lk, window, sinks)}
        total = sum(w.values())
        assert float(lse[0, t]) == pytest.approx(math.log(total) if w else -math.inf, rel=1e-12)
        torch.testing.assert_close(o[t, 0], sum((x / total * v[j, 0] for j, x in w.items()), torch.zeros(8, dtype=torch.float64)), rtol=1e-12, atol=1e-12)


@pytest.mark.parametrize("window, sinks", [(1, 0), (3, 2)])
def test_windows_gradients_against_differences(ragged_oracle, window, sinks):
    g = torch.Generator().manual_seed(2)
    at, h = [0, 5, 5, 12], 1e-6
    x = [torch.randn(12, n, 4, generator=g, dtype=torch.float64) for n in (4, 2, 2)]
    do = torch.randn(12, 4, 4, generator=g, dtype=torch.float64)
    loss = lambda *x: float((ragged_oracle.ragged_fwd(*x, at, at, True, 0.7, BF16, window=window, sinks=sinks)[0] * do).sum())
    grads, _ = ragged_oracle.ragged_bwd(*x, do, at, at, True, 0.7, BF16, window=window, sinks=sinks)
    for i in range(3):
        way = torch.randn(x[i].shape, generator=g, dtype=torch.float64)
        up, down = (loss(*(y + s * h * way if j == i else y for j, y in enumerate(x))) for s in (1, -1))
        assert (up - down) / (2 * h) == pytest.approx(float((grads[i] * way).sum()), abs=1e-7)


@pytest.mark.parametrize("interleaved", [False, True])
def test_turns_are_products_of_complex_numbers(ragged_oracle, interleaved):
    g = torch.Generator().manual_seed(3)
    x, freqs, positions = torch.randn(6, 2, 16, generator=g), torch.rand(2, 4, generator=g), torch.randint(-9, 99, (6, 2), generator=g)
    y, far = ragged_oracle.turned(x, None, 0.0, positions, freqs, interleaved)
    a, b = (slice(0, 8, 2), slice(1, 8, 2)) if interleaved else (slice(0, 4), slice(4, 8))
    z = torch.complex(x[..., a].double(), x[..., b].double()) * torch.exp(1j * (positions.double() @ freqs.double()))[:, None]
    torch.testing.assert_close(torch.complex(y[..., a], y[..., b]), z, rtol=1e-12, atol=1e-12)
    assert torch.equal(y[..., 8:], x[..., 8:].double()) and (far[..., 8:] == 0).all() and (far[..., :8] > 0).all()
