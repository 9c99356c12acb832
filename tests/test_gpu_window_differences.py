"""Gradients with a window against differences of the kernels' own forward.

The inputs lie on a grid of 2^-6 that fp16 holds, and are moved by h = 2^-6 along the signs of the gradient: every moved input is exact.  The loss is sum dout (o + rest), in 64 bits.  Its difference may be off by what
the forward's bounds allow for both of its ends, the gradient's product with the direction by the gradient's bounds (oracle/ragged_oracle.py); what the difference quotient itself leaves out, terms from h^3 on, is taken
from the formula in 64 bits at the same points."""
import pytest
import torch

from test_gpu_ragged import FP16, cu, offsets, rows

pytestmark = pytest.mark.gpu
H = 2.0 ** -6


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("lens, window, sinks", [([9, 30], 6, 2), ([150], 40, 0), ([70, 1, 33], 1, 1), ([40, 33], None, 0)])
def test_gradients_against_differences_of_the_forward(pkg, ragged_oracle, gpu, lens, window, sinks, D):
    at, n, heads = cu(lens), sum(lens), (4, 2, 2)
    x = [(rows(n, h, D, torch.float32, gpu, i) / H).round().mul(H).clamp(-8, 8) for i, h in enumerate(heads)]
    g, on, c = rows(n, 4, D, FP16, gpu, 9), offsets(at, gpu), D ** -0.5

    def forward(y):
        y = [t.to(FP16) for t in y]
        rest = torch.zeros_like(y[0])
        o, lse = pkg.ragged_fwd(*y, on, causal=True, rest=rest, window=window, sinks=sinks)
        O, _, tol, _ = ragged_oracle.ragged_fwd(*y, at, at, True, c, FP16, rest=True, window=window, sinks=sinks)
        G = g.double().cpu()
        return float(((o.double() + rest.double()).cpu() * G).sum()), float((O * G).sum()), float((tol * G.abs()).sum()), (o, lse, rest)

    _, _, _, (o, lse, rest) = forward(x)
    got = pkg.ragged_bwd(*(t.to(FP16) for t in x), o, lse, g, on, causal=True, rest=rest, window=window, sinks=sinks)
    want, tols = ragged_oracle.ragged_bwd(*(t.to(FP16) for t in x), g, at, at, True, c, FP16, rest=True, window=window, sinks=sinks)
    for i, name in enumerate(("dq", "dk", "dv")):
        d = want[i].sign()
        up, down = (forward([t + s * H * d.float().to(gpu) if j == i else t for j, t in enumerate(x)]) for s in (1, -1))
        left_out = abs((up[1] - down[1]) - 2 * H * float((want[i] * d).sum()))
        bound = up[2] + down[2] + left_out + 2 * H * float((tols[i] * d.abs()).sum())
        size = 2 * H * float((want[i] * d).sum())
        off = abs((up[0] - down[0]) - 2 * H * float((got[i].double().cpu() * d).sum()))
        assert off <= bound, (name, off, bound, size)
        assert name != "dv" or bound < 0.5 * size, (name, bound, size)          # (a gradient of another size would be found)
