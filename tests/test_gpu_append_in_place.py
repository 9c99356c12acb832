"""Queries turned in place, in a fused projection, and outputs that would lie over what other workgroups read."""
import pytest
import torch

from test_gpu_cache import BF16, INT8, empty, tables
from test_gpu_ragged import cu, offsets, rows

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", [BF16, INT8])
def test_in_place_in_a_fused_projection(pkg, gpu, kind):
    lens, new, page, D = [90, 200], [50, 7], 32, 64
    table, pages = tables(lens, page, gpu)
    a, b = (empty(pkg, pages, 2, page, D, kind, gpu) for _ in range(2))
    for c in (a, b):
        for x in (c.k, c.v, c.k_scale, c.v_scale):
            if x is not None:
                x.zero_()
    fused = rows(57, 8, D, BF16, gpu, 0)
    q, k, v = fused[:, :4], fused[:, 4:6], fused[:, 6:]
    freqs, on, n = 0.1 ** torch.arange(32, device=gpu), offsets(cu(new), gpu), offsets(lens, gpu)
    want = pkg.cache_append(a, q, k, v, table, n, on, freqs=freqs)
    refused = fused.clone()
    for out in (refused[:, 1:5], refused[:, 4:], refused[:, 2:6], refused.view(-1)[8:8 + 56 * 512].view(56, 8, D)[:, :4]):
        r = slice(0, out.shape[0])
        with pytest.raises(ValueError):
            pkg.cache_append(b, refused[r, :4], refused[r, 4:6], refused[r, 6:], table, n, on, freqs=freqs, out=out)
    assert torch.equal(refused, fused)
    kv = fused[:, 4:].clone()
    assert pkg.cache_append(b, q, k, v, table, n, on, freqs=freqs, out=q).data_ptr() == q.data_ptr()
    assert torch.equal(q, want) and torch.equal(fused[:, 4:], kv) and torch.equal(a.k, b.k) and torch.equal(a.v, b.v)
    # and over the queries once more
    o = pkg.cache_attention(q, b, table, n, cu=on)[0]
    with pytest.raises(ValueError):
        pkg.cache_attention(fused[:, :4], b, table, n, cu=on, out=fused[:, 1:5])
    assert torch.equal(pkg.cache_attention(q, b, table, n, cu=on, out=q)[0], o) and torch.equal(q, o)
