"""Many keys of little weight beside one that outweighs each of them by 2^25.5: together they are a
visible share of the row, which the 16-bit probabilities must not lose."""
from __future__ import annotations

import math

import pytest

from test_serving_operators_gpu import E, Paged, _half_step, _tiny

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("new", [1, 3, 64])
@pytest.mark.parametrize("name", ["fp16", "bf16"])
def test_small_weights_together(cuda, name, new):
    """Key 0 scores 0 and holds v = 0, all others score log2-units w = -25.5 and hold v = 1, so a row over n + 1
    keys is n 2^w / (1 + n 2^w). 64 sequences share the pages, so that a CTA goes over most of a row itself.

    Bound. A probability is rounded by u of it or half a subnormal of the type, t, where the reference is at
    2^-7 (fp16) of the largest weight or above: t 2^-7 a key, n of them. Its exponent has three fp32
    roundings of at most 26 (score, scale, reference), 26 * 3 e in log2 units, and the exponential 2^-21;
    the sums over n keys carry n e each, numerator and denominator; one more rounding of the result."""
    import torch
    heads, dim, cached, sequences = 8, 64, 131_072, 64
    paged = Paged(cuda, [(new, cached)] + [(new, new)] * (sequences - 1), heads, dim, 256, name, spare_pages=0)
    paged.table[1:] = paged.table[0]
    paged.lengths[1:] = cached
    paged.k.zero_()
    paged.k[..., 0] = -17.671875  # to the type; `score` is what it became
    score = float(paged.k[0, 0, 0, 0])
    at = int(paged.tables[0][0])
    paged.k[at, :, 0, 0] = 0.0
    paged.v.fill_(1.0)
    paged.v[at, :, 0] = 0.0
    q = torch.zeros(paged.tokens, heads, dim, device=cuda, dtype=paged.dtype)
    q[..., 0] = 1.0
    q = q.view(paged.tokens, heads * dim)
    out, lse = torch.empty_like(q), torch.empty(paged.tokens, heads, device=cuda)
    paged.attention(q, heads, out, lse, scale=1.0)
    torch.cuda.synchronize()
    assert int(paged.status) == 0
    n = torch.arange(cached - new, cached, device=cuda, dtype=torch.float64).repeat(sequences)[:, None]  # keys of weight 2^w
    weight = math.exp(score)
    want = n * weight / (1 + n * weight)
    u, tiny = _half_step(paged.dtype), _tiny(paged.dtype)
    below = 2.0 ** -7 if name == "fp16" else 1.0
    relative = math.log(2) * 3 * 26 * E + 2.0 ** -21 + n * E
    bound = n * tiny * below + (2 * relative + u) * want * 1.01 + u * want + tiny
    assert float(bound.max()) < 0.1 * float(want.min())  # far from losing them
    error = (out.double() - want).abs()
    assert float((error - bound).max()) <= 0, (float(error.max()), float(bound.max()))
    lse_want = torch.log2(1 + n * weight)
    # A running sum that holds key 0's weight rounds by e of the whole sum, so by more than a small weight's
    # own, at each addition: two a 64-key block in the form for few rows (sums of 2 probabilities), one a
    # 128-key block in the other, and at most 400 more inside a block and between lanes, warps and CTAs.
    # log2's own 2 ulp, and the reference, up to 7 in magnitude, is added to it.
    sums = (n / 32 + 400) * E * (1 + n * weight)
    excess = (lse.double() - lse_want).abs() - 1.45 * (relative * n * weight + sums) - 32 * E
    assert float(excess.max()) <= 0
