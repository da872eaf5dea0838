"""Scores so large that fp32 holds them in steps of 16 log2 units: the running reference of a row must
follow each step, or the probabilities pass fp16's range."""
from __future__ import annotations

import math

import pytest

from test_serving_operators_gpu import Paged, _half_step

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("new", [1, 4, 100])
@pytest.mark.parametrize("name", ["fp16", "bf16"])
def test_scores_that_rise_in_steps_of_16(cuda, name, new):
    """Keys 128 g .. 128 g + 127 score 2^27 + 16 g log2 units (q . k = 2^20 + g / 8, exact in fp32, times a
    scale of 128 log2 units, whose fp32 product has steps of 16), so all but 2^-16 of a row's weight is on
    the last group, which holds v = 8; the others hold 0."""
    import torch
    heads, dim, cached, sequences = 8, 64, 1024, 40
    paged = Paged(cuda, [(new, cached)] * sequences, heads, dim, 128, name, spare_pages=0)
    group = torch.arange(cached, device=cuda) // 128
    key = torch.zeros(heads, cached, dim, device=cuda)
    key[..., 0], key[..., 1] = 1024.0, group / 8
    value = torch.zeros(heads, cached, dim, device=cuda)
    value[:, group == group.max()] = 8.0
    for ids in paged.tables:
        paged.write(paged.k, ids, key.to(paged.dtype))
        paged.write(paged.v, ids, value.to(paged.dtype))
    q = torch.zeros(paged.tokens, heads, dim, device=cuda, dtype=paged.dtype)
    q[..., 0], q[..., 1] = 1024.0, 1.0
    q = q.view(paged.tokens, heads * dim)
    out, lse = torch.empty_like(q), torch.empty(paged.tokens, heads, device=cuda)
    paged.attention(q, heads, out, lse, scale=128 * math.log(2))
    torch.cuda.synchronize()
    assert int(paged.status) == 0
    seen = cached - new + torch.arange(new, device=cuda).repeat(sequences) + 1  # keys of a row; the last group's among them
    last = (seen - (cached - 128)).double()[:, None]
    assert float(last.min()) >= 1
    # the groups before: 128 keys of 2^-16, 2^-32 .. each against one of weight 1; u of the result
    bound = 8.0 * (129 * 2.0 ** -16 / last + _half_step(paged.dtype) + 2.0 ** -18)
    assert float(((out.double() - 8.0).abs() - bound).max()) <= 0
    want = 2.0 ** 27 + 16 * 7 + torch.log2(last)
    assert float((lse.double() - want).abs().max()) <= 32  # two steps of fp32
