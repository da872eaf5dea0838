"""Values of V that are not finite, behind a long cache: a row that does not see them is that of a clean
cache, bit for bit, and so are the other sequences of the batch; no wait inside the kernels runs out
while the rows that do see them are put right."""
from __future__ import annotations

import math

import pytest

from test_serving_operators_gpu import SENTINEL, Paged

pytestmark = pytest.mark.gpu

# sequences, window, position of the bad value from the end of sequence 0's cache
CASES = {
    "few, new token": ([(4, 131_072), (1, 9000), (3, 70)], 0, 3),
    "few, last token": ([(2, 100_001), (1, 9000)], 0, 1),
    "few, window's end": ([(6, 60_000), (1, 9000)], 30_000, 30_003),
    "few, seen by all": ([(4, 131_072), (1, 9000)], 0, 70_000),
    "chunk, new token": ([(512, 65_536), (300, 2000), (33, 5000)], 0, 200),
    "chunk, last token": ([(130, 131_072), (300, 2000)], 0, 1),
    "chunk, window's end": ([(400, 40_000), (300, 2000)], 20_000, 20_150),
    "chunk, seen by all": ([(300, 40_000), (300, 2000)], 0, 30_000),
}


@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("name", sorted(CASES))
def test_a_bad_value_behind_a_long_cache(cuda, name, bad):
    import torch
    sequences, window, back = CASES[name]
    heads, kv_heads, dim, page, column = 28, 4, 128, 64, 37
    paged = Paged(cuda, sequences, kv_heads, dim, page, "fp16", window=window)
    q = torch.randn(paged.tokens, heads * dim, generator=paged.generator, device=cuda).half()

    def call():
        out, lse = torch.full_like(q, SENTINEL), torch.full((paged.tokens, heads), SENTINEL, device=cuda)
        paged.attention(q, heads, out, lse)
        torch.cuda.synchronize()
        assert int(paged.status) == 0
        return out, lse

    clean, clean_lse = call()
    new, cached = sequences[0]
    at = cached - back
    paged.v[int(paged.tables[0][at // page]), :, at % page, column] = bad
    out, lse = call()
    position = torch.arange(cached - new, cached, device=cuda)
    sees = (position >= at) & (position - at < (window or cached))
    assert 0 < int(sees.sum())
    blind = torch.ones(paged.tokens, dtype=torch.bool, device=cuda)
    blind[:new] = ~sees
    assert torch.equal(lse, clean_lse)
    assert torch.equal(out[blind], clean[blind])
    rows, clean_rows = (x[~blind].view(-1, heads, dim) for x in (out, clean))
    assert not torch.isfinite(rows[..., column]).any()
    keep = [d for d in range(dim) if d != column]
    assert torch.equal(rows[..., keep], clean_rows[..., keep])
