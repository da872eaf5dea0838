"""Offsets that decrease somewhere: the sequences they spoil are left out by the append, the others are
appended whole, however the search for a row's sequence is misled by them."""
from __future__ import annotations

import ctypes

import pytest

from test_serving_operators_gpu import SENTINEL, Paged, _lib, _stream

pytestmark = pytest.mark.gpu


def check_append(cuda, offsets, token_count, kv_lengths, valid, refused=(), heads=2):
    """Every sequence in `valid` is appended (no rotation: k, v and q are copies); other rows, and slots no
    valid sequence's new token owns, keep what they held. `refused` ones get a negative length."""
    import torch
    native = _lib()
    kv_heads, dim, page = 2, 64, 16
    paged = Paged(cuda, [(0, n) for n in kv_lengths], kv_heads, dim, page, "fp16", fill=False)
    paged.offsets = torch.tensor(offsets, dtype=torch.int32, device=cuda)
    paged.batch.q_offsets, paged.batch.token_count = paged.offsets.data_ptr(), token_count
    paged.batch.max_query_tokens = token_count
    for s in refused:
        paged.lengths[s] = -1
    qkv = torch.randn(token_count, (heads + 2 * kv_heads) * dim, generator=paged.generator, device=cuda).half()
    q = torch.full((token_count, heads * dim), SENTINEL, device=cuda, dtype=torch.float16)
    k_want, v_want, q_want = paged.k.clone(), paged.v.clone(), q.clone()
    for s in valid:
        begin, end = offsets[s], offsets[s + 1]
        for token in range(begin, end):
            position = kv_lengths[s] - (end - token)
            at, slot = int(paged.tables[s][position // page]), position % page
            row = qkv[token].view(-1, dim)
            q_want[token] = row[:heads].flatten()
            k_want[at, :, slot], v_want[at, :, slot] = row[heads:heads + kv_heads], row[heads + kv_heads:]
    native.check(native.lib.ar_paged_append(
        ctypes.byref(paged.cache), ctypes.byref(paged.batch), qkv.data_ptr(), qkv.shape[1], None, heads, q.data_ptr(),
        heads * dim, None, None, 0, 0, 0, paged.status.data_ptr(), _stream()))
    torch.cuda.synchronize()
    assert int(paged.status) == (4 if len(valid) < len(kv_lengths) else 0)
    assert torch.equal(q, q_want)
    for got, want in ((paged.k, k_want), (paged.v, v_want)):
        assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(), want.nan_to_num())


@pytest.mark.parametrize("offsets,tokens,valid", [
    ([0, 4, 100, 8, 12], 12, [0, 3]), ([0, 10, 3], 12, [0]), ([5, 6, 0, 4], 9, [0, 2]), ([7, 0, 3, 9, 5, 7], 8, [1, 4]),
    ([0, 3, -8, 4, 6], 6, [0, 3]), ([0, 2, 2, 5], 9, [0, 1, 2]), ([3, 3, 6], 9, [0, 1])])
@pytest.mark.parametrize("rows", [1, 60])
def test_append_of_the_sequences_that_are_in_range(cuda, offsets, tokens, valid, rows):
    """`rows` rows for each one of the case: both sizes of the kernel."""
    offsets = [rows * n for n in offsets]
    check_append(cuda, offsets, rows * tokens, [max(offsets) + 50 + 3 * s for s in range(len(offsets) - 1)], valid)


@pytest.mark.parametrize("at,value", [(500, 10**6), (500, -1), (1, 900), (31, 2000), (999, 10**6), (640, 3)])
def test_append_of_a_thousand_sequences_around_a_bad_offset(cuda, at, value):
    """Two rows a sequence; the bad offset spoils its two neighbours, and the search probes it or not."""
    offsets = [2 * s for s in range(1001)]
    offsets[at] = value
    in_range = [s for s in range(1000) if 0 <= offsets[s] <= offsets[s + 1] <= 2010]
    # a sequence that the bad offset stretches over others' rows is in range: its length is refused instead
    stretched = [s for s in in_range if offsets[s + 1] - offsets[s] != 2]
    check_append(cuda, offsets, 2010, [2 + s % 40 for s in range(1000)], [s for s in in_range if s not in stretched], stretched)
