"""Waits of the paged attention kernels that run out end in status 3, not in a hang, and touch nothing
but the call's rows; the device works on. ar_paged_attention_wait_selftest stops loading at a chosen key
block (no fault is involved: the copies that the kernel waits for are simply not issued)."""
from __future__ import annotations

import ctypes
import time

import pytest

from test_serving_operators_gpu import SENTINEL, Paged, _lib, _stream

pytestmark = pytest.mark.gpu

# about a dozen key blocks a CTA and several (sequence, KV head) ends in each
FEW = {"singles": [(1, 700 + 40 * i) for i in range(40)], "four drafted": [(4, 90 + 45 * i) for i in range(30)]}


def gives_up(paged, heads, blocks, window):
    """One call whose waits run out: status 3, only rows that a sequence owns are written. Its seconds."""
    import torch
    native = _lib()
    width = heads * paged.head_dim
    q = torch.randn(paged.tokens, width, generator=paged.generator, device=paged.device).to(paged.dtype)
    before = [x.clone() for x in (q, paged.k, paged.v)]
    out = torch.full((paged.tokens, width + 8), SENTINEL, device=paged.device, dtype=paged.dtype)
    lse = torch.full((paged.tokens, heads), SENTINEL, device=paged.device)
    needed = native.lib.ar_paged_attention_workspace(ctypes.byref(paged.cache), ctypes.byref(paged.batch), heads)
    workspace = torch.full((needed // 4 + 64,), SENTINEL, device=paged.device)
    paged.status.zero_()
    torch.cuda.synchronize()
    start = time.monotonic()
    native.check(native.lib.ar_paged_attention_wait_selftest(
        ctypes.byref(paged.cache), ctypes.byref(paged.batch), q.data_ptr(), width, heads, window, out.data_ptr(), width + 8,
        lse.data_ptr(), workspace.data_ptr(), needed, blocks, paged.status.data_ptr(), _stream()))
    torch.cuda.synchronize()
    elapsed = time.monotonic() - start
    assert int(paged.status) == 3
    assert (out[paged.rows:] == SENTINEL).all() and (out[:, width:] == SENTINEL).all() and (lse[paged.rows:] == SENTINEL).all()
    assert (workspace[needed // 4:] == SENTINEL).all()
    for x, y in zip((q, paged.k, paged.v), before):
        assert torch.equal(x.nan_to_num(), y.nan_to_num())
    return elapsed


def check_waits(cuda, sequences, heads, kv_heads, head_dim, page, window, name, choices):
    import torch
    paged = Paged(cuda, sequences, kv_heads, head_dim, page, name, extra_rows=3, window=window)
    q = torch.randn(paged.tokens, heads * head_dim, generator=paged.generator, device=cuda).to(paged.dtype)

    def call():
        out, lse = torch.full_like(q, SENTINEL), torch.full((paged.tokens, heads), SENTINEL, device=cuda)
        paged.status.zero_()
        paged.attention(q, heads, out, lse)
        torch.cuda.synchronize()
        assert int(paged.status) == 0
        return out, lse

    out, lse = call()
    for blocks in choices:
        elapsed = gives_up(paged, heads, blocks, window)
        # the CTAs, all resident, wait at the same time, each until its first wait runs out
        assert 0.4 < elapsed < 3.0, (blocks, elapsed)
        again, again_lse = call()
        assert torch.equal(again, out) and torch.equal(again_lse, lse), blocks


@pytest.mark.parametrize("blocks", [0, 1, 2, 5])
@pytest.mark.parametrize("name", sorted(FEW))
def test_few_row_waits_that_run_out(cuda, name, blocks):
    check_waits(cuda, FEW[name], 28, 4, 128, 16, 0, "fp16", [blocks])


def test_few_row_waits_that_run_out_at_64_with_a_window(cuda):
    check_waits(cuda, FEW["singles"], 8, 8, 64, 64, 300, "bf16", [2, 2])


CHUNKS = [(300, 4000), (512, 2500), (130, 130), (700, 1900), (64, 3000), (257, 300)]


@pytest.mark.parametrize("blocks", [0, 1, 2, 3, 5])
@pytest.mark.parametrize("heads,kv_heads,head_dim,page,window,name", [(28, 4, 128, 64, 0, "fp16"), (16, 16, 64, 16, 500, "bf16")])
def test_chunk_waits_that_run_out(cuda, heads, kv_heads, head_dim, page, window, name, blocks):
    """Part of a CTA's loads are under way, or none, when the MMA and softmax warps give up."""
    check_waits(cuda, CHUNKS, heads, kv_heads, head_dim, page, window, name, [blocks])


def test_both_forms_of_a_mixed_batch_run_out(cuda):
    """The few-row kernel's waits run out and then the chunk kernel's, one after the other."""
    check_waits(cuda, CHUNKS + FEW["singles"], 28, 4, 128, 16, 0, "bf16", [2])
