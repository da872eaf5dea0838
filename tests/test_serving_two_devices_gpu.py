"""A call runs on the device that holds its arrays, whichever is current: every serving operator on a
second GPU's arrays and stream while the first one is current."""
from __future__ import annotations

import ctypes

import pytest

from test_serving_operators_gpu import E, Paged, _half_step, _lib, check_attention

pytestmark = pytest.mark.gpu


def test_arrays_on_another_device_than_the_current_one(cuda):
    import torch
    if torch.cuda.device_count() < 2:
        pytest.skip("needs two GPUs")
    native, other = _lib(), torch.device("cuda:1")
    heads, kv_heads, dim, page, positions = 14, 2, 128, 16, 512
    paged = Paged(other, [(1, 300), (40, 170), (3, 9)], kv_heads, dim, page, "fp16")
    stream = torch.cuda.Stream(device=other)
    cos, sin = (torch.empty(positions, dim // 2, device=other) for _ in range(2))
    qkv = torch.randn(paged.tokens, (heads + 2 * kv_heads) * dim, generator=paged.generator, device=other).half()
    q, turned = (torch.empty(paged.tokens, heads * dim, dtype=torch.float16, device=other) for _ in range(2))
    out, lse = torch.empty_like(q), torch.empty(paged.tokens, heads, device=other)
    workspace = torch.empty(64 << 20, dtype=torch.uint8, device=other)
    at = torch.cat([torch.arange(cached - new, cached) for new, cached in paged.sequences]).to(other, torch.int32)
    torch.cuda.synchronize(other)
    torch.cuda.set_device(0)
    scaling = native.RopeScalingStruct(1e4, dim, 0, 1.0, 0.0, 0.0, 0, 0.0)
    native.check(native.lib.ar_rope_table_scaled(ctypes.byref(scaling), positions, cos.data_ptr(), sin.data_ptr(), stream.cuda_stream))
    native.check(native.lib.ar_rotary_positions(
        qkv.data_ptr(), qkv.shape[1], dim, turned.data_ptr(), heads * dim, dim, at.data_ptr(), paged.tokens, heads, dim, dim, 0, 0,
        cos.data_ptr(), sin.data_ptr(), positions, paged.status.data_ptr(), 1, stream.cuda_stream))
    native.check(native.lib.ar_paged_append(
        ctypes.byref(paged.cache), ctypes.byref(paged.batch), qkv.data_ptr(), qkv.shape[1], None, heads, q.data_ptr(), heads * dim,
        cos.data_ptr(), sin.data_ptr(), positions, dim, 0, paged.status.data_ptr(), stream.cuda_stream))
    paged.attention(q, heads, out, lse, workspace=workspace, stream=stream.cuda_stream)
    assert torch.cuda.current_device() == 0
    torch.cuda.synchronize(other)
    assert int(paged.status) == 0
    assert torch.equal(q, turned)  # the same rotation of the same values
    angle = torch.outer(at.double(), 1e4 ** (-torch.arange(0, dim, 2, dtype=torch.float64, device=other) / dim))[:, None]
    a, b = (x.view(-1, heads, dim // 2).double() for x in qkv.view(paged.tokens, -1, 2, dim // 2)[:, :heads].unbind(2))
    want = torch.cat((a * angle.cos() - b * angle.sin(), b * angle.cos() + a * angle.sin()), dim=-1)
    size = torch.cat((a.abs() + b.abs(),) * 2, dim=-1)
    error = (q.view(-1, heads, dim).double() - want).abs()
    assert (error <= _half_step(torch.float16) * want.abs() + 8 * E * size + 2.0 ** -25).all()
    check_attention(paged, q, out, lse, heads)
