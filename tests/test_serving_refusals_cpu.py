"""Refusals of the serving operators that guard the kernels against accesses they could not make: every
call fails its checks on the host (AR_ERR_INVALID with a message), so none reaches a device."""
from __future__ import annotations

import ctypes

import pytest

from attnrank import _native
from test_serving_operators_cpu import ADDRESS, APPEND, ATTENTION, ROTARY, append, attention, descriptors

lib = _native.lib


def rotary(change, status=None):
    a = {**ROTARY, **change}
    return lib.ar_rotary_positions(a["x"], a["xt"], a["xh"], a["out"], a["ot"], a["oh"], a["positions"], a["tokens"],
                                   a["heads"], a["head_dim"], a["rotary"], 0, 0, a["cos"], a["sin"], a["table"], status,
                                   a["dtype"], None)


def refused(code, message):
    text = lib.ar_last_error().decode()
    assert code == _native.AR_ERR_INVALID and message in text, (code, text)


@pytest.mark.parametrize("off", [1, 2, 3])
@pytest.mark.parametrize("name", ["positions", "cos", "sin"])
def test_rotary_arrays_of_32_bits_are_aligned(name, off):
    refused(rotary({name: ADDRESS + off}), "4-byte aligned")


@pytest.mark.parametrize("off", [1, 2, 3])
@pytest.mark.parametrize("name", ["offsets", "lengths", "table"])
def test_batch_arrays_are_aligned(name, off):
    for call in (append, attention):
        refused(call({name: ADDRESS + off}), "4-byte aligned")
    assert lib.ar_paged_attention_workspace(*descriptors({name: ADDRESS + off}), 28) == -1


@pytest.mark.parametrize("off", [1, 2, 3])
def test_status_words_and_lse_are_aligned(off):
    refused(rotary({}, status=ADDRESS + off), "device_status")
    a, (cache, batch) = APPEND, descriptors({})
    refused(lib.ar_paged_append(cache, batch, a["qkv"], a["qkv_stride"], None, a["heads"], a["q_out"], a["q_stride"], a["cos"],
                                a["sin"], a["positions"], a["rotary"], 0, ADDRESS + off, None), "device_status")
    a = ATTENTION
    for lse, status, message in ((ADDRESS + off, None, "lse"), (None, ADDRESS + off, "device_status")):
        refused(lib.ar_paged_attention(cache, batch, a["q"], a["q_stride"], a["heads"], a["scale"], a["window"], a["out"],
                                       a["out_stride"], lse, a["workspace"], a["bytes"], status, None), message)


def share_elements(tokens, token_stride, heads, head_stride, head_dim):
    seen = set()
    for t in range(tokens):
        for h in range(heads):
            row = range(t * token_stride + h * head_stride, t * token_stride + h * head_stride + head_dim)
            if not seen.isdisjoint(row):
                return True
            seen.update(row)
    return False


def test_rotary_output_rows_never_overlap():
    """Every stride pair of small shapes against the elements themselves: refused where two rows share
    one. The others fail a later check here (the status word), so that no call reaches a device."""
    outcomes = set()
    for head_dim in (2, 3, 5):
        for tokens in (1, 2, 3, 7):
            for heads in (1, 2, 3, 4):
                for ot in range(head_dim, 5 * head_dim + 2):
                    for oh in range(head_dim, 5 * head_dim + 2):
                        code = rotary(dict(tokens=tokens, heads=heads, head_dim=head_dim, rotary=2, ot=ot, oh=oh), status=ADDRESS + 1)
                        overlap = share_elements(tokens, ot, heads, oh, head_dim)
                        refused(code, "rows overlap" if overlap else "device_status")
                        outcomes.add(overlap)
    assert outcomes == {True, False}


@pytest.mark.parametrize("change", [dict(tokens=2**31 - 1, ot=2**62, oh=128), dict(tokens=2**31 - 1, ot=128, oh=2**62),
                                    dict(tokens=1, heads=65536, ot=0, oh=2**47)])
def test_large_strides_do_not_overflow_the_check(change):
    refused(rotary(change, status=ADDRESS + 1), "device_status")


def test_sequence_counts_whose_indexes_would_overflow_are_refused():
    for call in (append, attention):
        refused(call(dict(sequences=(1 << 30) + 1)), "2^30")
        refused(call(dict(sequences=2**31 - 1)), "2^30")
    assert lib.ar_paged_attention_workspace(*descriptors(dict(sequences=2**31 - 1)), 28) == -1
    assert lib.ar_paged_attention_workspace(*descriptors(dict(sequences=1 << 30)), 28) > 0


@pytest.mark.parametrize("heads,kv_heads,head_dim,most", [(28, 4, 128, 1), (32, 8, 128, 4096), (128, 1, 64, 7), (5, 5, 64, 300)])
def test_workspace_does_not_depend_on_the_batch_and_is_required_whole(heads, kv_heads, head_dim, most):
    """One size for any number of sequences and rows that reach the bound, and for its wider pools; a byte
    less, a misaligned address or none is refused."""
    shape = dict(kv_heads=kv_heads, head_dim=head_dim, most=most)
    sizes = {lib.ar_paged_attention_workspace(*descriptors({**shape, **more}), heads)
             for more in (dict(sequences=1, tokens=most), dict(sequences=500, tokens=5000), dict(sequences=500, tokens=5000, pages=99, stride=70))}
    assert len(sizes) == 1
    needed = sizes.pop()
    assert 0 < needed <= 64 << 20
    row = heads * head_dim
    call = dict(**shape, heads=heads, q_stride=row, out_stride=row, sequences=500, tokens=5000)
    refused(attention({**call, "bytes": needed - 1}), f"workspace of {needed} bytes")
    refused(attention({**call, "bytes": 0}), "workspace")
    refused(attention({**call, "workspace": ADDRESS + 8, "bytes": needed}), "workspace")
    refused(attention({**call, "workspace": None, "bytes": needed}), "workspace")
