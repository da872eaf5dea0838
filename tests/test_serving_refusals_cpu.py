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
