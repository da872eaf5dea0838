"""Serving operators on a host without a GPU: the scaled rotary frequencies against their formulas in
64 bits, and every refusal of a bad argument (AR_ERR_INVALID with a message, before any device work).
No call here reaches a kernel."""
from __future__ import annotations

import ctypes
import math

import numpy as np
import pytest

from attnrank import _native

lib = _native.lib
F16, BF16 = _native.DTYPE_F16, _native.DTYPE_BF16
ADDRESS = 4096  # never dereferenced: each call below fails its checks first


def scaling(theta=10000.0, rotary_dim=128, kind=_native.ROPE_NONE, factor=1.0, low=1.0, high=4.0, original=8192,
            attention_factor=0.0):
    return _native.RopeScalingStruct(theta, rotary_dim, kind, factor, low, high, original, attention_factor)


def frequencies(s):
    out = np.zeros(max(s.rotary_dim // 2, 1), dtype=np.float64)
    multiplier = ctypes.c_double(0.0)
    _native.check(lib.ar_rope_frequencies(ctypes.byref(s), out.ctypes.data, ctypes.byref(multiplier)))
    return out, multiplier.value


def expected(s):
    """The header's formulas, one pair at a time."""
    r, theta = s.rotary_dim, float(s.theta)
    factor, low, high, window = float(s.factor), float(s.low), float(s.high), s.original_positions
    out = []
    for i in range(r // 2):
        f = theta ** (-2.0 * i / r)
        if s.kind == _native.ROPE_LINEAR:
            f = f / factor
        elif s.kind == _native.ROPE_BANDS:
            t = window * f / (2 * math.pi)
            m = (t - low) / (high - low)
            f = f / factor if t <= low else f if t >= high else m * f + (1 - m) * f / factor
        elif s.kind == _native.ROPE_YARN:
            def c(b):
                return r * math.log(window / (2 * math.pi * b)) / (2 * math.log(theta))
            a, b = max(math.floor(c(high)), 0), min(math.ceil(c(low)), r - 1)
            g = min(max((i - a) / max(b - a, 0.001), 0.0), 1.0)
            f = g * f / factor + (1 - g) * f
        out.append(f)
    multiplier = 0.1 * math.log(factor) + 1 if s.kind == _native.ROPE_YARN else 1.0
    return np.array(out), s.attention_factor or multiplier


@pytest.mark.parametrize("s", [
    scaling(), scaling(rotary_dim=2), scaling(theta=1e6, rotary_dim=512), scaling(rotary_dim=34, theta=1.5),
    scaling(kind=_native.ROPE_LINEAR, factor=4.0), scaling(kind=_native.ROPE_LINEAR, factor=1.0, attention_factor=0.5),
    scaling(theta=5e5, kind=_native.ROPE_BANDS, factor=8.0),
    scaling(theta=5e5, kind=_native.ROPE_BANDS, factor=8.0, original=1),
    scaling(theta=1e6, kind=_native.ROPE_YARN, factor=4.0, high=32.0, original=32768),
    scaling(theta=1e4, rotary_dim=64, kind=_native.ROPE_YARN, factor=40.0, high=32.0, original=4096, attention_factor=1.25),
    scaling(theta=1e4, rotary_dim=16, kind=_native.ROPE_YARN, factor=2.0, high=32.0, original=16),
], ids=lambda s: f"kind{s.kind}-r{s.rotary_dim}-s{s.factor:g}-L{s.original_positions}")
def test_frequencies_follow_their_formulas(s):
    got, multiplier = frequencies(s)
    want, want_multiplier = expected(s)
    # a handful of fp64 roundings (exp of up to 14 in magnitude loses four bits)
    np.testing.assert_allclose(got, want, rtol=1e-13)
    assert multiplier == pytest.approx(want_multiplier, rel=1e-13)


def test_multiplier_pointer_may_be_null():
    out = np.zeros(64)
    assert lib.ar_rope_frequencies(ctypes.byref(scaling()), out.ctypes.data, None) == _native.AR_OK
    assert out[0] == 1.0


BAD_SCALINGS = {
    "odd rotary_dim": (scaling(rotary_dim=63), "even"),
    "rotary_dim zero": (scaling(rotary_dim=0), "even"),
    "rotary_dim large": (scaling(rotary_dim=514), "even"),
    "theta one": (scaling(theta=1.0), "theta"),
    "theta nan": (scaling(theta=math.nan), "theta"),
    "theta infinite": (scaling(theta=math.inf), "theta"),
    "kind": (scaling(kind=4), "kind"),
    "kind negative": (scaling(kind=-1), "kind"),
    "factor below one": (scaling(kind=_native.ROPE_LINEAR, factor=0.5), "factor"),
    "factor nan": (scaling(kind=_native.ROPE_YARN, factor=math.nan), "factor"),
    "window": (scaling(kind=_native.ROPE_BANDS, original=0), "original_positions"),
    "bands reversed": (scaling(kind=_native.ROPE_BANDS, low=4.0, high=4.0), "low and high"),
    "bands low zero": (scaling(kind=_native.ROPE_YARN, low=0.0), "low and high"),
    "bands high infinite": (scaling(kind=_native.ROPE_YARN, high=math.inf), "low and high"),
    "attention factor": (scaling(attention_factor=-1.0), "attention_factor"),
}


@pytest.mark.parametrize("name", sorted(BAD_SCALINGS))
def test_bad_scalings_are_refused_by_both_entry_points(name):
    s, message = BAD_SCALINGS[name]
    out = np.zeros(512)
    for call in (lambda: lib.ar_rope_frequencies(ctypes.byref(s), out.ctypes.data, None),
                 lambda: lib.ar_rope_table_scaled(ctypes.byref(s), 16, ADDRESS, ADDRESS, None)):
        assert call() == _native.AR_ERR_INVALID
        assert message in lib.ar_last_error().decode()


TABLE = dict(positions=16, cos=ADDRESS, sin=ADDRESS)
BAD_TABLES = {
    "negative positions": (dict(positions=-1), "positions"),
    "too many positions": (dict(positions=(1 << 30) + 1), "positions"),
    "null cos": (dict(cos=None), "16-byte aligned"),
    "unaligned sin": (dict(sin=ADDRESS + 4), "16-byte aligned"),
}


@pytest.mark.parametrize("name", sorted(BAD_TABLES))
def test_rope_table_refusals(name):
    change, message = BAD_TABLES[name]
    a = {**TABLE, **change}
    assert lib.ar_rope_table_scaled(ctypes.byref(scaling()), a["positions"], a["cos"], a["sin"], None) == _native.AR_ERR_INVALID
    assert message in lib.ar_last_error().decode()
    assert lib.ar_rope_table_scaled(None, 16, ADDRESS, ADDRESS, None) == _native.AR_ERR_INVALID


ROTARY = dict(x=ADDRESS, xt=512, xh=128, out=2 * ADDRESS, ot=512, oh=128, positions=ADDRESS, tokens=3, heads=4, head_dim=128,
              rotary=64, cos=ADDRESS, sin=ADDRESS, table=16, dtype=F16)
BAD_ROTARY = {
    "fp32": (dict(dtype=0), "dtype"),
    "negative tokens": (dict(tokens=-1), "counts"),
    "negative heads": (dict(heads=-1), "counts"),
    "too many heads": (dict(heads=65537), "65536"),
    "negative table": (dict(table=-1), "counts"),
    "head_dim": (dict(head_dim=1025), "head_dim"),
    "odd rotary": (dict(rotary=63), "even"),
    "rotary beyond head": (dict(rotary=130), "even"),
    "rotary zero": (dict(rotary=0), "even"),
    "null x": (dict(x=None), "null"),
    "null out": (dict(out=None), "null"),
    "null positions": (dict(positions=None), "null"),
    "null tables": (dict(cos=None), "null"),
    "odd address": (dict(x=ADDRESS + 1), "aligned"),
    "negative stride": (dict(xt=-512), "negative"),
    "overlapping out heads": (dict(oh=64), "overlap"),
    "overlapping out tokens": (dict(ot=64), "overlap"),
    "in place with other strides": (dict(out=ADDRESS, ot=1024), "in place"),
}


@pytest.mark.parametrize("name", sorted(BAD_ROTARY))
def test_rotary_refusals(name):
    change, message = BAD_ROTARY[name]
    a = {**ROTARY, **change}
    status = lib.ar_rotary_positions(a["x"], a["xt"], a["xh"], a["out"], a["ot"], a["oh"], a["positions"], a["tokens"],
                                     a["heads"], a["head_dim"], a["rotary"], 0, 0, a["cos"], a["sin"], a["table"], None,
                                     a["dtype"], None)
    assert status == _native.AR_ERR_INVALID
    text = lib.ar_last_error().decode()
    assert message in text and "rotary_positions" in text


CACHE = dict(k=ADDRESS, v=ADDRESS, pages=10, page=16, kv_heads=4, head_dim=128, dtype=F16)
BATCH = dict(sequences=2, tokens=5, most=4, stride=3, offsets=ADDRESS, lengths=ADDRESS, table=ADDRESS)
APPEND = dict(qkv=ADDRESS, qkv_stride=36 * 128, bias=None, heads=28, q_out=2 * ADDRESS, q_stride=28 * 128, cos=ADDRESS,
              sin=ADDRESS, positions=64, rotary=128)
ATTENTION = dict(q=ADDRESS, q_stride=28 * 128, heads=28, scale=0.0, window=0, out=2 * ADDRESS, out_stride=28 * 128,
                 workspace=ADDRESS, bytes=64 << 20)


def descriptors(change):
    c = {**CACHE, **{k: v for k, v in change.items() if k in CACHE}}
    b = {**BATCH, **{k: v for k, v in change.items() if k in BATCH}}
    cache = _native.PagedCacheStruct(c["k"], c["v"], c["pages"], c["page"], c["kv_heads"], c["head_dim"], c["dtype"])
    batch = _native.PagedBatchStruct(b["sequences"], b["tokens"], b["most"], b["stride"], b["offsets"], b["lengths"], b["table"])
    return (None if change.get("cache", 1) is None else ctypes.byref(cache),
            None if change.get("batch", 1) is None else ctypes.byref(batch))


def append(change):
    a = {**APPEND, **change}
    cache, batch = descriptors(change)
    return lib.ar_paged_append(cache, batch, a["qkv"], a["qkv_stride"], a["bias"], a["heads"], a["q_out"], a["q_stride"],
                               a["cos"], a["sin"], a["positions"], a["rotary"], 0, None, None)


def attention(change):
    a = {**ATTENTION, **change}
    cache, batch = descriptors(change)
    return lib.ar_paged_attention(cache, batch, a["q"], a["q_stride"], a["heads"], a["scale"], a["window"], a["out"],
                                  a["out_stride"], None, a["workspace"], a["bytes"], None, None)


BAD_DESCRIPTORS = {
    "null cache": (dict(cache=None), "null cache"),
    "null batch": (dict(batch=None), "null batch"),
    "fp32 cache": (dict(dtype=0), "dtype"),
    "head_dim 96": (dict(head_dim=96), "head_dim"),
    "page of 8": (dict(page=8), "page_size"),
    "page of 24": (dict(page=24), "page_size"),
    "page of 2048": (dict(page=2048), "page_size"),
    "no kv heads": (dict(kv_heads=0), "kv_heads"),
    "no pages": (dict(pages=0), "page_count"),
    "pool of 2^31 rows": (dict(pages=1 << 25, page=16, kv_heads=4), "2^31 rows"),
    "null pages": (dict(v=None), "16-byte aligned"),
    "unaligned pages": (dict(k=ADDRESS + 8), "16-byte aligned"),
    "negative sequences": (dict(sequences=-1), "not be negative"),
    "negative tokens": (dict(tokens=-1), "not be negative"),
    "no query bound": (dict(most=0), "max_query_tokens"),
    "no table row": (dict(stride=0), "page_table_stride"),
    "null offsets": (dict(offsets=None), "null batch array"),
    "null lengths": (dict(lengths=None), "null batch array"),
    "null table": (dict(table=None), "null batch array"),
}


@pytest.mark.parametrize("name", sorted(BAD_DESCRIPTORS))
def test_cache_and_batch_refusals_are_the_same_for_append_and_attention(name):
    change, message = BAD_DESCRIPTORS[name]
    for call, who in ((append, "paged_append"), (attention, "paged_attention")):
        assert call(change) == _native.AR_ERR_INVALID
        text = lib.ar_last_error().decode()
        assert message in text and who in text, text
    cache, batch = descriptors(change)
    assert lib.ar_paged_attention_workspace(cache, batch, 28) == -1


BAD_APPENDS = {
    "negative heads": (dict(heads=-1), "query_heads"),
    "short row": (dict(qkv_stride=35 * 128), "qkv_stride"),
    "odd stride": (dict(qkv_stride=36 * 128 + 4), "qkv_stride"),
    "rotary 24": (dict(rotary=24), "rotary_dim"),
    "rotary beyond head": (dict(rotary=144), "rotary_dim"),
    "negative table": (dict(positions=-1), "table_positions"),
    "null table": (dict(sin=None), "tables"),
    "unaligned table": (dict(cos=ADDRESS + 8), "tables"),
    "unaligned q_out": (dict(q_out=ADDRESS + 2), "q_out"),
    "short q_out": (dict(q_stride=27 * 128), "q_out_stride"),
    "in place with another stride": (dict(q_out=ADDRESS), "in place"),
    "null qkv": (dict(qkv=None), "qkv"),
    "unaligned qkv": (dict(qkv=ADDRESS + 8), "qkv"),
    "unaligned bias": (dict(bias=ADDRESS + 4), "bias"),
}


@pytest.mark.parametrize("name", sorted(BAD_APPENDS))
def test_append_refusals(name):
    change, message = BAD_APPENDS[name]
    assert append(change) == _native.AR_ERR_INVALID
    assert message in lib.ar_last_error().decode()


BAD_ATTENTIONS = {
    "heads not a multiple": (dict(heads=30), "multiple of kv_heads"),
    "no heads": (dict(heads=0), "multiple of kv_heads"),
    "group of 129": (dict(heads=129, kv_heads=1, q_stride=129 * 128, out_stride=129 * 128), "128 times"),
    "short q": (dict(q_stride=27 * 128), "q_stride"),
    "odd q stride": (dict(q_stride=28 * 128 + 4), "q_stride"),
    "short out": (dict(out_stride=27 * 128), "out_stride"),
    "negative scale": (dict(scale=-0.5), "scale"),
    "nan scale": (dict(scale=math.nan), "scale"),
    "scale beyond fp32 in log2": (dict(scale=3e38), "normal"),
    "subnormal scale": (dict(scale=1e-45), "normal"),
    "2^24 + 1 new tokens": (dict(most=(1 << 24) + 1, tokens=(1 << 24) + 1), "2^24"),
    "negative window": (dict(window=-1), "sliding_window"),
    "null q": (dict(q=None), "q and out"),
    "unaligned out": (dict(out=ADDRESS + 8), "q and out"),
    "in place": (dict(out=ADDRESS), "overlap"),
}


@pytest.mark.parametrize("name", sorted(BAD_ATTENTIONS))
def test_attention_refusals(name):
    change, message = BAD_ATTENTIONS[name]
    assert attention(change) == _native.AR_ERR_INVALID
    assert message in lib.ar_last_error().decode()


def test_empty_calls_succeed_without_a_device():
    """No tokens or no sequences: nothing to launch, so null buffers are fine."""
    assert append(dict(tokens=0, qkv=None)) == _native.AR_OK
    assert append(dict(sequences=0, offsets=None, lengths=None, table=None, qkv=None)) == _native.AR_OK
    assert attention(dict(tokens=0, q=None, out=None, workspace=None, bytes=0)) == _native.AR_OK
    assert lib.ar_rope_table_scaled(ctypes.byref(scaling()), 0, None, None, None) == _native.AR_OK
    assert lib.ar_rotary_positions(None, 0, 0, None, 0, 0, None, 0, 4, 128, 64, 0, 0, None, None, 0, None, F16, None) == _native.AR_OK


@pytest.mark.parametrize("heads,kv_heads,head_dim,most", [(28, 4, 128, 1), (32, 8, 128, 4096), (128, 1, 64, 7), (5, 5, 64, 300)])
def test_workspace_is_bounded_and_independent_of_the_batch(heads, kv_heads, head_dim, most):
    sizes = set()
    for sequences, tokens in ((1, most), (500, 5000)):
        cache, batch = descriptors(dict(kv_heads=kv_heads, head_dim=head_dim, most=most, sequences=sequences, tokens=tokens))
        sizes.add(lib.ar_paged_attention_workspace(cache, batch, heads))
    assert all(0 <= size <= 64 << 20 for size in sizes)


def test_structures_match_the_header_layout():
    """Field order and types of the serving operators' structures against their typedefs."""
    import re

    from test_library import HEADER, _c_declarations, _ctype_of, _same
    text = _c_declarations(HEADER.read_text())
    for c_name, structure in {"ar_rope_scaling": _native.RopeScalingStruct, "ar_paged_cache": _native.PagedCacheStruct,
                              "ar_paged_batch": _native.PagedBatchStruct}.items():
        body = re.search(r"typedef struct\s*\{([^}]*)\}\s*" + c_name + r"\s*;", text)
        fields = [f.strip() for f in body.group(1).split(";") if f.strip()]
        assert [f.split()[-1].lstrip("*") for f in fields] == [n for n, _ in structure._fields_], c_name
        for c_field, (field_name, ctype) in zip(fields, structure._fields_):
            assert _same(_ctype_of(c_field), ctype), f"{c_name}.{field_name}"
