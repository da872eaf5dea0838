"""Serving operators on a B200 against plain implementations in 64 bits: scaled rotary tables, rotary
positions, the append to a paged KV cache, the attention over it, and a run of them together.

Every tolerance is a bound derived from the arithmetic, written at the function that gives it, with
u = torch.finfo(type).eps / 2 for one rounding to the type and e = 2^-24 for one fp32 rounding. Slots
and pages that no position owns hold NaN, page-table entries no position needs hold numbers outside
the pool, and rows no sequence owns hold a sentinel that must survive.
"""
from __future__ import annotations

import ctypes
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
SENTINEL = 7.5


def _lib():
    from attnrank import _native
    return _native


def _types(name):
    import torch
    return {"fp16": (torch.float16, 1), "bf16": (torch.bfloat16, 2)}[name]


def _stream():
    import torch
    return torch.cuda.current_stream().cuda_stream


def _half_step(dtype):
    import torch
    return torch.finfo(dtype).eps / 2


def _tiny(dtype):
    """Half of the smallest subnormal: what rounding adds near zero."""
    import torch
    info = torch.finfo(dtype)
    return info.tiny * info.eps / 2


def assert_within(got, want, bound, what=""):
    import torch
    got, want = got.double(), want.double()
    if got.numel() == 0:
        return
    assert torch.isfinite(got).all(), f"{what}: not finite"
    excess = (got - want).abs() - bound
    worst = excess.argmax()
    assert (excess <= 0).all(), (f"{what}: {int((excess > 0).sum())} of {excess.numel()} outside; worst got "
                                 f"{got.flatten()[worst]:.8g} want {want.flatten()[worst]:.8g} bound "
                                 f"{torch.as_tensor(bound).expand_as(want).flatten()[worst]:.3g}")


# ------------------------------------------------------------------------------------------ tables
@pytest.mark.parametrize("kind,rotary,positions,theta,factor,high", [
    (0, 128, 1000, 1e4, 1.0, 4.0), (0, 2, 7, 1e6, 1.0, 4.0), (1, 34, 333, 1e4, 4.0, 4.0), (2, 128, 5000, 5e5, 8.0, 4.0),
    (3, 64, 100_003, 1e6, 4.0, 32.0), (3, 512, 129, 1e4, 40.0, 32.0), (0, 6, 1, 1e4, 1.0, 4.0), (0, 2, 3_000_000, 1e4, 1.0, 4.0)])
def test_table(cuda, kind, rotary, positions, theta, factor, high):
    """The angle is p times an fp64 frequency in turns: relative error under 2^-50, so under p 2^-50
    turns; the remainder r of at most half a turn takes one fp32 rounding (pi e radians at most);
    sincospi and the product with the multiplier A two ulp each (4 e A), the multiplier's own rounding
    e A."""
    import torch
    native = _lib()
    s = native.RopeScalingStruct(theta, rotary, kind, factor, 1.0, high, 8192, 0.0)
    f, multiplier = np.zeros(rotary // 2), ctypes.c_double()
    native.check(native.lib.ar_rope_frequencies(ctypes.byref(s), f.ctypes.data, ctypes.byref(multiplier)))
    half = positions * (rotary // 2)  # the values behind the tables must survive
    cos, sin = torch.full((half + 8,), SENTINEL, device=cuda), torch.full((half + 8,), SENTINEL, device=cuda)
    native.check(native.lib.ar_rope_table_scaled(ctypes.byref(s), positions, cos.data_ptr(), sin.data_ptr(), _stream()))
    angle = torch.outer(torch.arange(positions, dtype=torch.float64, device=cuda), torch.from_numpy(f).to(cuda)).flatten()
    a = multiplier.value
    bound = a * (math.pi * E + 5 * E + 2 * math.pi * positions * 2.0 ** -50)
    assert_within(cos[:half], a * angle.cos(), bound, "cos")
    assert_within(sin[:half], a * angle.sin(), bound, "sin")
    assert (cos[half:] == SENTINEL).all() and (sin[half:] == SENTINEL).all()


def test_unscaled_table_agrees_with_the_existing_one(cuda):
    """ar_rope_table forms the angle in fp32: off by the product's rounding, p f e, and the frequency's
    own (about eight fp32 roundings of it through pow), so p f 9 e in all beside the functions' ulps."""
    import torch
    native = _lib()
    positions, rotary, theta = 600, 128, 1e6
    s = native.RopeScalingStruct(theta, rotary, 0, 1.0, 0.0, 0.0, 0, 0.0)
    new, old = (torch.empty(2, positions, rotary // 2, device=cuda) for _ in range(2))
    native.check(native.lib.ar_rope_table_scaled(ctypes.byref(s), positions, new[0].data_ptr(), new[1].data_ptr(), _stream()))
    native.check(native.lib.ar_rope_table(old[0].data_ptr(), old[1].data_ptr(), positions, rotary, theta, _stream()))
    f = theta ** (-torch.arange(0, rotary, 2, dtype=torch.float64, device=cuda) / rotary)
    angle = torch.outer(torch.arange(positions, dtype=torch.float64, device=cuda), f)
    assert_within(new, old, 9 * E * angle + 16 * E, "tables")


# ---------------------------------------------------------------------------------------- rotation
def rotate64(x, cos, sin, rotary, interleaved):
    """(rotated x, sum of the magnitudes of its two products) in 64 bits; cos, sin [tokens, rotary/2]."""
    import torch
    half = rotary // 2
    index = torch.arange(half, device=x.device)
    a_at, b_at = (2 * index, 2 * index + 1) if interleaved else (index, index + half)
    y, size = x.clone(), x.abs()
    c, s = cos[:, None], sin[:, None]
    a, b = x[..., a_at], x[..., b_at]
    y[..., a_at], y[..., b_at] = a * c - b * s, b * c + a * s
    size[..., a_at], size[..., b_at] = (a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs()
    return y, size


def rotation_bound(y, size, dtype):
    """Two products and a sum in fp32 (3 e of the products' magnitudes; a bias adds one more, 4 e), one
    rounding to the type."""
    u = _half_step(dtype)
    return u * y.abs() + (1 + u) * 4 * E * size + _tiny(dtype)


ROTARY_CASES = [  # tokens, heads, head_dim, rotary, interleaved, inverse, dtype, padding of x and out (elements)
    (1, 1, 128, 128, False, False, "fp16", 0), (1, 28, 128, 64, True, False, "bf16", 0), (33, 7, 64, 64, False, True, "bf16", 0),
    (300, 5, 80, 80, True, True, "fp16", 0), (300, 5, 80, 32, False, False, "fp16", 8), (17, 3, 96, 96, False, False, "bf16", 8),
    (17, 3, 96, 94, False, False, "fp16", 0), (17, 3, 96, 30, True, False, "fp16", 1), (9, 2, 7, 2, False, True, "bf16", 0),
    (9, 2, 7, 6, True, False, "fp16", 3), (5, 1, 1024, 1024, False, False, "fp16", 0), (2000, 40, 128, 128, False, False, "bf16", 0),
    (4100, 32, 128, 130 - 2, True, False, "fp16", 0), (2500, 9, 192, 66, False, False, "bf16", 0), (2, 2, 2, 2, True, False, "fp16", 0)]


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("tokens,heads,head_dim,rotary,interleaved,inverse,name,pad", ROTARY_CASES)
def test_rotary_positions(cuda, tokens, heads, head_dim, rotary, interleaved, inverse, name, pad, in_place):
    import torch
    native = _lib()
    dtype, code = _types(name)
    g = torch.Generator(device=cuda).manual_seed(tokens * 31 + head_dim + rotary)
    table = 2 * tokens + 50
    cos, sin = (torch.randn(table, rotary // 2, generator=g, device=cuda) for _ in range(2))
    positions = torch.randint(0, table, (tokens,), generator=g, device=cuda, dtype=torch.int32)
    row, token = head_dim + pad, heads * (head_dim + pad) + 3 * pad
    x = torch.full((tokens * token + 16,), SENTINEL, device=cuda, dtype=dtype)
    xs = x.as_strided((tokens, heads, head_dim), (token, row, 1))
    xs.copy_(torch.randn(tokens, heads, head_dim, generator=g, device=cuda))
    before = xs.clone()
    out = x if in_place else torch.full_like(x, SENTINEL)
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    native.check(native.lib.ar_rotary_positions(x.data_ptr(), token, row, out.data_ptr(), token, row, positions.data_ptr(),
                                                tokens, heads, head_dim, rotary, interleaved, inverse, cos.data_ptr(),
                                                sin.data_ptr(), table, status.data_ptr(), code, _stream()))
    at = positions.long()
    sign = -1.0 if inverse else 1.0
    want, size = rotate64(before.double(), cos.double()[at], sign * sin.double()[at], rotary, interleaved)
    got = out.as_strided((tokens, heads, head_dim), (token, row, 1))
    assert_within(got, want, rotation_bound(want, size, dtype), "rotation")
    assert torch.equal(got[..., rotary:], before[..., rotary:])
    assert int(status) == 0
    got.fill_(SENTINEL)
    assert (out == SENTINEL).all(), "values between the rows were written"
    if not in_place:
        assert torch.equal(xs, before)


def test_rotary_gradient_is_the_inverse_rotation(cuda):
    """d/dx of sum(w . rotation(x)) is the inverse rotation of w: against the formula's gradient in 64
    bits, and against differences. The rotation is linear, so a difference quotient over a step of 1
    of an fp16 x whose values are multiples of 1/8 has only the roundings of its two outputs."""
    import torch
    native = _lib()
    tokens, heads, head_dim, rotary, table = 6, 3, 32, 16, 64
    g = torch.Generator(device=cuda).manual_seed(5)
    angle = 2 * math.pi * torch.rand(table, rotary // 2, generator=g, device=cuda, dtype=torch.float64)
    cos, sin = angle.cos().float(), angle.sin().float()
    positions = torch.randint(0, table, (tokens,), generator=g, device=cuda, dtype=torch.int32)

    def call(x, inverse, interleaved):
        out = torch.empty_like(x)
        native.check(native.lib.ar_rotary_positions(x.data_ptr(), heads * head_dim, head_dim, out.data_ptr(), heads * head_dim,
                                                    head_dim, positions.data_ptr(), tokens, heads, head_dim, rotary,
                                                    interleaved, inverse, cos.data_ptr(), sin.data_ptr(), table, None, 1,
                                                    _stream()))
        return out

    at = positions.long()
    for interleaved in (False, True):
        w = torch.randn(tokens, heads, head_dim, generator=g, device=cuda).half()
        x = torch.randint(-16, 17, w.shape, generator=g, device=cuda).half() / 8
        got = call(w, True, interleaved)
        leaf = x.double().requires_grad_()
        half = rotary // 2
        index = torch.arange(half, device=cuda)
        a_at, b_at = (2 * index, 2 * index + 1) if interleaved else (index, index + half)
        c, s = cos.double()[at][:, None], sin.double()[at][:, None]
        a, b = leaf[..., a_at], leaf[..., b_at]
        loss = ((a * c - b * s) * w.double()[..., a_at]).sum() + ((b * c + a * s) * w.double()[..., b_at]).sum()
        (loss + (leaf[..., rotary:] * w.double()[..., rotary:]).sum()).backward()
        _, size = rotate64(w.double(), cos.double()[at], -sin.double()[at], rotary, interleaved)
        assert_within(got, leaf.grad, rotation_bound(leaf.grad, size, torch.float16), "gradient")
        for column in (0, half, rotary - 1, rotary, head_dim - 1):
            step = torch.zeros_like(x)
            step[..., column] = 1.0
            up, down = call(x + step, False, interleaved).double(), call(x, False, interleaved).double()
            difference = ((up - down) * w.double()).sum(-1)
            # each output is off by u of it plus fp32's 4 e; x and x + 1 are exact in fp16
            slack = ((up.abs() + down.abs()) * (2.0 ** -11 + 8 * E) * w.double().abs()).sum(-1) * 1.01 + 1e-6
            bound = slack + 2.0 ** -11 * got[..., column].double().abs() + 8 * E * size[..., column]
            assert_within(difference, got[..., column].double(), bound, f"difference along {column}")


def test_rotary_position_outside_the_table_is_reported_and_left_out(cuda):
    import torch
    native = _lib()
    for pad in (0, 1):  # both forms of the kernel
        x = torch.randn(4, 2, 32 + pad, device=cuda).half()
        out = torch.full_like(x, SENTINEL)
        cos, sin = torch.ones(10, 16, device=cuda), torch.zeros(10, 16, device=cuda)
        positions = torch.tensor([3, 10, -1, 9], dtype=torch.int32, device=cuda)
        status = torch.zeros(1, dtype=torch.int32, device=cuda)
        native.check(native.lib.ar_rotary_positions(x.data_ptr(), 2 * (32 + pad), 32 + pad, out.data_ptr(), 2 * (32 + pad),
                                                    32 + pad, positions.data_ptr(), 4, 2, 32, 32, 0, 0, cos.data_ptr(),
                                                    sin.data_ptr(), 10, status.data_ptr(), 1, _stream()))
        assert int(status) == 2
        assert torch.equal(out[[0, 3], :, :32], x[[0, 3], :, :32]) and (out[[1, 2]] == SENTINEL).all()


# --------------------------------------------------------------------------------------- the cache
class Paged:
    """A paged cache and a batch over it: `sequences` is [(new tokens, cached tokens after the append)].
    Pages lie in random order behind `first_page`; what no position owns is NaN or out of range."""

    def __init__(self, device, sequences, kv_heads, head_dim, page, name, seed=0, extra_rows=0, spare_pages=3, window=0,
                 first_page=0, most=None, fill=True):
        import torch
        native = _lib()
        self.dtype, self.code = _types(name)
        self.device, self.sequences, self.page, self.window = device, sequences, page, window
        self.kv_heads, self.head_dim = kv_heads, head_dim
        g = torch.Generator(device="cpu").manual_seed(seed)
        counts = [-(-t // page) for _, t in sequences]
        total = sum(counts) + spare_pages
        order = (torch.randperm(total, generator=g) + first_page).int()
        width = max(counts + [1]) + 1
        self.tables = []
        table, at = torch.full((max(len(sequences), 1), width), -7, dtype=torch.int32), 0
        for s, ((new, cached), n) in enumerate(zip(sequences, counts)):
            ids = order[at:at + n]
            at += n
            self.tables.append(ids.long())
            # pages wholly before every new token's window are gone
            gone = max(0, cached - new - window + 1) // page if window else 0
            table[s, gone:n] = ids[gone:]
            if s % 2:
                table[s, :gone] = total + first_page + 12345
        self.pages = total + first_page
        shape = (self.pages, kv_heads, page, head_dim)
        if first_page:  # a large pool: only its end is used
            self.k, self.v = (torch.empty(shape, dtype=self.dtype, device=device) for _ in range(2))
            self.k[first_page:], self.v[first_page:] = math.nan, math.nan
        else:
            self.k, self.v = (torch.full(shape, math.nan, dtype=self.dtype, device=device) for _ in range(2))
        gd = torch.Generator(device=device).manual_seed(seed)
        self.generator = gd
        if fill:
            for (new, cached), ids in zip(sequences, self.tables):
                for pool in (self.k, self.v):
                    values = torch.randn(kv_heads, cached, head_dim, generator=gd, device=device).to(self.dtype)
                    self.write(pool, ids, values, window and max(0, cached - new - window + 1))
        offsets = np.concatenate([[0], np.cumsum([n for n, _ in sequences])]).astype(np.int32)
        self.rows = int(offsets[-1])
        self.tokens = self.rows + extra_rows
        self.offsets = torch.from_numpy(offsets).to(device)
        self.lengths = torch.tensor([t for _, t in sequences] or [0], dtype=torch.int32, device=device)
        self.table = table.to(device)
        self.status = torch.zeros(1, dtype=torch.int32, device=device)
        self.most = most if most is not None else max([n for n, _ in sequences] + [1])
        self.cache = native.PagedCacheStruct(self.k.data_ptr(), self.v.data_ptr(), self.pages, page, kv_heads, head_dim, self.code)
        self.batch = native.PagedBatchStruct(len(sequences), self.tokens, self.most, width, self.offsets.data_ptr(),
                                             self.lengths.data_ptr(), self.table.data_ptr())

    def write(self, pool, ids, values, first=0):
        """values [kv_heads, cached, head_dim] into their slots, from position `first` on."""
        cached = values.shape[1]
        for i, page in enumerate(ids.tolist()):
            lo, hi = max(i * self.page, first), min((i + 1) * self.page, cached)
            if lo < hi:
                pool[page, :, lo - i * self.page:hi - i * self.page] = values[:, lo:hi]

    def read(self, pool, s):
        """[kv_heads, cached, head_dim] of sequence s in 64 bits."""
        cached = self.sequences[s][1]
        ids = self.tables[s].to(self.device)
        return pool[ids].permute(1, 0, 2, 3).reshape(self.kv_heads, -1, self.head_dim)[:, :cached].double()

    def attention(self, q, heads, out, lse, scale=0.0, workspace=None, stream=None):
        import torch
        native = _lib()
        needed = native.lib.ar_paged_attention_workspace(ctypes.byref(self.cache), ctypes.byref(self.batch), heads)
        assert 0 <= needed <= 64 << 20
        if workspace is None:  # whatever an earlier call left there means nothing
            workspace = torch.full((needed // 4 + 4,), math.nan, device=self.device)
            self.workspace = workspace
        native.check(native.lib.ar_paged_attention(
            ctypes.byref(self.cache), ctypes.byref(self.batch), q.data_ptr(), q.stride(0), heads, scale, self.window,
            out.data_ptr(), out.stride(0), None if lse is None else lse.data_ptr(), workspace.data_ptr(), needed,
            self.status.data_ptr(), _stream() if stream is None else stream))


def attention64(q, k, v, position, window, scale, group, dtype):
    """Rows [n, heads, D] over k, v [kv_heads, cached, D] in 64 bits: (out, lse2, bound of out, bound of
    lse2). Masked positions do not enter, whatever they hold.

    Bounds. A score is a sum of D fp32 products of exact 16-bit values: off by at most
    (D + 2) e sum|q_d k_d|, times scale; its place in the exponent adds a few roundings of |w| and of
    the running maximum (8 e of the largest |w|). A weight's relative error d is that, twice (its own
    and the maximum's), the exponential's own error (2^-21), and the rescalings of the partial sums
    (2^-21 more). Numerator and denominator each carry d; n additions add n e. The probability is
    rounded to the type: u of it, or half a subnormal of the type where it is that small relative to
    the row's largest. The result takes one more rounding."""
    import torch
    u, tiny = _half_step(dtype), _tiny(dtype)
    n, heads, dim = q.shape
    if k.shape[1] == 0:  # nothing cached: one position that no row sees
        k, v = (x.new_zeros(x.shape[0], 1, dim) for x in (k, v))
    cached = k.shape[1]
    key = torch.arange(cached, device=q.device)
    seen = key <= position[:, None]
    if window:
        seen &= key > position[:, None] - window
    outs, sums, out_bounds, sum_bounds = [], [], [], []
    for h in range(heads):
        kh, vh = k[h // group], v[h // group]
        w = (scale * (q[:, h] @ torch.nan_to_num(kh, 0, 0, 0).T)).masked_fill(~seen, -math.inf)
        size = (scale * (q[:, h].abs() @ torch.nan_to_num(kh, 0, 0, 0).abs().T)).masked_fill(~seen, 0.0).amax(1, keepdim=True)
        top = w.amax(1, keepdim=True)
        p = torch.where(seen, (w - torch.where(top == -math.inf, 0.0, top)).exp(), 0.0)
        total = p.sum(1, keepdim=True)
        safe = torch.where(total > 0, total, 1.0)
        vz = torch.nan_to_num(vh, 0, 0, 0)
        out = (p @ vz) / safe
        spread = (p @ vz.abs()) / safe
        biggest = w.masked_fill(~seen, 0.0).abs().amax(1, keepdim=True)
        d = 2 * (dim + 2) * E * size + 16 * E * biggest + 2.0 ** -20
        rest = tiny * (seen.double() @ vz.abs())
        outs.append(out)
        out_bounds.append((1 + u) * ((2 * d + u + 2 * cached * E) * spread + rest) + u * out.abs() + tiny)
        lse = (torch.where(top == -math.inf, 0.0, top) + safe.log()) / math.log(2.0)
        sums.append(torch.where(total > 0, lse, -math.inf)[:, 0])
        sum_bounds.append((1.45 * (d + cached * E) + 4 * E * lse.abs() + 4 * E)[:, 0])
    return (torch.stack(outs, 1), torch.stack(sums, 1), torch.stack(out_bounds, 1), torch.stack(sum_bounds, 1))


def check_attention(paged, q, out, lse, heads, scale=None, rows_of=None):
    import torch
    group, dim = heads // paged.kv_heads, paged.head_dim
    scale = 1 / math.sqrt(dim) if scale is None else scale
    start = 0
    for s, (new, cached) in enumerate(paged.sequences):
        if new and (rows_of is None or s in rows_of):
            rows = slice(start, start + new)
            position = torch.arange(cached - new, cached, device=q.device)
            k, v = paged.read(paged.k, s), paged.read(paged.v, s)
            want, want_lse, bound, lse_bound = attention64(q[rows].double().view(new, heads, dim), k, v, position, paged.window,
                                                           scale, group, paged.dtype)
            assert_within(out[rows].reshape(new, heads, dim), want, bound, f"out of sequence {s}")
            if lse is not None:
                empty = want_lse == -math.inf
                assert (lse[rows][empty] == -math.inf).all()
                assert_within(torch.where(empty, 0.0, lse[rows].double()), torch.where(empty, 0.0, want_lse), lse_bound,
                              f"lse of sequence {s}")
        start += new


def run_attention(cuda, sequences, heads, kv_heads, head_dim, page, window, name, seed=1, strided=False, with_lse=True,
                  scale=0.0, gain=1.0, most=None, **more):
    import torch
    paged = Paged(cuda, sequences, kv_heads, head_dim, page, name, seed=seed, extra_rows=3, window=window, most=most, **more)
    width = heads * head_dim
    stride = width + (264 if strided else 0)
    q = torch.full((paged.tokens, stride), math.nan, device=cuda, dtype=paged.dtype)
    q[:, :width] = gain * torch.randn(paged.tokens, width, generator=paged.generator, device=cuda)
    q[paged.rows:] = math.nan  # rows no sequence owns
    out = torch.full((paged.tokens, width + (40 if strided else 0)), SENTINEL, device=cuda, dtype=paged.dtype)
    lse = torch.full((paged.tokens, heads), SENTINEL, device=cuda) if with_lse else None
    paged.attention(q, heads, out, lse, scale)
    torch.cuda.synchronize()
    assert int(paged.status) == 0
    check_attention(paged, q[:, :width], out[:, :width], lse, heads, scale or None)
    assert (out[paged.rows:] == SENTINEL).all() and (out[:, width:] == SENTINEL).all()
    if with_lse:
        assert (lse[paged.rows:] == SENTINEL).all()
    return paged, q, out, lse


SINGLES = [(1, n) for n in (1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 700, 1300)]
ATTENTION_CASES = {
    # sequences, heads, kv_heads, head_dim, page, window, dtype
    "single": ([(1, 1)], 28, 4, 128, 16, 0, "fp16"),
    "singles": (SINGLES, 28, 4, 128, 16, 0, "bf16"),
    "singles wide pages": (SINGLES, 32, 8, 128, 1024, 0, "fp16"),
    "singles 64": (SINGLES, 8, 8, 64, 32, 0, "bf16"),
    "singles one kv head": (SINGLES, 16, 1, 64, 128, 0, "fp16"),
    "singles window": (SINGLES, 28, 4, 128, 16, 100, "fp16"),
    "singles window one": (SINGLES, 4, 4, 128, 64, 1, "bf16"),
    "idle slots": ([(0, 0), (1, 40), (0, 33), (0, 0), (1, 1), (0, 5)], 28, 4, 128, 16, 0, "fp16"),
    "two and three": ([(2, 2), (3, 50), (2, 333), (1, 9), (3, 3)], 28, 4, 128, 16, 0, "fp16"),
    "four drafted": ([(4, 4), (4, 700), (4, 64), (4, 131)], 28, 4, 128, 64, 0, "bf16"),
    "four drafted window": ([(4, 4), (4, 700), (4, 64), (4, 131)], 28, 4, 128, 16, 37, "fp16"),
    "six of a group of five": ([(6, 100), (5, 5), (1, 2)], 40, 8, 128, 32, 0, "fp16"),
    "group of 128": ([(1, 300), (2, 200), (3, 3)], 128, 1, 128, 16, 0, "bf16"),
    "group of 33": ([(1, 300), (1, 17), (1, 1)], 66, 2, 64, 16, 0, "fp16"),
    "chunk": ([(130, 130)], 4, 2, 128, 16, 0, "fp16"),
    "chunk behind": ([(130, 1000)], 28, 4, 128, 64, 0, "bf16"),
    "chunks ragged": ([(33, 40), (1, 500), (300, 900), (0, 10), (64, 64), (129, 256), (17, 17)], 28, 4, 128, 16, 0, "fp16"),
    "chunks ragged 64": ([(33, 40), (1, 500), (300, 900), (0, 10), (64, 64), (129, 256)], 12, 2, 64, 256, 0, "bf16"),
    "chunks window": ([(33, 40), (1, 500), (300, 900), (128, 640), (64, 64)], 32, 8, 128, 32, 75, "fp16"),
    "chunks window 64": ([(33, 400), (1, 500), (300, 900), (128, 640)], 5, 5, 64, 16, 200, "bf16"),
    "chunk of one head": ([(257, 300), (5, 900)], 1, 1, 128, 128, 0, "fp16"),
    "chunk many heads": ([(40, 170), (41, 41)], 96, 2, 128, 16, 0, "fp16"),
    "chunk group of 100": ([(9, 170), (41, 41)], 100, 1, 64, 512, 0, "bf16"),
    "fewer cached than new": ([(10, 4), (50, 3), (3, 0), (200, 130), (1, 0), (5, 5)], 8, 2, 128, 16, 0, "fp16"),
    "fewer cached than new window": ([(10, 4), (50, 3), (3, 0), (200, 130), (1, 0)], 28, 4, 64, 16, 7, "bf16"),
    "single none cached": ([(1, 0), (1, 5), (1, 0)], 28, 4, 128, 16, 0, "fp16"),
    "forty rows": ([(6, 100), (5, 700), (1, 64), (6, 6), (3, 65)], 28, 4, 128, 16, 0, "fp16"),
    "forty rows window": ([(6, 100), (5, 700), (1, 64), (6, 6), (3, 65)], 28, 4, 64, 32, 50, "bf16"),
    "largest window": ([(10, 4), (50, 3), (3, 0), (200, 130), (1, 0), (5, 5)], 8, 2, 128, 16, 2**31 - 1, "fp16"),
    "largest window few": ([(4, 1), (3, 0), (4, 200), (1, 0), (2, 2)], 8, 2, 64, 16, 2**31 - 1, "bf16"),
    "long": ([(1, 20_000), (2, 9000)], 28, 4, 128, 64, 0, "fp16"),
    "long chunk": ([(100, 9000)], 14, 2, 128, 64, 0, "bf16"),
    "long chunk window": ([(700, 9000)], 14, 2, 128, 16, 3000, "bf16"),
}


@pytest.mark.parametrize("name", sorted(ATTENTION_CASES))
def test_paged_attention(cuda, name):
    run_attention(cuda, *ATTENTION_CASES[name])


@pytest.mark.parametrize("name", ["singles", "chunks ragged", "fewer cached than new", "chunks window 64"])
def test_paged_attention_strided_rows(cuda, name):
    run_attention(cuda, *ATTENTION_CASES[name], strided=True)


@pytest.mark.parametrize("name", ["singles", "chunks ragged"])
def test_paged_attention_without_lse_and_with_a_scale(cuda, name):
    run_attention(cuda, *ATTENTION_CASES[name], with_lse=False, scale=0.03125)


@pytest.mark.parametrize("gain", [0.0, 30.0])
@pytest.mark.parametrize("name", ["singles", "four drafted", "chunks ragged", "chunks window"])
def test_paged_attention_flat_and_peaked_rows(cuda, name, gain):
    """All scores equal, and scores of a hundred and more whose maximum moves from tile to tile."""
    run_attention(cuda, *ATTENTION_CASES[name], gain=gain)


@pytest.mark.parametrize("chunk", [1, 4, 200])
def test_paged_attention_rising_scores(cuda, chunk):
    """Every key scores higher than the one before it, so the running maximum moves in every tile."""
    import torch
    cached, heads, kv_heads, dim = 1500, 8, 2, 128
    paged = Paged(cuda, [(chunk, cached)], kv_heads, dim, 16, "fp16", seed=3)
    ramp = torch.linspace(-8, 8, cached, device=cuda).half()
    keys = torch.zeros(kv_heads, cached, dim, device=cuda, dtype=torch.float16)
    keys[..., 0] = ramp
    paged.write(paged.k, paged.tables[0], keys)
    q = torch.zeros(paged.tokens, heads * dim, device=cuda, dtype=torch.float16)
    q.view(-1, heads, dim)[..., 0] = 64.0
    out, lse = torch.empty_like(q), torch.empty(paged.tokens, heads, device=cuda)
    paged.attention(q, heads, out, lse)
    check_attention(paged, q, out, lse, heads)


@pytest.mark.parametrize("chunk", [1, 5, 60])
def test_paged_attention_shared_prefix_pages(cuda, chunk):
    """Sequences whose first pages are the same ones: the instruction all prompts begin with."""
    import torch
    heads, kv_heads, dim, page, prefix = 14, 2, 128, 16, 96
    paged = Paged(cuda, [(chunk, prefix + 70), (chunk, prefix + chunk), (chunk, prefix + 300)], kv_heads, dim, page, "fp16", seed=4)
    for s in (1, 2):
        paged.tables[s][:prefix // page] = paged.tables[0][:prefix // page]
        paged.table[s, :prefix // page] = paged.table[0, :prefix // page]
    q = torch.randn(paged.tokens, heads * dim, generator=paged.generator, device=cuda).half()
    out, lse = torch.empty_like(q), torch.empty(paged.tokens, heads, device=cuda)
    paged.attention(q, heads, out, lse)
    assert int(paged.status) == 0
    check_attention(paged, q, out, lse, heads)


def test_paged_attention_many_sequences(cuda):
    rng = np.random.default_rng(0)
    for most, count in ((1, 1500), (5, 1100), (40, 700)):
        sequences = [(n, n + int(rng.integers(0, 60))) for n in rng.integers(0, most + 1, count).tolist()]
        run_attention(cuda, sequences, 4, 2, 64, 16, 0, "fp16", seed=most)


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("sequences,window", [([(4, 70)], 0), ([(4, 70)], 8), ([(60, 200)], 0), ([(60, 200)], 20)])
def test_values_a_row_does_not_see_do_not_touch_it(cuda, sequences, window, bad):
    """A NaN or infinity in the key and value of one new token: rows before it (and rows whose window
    has passed it) are those of a clean cache, bit for bit; rows that see it are not finite."""
    import torch
    heads, kv_heads, dim, page = 14, 2, 128, 16
    new, cached = sequences[0]
    clean = run_attention(cuda, sequences, heads, kv_heads, dim, page, window, "fp16", seed=9)
    for which in ("k", "v"):
        paged = Paged(cuda, sequences, kv_heads, dim, page, "fp16", seed=9, extra_rows=3, window=window)
        at = cached - new + new // 2
        pool = paged.k if which == "k" else paged.v
        pool[int(paged.tables[0][at // page]), :, at % page, 5] = bad
        out, lse = torch.full_like(clean[2], SENTINEL), torch.full_like(clean[3], SENTINEL)
        q = clean[1].clone()
        q[:, :heads * dim] = torch.where(clean[1].isnan(), clean[1], clean[1].abs() + 0.125)  # no sign change, no zero
        reference_out, reference_lse = torch.full_like(out, SENTINEL), torch.full_like(lse, SENTINEL)
        clean[0].attention(q, heads, reference_out, reference_lse)
        paged.attention(q, heads, out, lse)
        position = torch.arange(cached - new, cached)
        sees = (position >= at) & ((position < at + window) if window else torch.ones(new, dtype=torch.bool))
        blind = (~sees).nonzero()[:, 0].to(cuda)
        assert torch.equal(out[blind], reference_out[blind]) and torch.equal(lse[blind], reference_lse[blind]), which
        rows = out[:new][sees.to(cuda)].view(-1, heads, dim)
        if which == "v":
            assert not torch.isfinite(rows[..., 5]).any()
            keep = [d for d in range(dim) if d != 5]
            assert torch.equal(rows[..., keep], reference_out[:new][sees.to(cuda)].view(-1, heads, dim)[..., keep])
        elif bad == math.inf or math.isnan(bad):  # q > 0, so a key of -inf scores -inf: weight 0
            assert not torch.isfinite(rows).any()


@pytest.mark.parametrize("chunk", [1, 70])
def test_paged_attention_bits_repeat(cuda, chunk):
    import torch
    sequences = [(chunk, 3000 + 100 * i) for i in range(5)] + [(1, 77)]
    paged, q, out, lse = run_attention(cuda, sequences, 28, 4, 128, 16, 0, "bf16")
    for _ in range(3):
        again, again_lse = torch.full_like(out, SENTINEL), torch.full_like(lse, SENTINEL)
        paged.attention(q, 28, again, again_lse)
        assert torch.equal(again, out) and torch.equal(again_lse, lse)


def test_offsets_past_32_bits(cuda):
    """Pages behind 2^31 elements of the pool, for the append and the attention."""
    import torch
    native = _lib()
    kv_heads, dim, page, heads = 2, 128, 1024, 4
    first = (1 << 31) // (kv_heads * dim * page) + 2
    for sequences in ([(1, 2100), (1, 30)], [(70, 2100), (33, 33)]):
        paged = Paged(cuda, sequences, kv_heads, dim, page, "fp16", first_page=first, seed=2)
        width = (heads + 2 * kv_heads) * dim
        qkv = torch.randn(paged.tokens, width, generator=paged.generator, device=cuda).half()
        q = torch.empty(paged.tokens, heads * dim, device=cuda, dtype=torch.float16)
        native.check(native.lib.ar_paged_append(ctypes.byref(paged.cache), ctypes.byref(paged.batch), qkv.data_ptr(), width, None,
                                                heads, q.data_ptr(), heads * dim, None, None, 0, 0, 0, paged.status.data_ptr(),
                                                _stream()))
        start = 0
        for s, (new, cached) in enumerate(sequences):
            for pool, column in ((paged.k, heads), (paged.v, heads + kv_heads)):
                want = qkv[start:start + new].view(new, -1, dim)[:, column:column + kv_heads].transpose(0, 1)
                assert torch.equal(paged.read(pool, s)[:, cached - new:], want.double())
            start += new
        out, lse = torch.empty_like(q), torch.empty(paged.tokens, heads, device=cuda)
        paged.attention(q, heads, out, lse)
        check_attention(paged, q, out, lse, heads)
        assert int(paged.status) == 0
        del paged


# ------------------------------------------------------------------------------ refusals on device
BAD_BATCHES = {
    "rows past the call's": dict(offsets=[0, 2, 9, 10]),
    "decreasing": dict(offsets=[0, 4, 2, 6]),
    "negative offset": dict(offsets=[0, -3, 2, 6]),
    "negative length": dict(lengths=[20, -1, 30]),
    "length beyond the row": dict(lengths=[20, 1000, 30]),
    "more than max_query_tokens": dict(offsets=[0, 1, 6, 6], most=4),
    "huge length": dict(lengths=[20, 2**31 - 1, 30]),
}


@pytest.mark.parametrize("heads", [4, 64])
@pytest.mark.parametrize("name", sorted(BAD_BATCHES))
def test_bad_batches_are_reported_and_left_out(cuda, name, heads):
    """Sequence 1 is out of range: status 4, no fault, its rows untouched, sequence 0 computed."""
    import torch
    native = _lib()
    change = BAD_BATCHES[name]
    paged = Paged(cuda, [(2, 20), (3, 25), (1, 30)], 2, 64, 16, "fp16", most=change.get("most"))
    if "offsets" in change:
        paged.offsets.copy_(torch.tensor(change["offsets"], dtype=torch.int32))
    if "lengths" in change:
        paged.lengths.copy_(torch.tensor(change["lengths"], dtype=torch.int32))
    q = torch.randn(paged.tokens, heads * 64, device=cuda).half()
    out, lse = torch.full_like(q, SENTINEL), torch.full((paged.tokens, heads), SENTINEL, device=cuda)
    paged.attention(q, heads, out, lse)
    torch.cuda.synchronize()
    assert int(paged.status) == 4
    first = change.get("offsets", [0, 2])[1]
    if first == 2:
        check_attention(paged, q, out, lse, heads, rows_of=[0])
    if "lengths" in change:
        assert (out[2:5] == SENTINEL).all() and (lse[2:5] == SENTINEL).all()
    k, v = paged.k.clone(), paged.v.clone()
    paged.status.zero_()
    qkv = torch.randn(paged.tokens, (heads + 4) * 64, device=cuda).half()
    native.check(native.lib.ar_paged_append(ctypes.byref(paged.cache), ctypes.byref(paged.batch), qkv.data_ptr(),
                                            (heads + 4) * 64, None, heads, out.data_ptr(), heads * 64, None, None, 0, 0, 0,
                                            paged.status.data_ptr(), _stream()))
    torch.cuda.synchronize()
    assert int(paged.status) == 4
    if "lengths" in change:
        ids = paged.tables[1].to(cuda)
        assert torch.equal(paged.k[ids].nan_to_num(), k[ids].nan_to_num()) and torch.equal(paged.v[ids].nan_to_num(), v[ids].nan_to_num())


@pytest.mark.parametrize("new", [1, 300])
def test_idle_sequences_out_of_range_are_reported(cuda, new):
    """Sequence 1 has no new tokens and a negative length: no row leads to it, both operators report it."""
    import torch
    native = _lib()
    paged = Paged(cuda, [(new, 320), (0, 25), (1, 30)], 2, 64, 16, "fp16")
    paged.lengths[1] = -1
    q = torch.randn(paged.tokens, 4 * 64, device=cuda).half()
    out, lse = torch.full_like(q, SENTINEL), torch.full((paged.tokens, 4), SENTINEL, device=cuda)
    paged.attention(q, 4, out, lse)
    torch.cuda.synchronize()
    assert int(paged.status) == 4
    check_attention(paged, q, out, lse, 4, rows_of=[0, 2])
    paged.status.zero_()
    qkv = torch.randn(paged.tokens, 8 * 64, device=cuda).half()
    native.check(native.lib.ar_paged_append(ctypes.byref(paged.cache), ctypes.byref(paged.batch), qkv.data_ptr(), 8 * 64, None,
                                            4, None, 0, None, None, 0, 0, 0, paged.status.data_ptr(), _stream()))
    torch.cuda.synchronize()
    assert int(paged.status) == 4
    row = qkv[-1].view(8, 64)
    page = int(paged.tables[2][29 // 16])
    assert torch.equal(paged.k[page, :, 29 % 16], row[4:6]) and torch.equal(paged.v[page, :, 29 % 16], row[6:])


@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("page_id", [-1, 10**6, 2**31 - 1, -2**31])
def test_page_ids_outside_the_pool_are_reported(cuda, page_id, new):
    import torch
    native = _lib()
    paged = Paged(cuda, [(new, 100), (new, 90)], 2, 128, 16, "fp16")
    last = paged.table[1, 5].clone()
    paged.table[1, 5] = page_id  # positions 80..89 of sequence 1
    q = torch.randn(paged.tokens, 8 * 128, device=cuda).half()
    out, lse = torch.full_like(q, SENTINEL), torch.full((paged.tokens, 8), SENTINEL, device=cuda)
    paged.attention(q, 8, out, lse)
    torch.cuda.synchronize()
    assert int(paged.status) == 4
    check_attention(paged, q, out, lse, 8, rows_of=[0])
    paged.status.zero_()
    before = paged.k.clone()
    qkv = torch.randn(paged.tokens, 12 * 128, device=cuda).half()
    native.check(native.lib.ar_paged_append(ctypes.byref(paged.cache), ctypes.byref(paged.batch), qkv.data_ptr(), 12 * 128, None,
                                            8, None, 0, None, None, 0, 0, 0, paged.status.data_ptr(), _stream()))
    torch.cuda.synchronize()
    assert int(paged.status) == 4
    assert torch.equal(paged.k[int(last)].nan_to_num(), before[int(last)].nan_to_num())


# ----------------------------------------------------------------------------------------- append
APPEND_CASES = {
    # sequences, heads, kv_heads, head_dim, page, rotary, interleaved, bias, dtype, q ("out", "place", "none")
    "one": ([(1, 1)], 28, 4, 128, 16, 128, False, True, "fp16", "out"),
    "singles": ([(1, n) for n in (1, 16, 17, 200)], 28, 4, 128, 16, 128, False, True, "bf16", "out"),
    "idle": ([(0, 0), (1, 9), (0, 30), (2, 2)], 4, 4, 64, 32, 64, True, False, "fp16", "place"),
    "partial": ([(3, 40), (50, 64), (1, 1)], 32, 8, 128, 64, 64, False, False, "bf16", "out"),
    "partial interleaved": ([(3, 40), (50, 64), (1, 1)], 32, 8, 128, 64, 32, True, True, "fp16", "place"),
    "no rotation": ([(3, 40), (50, 64)], 5, 5, 64, 16, 0, False, True, "bf16", "out"),
    "no rotation no bias": ([(3, 40), (50, 64)], 5, 5, 64, 16, 0, False, False, "fp16", "none"),
    "keys and values alone": ([(3, 40), (50, 64)], 0, 3, 128, 16, 128, False, False, "fp16", "none"),
    "queries left alone": ([(3, 40), (50, 64)], 6, 3, 128, 16, 128, True, True, "fp16", "none"),
    "many": ([(200, 300), (7, 7), (400, 1000), (123, 500)], 28, 4, 128, 16, 128, False, True, "fp16", "out"),
    "many interleaved": ([(200, 300), (7, 7), (400, 1000), (122, 500)], 9, 3, 64, 1024, 64, True, False, "bf16", "place"),
    "fewer cached than new": ([(10, 4), (400, 33), (3, 0), (1, 5)], 8, 2, 128, 16, 128, False, False, "fp16", "out"),
}


@pytest.mark.parametrize("name", sorted(APPEND_CASES))
def test_paged_append(cuda, name):
    import torch
    native = _lib()
    sequences, heads, kv_heads, dim, page, rotary, interleaved, with_bias, dtype_name, where = APPEND_CASES[name]
    paged = Paged(cuda, sequences, kv_heads, dim, page, dtype_name, seed=4, extra_rows=2)
    g, dtype = paged.generator, paged.dtype
    width = (heads + 2 * kv_heads) * dim
    stride = width + 24
    qkv = torch.full((paged.tokens, stride), SENTINEL, device=cuda, dtype=dtype)
    qkv[:, :width] = torch.randn(paged.tokens, width, generator=g, device=cuda)
    before, k_before, v_before = qkv.clone(), paged.k.clone(), paged.v.clone()
    bias = 0.3 * torch.randn(width, generator=g, device=cuda) if with_bias else None
    table = max(t for _, t in sequences)
    cos, sin = (torch.randn(table, max(rotary // 2, 1), generator=g, device=cuda) for _ in range(2))
    q_out = {"out": torch.full((paged.tokens, heads * dim + 8), SENTINEL, device=cuda, dtype=dtype), "place": qkv, "none": None}[where]
    native.check(native.lib.ar_paged_append(
        ctypes.byref(paged.cache), ctypes.byref(paged.batch), qkv.data_ptr(), stride, None if bias is None else bias.data_ptr(),
        heads, None if q_out is None else q_out.data_ptr(), 0 if q_out is None else q_out.stride(0),
        cos.data_ptr() if rotary else None, sin.data_ptr() if rotary else None, table if rotary else 0, rotary, interleaved,
        paged.status.data_ptr(), _stream()))
    torch.cuda.synchronize()
    assert int(paged.status) == 0
    k_want, v_want = k_before.double(), v_before.double()
    k_bound, v_bound = torch.zeros_like(k_want), torch.zeros_like(v_want)
    start = 0
    for s, (new, cached) in enumerate(sequences):
        position = torch.arange(cached - new, cached, device=cuda)
        keep = position >= 0
        x = before[start:start + new, :width].double()[keep]
        size = x.abs()
        if with_bias:
            x, size = x + bias.double(), size + bias.double().abs()
        x, size = x.view(len(x), width // dim, dim), size.view(len(x), width // dim, dim)
        position = position[keep]
        turned, turned_size = x.clone(), size.clone()
        if rotary:
            turned, _ = rotate64(x, cos.double()[position], sin.double()[position], rotary, interleaved)
            _, turned_size = rotate64(size, cos.double().abs()[position], sin.double().abs()[position], rotary, interleaved)
        bound = rotation_bound(turned, turned_size, dtype)
        plain_bound = _half_step(dtype) * x.abs() + 2 * E * size + _tiny(dtype)
        if q_out is not None and heads:
            got = q_out[start:start + new, :heads * dim][keep].view(-1, heads, dim)
            assert_within(got, turned[:, :heads], bound[:, :heads], f"q of sequence {s}")
            rest = q_out[start:start + new, :heads * dim][~keep]
            assert (rest == SENTINEL).all() if where == "out" else torch.equal(rest, before[start:start + new, :heads * dim][~keep])
        if len(position):
            ids, slot = paged.tables[s].to(cuda)[position // page], position % page
            k_want[ids, :, slot], k_bound[ids, :, slot] = turned[:, heads:heads + kv_heads], bound[:, heads:heads + kv_heads]
            v_want[ids, :, slot], v_bound[ids, :, slot] = x[:, heads + kv_heads:], plain_bound[:, heads + kv_heads:]
        start += new
    for got, want, bound, what in ((paged.k, k_want, k_bound, "k"), (paged.v, v_want, v_bound, "v")):
        assert torch.equal(got.isnan(), want.isnan()), f"{what}: a slot no new token owns was written"
        assert_within(got.nan_to_num(), want.nan_to_num(), bound, what)
    if where == "out":
        assert (q_out[paged.rows:] == SENTINEL).all() and (q_out[:, heads * dim:] == SENTINEL).all()
    if where == "place":
        assert torch.equal(qkv[:, heads * dim:], before[:, heads * dim:]) and torch.equal(qkv[paged.rows:], before[paged.rows:])
    else:
        assert torch.equal(qkv, before)


def test_append_position_past_the_table_is_reported_and_left_out(cuda):
    import torch
    native = _lib()
    paged = Paged(cuda, [(4, 20)], 2, 64, 16, "fp16")
    k, v = paged.k.clone(), paged.v.clone()
    qkv = torch.randn(4, 6 * 64, device=cuda).half()
    q = torch.full((4, 128), SENTINEL, device=cuda, dtype=torch.float16)
    cos, sin = torch.ones(18, 32, device=cuda), torch.zeros(18, 32, device=cuda)
    native.check(native.lib.ar_paged_append(ctypes.byref(paged.cache), ctypes.byref(paged.batch), qkv.data_ptr(), 384, None, 2,
                                            q.data_ptr(), 128, cos.data_ptr(), sin.data_ptr(), 18, 64, 0, paged.status.data_ptr(),
                                            _stream()))
    torch.cuda.synchronize()
    assert int(paged.status) == 2
    got = paged.read(paged.k, 0)
    assert torch.equal(got[:, 16:18], qkv[:2].view(2, 6, 64)[:, 2:4].transpose(0, 1).double())  # cos 1, sin 0
    page = int(paged.tables[0][1])
    assert torch.equal(paged.k[page, :, 2:4], k[page, :, 2:4]) and torch.equal(paged.v[page, :, 2:4], v[page, :, 2:4])
    assert (q[2:] == SENTINEL).all() and torch.equal(q[:2], qkv[:2, :128])


# ----------------------------------------------------------------------------------- runs together
def _serve(native, paged, qkv, heads, table, q, out, lse, workspace, stream):
    """One layer's step as a serving loop makes it: append with rotation, then attention."""
    width = (heads + 2 * paged.kv_heads) * paged.head_dim
    cos, sin, positions = table
    native.check(native.lib.ar_paged_append(ctypes.byref(paged.cache), ctypes.byref(paged.batch), qkv.data_ptr(), width, None,
                                            heads, q.data_ptr(), heads * paged.head_dim, cos.data_ptr(), sin.data_ptr(), positions,
                                            paged.head_dim, 0, paged.status.data_ptr(), stream))
    paged.attention(q, heads, out, lse, workspace=workspace, stream=stream)


@pytest.mark.parametrize("name", ["fp16", "bf16"])
def test_chunked_prefill_and_decode_equal_the_packed_prefill(cuda, name):
    """Two prompts fed as chunks, then token by token, through table, append and attention: every row's
    output is the 64-bit attention over the rotated and rounded q, k, v, and agrees with
    ar_rotary_embedding + ar_causal_attention over the packed prompts, whose rows each lie within the
    same bound of the same values (so within twice it of each other), plus what the rotation of two
    tables can differ by: one rounding step of q, k (2 u of the score's magnitude sum, twice)."""
    import torch
    native = _lib()
    dtype, code = _types(name)
    heads, kv_heads, dim, page = 28, 4, 128, 16
    lengths, chunks = [389, 250], [(128, 1), (200, 149), (40, 99), (20, 1), (1, 0)]
    width = (heads + 2 * kv_heads) * dim
    g = torch.Generator(device=cuda).manual_seed(8)
    total = sum(lengths)
    qkv = torch.randn(total, width, generator=g, device=cuda).to(dtype)
    rows = [qkv[:lengths[0]], qkv[lengths[0]:]]
    scaling = native.RopeScalingStruct(1e6, dim, 0, 1.0, 0.0, 0.0, 0, 0.0)
    cos, sin = (torch.empty(512, dim // 2, device=cuda) for _ in range(2))
    native.check(native.lib.ar_rope_table_scaled(ctypes.byref(scaling), 512, cos.data_ptr(), sin.data_ptr(), _stream()))
    paged = Paged(cuda, [(1, n) for n in lengths], kv_heads, dim, page, name, fill=False, extra_rows=512)
    outs, sums, queries = ([torch.empty(n, heads * w, device=cuda, dtype=t) for n in lengths]
                           for w, t in ((dim, dtype), (1, torch.float32), (dim, dtype)))
    fed = [0, 0]
    workspace = torch.empty(64 << 20, dtype=torch.uint8, device=cuda)
    while fed != lengths:
        step = chunks.pop(0) if chunks else (1, 1)
        new = [min(n, l - f) for n, l, f in zip(step, lengths, fed)]
        batch = torch.cat([r[f:f + n] for r, f, n in zip(rows, fed, new)])
        paged.offsets.copy_(torch.tensor([0, new[0], sum(new)], dtype=torch.int32))
        paged.lengths.copy_(torch.tensor([f + n for f, n in zip(fed, new)], dtype=torch.int32))
        paged.batch.token_count, paged.batch.max_query_tokens = len(batch), max(new)
        q = torch.empty(len(batch), heads * dim, device=cuda, dtype=dtype)
        out, lse = torch.empty_like(q), torch.empty(len(batch), heads, device=cuda)
        _serve(native, paged, batch, heads, (cos, sin, 512), q, out, lse, workspace, _stream())
        for i, at in ((0, 0), (1, new[0])):
            piece = slice(at, at + new[i])
            outs[i][fed[i]:fed[i] + new[i]], sums[i][fed[i]:fed[i] + new[i]] = out[piece], lse[piece]
            queries[i][fed[i]:fed[i] + new[i]] = q[piece]
            fed[i] += new[i]
    assert int(paged.status) == 0
    packed = qkv.clone()
    old_cos, old_sin = (torch.empty(512, dim // 2, device=cuda) for _ in range(2))
    positions = torch.cat([torch.arange(n, dtype=torch.int32) for n in lengths]).to(cuda)
    native.check(native.lib.ar_rope_table(old_cos.data_ptr(), old_sin.data_ptr(), 512, dim, 1e6, _stream()))
    native.check(native.lib.ar_rotary_embedding(packed.data_ptr(), None, positions.data_ptr(), total, heads, kv_heads, dim,
                                                old_cos.data_ptr(), old_sin.data_ptr(), 512, None, code, _stream()))
    offsets = torch.tensor([0, lengths[0], total], dtype=torch.int32)
    device_offsets = offsets.to(cuda)
    prefill, prefill_lse = torch.empty(total, heads * dim, device=cuda, dtype=dtype), torch.empty(total, heads, device=cuda)
    native.check(native.lib.ar_causal_attention(packed.data_ptr(), prefill.data_ptr(), prefill_lse.data_ptr(), offsets.data_ptr(),
                                                device_offsets.data_ptr(), 2, heads, kv_heads, dim, 0, code, _stream()))
    start, u = 0, _half_step(dtype)
    for i, n in enumerate(lengths):
        paged.sequences = [(m, m) for m in lengths]
        k, v = paged.read(paged.k, i), paged.read(paged.v, i)
        q = queries[i].double().view(n, heads, dim)
        want, want_lse, bound, lse_bound = attention64(q, k, v, torch.arange(n, device=cuda), 0, dim ** -0.5, heads // kv_heads, dtype)
        assert_within(outs[i].view(n, heads, dim), want, bound, f"prompt {i}")
        assert_within(sums[i], want_lse, lse_bound, f"lse of prompt {i}")
        size = torch.stack([(q[:, h].abs() @ k[h // 7].abs().T).amax(1) for h in range(heads)], 1) * dim ** -0.5
        spread = v.abs().amax()
        assert_within(prefill[start:start + n].view(n, heads, dim), want, bound + 4 * u * size[..., None] * 2 * spread, f"packed {i}")
        assert_within(prefill_lse[start:start + n], want_lse, lse_bound + 1.45 * 4 * u * size, f"packed lse {i}")
        start += n


@pytest.mark.parametrize("chunk", [1, 60])
def test_captured_step_replays_with_new_lengths(cuda, chunk):
    """append + attention captured once; lengths, offsets and page table change between replays, and an
    eager call with its own workspace runs in between."""
    import torch
    native = _lib()
    heads, kv_heads, dim, page, name = 28, 4, 128, 16, "fp16"
    full = [(chunk, 700), (chunk, 300), (chunk, 90)]
    paged = Paged(cuda, full, kv_heads, dim, page, name, seed=6)
    table = torch.empty(2, 800, dim // 2, device=cuda)
    scaling = native.RopeScalingStruct(1e4, dim, 1, 2.0, 0.0, 0.0, 0, 0.0)
    native.check(native.lib.ar_rope_table_scaled(ctypes.byref(scaling), 800, table[0].data_ptr(), table[1].data_ptr(), _stream()))
    qkv = torch.randn(paged.tokens, (heads + 2 * kv_heads) * dim, generator=paged.generator, device=cuda).half()
    q = torch.empty(paged.tokens, heads * dim, device=cuda, dtype=torch.float16)
    out, lse = torch.empty_like(q), torch.empty(paged.tokens, heads, device=cuda)
    spaces = [torch.empty(64 << 20, dtype=torch.uint8, device=cuda) for _ in range(2)]
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _serve(native, paged, qkv, heads, (table[0], table[1], 800), q, out, lse, spaces[0], side.cuda_stream)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        _serve(native, paged, qkv, heads, (table[0], table[1], 800), q, out, lse, spaces[0], torch.cuda.current_stream().cuda_stream)
    for lengths in ([700, 300, 90], [650, 299, 61], [chunk, chunk, chunk]):
        paged.lengths.copy_(torch.tensor(lengths, dtype=torch.int32))
        qkv.copy_(torch.randn(qkv.shape, generator=paged.generator, device=cuda))
        out.fill_(SENTINEL)
        graph.replay()
        graph_out, graph_lse, graph_q, k = out.clone(), lse.clone(), q.clone(), paged.k.clone()
        out.fill_(SENTINEL)
        _serve(native, paged, qkv, heads, (table[0], table[1], 800), q, out, lse, spaces[1], _stream())
        assert torch.equal(out, graph_out) and torch.equal(lse, graph_lse) and torch.equal(q, graph_q)
        assert torch.equal(paged.k.nan_to_num(), k.nan_to_num())
        paged.sequences = [(chunk, n) for n in lengths]
        check_attention(paged, q, out, lse, heads)
    assert int(paged.status) == 0


def test_two_streams_with_their_own_workspaces(cuda):
    import torch
    heads = 28
    jobs = []
    for seed, sequences in ((1, [(1, 3000), (1, 50)]), (2, [(90, 2000), (1, 700)])):
        paged = Paged(cuda, sequences, 4, 128, 16, "fp16", seed=seed)
        q = torch.randn(paged.tokens, heads * 128, generator=paged.generator, device=cuda).half()
        out, lse = torch.empty_like(q), torch.empty(paged.tokens, heads, device=cuda)
        jobs.append((paged, q, out, lse, torch.cuda.Stream(), torch.empty(64 << 20, dtype=torch.uint8, device=cuda)))
    torch.cuda.synchronize()
    for _ in range(20):
        for paged, q, out, lse, stream, workspace in jobs:
            paged.attention(q, heads, out, lse, workspace=workspace, stream=stream.cuda_stream)
    torch.cuda.synchronize()
    for paged, q, out, lse, *_ in jobs:
        check_attention(paged, q, out, lse, heads)


def test_workspace_is_required_where_needed(cuda):
    import torch
    native = _lib()
    paged = Paged(cuda, [(1, 100)], 4, 128, 16, "fp16")
    needed = native.lib.ar_paged_attention_workspace(ctypes.byref(paged.cache), ctypes.byref(paged.batch), 28)
    q = torch.zeros(1, 28 * 128, device=cuda, dtype=torch.float16)
    out = torch.empty_like(q)
    if needed > 0:
        status = native.lib.ar_paged_attention(ctypes.byref(paged.cache), ctypes.byref(paged.batch), q.data_ptr(), 28 * 128, 28, 0.0,
                                               0, out.data_ptr(), 28 * 128, None, None, 0, None, _stream())
        assert status == native.AR_ERR_INVALID and "workspace" in native.lib.ar_last_error().decode()
