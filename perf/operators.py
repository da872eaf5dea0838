"""Cases of the serving operators: scaled rotary tables, rotary positions, the append to a paged KV
cache and the attention over it. `run` computes a case in plain torch, or with `own` set through
this repository's library."""
import ctypes
import functools
import math
import os
import random
import sys

import torch

own = False

TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
CODES = {"fp16": 1, "bf16": 2}  # AR_DTYPE_F16, AR_DTYPE_BF16
KINDS = {"none": 0, "linear": 1, "bands": 2, "yarn": 3}  # AR_ROPE_*
WORKSPACE = 64 << 20  # bytes; enough for every ar_paged_attention call on one GPU


# ------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # the cos/sin table of an engine's whole window, frequencies stretched by wavelength
        {"name": "table_bands_8k", "op": "table", "kind": "bands", "theta": 500000.0, "rotary": 128, "positions": 8192,
         "factor": 8.0, "low": 1.0, "high": 4.0, "original": 8192},
        # the table of a 128K window, half of each head rotated
        {"name": "table_yarn_128k", "op": "table", "kind": "yarn", "theta": 1000000.0, "rotary": 64, "positions": 131072,
         "factor": 4.0, "low": 1.0, "high": 32.0, "original": 32768},
        # one generated token's query heads: the smallest call, launch latency
        {"name": "rotary_one_token", "op": "rotary", "tokens": 1, "heads": 28, "head_dim": 128, "rotary": 128,
         "interleaved": False, "inverse": False, "dtype": "fp16", "table": 4096},
        # a packed prefill batch, pairs side by side, half of each head rotated
        {"name": "rotary_prefill_partial", "op": "rotary", "tokens": 16384, "heads": 32, "head_dim": 128, "rotary": 64,
         "interleaved": True, "inverse": False, "dtype": "bf16", "table": 8192},
        # 32 answers generated together: one new token each
        {"name": "append_decode_32", "op": "append", "sequences": 32, "chunk": 1, "singles": 1.0, "history": 2048,
         "heads": 28, "kv_heads": 4, "head_dim": 128, "rotary": 128, "interleaved": False, "bias": True, "page": 16,
         "dtype": "bf16", "lengths": 3},
        # ragged prompt chunks of a prefill batch
        {"name": "append_prefill_ragged", "op": "append", "sequences": 9, "chunk": 2048, "singles": 0.0, "history": 1000,
         "heads": 32, "kv_heads": 8, "head_dim": 128, "rotary": 128, "interleaved": False, "bias": False, "page": 64,
         "dtype": "fp16", "lengths": 5},
        # one answer after one prompt: latency
        {"name": "attn_decode_one", "op": "attention", "sequences": 1, "chunk": 1, "singles": 1.0, "history": 1096,
         "fixed": True, "heads": 28, "kv_heads": 4, "head_dim": 128, "page": 16, "window": 0, "dtype": "fp16", "lengths": 1},
        # 64 answers generated together after contexts of all lengths: the cache's bandwidth
        {"name": "attn_decode_64", "op": "attention", "sequences": 64, "chunk": 1, "singles": 1.0, "history": 8191,
         "fixed": False, "heads": 32, "kv_heads": 8, "head_dim": 128, "page": 16, "window": 0, "dtype": "bf16", "lengths": 7},
        # four drafted tokens checked at once for 16 answers
        {"name": "attn_verify_4", "op": "attention", "sequences": 16, "chunk": 4, "singles": 0.0, "history": 4090,
         "fixed": False, "heads": 28, "kv_heads": 4, "head_dim": 128, "page": 64, "window": 0, "dtype": "fp16", "lengths": 11},
        # one 512-token prefill chunk behind 3.5K tokens of cache (the engine's prefill_chunk_tokens)
        {"name": "attn_chunk_512", "op": "attention", "sequences": 1, "chunk": 512, "singles": 0.0, "history": 3584,
         "fixed": True, "heads": 28, "kv_heads": 4, "head_dim": 128, "page": 64, "window": 0, "dtype": "fp16", "lengths": 13},
        # generation and prefill chunks in one batch, sliding window, no shared heads, 64-wide heads
        {"name": "attn_mixed_window", "op": "attention", "sequences": 19, "chunk": 400, "singles": 0.7, "history": 3000,
         "fixed": False, "heads": 16, "kv_heads": 16, "head_dim": 64, "page": 32, "window": 1000, "dtype": "bf16",
         "lengths": 17},
        # two whole 4K chunks behind up to 4K of cache: the tensor cores' rate
        {"name": "attn_prefill_4k", "op": "attention", "sequences": 2, "chunk": 4096, "singles": 0.0, "history": 4096,
         "fixed": True, "heads": 32, "kv_heads": 8, "head_dim": 128, "page": 128, "window": 0, "dtype": "bf16",
         "lengths": 19},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["table", "rotary", "append", "append", "attention", "attention", "attention"])
    if op == "table":
        return {"op": op, "kind": rng.choice(sorted(KINDS)), "theta": rng.choice([10000.0, 500000.0, 1000000.0]),
                "rotary": 2 * rng.randint(8, 128), "positions": _log(rng, 300, 130000), "factor": rng.choice([2.0, 4.0, 8.0]),
                "low": 1.0, "high": rng.choice([4.0, 32.0]), "original": rng.choice([4096, 8192, 32768])}
    if op == "rotary":
        head_dim = rng.choice([64, 80, 96, 128, 192, 256])
        heads = rng.choice([1, 4, 7, 8, 28, 32, 40])
        return {"op": op, "tokens": _log(rng, 1, max(2, 60_000_000 // (heads * head_dim))), "heads": heads, "head_dim": head_dim,
                "rotary": rng.choice([head_dim, head_dim // 2, 2 * rng.randint(4, head_dim // 2)]),
                "interleaved": rng.random() < 0.5, "inverse": rng.random() < 0.3, "dtype": rng.choice(sorted(TYPES)),
                "table": _log(rng, 512, 40000)}
    heads, kv_heads = rng.choice([(28, 4), (32, 8), (16, 16), (12, 2), (8, 1), (32, 4), (40, 8), (5, 5)])
    case = {"op": op, "sequences": _log(rng, 1, 96), "chunk": 1, "singles": 1.0, "history": _log(rng, 1, 12000),
            "heads": heads, "kv_heads": kv_heads, "head_dim": rng.choice([64, 128, 128]), "page": rng.choice([16, 32, 64, 128, 256]),
            "dtype": rng.choice(sorted(TYPES)), "lengths": rng.randint(0, 1 << 20)}
    if rng.random() < 0.65:
        case["chunk"], case["singles"] = _log(rng, 2, 4096), rng.choice([0.0, 0.0, 0.5, 0.9])
    if op == "append":
        case["rotary"] = case["head_dim"] // rng.choice([1, 1, 2])
        case["interleaved"], case["bias"] = rng.random() < 0.3, rng.random() < 0.5
        while case["sequences"] > 1 and (case["sequences"] * case["chunk"] > 20000
                                         or case["sequences"] * kv_heads * (case["history"] + case["chunk"]) > 1.5e6):
            case["sequences"] = (case["sequences"] + 1) // 2
    else:
        case["fixed"], case["window"] = rng.random() < 0.2, rng.choice([0, 0, _log(rng, 16, 6000)])
        reach = case["history"] + case["chunk"]
        while case["sequences"] > 1 and (case["sequences"] * heads * case["chunk"] * reach > 1.6e9
                                         or case["sequences"] * kv_heads * reach > 4.0e6):
            case["sequences"] = (case["sequences"] + 1) // 2
        while heads * case["chunk"] * (case["history"] + case["chunk"]) > 1.6e9:
            case["chunk"] //= 2
    return case


@functools.lru_cache(maxsize=64)
def _lengths(sequences, chunk, singles, history, fixed, lengths):
    """(new tokens, cached tokens after the append) of every sequence: a function of the case alone."""
    rng = random.Random(lengths)
    new, total = [], []
    for _ in range(sequences):
        n = 1 if rng.random() < singles else chunk if fixed else rng.randint(max(1, chunk // 4), chunk)
        before = history if fixed else rng.randint(history // 8, history)
        new.append(n)
        total.append(before + n)
    return tuple(new), tuple(total)


def _shape(case):
    return _lengths(case["sequences"], case["chunk"], case["singles"], case["history"], case.get("fixed", False), case["lengths"])


def _pairs(new, total, window):
    """Visible (query, key) pairs of one sequence, and the distinct keys they touch."""
    first = total - new  # position of the first new token
    if window <= 0 or window >= total:
        return new * first + new * (new + 1) // 2, total
    full = max(0, total - max(first, window - 1))  # queries that see `window` keys
    short = new - full
    return full * window + short * first + short * (short + 1) // 2, total - max(0, first - window + 1)


def work(case):
    if case["op"] == "table":
        values = case["positions"] * (case["rotary"] // 2)
        return {"bytes": 8 * values, "flops": 4 * values}
    if case["op"] == "rotary":
        values = case["tokens"] * case["heads"] * case["head_dim"]
        rows = min(case["tokens"], case["table"])
        return {"bytes": 4 * values + rows * case["rotary"] * 4 + 4 * case["tokens"],
                "flops": 3 * case["tokens"] * case["heads"] * case["rotary"]}
    new, total = _shape(case)
    tokens, width = sum(new), case["heads"] * case["head_dim"]
    if case["op"] == "append":
        values = tokens * (case["heads"] + 2 * case["kv_heads"]) * case["head_dim"]
        return {"bytes": 4 * values + tokens * case["rotary"] * 4,
                "flops": 3 * tokens * (case["heads"] + case["kv_heads"]) * case["rotary"]}
    seen = [_pairs(n, t, case["window"]) for n, t in zip(new, total)]
    return {"bytes": 4 * tokens * width + 4 * tokens * case["heads"] + 4 * case["kv_heads"] * case["head_dim"] * sum(k for _, k in seen),
            "flops": 4 * case["head_dim"] * case["heads"] * sum(p for p, _ in seen)}


# ------------------------------------------------------------------------------------------ inputs
def _frequencies(case):
    """Radians a position of each pair (64 bits, CPU) and the amplitude of the table."""
    rotary, theta, factor, original = case["rotary"], case["theta"], case["factor"], case["original"]
    i = torch.arange(rotary // 2, dtype=torch.float64)
    f = torch.exp(i * (-2.0 * math.log(theta) / rotary))
    if case["kind"] == "none":
        return f, 1.0
    if case["kind"] == "linear":
        return f / factor, 1.0
    if case["kind"] == "bands":
        turns = original * f / (2.0 * math.pi)  # rotations over the original window
        mix = ((turns - case["low"]) / (case["high"] - case["low"])).clamp(0.0, 1.0)
        return mix * f + (1.0 - mix) * f / factor, 1.0
    low, high = (rotary * math.log(original / (2.0 * math.pi * b)) / (2.0 * math.log(theta)) for b in (case["high"], case["low"]))
    low, high = max(math.floor(low), 0), min(math.ceil(high), rotary - 1)
    ramp = ((i - low) / max(high - low, 0.001)).clamp(0.0, 1.0)
    return ramp * f / factor + (1.0 - ramp) * f, 0.1 * math.log(factor) + 1.0


def _table(positions, rotary, theta):
    angle = torch.arange(positions, dtype=torch.float64, device="cuda")[:, None] * torch.exp(
        torch.arange(rotary // 2, dtype=torch.float64, device="cuda") * (-2.0 * math.log(theta) / rotary))
    return angle.cos().float(), angle.sin().float()


def prepare(case, seed):
    """Everything but the table comes from the seed; the table's frequencies are the case's, moved a
    little by the seed as a model's own theta would move them."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    host = random.Random(seed)
    s = dict(case)
    s["status"] = torch.zeros(1, dtype=torch.int32, device="cuda")
    if case["op"] == "table":
        s["theta"] = float(torch.tensor(case["theta"] * host.uniform(0.9, 1.1), dtype=torch.float32))
        s["cos"] = torch.empty(case["positions"], case["rotary"] // 2, device="cuda")
        s["sin"] = torch.empty_like(s["cos"])
        return s
    dtype = TYPES[case["dtype"]]
    if case["op"] == "rotary":
        s["x"] = torch.randn(case["tokens"], case["heads"], case["head_dim"], generator=g, device="cuda", dtype=dtype)
        s["out"] = torch.empty_like(s["x"])
        s["positions"] = torch.randint(0, case["table"], (case["tokens"],), generator=g, device="cuda", dtype=torch.int32)
        s["cos"], s["sin"] = _table(case["table"], case["rotary"], 1e6)
        return s
    new, total = _shape(case)
    page, kv_heads, head_dim = case["page"], case["kv_heads"], case["head_dim"]
    counts = [-(-t // page) for t in total]
    pages = sum(counts)
    s["tokens"], s["max_new"], s["max_total"], s["pages"] = sum(new), max(new), max(total), pages
    offsets = torch.zeros(len(new) + 1, dtype=torch.int64)
    offsets[1:] = torch.tensor(new).cumsum(0)
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)  # pages lie anywhere in the pool
    table = torch.full((len(new), max(counts)), -1, dtype=torch.int32)
    filled = torch.arange(max(counts))[None, :] < torch.tensor(counts)[:, None]
    table = table.to("cuda")
    table[filled.to("cuda")] = order
    s["page_table"] = table
    s["q_offsets"], s["kv_lengths"] = offsets.to("cuda", torch.int32), torch.tensor(total, dtype=torch.int32).to("cuda")
    s["k_pages"] = torch.randn(pages, kv_heads, page, head_dim, generator=g, device="cuda", dtype=dtype)
    s["v_pages"] = torch.randn(pages, kv_heads, page, head_dim, generator=g, device="cuda", dtype=dtype)
    if case["op"] == "append":
        width = (case["heads"] + 2 * kv_heads) * head_dim
        s["qkv"] = torch.randn(s["tokens"], width, generator=g, device="cuda", dtype=dtype)
        s["bias_values"] = 0.1 * torch.randn(width, generator=g, device="cuda") if case["bias"] else None
        s["q_out"] = torch.empty(s["tokens"], case["heads"], head_dim, device="cuda", dtype=dtype)
        s["cos"], s["sin"] = _table(s["max_total"], case["rotary"], 1e6)
    else:
        s["q"] = 1.5 * torch.randn(s["tokens"], case["heads"], head_dim, generator=g, device="cuda", dtype=dtype)
        s["out"] = torch.empty_like(s["q"])
        s["lse"] = torch.empty(s["tokens"], case["heads"], device="cuda")
        s["workspace"] = torch.empty(WORKSPACE, dtype=torch.uint8, device="cuda")
    return s


# ------------------------------------------------------------------------------------- plain forms
def _rotate(x, cos, sin, interleaved):
    """x [..., rotary] rotated; cos, sin [..., rotary / 2] (32 bits)."""
    if interleaved:
        a, b = x[..., 0::2], x[..., 1::2]
        return torch.stack((a * cos - b * sin, b * cos + a * sin), dim=-1).flatten(-2)
    half = x.shape[-1] // 2
    a, b = x[..., :half], x[..., half:]
    return torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1)


def _plain_table(s):
    f, amplitude = _frequencies(s)
    angle = torch.arange(s["positions"], dtype=torch.float64, device="cuda")[:, None] * f.to("cuda")
    return {"cos": (amplitude * angle.cos()).float(), "sin": (amplitude * angle.sin()).float()}


def _plain_rotary(s):
    at = s["positions"].long()
    cos, sin = s["cos"][at][:, None], s["sin"][at][:, None]
    x, r = s["x"].float(), s["rotary"]
    turned = _rotate(x[..., :r], cos, -sin if s["inverse"] else sin, s["interleaved"])
    s["out"].copy_(torch.cat((turned, x[..., r:]), dim=-1))
    return {"out": s["out"]}


def _token_places(s):
    """Sequence and position of every new token."""
    offsets, lengths = s["q_offsets"].long(), s["kv_lengths"].long()
    token = torch.arange(s["tokens"], device="cuda")
    sequence = torch.searchsorted(offsets, token, right=True) - 1
    return sequence, token - offsets[sequence + 1] + lengths[sequence]


def _plain_append(s):
    heads, kv_heads, head_dim, r = s["heads"], s["kv_heads"], s["head_dim"], s["rotary"]
    x = s["qkv"].float()
    if s["bias_values"] is not None:
        x = x + s["bias_values"]
    x = x.view(s["tokens"], heads + 2 * kv_heads, head_dim)
    sequence, position = _token_places(s)
    cos, sin = s["cos"][position][:, None], s["sin"][position][:, None]
    turned = x[:, :heads + kv_heads]
    turned = torch.cat((_rotate(turned[..., :r], cos, sin, s["interleaved"]), turned[..., r:]), dim=-1).to(s["qkv"].dtype)
    page, slot = s["page_table"][sequence, position // s["page"]].long(), position % s["page"]
    s["q_out"].copy_(turned[:, :heads])
    s["k_pages"][page, :, slot] = turned[:, heads:]
    s["v_pages"][page, :, slot] = x[:, heads + kv_heads:].to(s["qkv"].dtype)
    return {"q": s["q_out"], "k_pages": s["k_pages"], "v_pages": s["v_pages"]}


def _plain_attention(s):
    heads, kv_heads, head_dim = s["heads"], s["kv_heads"], s["head_dim"]
    sequences, group, most = s["page_table"].shape[0], heads // kv_heads, s["max_new"]
    sequence, position = _token_places(s)
    row = torch.arange(s["tokens"], device="cuda") - s["q_offsets"].long()[sequence]
    q = torch.zeros(sequences, most, heads, head_dim, device="cuda")
    q[sequence, row] = s["q"].float()
    q = q.view(sequences, most, kv_heads, group, head_dim).permute(0, 2, 1, 3, 4).reshape(sequences, kv_heads, most * group, head_dim)
    at = s["page_table"].clamp(min=0).long()
    k = s["k_pages"][at].float().permute(0, 2, 1, 3, 4).reshape(sequences, kv_heads, -1, head_dim)
    scores = q @ k.transpose(2, 3)
    del k
    scores *= 1.0 / math.sqrt(head_dim)
    key = torch.arange(scores.shape[-1], device="cuda")
    query = (s["kv_lengths"] - s["q_offsets"].diff()).long()[:, None] + torch.arange(most, device="cuda")  # position of row i
    hidden = key[None, None] > query[..., None]
    if s["window"]:
        hidden |= key[None, None] <= query[..., None] - s["window"]
    scores.view(sequences, kv_heads, most, group, -1).masked_fill_(hidden[:, None, :, None], -math.inf)
    top = scores.amax(dim=-1, keepdim=True)
    scores -= top
    scores.exp_()
    total = scores.sum(dim=-1, keepdim=True)
    v = s["v_pages"][at].float().permute(0, 2, 1, 3, 4).reshape(sequences, kv_heads, -1, head_dim)
    out = (scores @ v) / total
    lse = (top + total.log()) * (1.0 / math.log(2.0))

    def rows(x):
        return x.view(sequences, kv_heads, most, group, -1).permute(0, 2, 1, 3, 4).reshape(sequences, most, heads, -1)[sequence, row]

    s["out"].copy_(rows(out))
    s["lse"].copy_(rows(lse)[..., 0])
    return {"out": s["out"], "lse": s["lse"]}


# ----------------------------------------------------------------------------------- this library
@functools.lru_cache(maxsize=1)
def _native():
    sys.path.insert(0, os.path.join(os.getcwd(), "attention-rank_b200"))
    from attnrank import _native as native
    return native


def _handles(s):
    """The descriptors that a serving loop keeps beside its cache and its batch's metadata."""
    native = _native()
    cache = native.PagedCacheStruct(s["k_pages"].data_ptr(), s["v_pages"].data_ptr(), s["pages"], s["page"], s["kv_heads"],
                                    s["head_dim"], CODES[s["dtype"]])
    batch = native.PagedBatchStruct(s["page_table"].shape[0], s["tokens"], s["max_new"], s["page_table"].shape[1],
                                    s["q_offsets"].data_ptr(), s["kv_lengths"].data_ptr(), s["page_table"].data_ptr())
    s["handles"] = ctypes.byref(cache), ctypes.byref(batch)
    return s["handles"]


def _own(s):
    native = _native()
    lib, check, stream = native.lib, native.check, torch.cuda.current_stream().cuda_stream
    if s["op"] == "table":
        scaling = native.RopeScalingStruct(s["theta"], s["rotary"], KINDS[s["kind"]], s["factor"], s["low"], s["high"],
                                           s["original"], 0.0)
        check(lib.ar_rope_table_scaled(ctypes.byref(scaling), s["positions"], s["cos"].data_ptr(), s["sin"].data_ptr(), stream))
        return {"cos": s["cos"], "sin": s["sin"]}
    if s["op"] == "rotary":
        row = s["heads"] * s["head_dim"]
        check(lib.ar_rotary_positions(s["x"].data_ptr(), row, s["head_dim"], s["out"].data_ptr(), row, s["head_dim"],
                                      s["positions"].data_ptr(), s["tokens"], s["heads"], s["head_dim"], s["rotary"],
                                      s["interleaved"], s["inverse"], s["cos"].data_ptr(), s["sin"].data_ptr(), s["table"],
                                      s["status"].data_ptr(), CODES[s["dtype"]], stream))
        return {"out": s["out"]}
    cache, batch = s.get("handles") or _handles(s)
    if s["op"] == "append":
        bias = s["bias_values"].data_ptr() if s["bias_values"] is not None else None
        check(lib.ar_paged_append(cache, batch, s["qkv"].data_ptr(), s["qkv"].shape[1], bias, s["heads"], s["q_out"].data_ptr(),
                                  s["heads"] * s["head_dim"], s["cos"].data_ptr(), s["sin"].data_ptr(), s["max_total"],
                                  s["rotary"], s["interleaved"], s["status"].data_ptr(), stream))
        return {"q": s["q_out"], "k_pages": s["k_pages"], "v_pages": s["v_pages"]}
    row = s["heads"] * s["head_dim"]
    check(lib.ar_paged_attention(cache, batch, s["q"].data_ptr(), row, s["heads"], 0.0, s["window"], s["out"].data_ptr(), row,
                                 s["lse"].data_ptr(), s["workspace"].data_ptr(), WORKSPACE, s["status"].data_ptr(), stream))
    return {"out": s["out"], "lse": s["lse"]}


def run(state):
    if own:
        return _own(state)
    return {"table": _plain_table, "rotary": _plain_rotary, "append": _plain_append, "attention": _plain_attention}[state["op"]](state)


# ------------------------------------------------------------------------------- exact, in 64 bits
def _turn(x, angle_cos, angle_sin, rotary, interleaved):
    """Each pair of x [tokens, heads, head_dim] as a complex number times cos + i sin."""
    y = x.clone()
    half = rotary // 2
    first = torch.arange(half, device="cuda") * (2 if interleaved else 1)
    second = first + (1 if interleaved else half)
    turned = torch.complex(x[..., first], x[..., second]) * torch.complex(angle_cos, angle_sin)[:, None]
    y[..., first], y[..., second] = turned.real, turned.imag
    return y


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "table":
        half, theta, out = case["rotary"] // 2, s["theta"], []
        amplitude = 0.1 * math.log(case["factor"]) + 1.0 if case["kind"] == "yarn" else 1.0
        for i in range(half):
            f = theta ** (-2.0 * i / case["rotary"])
            slow = f / case["factor"]
            if case["kind"] == "linear":
                f = slow
            elif case["kind"] == "bands":
                wavelength = 2.0 * math.pi / f
                if wavelength > case["original"] / case["low"]:
                    f = slow
                elif wavelength >= case["original"] / case["high"]:
                    part = (case["original"] / wavelength - case["low"]) / (case["high"] - case["low"])
                    f = part * f + (1.0 - part) * slow
            elif case["kind"] == "yarn":
                def index(turns):
                    return case["rotary"] * math.log(case["original"] / (2.0 * math.pi * turns)) / (2.0 * math.log(theta))
                low, high = max(math.floor(index(case["high"])), 0), min(math.ceil(index(case["low"])), case["rotary"] - 1)
                share = min(max((i - low) / max(high - low, 0.001), 0.0), 1.0)
                f = share * slow + (1.0 - share) * f
            out.append(f)
        angle = torch.outer(torch.arange(case["positions"], dtype=torch.float64), torch.tensor(out, dtype=torch.float64))
        return {"cos": amplitude * angle.cos(), "sin": amplitude * angle.sin()}
    if case["op"] == "rotary":
        at = s["positions"].long()
        sign = -1.0 if case["inverse"] else 1.0
        return {"out": _turn(s["x"].double(), s["cos"].double()[at], sign * s["sin"].double()[at], case["rotary"], case["interleaved"])}
    new, total = _shape(case)
    heads, kv_heads, page = case["heads"], case["kv_heads"], case["page"]
    k_pages, v_pages = s["k_pages"].double(), s["v_pages"].double()
    start, outs, sums = 0, [], []
    for b, (n, t) in enumerate(zip(new, total)):
        position = torch.arange(t - n, t, device="cuda")
        own_pages = s["page_table"][b, : -(-t // page)].long()
        if case["op"] == "append":
            x = s["qkv"][start:start + n].double()
            if case["bias"]:
                x = x + s["bias_values"].double()
            x = x.view(n, heads + 2 * kv_heads, -1)
            cos, sin = s["cos"].double()[position], s["sin"].double()[position]
            outs.append(_turn(x[:, :heads], cos, sin, case["rotary"], case["interleaved"]))
            where, slot = own_pages[position // page], position % page
            k_pages[where, :, slot] = _turn(x[:, heads:heads + kv_heads], cos, sin, case["rotary"], case["interleaved"])
            v_pages[where, :, slot] = x[:, heads + kv_heads:]
        else:
            key = torch.arange(t, device="cuda")
            hidden = key > position[:, None]
            if case["window"]:
                hidden |= key < position[:, None] - case["window"] + 1
            out, lse = [], []
            for h in range(heads):
                k = k_pages[own_pages, h * kv_heads // heads].reshape(-1, case["head_dim"])[:t]
                v = v_pages[own_pages, h * kv_heads // heads].reshape(-1, case["head_dim"])[:t]
                score = torch.mm(s["q"][start:start + n, h].double(), k.T) / math.sqrt(case["head_dim"])
                score = score.masked_fill(hidden, -math.inf)
                lse.append(torch.logsumexp(score, dim=1) / math.log(2.0))
                out.append(torch.softmax(score, dim=1) @ v)
            outs.append(torch.stack(out, dim=1))
            sums.append(torch.stack(lse, dim=1))
        start += n
    if case["op"] == "append":
        return {"q": torch.cat(outs), "k_pages": k_pages, "v_pages": v_pages}
    return {"out": torch.cat(outs), "lse": torch.cat(sums)}
