"""Timed cases of the MXFP4 operators: 4-bit weights and a 4-bit paged K/V cache.

MXFP4 holds 32 consecutive values x in 17 bytes: one power-of-two scale s (e8m0) and 32
e2m1 codes (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives), two to a byte, the even
element in the low nibble. s = 2^(floor(log2(max|x|)) - 2), between 2^-125 and 2^125, and
a code is x / s rounded to nearest, ties to the even code, at most 6.

A case is a dict of plain values; its kind says which operator it goes through:

  quantize  rows to MXFP4 and back: mxfp4_quantize, mxfp4_dequantize
  linear    a projection with MXFP4 weights, its rows quantized within: mxfp4_linear
  cache     new K/V rows into MXFP4 pools and the sequences read back: kv_append, paged_gather
  decode    one new token per sequence over MXFP4 pools: paged_attention_decode
  prefill   ragged chunks of prompts over MXFP4 pools: paged_attention_prefill

`run` computes them from elementary torch operations in 32 bits, or, where `own` is true,
through the package's entry points. What is held in 4 bits is returned as its values.
"""

from __future__ import annotations

import math
import random

import torch

own = False

DEVICE = "cuda"
DTYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
CODES, SCALES = torch.float4_e2m1fn_x2, torch.float8_e8m0fnu
BLOCK = 32


def listed() -> list[dict]:
    return [
        # The activations of a small decode batch, at an odd count of rows: latency.
        dict(name="quantize_rows_fp32", kind="quantize", dtype="float32", rows=33, cols=2048),
        # The stacked gate/up weights of the 1.1B model, quantized when a model is loaded.
        dict(name="quantize_weights_bf16", kind="quantize", dtype="bfloat16", rows=11264,
             cols=2048),
        # The QKV projection of one running request of the 1.1B model.
        dict(name="linear_token_bf16", kind="linear", dtype="bfloat16", rows=1, cols=2048,
             out=2560),
        # Its gate/up projection for a middling batch of running requests.
        dict(name="linear_decode_fp16", kind="linear", dtype="float16", rows=48, cols=2048,
             out=11264),
        # Its down projection in an iteration with a few ragged chunks.
        dict(name="linear_chunks_bf16", kind="linear", dtype="bfloat16", rows=777, cols=5632,
             out=2048),
        # A wide projection of a packed iteration of 16 chunks of 512 tokens.
        dict(name="linear_prefill_bf16", kind="linear", dtype="bfloat16", rows=8192, cols=4096,
             out=8192),
        # A small fp32 layer: the newest token of a handful of requests, then their keys.
        dict(name="cache_step_fp32", kind="cache", dtype="float32", seqs=8, min_new=1, max_new=1,
             max_prior=512, heads=8, kv_heads=2, head_dim=64, block_size=16, lengths=1),
        # Chunks of 512 tokens behind cached prefixes at the Llama-3-8B layer shape.
        dict(name="cache_chunks_bf16", kind="cache", dtype="bfloat16", seqs=16, min_new=1,
             max_new=512, max_prior=2048, heads=32, kv_heads=8, head_dim=128, block_size=16,
             lengths=2),
        # One layer of a decode iteration at serving load (128 requests of the 1.1B shape),
        # blocks of 32 tokens, sequences without a key among them.
        dict(name="decode_serving_fp16", kind="decode", dtype="float16", seqs=128, min_keys=0,
             max_keys=1152, log_keys=False, heads=32, kv_heads=4, head_dim=64, block_size=32,
             lengths=3),
        # Long and short contexts of a full batch at the Llama-3-8B layer shape, the headline
        # batch of bench.py.
        dict(name="decode_long_bf16", kind="decode", dtype="bfloat16", seqs=256, min_keys=128,
             max_keys=8192, log_keys=True, heads=32, kv_heads=8, head_dim=128, block_size=16,
             lengths=0),
        # A few ragged chunks, odd ones among them, in fp32.
        dict(name="prefill_ragged_fp32", kind="prefill", dtype="float32", seqs=5, min_new=1,
             max_new=333, max_prior=1024, heads=32, kv_heads=4, head_dim=64, block_size=16,
             lengths=4),
        # Chunked prefill of a mixed iteration: chunks of 512 tokens behind cached prefixes.
        dict(name="prefill_chunks_bf16", kind="prefill", dtype="bfloat16", seqs=16, min_new=512,
             max_new=512, max_prior=2048, heads=32, kv_heads=8, head_dim=128, block_size=16,
             lengths=5),
    ]


def _between(rng: random.Random, low: int, high: int) -> int:
    """An integer of [low, high], uniform over its logarithm."""

    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


# (query heads, KV heads, head_dim) of the layers served: the small fp32 layer, the 1.1B
# layer and the Llama-3-8B layer, and one whose head is neither 64 nor 128 values.
LAYERS = ((8, 2, 64), (32, 4, 64), (32, 8, 128), (16, 4, 96))


def _draw_once(rng: random.Random) -> dict:
    kind = rng.choice(("quantize", "linear", "linear", "linear", "cache", "decode", "decode",
                       "prefill"))
    dtype = rng.choice(("bfloat16", "bfloat16", "float16", "float32"))
    if kind in ("quantize", "linear"):
        cols = BLOCK * _between(rng, 1, 176)
        case = dict(kind=kind, dtype=dtype, rows=_between(rng, 1, 8192), cols=cols)
        return case | ({"out": _between(rng, 1, 11264)} if kind == "linear" else {})
    heads, kv_heads, head_dim = rng.choice(LAYERS)
    case = dict(kind=kind, dtype=dtype, heads=heads, kv_heads=kv_heads, head_dim=head_dim,
                block_size=rng.choice((16, 16, 32, 5)), lengths=rng.randrange(1 << 30))
    if kind == "decode":
        high = _between(rng, 16, 8192)
        low = rng.choice((0, 1, min(high, 128)))
        return case | dict(seqs=_between(rng, 1, 256), min_keys=low, max_keys=high,
                           log_keys=low > 0 and rng.random() < 0.5)
    high = _between(rng, 1, 512)
    return case | dict(seqs=_between(rng, 1, 16), min_new=rng.randint(1, high), max_new=high,
                       max_prior=rng.choice((0, _between(rng, 16, 4096))))


def draw(rng: random.Random) -> dict:
    """A case of the listed ranges that costs no more than the largest listed one of its kind."""

    while True:
        case = _draw_once(rng)
        alike = [work(c) for c in listed() if c["kind"] == case["kind"]]
        cost = work(case)
        if all(cost[m] <= max(w[m] for w in alike) for m in ("bytes", "flops")):
            return case


# ------------------------------------------------------------------ lengths


def _lengths(case: dict) -> list[int]:
    """Keys of each decode sequence (its new token's among them)."""

    rng = random.Random(case["lengths"])
    low, high = case["min_keys"], case["max_keys"]
    if case["log_keys"]:
        return [_between(rng, low, high) for _ in range(case["seqs"])]
    return [rng.randint(low, high) for _ in range(case["seqs"])]


def _chunks(case: dict) -> list[tuple[int, int]]:
    """(new tokens, cached tokens before them) of each sequence."""

    rng = random.Random(case["lengths"])
    return [(rng.randint(case["min_new"], case["max_new"]), rng.randint(0, case["max_prior"]))
            for _ in range(case["seqs"])]


def work(case: dict) -> dict:
    """Bytes (inputs read once, outputs written once) and operations of one pass."""

    kind = case["kind"]
    elem = 4 if case["dtype"] == "float32" else 2
    packed = 17 / 32  # bytes of a value in MXFP4
    if kind == "quantize":
        n = case["rows"] * case["cols"]
        return {"bytes": n * (2 * elem + packed), "flops": 2 * n}
    if kind == "linear":
        m, k, n = case["rows"], case["cols"], case["out"]
        return {"bytes": elem * m * (k + n) + packed * n * k, "flops": 2 * m * k * n}
    row = 2 * case["kv_heads"] * case["head_dim"]  # values of a token's K and V rows
    q_row = case["heads"] * case["head_dim"]
    if kind == "decode":
        keys = sum(_lengths(case))
        return {"bytes": keys * row * packed + 2 * case["seqs"] * q_row * elem,
                "flops": 4 * keys * q_row}
    chunks = _chunks(case)
    new, keys = sum(t for t, _ in chunks), sum(t + p for t, p in chunks)
    if kind == "cache":
        # New rows in, their codes out; every row's codes in, its values out.
        return {"bytes": row * (new * (elem + packed) + keys * (packed + elem)),
                "flops": 2 * row * (new + keys)}
    return {"bytes": keys * row * packed + 2 * new * q_row * elem,
            "flops": 4 * q_row * sum(t * p + t * (t + 1) // 2 for t, p in chunks)}


# -------------------------------------------------------------- plain forms


def _scale_values(scales: torch.Tensor) -> torch.Tensor:
    """2^(byte - 127) of e8m0 bytes from 1 to 254, from its bits."""

    return (scales.int() << 23).view(torch.float32)


def _plain_quantize(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(..., K) finite values to packed codes (..., K/2) and scale bytes (..., K/32)."""

    blocks = x.float().unflatten(-1, (-1, BLOCK))
    largest = blocks.abs().amax(dim=-1)
    exponent = torch.frexp(largest).exponent - 1  # of a zero block: replaced below
    scales = torch.where(largest > 0, exponent + 125, 2).clamp(2, 252)
    scaled = blocks / _scale_values(scales).unsqueeze(-1)
    size = scaled.abs()
    # Borders between neighbouring codes: an even code's own, an odd code's neighbours'.
    codes = ((size > 0.25).to(torch.uint8) + (size >= 0.75) + (size > 1.25) + (size >= 1.75)
             + (size > 2.5) + (size >= 3.5) + (size > 5.0))
    codes = (codes | (torch.signbit(scaled).to(torch.uint8) << 3)).flatten(-2)
    return codes[..., 0::2] | (codes[..., 1::2] << 4), scales.to(torch.uint8)


def _plain_values(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """The fp32 values of packed codes and scale bytes."""

    table = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0,
                          -3.0, -4.0, -6.0], device=codes.device)
    pair = torch.stack((codes & 15, codes >> 4), dim=-1).flatten(-2)
    values = table[pair.int()].unflatten(-1, (-1, BLOCK))
    return (values * _scale_values(scales).unsqueeze(-1)).flatten(-2)


def _plain_rows(state: dict, name: str, width: int) -> torch.Tensor:
    """The first `width` positions behind every block table in fp32, (B, width, Hkv, Dh)."""

    blocks = state["block_tables"].long()
    codes = state[name + "_cache"].view(torch.uint8)[0][blocks]  # (B, W, Hkv, BS, Dh/2)
    scales = state[name[0] + "_scales"].view(torch.uint8)[0][blocks]
    rows = _plain_values(codes, scales).transpose(2, 3)
    return rows.flatten(1, 2)[:, :width]


def _plain_attention(query: torch.Tensor, state: dict, last: torch.Tensor) -> torch.Tensor:
    """query (B, T, Hq, Dh) fp32 over keys 0 .. last (B, T) of each row, none where it is -1."""

    b, t, hq, dh = query.shape
    keys, values = (_plain_rows(state, name, state["max_seq_len"]) for name in ("key", "value"))
    s, hkv = keys.shape[1:3]
    g = hq // hkv
    q = query.view(b, t, hkv, g, dh).permute(0, 2, 3, 1, 4).reshape(b * hkv, g * t, dh)
    k = keys.permute(0, 2, 3, 1).reshape(b * hkv, dh, s)
    v = values.permute(0, 2, 1, 3).reshape(b * hkv, s, dh)
    scores = torch.bmm(q, k).view(b, hkv, g, t, s) / math.sqrt(dh)
    seen = torch.arange(s, device=query.device) <= last.unsqueeze(-1)  # (B, T, S)
    scores = scores.masked_fill(~seen[:, None, None], -math.inf)
    largest = scores.amax(dim=-1, keepdim=True)
    weights = torch.exp(scores - torch.where(largest == -math.inf, 0.0, largest))
    total = weights.sum(dim=-1, keepdim=True)
    out = torch.bmm(weights.view(b * hkv, g * t, s), v).view(b, hkv, g, t, dh)
    out = torch.where(total > 0, out / total, 0.0)
    return out.permute(0, 3, 1, 2, 4).reshape(b, t, hq, dh)


# ------------------------------------------------------------------ inputs


class _Values:
    """Seeded inputs, drawn on the device."""

    def __init__(self, seed: int) -> None:
        self.rng = torch.Generator(device=DEVICE).manual_seed(seed)
        self.host = torch.Generator().manual_seed(seed)

    def normal(self, *shape: int) -> torch.Tensor:
        return torch.randn(shape, generator=self.rng, device=DEVICE)

    def rows(self, *shape: int) -> torch.Tensor:
        """Activations: rows of different sizes, a few of their columns larger than the rest."""

        size = torch.exp2(3.0 * torch.rand((*shape[:-1], 1), generator=self.rng, device=DEVICE))
        large = torch.rand(shape[-1:], generator=self.rng, device=DEVICE) < 0.02
        return self.normal(*shape) * size * torch.where(large, 8.0, 1.0)

    def tables(self, counts: list[int]) -> tuple[torch.Tensor, int]:
        """Disjoint block tables (B, W) out of one random order of the pool's blocks."""

        total = sum(counts)
        order = torch.randperm(total, generator=self.host).to(torch.int32)
        tables = torch.zeros((len(counts), max(max(counts), 1)), dtype=torch.int32)
        start = 0
        for b, count in enumerate(counts):
            tables[b, :count] = order[start:start + count]
            start += count
        return tables, max(total, 1)


def _sequences(case: dict, values: _Values, keys: list[int]) -> dict:
    """Pools that hold `keys[b]` positions of sequence b, their tables and lengths."""

    bs = case["block_size"]
    tables, blocks = values.tables([-(-n // bs) for n in keys])
    state = {"block_tables": tables.to(DEVICE), "host_tables": tables,
             "seq_lens": torch.tensor(keys, dtype=torch.int32, device=DEVICE),
             "max_seq_len": max(max(keys), 1)}
    for name in ("key", "value"):
        rows = values.rows(1, blocks, case["kv_heads"], bs, case["head_dim"])
        codes, scales = _plain_quantize(rows)
        state[name + "_cache"] = codes.view(CODES)
        state[name[0] + "_scales"] = scales.view(SCALES)
    order = sorted(range(len(keys)), key=lambda b: (-keys[b], b))
    state["seq_order"] = torch.tensor(order, dtype=torch.int32, device=DEVICE)
    return state


def prepare(case: dict, seed: int) -> dict:
    kind, dtype = case["kind"], DTYPES[case["dtype"]]
    values = _Values(seed)
    if kind == "quantize":
        x = values.rows(case["rows"], case["cols"]).to(dtype)
        return {"case": case, "inputs": x, "out": torch.empty_like(x)}
    if kind == "linear":
        codes, scales = _plain_quantize(values.normal(case["out"], case["cols"])
                                        / math.sqrt(case["cols"]))
        return {"case": case, "inputs": values.rows(case["rows"], case["cols"]).to(dtype),
                "codes": codes.view(CODES), "scales": scales.view(SCALES),
                "out": torch.empty((case["rows"], case["out"]), dtype=dtype, device=DEVICE)}
    if kind == "decode":
        keys = _lengths(case)
        state = _sequences(case, values, keys)
        shape = (len(keys), case["heads"], case["head_dim"])
    else:
        chunks = _chunks(case)
        state = _sequences(case, values, [t + p for t, p in chunks])
        new = [t for t, _ in chunks]
        cu = torch.tensor([0, *new]).cumsum(0)
        sequence = torch.repeat_interleave(torch.arange(len(new)), torch.tensor(new))
        index = torch.arange(sum(new)) - cu[sequence]  # of a token in its chunk
        position = index + torch.tensor([p for _, p in chunks])[sequence]
        state.update(cu_seqlens_q=cu.to(torch.int32).to(DEVICE), max_query_len=max(new),
                     sequence=sequence.to(DEVICE), index=index.to(DEVICE),
                     position=position.to(DEVICE))
        shape = (sum(new), case["heads"], case["head_dim"])
    if kind == "cache":
        bs, total = case["block_size"], sum(t + p for t, p in _chunks(case))
        slots = state["host_tables"][sequence, position // bs] * bs + position % bs
        state["slots"] = slots.to(torch.int64).to(DEVICE)
        cu = torch.zeros(case["seqs"] + 1, dtype=torch.int32, device=DEVICE)
        cu[1:] = state["seq_lens"].cumsum(0)
        state["cu_seqlens"] = cu
        row = torch.arange(total, device=DEVICE)
        state["row_sequence"] = torch.repeat_interleave(
            torch.arange(case["seqs"], device=DEVICE), state["seq_lens"].long())
        state["row_position"] = row - cu[state["row_sequence"]]
        for name in ("key", "value"):
            state[name] = values.rows(shape[0], case["kv_heads"], case["head_dim"]).to(dtype)
            state[name + "_out"] = torch.empty((total, case["kv_heads"], case["head_dim"]),
                                               dtype=dtype, device=DEVICE)
    else:
        state["query"] = values.normal(*shape).to(dtype)
        state["out"] = torch.empty_like(state["query"])
    state["case"] = case
    return state


# --------------------------------------------------------------------- run


def _plain(state: dict):
    case = state["case"]
    kind, dtype = case["kind"], DTYPES[case["dtype"]]
    if kind == "quantize":
        return _plain_values(*_plain_quantize(state["inputs"])).to(dtype)
    if kind == "linear":
        x = _plain_values(*_plain_quantize(state["inputs"]))
        weight = _plain_values(state["codes"].view(torch.uint8), state["scales"].view(torch.uint8))
        return (x @ weight.t()).to(dtype)
    if kind == "cache":
        bs = case["block_size"]
        blocks, rows = state["slots"] // bs, state["slots"] % bs
        k_codes, k_scales = _plain_quantize(state["key"])
        v_codes, v_scales = _plain_quantize(state["value"])
        state["key_cache"].view(torch.uint8)[0][blocks, :, rows] = k_codes
        state["k_scales"].view(torch.uint8)[0][blocks, :, rows] = k_scales
        state["value_cache"].view(torch.uint8)[0][blocks, :, rows] = v_codes
        state["v_scales"].view(torch.uint8)[0][blocks, :, rows] = v_scales
        at = state["row_sequence"], state["row_position"]
        return tuple(_plain_rows(state, name, state["max_seq_len"])[at].to(dtype)
                     for name in ("key", "value"))
    if kind == "decode":
        last = state["seq_lens"].long().unsqueeze(1) - 1
        return _plain_attention(state["query"].float().unsqueeze(1), state, last)[:, 0].to(dtype)
    # Chunks side by side, padded to the longest; padding tokens see the first key.
    b, t = case["seqs"], state["max_query_len"]
    query = torch.zeros((b, t, case["heads"], case["head_dim"]), device=DEVICE)
    query[state["sequence"], state["index"]] = state["query"].float()
    last = torch.zeros((b, t), dtype=torch.int64, device=DEVICE)
    last[state["sequence"], state["index"]] = state["position"]
    return _plain_attention(query, state, last)[state["sequence"], state["index"]].to(dtype)


def run(state: dict):
    if not own:
        return _plain(state)
    from tokserve_amd.kernels import ops

    kind = state["case"]["kind"]
    if kind == "quantize":
        codes, scales = ops.mxfp4_quantize(state["inputs"])
        return ops.mxfp4_dequantize(codes, scales, state["inputs"].dtype, out=state["out"])
    if kind == "linear":
        return ops.mxfp4_linear(state["inputs"], state["codes"], state["scales"],
                                out=state["out"])
    scales = {"k_scales": state["k_scales"], "v_scales": state["v_scales"]}
    pools = state["key_cache"], state["value_cache"]
    if kind == "cache":
        ops.kv_append(state["key"], state["value"], *pools, state["slots"], 0, **scales)
        ops.paged_gather(*pools, state["block_tables"], state["seq_lens"], state["cu_seqlens"], 0,
                         state["max_seq_len"], state["key_out"], state["value_out"], **scales)
        return state["key_out"], state["value_out"]
    if kind == "decode":
        return ops.paged_attention_decode(
            state["query"], *pools, state["block_tables"], state["seq_lens"], layer_index=0,
            max_seq_len=state["max_seq_len"], out=state["out"], seq_order=state["seq_order"],
            **scales)
    return ops.paged_attention_prefill(
        state["query"], *pools, state["block_tables"], state["seq_lens"], state["cu_seqlens_q"],
        layer_index=0, max_query_len=state["max_query_len"], max_seq_len=state["max_seq_len"],
        out=state["out"], seq_order=state["seq_order"], **scales)


# ------------------------------------------------------------------- exact


def _exact_rounded(x: torch.Tensor) -> torch.Tensor:
    """The values that (..., K) finite numbers have in MXFP4, in 64 bits."""

    blocks = x.double().unflatten(-1, (-1, BLOCK))
    largest = blocks.abs().amax(dim=-1, keepdim=True)
    power = torch.log2(torch.where(largest > 0, largest, 1.0)).floor()
    # log2 may round across a power of two: one step either way.
    power = power - (torch.exp2(power) > largest).double()
    power = power + (torch.exp2(power + 1.0) <= largest).double()
    scale = torch.exp2((power - 2.0).clamp(-125.0, 125.0))
    scaled = blocks / scale
    size = scaled.abs()
    step = torch.where(size < 2.0, 0.5, torch.where(size < 4.0, 1.0, 2.0)).double()
    size = (torch.round(size / step) * step).clamp(max=6.0)
    return (torch.copysign(size, scaled) * scale).flatten(-2)


def _exact_values(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """The values of packed codes and scale bytes, in 64 bits."""

    raw, power = codes.view(torch.uint8).int(), scales.view(torch.uint8).double() - 127.0
    raw = torch.stack((raw % 16, raw // 16), dim=-1).flatten(-2)
    magnitude = raw % 8
    exponent, mantissa = magnitude // 2, (magnitude % 2).double()
    value = torch.where(exponent > 0, (1.0 + mantissa / 2) * torch.exp2(exponent.double() - 1.0),
                        mantissa / 2)
    value = torch.where(raw >= 8, -value, value).unflatten(-1, (-1, BLOCK))
    return (value * torch.exp2(power).unsqueeze(-1)).flatten(-2)


def _exact_attention(query: torch.Tensor, keys: torch.Tensor, values: torch.Tensor):
    """query (T, Hq, Dh), the last T positions of keys and values (S, Hkv, Dh): causal."""

    t, hq, dh = query.shape
    s, hkv, _ = keys.shape
    g = hq // hkv
    q = query.view(t, hkv, g, dh).permute(1, 2, 0, 3).reshape(hkv, g * t, dh)
    scores = (q @ keys.permute(1, 2, 0).contiguous()).view(hkv, g, t, s) / math.sqrt(dh)
    hidden = torch.ones(t, s, dtype=torch.bool, device=query.device).triu(s - t + 1)
    probs = scores.masked_fill_(hidden, -math.inf).softmax(dim=-1).view(hkv, g * t, s)
    out = probs @ values.permute(1, 0, 2).contiguous()
    return out.view(hkv, g, t, dh).permute(2, 0, 1, 3).reshape(t, hq, dh)


def exact(case: dict, seed: int):
    kind = case["kind"]
    state = prepare(case, seed)
    if kind == "quantize":
        return _exact_rounded(state["inputs"])
    if kind == "linear":
        weight = _exact_values(state["codes"], state["scales"])
        return _exact_rounded(state["inputs"]) @ weight.t()
    bs = case["block_size"]
    pools = {name: _exact_values(state[name + "_cache"], state[name[0] + "_scales"])[0]
             for name in ("key", "value")}
    if kind == "cache":
        out = []
        for name, pool in pools.items():
            pool[state["slots"] // bs, :, state["slots"] % bs] = _exact_rounded(state[name])
            blocks = state["block_tables"].long()[state["row_sequence"],
                                                  state["row_position"] // bs]
            out.append(pool[blocks, :, state["row_position"] % bs])
        return tuple(out)
    out = state["query"].double()
    lengths = _lengths(case) if kind == "decode" else [t + p for t, p in _chunks(case)]
    counts = [1] * len(lengths) if kind == "decode" else [t for t, _ in _chunks(case)]
    start = 0
    for b, (length, count) in enumerate(zip(lengths, counts)):
        blocks = state["block_tables"][b, :-(-length // bs)].long()
        keys, vals = (pools[name][blocks].transpose(1, 2).flatten(0, 1)[:length]
                      for name in ("key", "value"))
        rows = out[start:start + count]
        rows.copy_(_exact_attention(rows.clone(), keys, vals) if length else torch.zeros_like(rows))
        start += count
    return out
