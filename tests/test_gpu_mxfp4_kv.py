"""MXFP4 K/V pools on the GPU: appends and the gather against the CPU definition
(oracle/mxfp4.py) bit for bit, attention against 64-bit attention of the decoded values.

Attention's tolerance, with A = sum p |v| of an output value: the scores are fp32 sums of Dh
products, off by at most (Dh + 8) 2^-23 of the sum of their magnitudes, and a probability by
that (times two, its own and the sum's); 2^x is good to 2^-22 and the sums of n keys to
(n / 32 + 32) 2^-23. A probability is rounded to the parts that the second product takes,
half a step of `P_STEP`; the result half a step of its type.
"""

import pytest
import torch

from oracle import mxfp4
from tokserve_amd.engine.paged.storage import PagedKVStorage
from tokserve_amd.kernels import ops

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]
CODES, SCALES = torch.float4_e2m1fn_x2, torch.float8_e8m0fnu


class Pool:
    """Pools of one or more layers with sequences in blocks of a random order; every unused
    row holds NaN scales and random codes."""

    def __init__(self, lengths, hkv, dh, block_size, device, seed=0, layers=1, layer=0,
                 extra_width=0, spread=3):
        g = torch.Generator().manual_seed(seed)
        counts = [-(-n // block_size) for n in lengths]
        blocks = sum(counts) + 2
        order = torch.randperm(blocks, generator=g)
        self.tables = torch.zeros(len(lengths), max([1, *counts]) + extra_width, dtype=torch.int32)
        shape = (layers, blocks, hkv, block_size)
        codes = [torch.randint(0, 256, (*shape, dh // 2), generator=g, dtype=torch.uint8)
                 for _ in range(2)]
        scales = [torch.full((*shape, dh // 32), 255, dtype=torch.uint8) for _ in range(2)]
        self.rows = []  # per sequence: K and V (n, Hkv, Dh) as float64
        at = 0
        for b, n in enumerate(lengths):
            self.tables[b, :counts[b]] = order[at:at + counts[b]]
            at += counts[b]
            block = self.tables[b].long()[torch.arange(n) // block_size]
            offset = torch.arange(n) % block_size
            pair = []
            for c, s in zip(codes, scales):
                x = torch.randn(n, hkv, dh, generator=g)
                x = x * 2.0 ** (spread * torch.rand(n, hkv, 1, generator=g) - spread / 2)
                x_codes, x_scales = mxfp4.quantize(x)
                c[layer][block, :, offset] = x_codes
                s[layer][block, :, offset] = x_scales
                pair.append(mxfp4.values(x_codes, x_scales))
            self.rows.append(pair)
        self.key, self.value = (c.to(device).view(CODES) for c in codes)
        self.scales = {"k_scales": scales[0].to(device).view(SCALES),
                       "v_scales": scales[1].to(device).view(SCALES)}
        self.lens = torch.tensor(lengths, dtype=torch.int32, device=device)
        self.block_tables = self.tables.to(device)
        self.layer = layer


P_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -22}


def _check_attention(got, query, keys, vals, scale=None):
    """got (T, Hq, Dh) against 64-bit attention of query over keys and vals (S, Hkv, Dh)."""

    if keys.shape[0] == 0:
        assert not got.any()
        return
    exact, size, scores = mxfp4.attention(query, keys, vals, scale)
    dh, n, dtype = query.shape[-1], keys.shape[0], got.dtype
    share = (2 * (dh + 8) * scores + n / 32 + 32) * 2.0 ** -23 + 2.0 ** -22
    limit = (share[..., None] + P_STEP[dtype]) * size + torch.finfo(dtype).eps / 2 * exact.abs()
    error = (got.cpu().double() - exact).abs()
    assert bool((error <= limit + torch.finfo(dtype).tiny).all()), (error / limit).max()


# ------------------------------------------------------------------ the cache


def _slots(pool, block_size, starts, counts):
    out = []
    for b, (start, count) in enumerate(zip(starts, counts)):
        p = torch.arange(start, start + count)
        out.append(pool.tables[b].long()[p // block_size] * block_size + p % block_size)
    return torch.cat(out)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dh,block_size", [(32, 16), (64, 16), (96, 5), (128, 32), (128, 1)])
def test_append_and_gather(device, dtype, dh, block_size) -> None:
    """Rows land in their slots and nowhere else, negative and foreign slots nowhere; the
    gather reads the values back."""

    lengths, hkv = [37, 1, 0, 64], 3
    pool = Pool(lengths, hkv, dh, block_size, device, layers=2, layer=1)
    g = torch.Generator().manual_seed(dh)
    new = [torch.randn(12, hkv, dh, generator=g).to(dtype) for _ in range(2)]
    new[0][2, 1, 3] = float("nan")
    new[1][4, 0] = 0.0
    slots = _slots(pool, block_size, [30, 0, 0, 60], [7, 1, 0, 4])
    slots[5], slots[9] = -1, pool.key.shape[1] * block_size
    want = [pool.key.view(torch.uint8).cpu(), pool.value.view(torch.uint8).cpu()]
    want_scales = [s.view(torch.uint8).cpu() for s in pool.scales.values()]
    kept = [t for t in range(12) if t not in (5, 9)]
    for x, codes, scales in zip(new, want, want_scales):
        x_codes, x_scales = mxfp4.quantize(x[kept])
        at = slots[kept]
        codes[1][at // block_size, :, at % block_size] = x_codes
        scales[1][at // block_size, :, at % block_size] = x_scales
    # (rows of a wider buffer, as a fused projection leaves them)
    wide = torch.cat((new[0], new[1]), dim=1).to(device)
    ops.kv_append(wide[:, :hkv], wide[:, hkv:], pool.key, pool.value, slots.to(device), 1,
                  **pool.scales)
    for got, codes in zip((pool.key, pool.value), want):
        assert torch.equal(got.view(torch.uint8).cpu(), codes)
    for got, scales in zip(pool.scales.values(), want_scales):
        assert torch.equal(got.view(torch.uint8).cpu(), scales)

    total = sum(lengths)
    cu = torch.tensor([0, *torch.tensor(lengths).cumsum(0).tolist()[:-1], total], dtype=torch.int32)
    out = torch.full((2, total + 2, hkv, dh), 7.0, dtype=dtype, device=device)
    ops.paged_gather(pool.key, pool.value, pool.block_tables, pool.lens, (cu + 1).to(device), 1,
                     max(lengths), out[0], out[1], **pool.scales)
    for side, codes, scales in zip(out.cpu(), want, want_scales):
        rows = []
        for b, n in enumerate(lengths):
            p = torch.arange(n)
            at = pool.tables[b].long()[p // block_size], p % block_size
            rows.append(mxfp4.values(codes[1][at[0], :, at[1]], scales[1][at[0], :, at[1]]))
        torch.testing.assert_close(side[1:-1], torch.cat(rows).to(dtype), rtol=0, atol=0,
                                   equal_nan=True)
        assert bool((side[0] == 7.0).all()) and bool((side[-1] == 7.0).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dh", [32, 64, 96, 128])
@pytest.mark.parametrize("in_place", [True, False])
def test_rope_append_is_rope_then_append(device, dtype, dh, in_place) -> None:
    hq, hkv, n, block_size = 6, 2, 9, 4
    g = torch.Generator().manual_seed(dh)
    query, key, value = (torch.randn(n, h, dh, generator=g).to(dtype).to(device)
                         for h in (hq, hkv, hkv))
    positions = torch.tensor([0, 1, 2, 7, 3, 900, 77, 50, 4], device=device)
    table = ops.RotaryTable(dh, theta=1e4, max_position=1000, dtype=dtype, device=device)
    slots = torch.tensor([0, 5, -1, 9, 2, 11, 3, 7, 8], device=device)
    storages = [PagedKVStorage(num_layers=1, num_blocks=3, num_key_value_heads=hkv, device=device,
                               block_size=block_size, head_dim=dh, dtype=dtype, kv_dtype=CODES)
                for _ in range(2)]
    for s in storages:
        for t in (s.key_storage, s.value_storage, s.key_scales, s.value_scales):
            t.view(torch.uint8).fill_(77)
    rotated_q, rotated_k = ops.rope(query.transpose(0, 1)[None], key.transpose(0, 1)[None],
                                    positions, table)
    rotated_q, rotated_k = (x[0].transpose(0, 1) for x in (rotated_q, rotated_k))
    storages[0].write_slots(0, slots, rotated_k, value)
    q_out = None if in_place else torch.zeros_like(query)
    k_out = key if in_place else torch.zeros_like(key)
    got = ops.rope_kv_append(query, key, value, positions, table, storages[1].key_storage,
                             storages[1].value_storage, slots, 0, query_out=q_out, key_out=k_out,
                             **storages[1].scales)
    assert torch.equal(got, rotated_q) and torch.equal(k_out, rotated_k)
    for name in ("key_storage", "value_storage", "key_scales", "value_scales"):
        assert torch.equal(getattr(storages[0], name).view(torch.uint8),
                           getattr(storages[1], name).view(torch.uint8)), name


# -------------------------------------------------------------------- decode

LENGTHS = [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 200, 333, 517]
LAYOUTS = [(8, 2, 64, 16), (32, 4, 64, 32), (32, 8, 128, 16), (16, 1, 128, 48), (4, 4, 32, 16),
           (6, 2, 96, 16), (8, 8, 96, 5), (8, 2, 128, 1), (4, 2, 64, 7), (3, 1, 32, 3)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq,hkv,dh,block_size", LAYOUTS)
def test_decode(device, dtype, hq, hkv, dh, block_size) -> None:
    """Every length around a tile's and a page's end, unsplit and in splits of a few blocks."""

    pool = Pool(LENGTHS, hkv, dh, block_size, device, seed=dh + hq, layers=2, layer=1,
                extra_width=3)
    g = torch.Generator().manual_seed(7)
    query = torch.randn(len(LENGTHS), hq, dh, generator=g).to(dtype)
    wide = torch.cat((query, query), dim=1).to(device)
    for pages in (0, max(1, 64 // block_size), 10_000):
        out = ops.paged_attention_decode(
            wide[:, :hq], pool.key, pool.value, pool.block_tables, pool.lens, layer_index=1,
            max_seq_len=max(LENGTHS), pages_per_split=pages,
            seq_order=ops.longest_first(LENGTHS, device) if pages else None, **pool.scales)
        for b in range(len(LENGTHS)):
            _check_attention(out[b:b + 1], query[b:b + 1], *pool.rows[b])


@pytest.mark.parametrize("dtype", DTYPES)
def test_decode_of_long_sequences(device, dtype) -> None:
    lengths = [4097, 8192, 2000]
    pool = Pool(lengths, 2, 128, 16, device, seed=3)
    query = torch.randn(3, 8, 128, generator=torch.Generator().manual_seed(1)).to(dtype)
    out = ops.paged_attention_decode(query.to(device), pool.key, pool.value, pool.block_tables,
                                     pool.lens, layer_index=0, max_seq_len=8192, **pool.scales)
    for b in range(3):
        _check_attention(out[b:b + 1], query[b:b + 1], *pool.rows[b])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("block_size,pages,bound", [(16, 600, 9000), (48, 0, 9000), (5, 2000, 9000),
                                                    (100, 0, 2100), (32, 0, 12288), (16, 0, 2048)])
def test_decode_of_long_splits(device, dtype, block_size, pages, bound) -> None:
    """Splits of thousands of keys (a wave's tiles pass one look-up of pages), and the bound's
    own choice, of every kind of block."""

    lengths = [min(n, bound) for n in (9000, 4096, 4097, 2047, 31, 0)]
    pool = Pool(lengths, 1, 64, block_size, device, seed=bound + block_size,
                extra_width=-(-bound // block_size) - -(-max(lengths) // block_size))
    query = torch.randn(6, 3, 64, generator=torch.Generator().manual_seed(2)).to(dtype)
    out = ops.paged_attention_decode(query.to(device), pool.key, pool.value, pool.block_tables,
                                     pool.lens, layer_index=0, max_seq_len=bound,
                                     pages_per_split=pages, **pool.scales)
    for b in range(6):
        _check_attention(out[b:b + 1], query[b:b + 1], *pool.rows[b])


@pytest.mark.parametrize("dtype", DTYPES)
def test_decode_of_extreme_values(device, dtype) -> None:
    """Scores far apart (a reference that moves late), a zero query, a negative scale, and
    NaN or infinite inputs in one sequence, which stay in it."""

    lengths = [300, 300, 300, 300, 100]
    pool = Pool(lengths, 1, 64, 16, device, seed=4, spread=8)
    query = torch.randn(5, 4, 64, generator=torch.Generator().manual_seed(2))
    query[0] *= 30.0
    query[1] = 0.0
    query[3, 2, 7] = float("nan")
    query[4, 1, 0] = float("inf")
    query = query.to(dtype)
    for scale in (None, -0.3):
        out = ops.paged_attention_decode(query.to(device), pool.key, pool.value, pool.block_tables,
                                         pool.lens, layer_index=0, max_seq_len=300, scale=scale,
                                         **pool.scales).cpu()
        for b in range(3):
            _check_attention(out[b:b + 1], query[b:b + 1], *pool.rows[b], scale)
        assert torch.isnan(out[3, 2]).all() and not torch.isnan(out[3, [0, 1, 3]]).any()
        assert torch.isnan(out[4, 1]).all() and not torch.isnan(out[4, [0, 2, 3]]).any()


def test_decode_reads_a_nan_block_only_where_it_is(device) -> None:
    """A value row with a NaN makes its block's output dims NaN for its sequence's heads."""

    pool = Pool([40, 40], 2, 64, 16, device, seed=5)
    row = torch.zeros(1, 2, 64)
    row[0, 1, 40] = float("nan")
    at = int(pool.tables[0, 2]) * 16 + 1  # position 33 of the first sequence
    ops.kv_append(torch.zeros(1, 2, 64, device=device), row.to(device), pool.key, pool.value,
                  torch.tensor([at], device=device), 0, **pool.scales)
    query = torch.randn(2, 4, 64, device=device)
    out = ops.paged_attention_decode(query, pool.key, pool.value, pool.block_tables, pool.lens,
                                     layer_index=0, max_seq_len=40, **pool.scales).cpu()
    nan = torch.zeros(2, 4, 64, dtype=torch.bool)
    nan[0, 2:, 32:] = True
    assert torch.equal(torch.isnan(out), nan)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq,hkv,dh,block_size", [(32, 8, 128, 16), (8, 2, 64, 16), (6, 2, 96, 5)])
def test_rope_append_decode_is_its_parts(device, dtype, hq, hkv, dh, block_size) -> None:
    lengths = [1, 16, 33, 200, 700]
    n = len(lengths)
    g = torch.Generator().manual_seed(11)
    query, key, value = (torch.randn(n, h, dh, generator=g).to(dtype).to(device)
                         for h in (hq, hkv, hkv))
    table = ops.RotaryTable(dh, theta=1e4, max_position=1000, dtype=dtype, device=device)
    positions = torch.tensor([x - 1 for x in lengths], device=device)
    results = []
    for fused in (True, False):
        pool = Pool(lengths, hkv, dh, block_size, device, seed=6)
        slots = _slots(pool, block_size, [x - 1 for x in lengths], [1] * n).to(device)
        slots[2] = -1
        more = dict(layer_index=0, max_seq_len=700, **pool.scales)
        before = query.clone()
        if fused:
            out = ops.rope_append_paged_decode(query, key, value, positions, table, pool.key,
                                               pool.value, slots, pool.block_tables, pool.lens,
                                               **more)
            assert torch.equal(query, before)
        else:
            q = ops.rope_kv_append(query.clone(), key, value, positions, table, pool.key,
                                   pool.value, slots, 0, **pool.scales)
            out = ops.paged_attention_decode(q, pool.key, pool.value, pool.block_tables,
                                             pool.lens, **more)
        results.append([out] + [t.view(torch.uint8) for t in (pool.key, pool.value,
                                                              *pool.scales.values())])
    for a, b in zip(*results):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq,hkv,dh,block_size,pages", [
    (8, 2, 64, 16, 2), (4, 1, 128, 32, 0), (16, 1, 32, 16, 1), (6, 2, 96, 48, 0), (8, 8, 64, 5, 7)])
def test_rope_append_decode_at_the_edges(device, dtype, hq, hkv, dh, block_size, pages) -> None:
    """The new row first, last or alone in a tile and in a split, of sequences without keys, and
    of rows that are not 16-byte aligned: the two calls' results bit for bit, pools included."""

    lengths = [0, 1, 32, 33, 64, 65, 127, 128, 129, 320, 321, 2100]
    n = len(lengths)
    g = torch.Generator().manual_seed(12)
    table = ops.RotaryTable(dh, theta=1e4, max_position=4000, dtype=dtype, device=device)
    positions = torch.tensor([max(x - 1, 0) for x in lengths], device=device)
    for shift in (0, 1):  # elements off the alignment
        rows = []
        for h in (hq, hkv, hkv):
            flat = torch.randn(n * h * (dh + 8) + 1, generator=g).to(dtype).to(device)
            rows.append(flat[shift:shift + n * h * (dh + 8)].view(n, h, dh + 8)[..., :dh])
        query, key, value = rows
        results = []
        for fused in (True, False):
            pool = Pool(lengths, hkv, dh, block_size, device, seed=6)
            slots = _slots(pool, block_size, [max(x - 1, 0) for x in lengths], [1] * n).to(device)
            slots[0] = -1
            slots[6] = pool.key.shape[1] * block_size  # (past the pools: left out)
            more = dict(layer_index=0, max_seq_len=2100, pages_per_split=pages, **pool.scales)
            before = query.clone()
            if fused:
                out = ops.rope_append_paged_decode(query, key, value, positions, table, pool.key,
                                                   pool.value, slots, pool.block_tables,
                                                   pool.lens, **more)
                assert torch.equal(query, before)
            else:
                q = ops.rope_kv_append(query.clone(), key, value, positions, table, pool.key,
                                       pool.value, slots, 0, **pool.scales)
                out = ops.paged_attention_decode(q, pool.key, pool.value, pool.block_tables,
                                                 pool.lens, **more)
            results.append([out] + [t.view(torch.uint8) for t in (pool.key, pool.value,
                                                                  *pool.scales.values())])
        for a, b in zip(*results):
            assert torch.equal(a, b)
        assert not results[0][0][0].any()


def test_rope_append_decode_under_a_short_bound(device) -> None:
    """max_seq_len below a sequence's length (48 of 100 keys): the two calls' results."""

    pool_of = lambda: Pool([100, 20], 2, 64, 16, device, seed=3)  # noqa: E731
    g = torch.Generator().manual_seed(4)
    query, key, value = (torch.randn(2, h, 64, generator=g).to(device) for h in (4, 2, 2))
    table = ops.RotaryTable(64, theta=1e4, max_position=200, dtype=torch.float32, device=device)
    positions = torch.tensor([99, 19], device=device)
    fused, apart = pool_of(), pool_of()
    slots = _slots(fused, 16, [99, 19], [1, 1]).to(device)
    out = ops.rope_append_paged_decode(query, key, value, positions, table, fused.key, fused.value,
                                       slots, fused.block_tables, fused.lens, layer_index=0,
                                       max_seq_len=48, **fused.scales)
    q = ops.rope_kv_append(query.clone(), key, value, positions, table, apart.key, apart.value,
                           slots, 0, **apart.scales)
    want = ops.paged_attention_decode(q, apart.key, apart.value, apart.block_tables, apart.lens,
                                      layer_index=0, max_seq_len=48, **apart.scales)
    assert torch.equal(out, want)
    assert torch.equal(fused.key.view(torch.uint8), apart.key.view(torch.uint8))


# ------------------------------------------------------------------- prefill


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq,hkv,dh,block_size", [(8, 2, 64, 16), (32, 8, 128, 16), (6, 2, 96, 16),
                                                  (4, 2, 64, 5), (4, 1, 32, 32)])
def test_prefill(device, dtype, hq, hkv, dh, block_size) -> None:
    chunks = [(1, 0), (1, 40), (33, 0), (64, 100), (5, 17), (130, 3)]
    lengths = [t + p for t, p in chunks]
    pool = Pool(lengths, hkv, dh, block_size, device, seed=8, extra_width=4)
    new = [t for t, _ in chunks]
    cu = torch.tensor([0, *torch.tensor(new).cumsum(0).tolist()], dtype=torch.int32, device=device)
    query = torch.randn(sum(new), hq, dh, generator=torch.Generator().manual_seed(3)).to(dtype)
    out = ops.paged_attention_prefill(
        query.to(device), pool.key, pool.value, pool.block_tables, pool.lens, cu, layer_index=0,
        max_query_len=max(new), max_seq_len=max(lengths), **pool.scales)
    start = 0
    for b, t in enumerate(new):
        rows = [x.to(dtype).double() for x in pool.rows[b]]  # as the scratch pages hold them
        _check_attention(out[start:start + t], query[start:start + t], *rows)
        start += t


# (Few rows; many: the waves of a workgroup share their keys; many of a sequence and many keys
# in 16 bits, Dh 64 or 128 and blocks of a multiple of 16: over the decoded pages.)
FORMS = [((6, 2, 96, 16), [(40, 30), (7, 100), (33, 0)]), ((8, 1, 32, 5), [(20, 300), (1, 0)]),
         ((32, 8, 128, 16), [(113, 40 * k) for k in range(8)]),
         ((64, 4, 32, 16), [(300, 70), (1, 9), (160, 0)]),
         ((48, 3, 96, 24), [(590, 33), (12, 1100)]), ((64, 8, 64, 7), [(460, 129)]),
         ((32, 2, 128, 48), [(900, 21)]), ((8, 1, 64, 16), [(260, 1090), (3, 40), (130, 0)]),
         ((32, 4, 64, 32), [(129, 17), (150, 60)]), ((16, 1, 64, 32), [(300, 700)]),
         ((8, 1, 128, 16), [(260, 1090), (3, 40), (130, 0)])]


def _prefill(device, dtype, sizes, chunks, nan_at=None, short=None, **kw):
    """One call, each sequence checked; behind the last query and between heads nothing is
    written. nan_at: (sequence, key, head, block of V) that is NaN; short: a sequence of that
    many keys, fewer than its queries."""

    hq, hkv, dh, block_size = sizes
    lengths = [t + p for t, p in chunks]
    if short is not None:
        lengths[-1] = short
    pool = Pool(lengths, hkv, dh, block_size, device, seed=17, extra_width=3)
    if nan_at is not None:
        b, key, head, block = nan_at
        at = pool.tables[b, key // block_size].item(), head, key % block_size, block
        raw = pool.scales["v_scales"].view(torch.uint8)
        raw[pool.layer][at] = 255
    new = [t for t, _ in chunks]
    cu = torch.tensor([0, *torch.tensor(new).cumsum(0).tolist()], dtype=torch.int32, device=device)
    g = torch.Generator().manual_seed(5)
    query = torch.randn(sum(new), hq, dh, generator=g).to(dtype)
    canvas = torch.full((sum(new) + 3, hq, dh + 8), 7.0, dtype=dtype, device=device)
    out = canvas[:sum(new), :, :dh]
    got = ops.paged_attention_prefill(
        query.to(device), pool.key, pool.value, pool.block_tables, pool.lens, cu, layer_index=0,
        max_query_len=max(new), max_seq_len=max(lengths), out=out,
        seq_order=ops.longest_first(lengths, device), **kw, **pool.scales)
    assert got is out
    assert bool((canvas[sum(new):] == 7).all()) and bool((canvas[:, :, dh:] == 7).all())
    at = 0
    for b, t in enumerate(new):
        rows, x = out[at:at + t].cpu(), query[at:at + t]
        at += t
        none = max(0, t - lengths[b])  # rows of no keys
        assert not rows[:none].any()
        rows, x = rows[none:], x[none:]
        if nan_at is not None and nan_at[0] == b:
            _, key, head, block = nan_at
            first = max(0, key - (lengths[b] - t))
            hit = torch.zeros(rows.shape, dtype=torch.bool)
            group = hq // hkv
            hit[first:, head * group:(head + 1) * group, 32 * block:32 * block + 32] = True
            assert torch.equal(rows.isnan(), hit)
            # (The key's other blocks are as they were: the rest is checked against them.)
            exact = mxfp4.attention(x, *pool.rows[b], kw.get("scale"))[0]
            rows = torch.where(hit, exact.to(dtype), rows)
        _check_attention(rows, x, *pool.rows[b], kw.get("scale"))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("sizes,chunks", FORMS)
def test_prefill_in_every_form(device, dtype, sizes, chunks) -> None:
    _prefill(device, dtype, sizes, chunks)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("sizes,chunks", FORMS)
def test_prefill_reads_a_nan_block_only_where_it_is_seen(device, dtype, sizes, chunks) -> None:
    """A value block of the first sequence that is NaN, in the middle of its queries."""

    tokens, prior = chunks[0]
    _prefill(device, dtype, sizes, chunks,
             nan_at=(0, prior + tokens // 2, sizes[1] - 1, sizes[2] // 32 - 1))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("sizes,chunks", [FORMS[0], FORMS[3], FORMS[7], FORMS[10]])
def test_prefill_of_more_queries_than_keys(device, dtype, sizes, chunks) -> None:
    for short in (0, chunks[-1][0] // 2):
        _prefill(device, dtype, sizes, chunks, short=short)


@pytest.mark.parametrize("sizes,chunks", [FORMS[0], FORMS[3], FORMS[7], FORMS[10]])
@pytest.mark.parametrize("scale", [0.0, -0.3])
def test_attention_of_any_scale(device, sizes, chunks, scale) -> None:
    _prefill(device, torch.bfloat16, sizes, chunks, scale=scale)
    pool = Pool([40, 3], sizes[1], sizes[2], 16, device, seed=4)
    query = torch.randn(2, sizes[0], sizes[2], generator=torch.Generator().manual_seed(1))
    out = ops.paged_attention_decode(query.to(device), pool.key, pool.value, pool.block_tables,
                                     pool.lens, layer_index=0, max_seq_len=40, scale=scale,
                                     **pool.scales)
    for b in range(2):
        _check_attention(out[b:b + 1], query[b:b + 1], *pool.rows[b], scale)


def test_refused_appends_and_gathers(device) -> None:
    """By the operators themselves; nothing is written."""

    def on(*shape, dtype=torch.float32):
        return torch.zeros(shape, dtype=torch.uint8 if dtype.itemsize == 1 else dtype,
                           device=device).view(dtype)

    def pools(dh=64, dtype=CODES):
        return on(1, 4, 2, 16, dh // 2, dtype=dtype), on(1, 4, 2, 16, dh // 2, dtype=dtype)

    rows, slots = on(3, 2, 64) + 1, on(3, dtype=torch.int64)
    kv = pools()
    scales = {n: on(1, 4, 2, 16, 2, dtype=SCALES) for n in ("k_scales", "v_scales")}

    def refused(kind, match, *args, **kw):
        with pytest.raises(kind, match=match):
            ops.kv_append(*args, **kw)

    refused(ValueError, "need k_scales and v_scales", rows, rows, *kv, slots, 0)
    refused(ValueError, "go together", rows, rows, *kv, slots, 0, k_scales=scales["k_scales"])
    refused(TypeError, "float8_e8m0fnu", rows, rows, *kv, slots, 0, k_scales=scales["k_scales"],
            v_scales=on(1, 4, 2, 16, 2))
    refused(ValueError, "Dh / 32", rows, rows, *kv, slots, 0, k_scales=scales["k_scales"],
            v_scales=on(1, 4, 2, 16, dtype=SCALES))
    refused(ValueError, "head_dim of 32", on(3, 2, 160), on(3, 2, 160), *pools(160), slots, 0,
            **scales)
    refused(ValueError, "fp8 KV pools only", rows, rows, *kv, slots, 0, k_scale=2.0, **scales)
    refused(ValueError, "must match the pool's", on(3, 2, 32), on(3, 2, 32), *kv, slots, 0, **scales)
    refused(ValueError, "same dtype", rows, rows, kv[0], on(1, 4, 2, 16, 32, dtype=torch.uint8),
            slots, 0, **scales)
    refused(ValueError, "contiguous", rows, rows, *(p[:, ::2] for p in kv), slots, 0, **scales)
    refused(ValueError, "storage dtype", rows, rows.half(), *kv, slots, 0, **scales)
    refused(ValueError, "storage dtype", rows.double(), rows.double(), *kv, slots, 0, **scales)
    refused(ValueError, "slot_mapping must have shape", rows, rows, *kv, slots[:2], 0, **scales)
    refused(TypeError, "slot_mapping must be torch.int64", rows, rows, *kv, slots.int(), 0, **scales)
    refused(ValueError, "requires HIP device", rows.cpu(), rows, *kv, slots, 0, **scales)
    refused(ValueError, "requires HIP device", rows, rows, *kv, slots.cpu(), 0, **scales)
    refused(IndexError, None, rows, rows, *kv, slots, 1, **scales)
    tables, lens, cu = (on(*s, dtype=torch.int32) for s in ((2, 3), (2,), (3,)))
    out = on(5, 2, 64), on(5, 2, 64)

    def no_gather(kind, match, *args, **kw):
        with pytest.raises(kind, match=match):
            ops.paged_gather(*args, **kw)

    no_gather(ValueError, "block_tables must have", *kv, tables[0], lens, cu, 0, 40, *out, **scales)
    no_gather(TypeError, "seq_lens must be torch.int32", *kv, tables, lens.long(), cu, 0, 40, *out,
              **scales)
    no_gather(ValueError, "an entry per row", *kv, tables, lens[:1], cu, 0, 40, *out, **scales)
    no_gather(ValueError, "outputs must have shape", *kv, tables, lens, cu, 0, 40, out[0][..., :32],
              out[1][..., :32], **scales)
    no_gather(ValueError, "share shape and strides", *kv, tables, lens, cu, 0, 40, out[0],
              out[1][:4], **scales)
    no_gather(ValueError, "outputs must match", *kv, tables, lens, cu, 0, 40, out[0], out[1].half(),
              **scales)
    no_gather(ValueError, None, *kv, tables, lens, cu, 0, 49, *out, **scales)  # (past the tables)
    for t in (*kv, *scales.values()):
        assert not t.view(torch.uint8).any()


def test_refused_attention(device) -> None:
    """By the operators themselves, before anything is launched: out is as it was."""

    pool = Pool([40, 3], 2, 64, 16, device, seed=4)
    tables, lens = pool.block_tables, pool.lens
    cu = torch.tensor([0, 1, 2], dtype=torch.int32, device=device)
    query = torch.randn(2, 4, 64, device=device)
    out = torch.full((2, 4, 64), 5.0, device=device)
    base = dict(query=query, key_cache=pool.key, value_cache=pool.value, block_tables=tables,
                seq_lens=lens, layer_index=0, max_seq_len=40, out=out, **pool.scales)
    cases = [
        (ValueError, "Hq, Dh\\) with the pool's Dh", dict(query=query[..., :32])),
        (TypeError, "query must be float32", dict(query=query.double(), out=out.double())),
        (ValueError, "divisible by KV head", dict(query=query[:, :3], out=out[:, :3])),
        (ValueError, "out must match query", dict(out=out[:1])),
        (ValueError, "out must match query", dict(out=out.half())),
        (ValueError, "out must match query", dict(out=out.transpose(1, 2).contiguous().transpose(1, 2))),
        (ValueError, "must match query", dict(block_tables=tables[:1])),
        (ValueError, "must match query", dict(block_tables=tables[0])),
        (TypeError, "block_tables must be torch.int32", dict(block_tables=tables.long())),
        (TypeError, "seq_lens must be torch.int32", dict(seq_lens=lens.long())),
        (ValueError, "seq_order must have shape", dict(seq_order=lens[:1])),
        (TypeError, "seq_order must be torch.int32", dict(seq_order=lens.long())),
        (ValueError, "requires HIP device", dict(seq_lens=lens.cpu())),
        (ValueError, "requires HIP device", dict(query=query.cpu())),
        (ValueError, "need k_scales", dict(k_scales=None, v_scales=None)),
        (ValueError, "go together", dict(v_scales=None)),
        (ValueError, "fp8 KV pools only", dict(k_scale=2.0)),
        (IndexError, None, dict(layer_index=1)),
        (ValueError, None, dict(max_seq_len=49)),
    ]
    for kind, match, change in cases:
        for op in ("decode", "prefill"):
            args = base | change
            extra = dict(cu_seqlens_q=cu, max_query_len=1) if op == "prefill" else {}
            with pytest.raises(kind, match=match):
                getattr(ops, f"paged_attention_{op}")(**args, **extra)
    with pytest.raises(ValueError, match="cu_seqlens_q"):
        ops.paged_attention_prefill(**base, cu_seqlens_q=cu[:2], max_query_len=1)
    with pytest.raises(ValueError, match="uint8"):
        ops.paged_attention_decode(**base, workspace=torch.empty(8, device=device))
    with pytest.raises(ValueError, match="workspace"):
        ops.paged_attention_decode(**base, pages_per_split=1,
                                   workspace=torch.empty(8, dtype=torch.uint8, device=device))
    assert bool((out == 5).all())
    # Strided queries are taken as they are.
    wide = torch.randn(2, 4, 128, device=device)
    again = ops.paged_attention_decode(**(base | dict(query=wide[..., ::2], out=None)))
    assert torch.equal(again, ops.paged_attention_decode(
        **(base | dict(query=wide[..., ::2].contiguous(), out=None))))


# ------------------------------------------------------ the operators together


@pytest.mark.parametrize("sizes,chunks", [FORMS[0], FORMS[3], FORMS[10]])
def test_attention_from_graphs_and_on_two_streams(device, sizes, chunks) -> None:
    """A prefill of each form and a split decode: captured and replayed among eager calls, and
    two at once on two streams, each with scratch memory of its own."""

    hq, hkv, dh, block_size = sizes
    lengths = [t + p for t, p in chunks]
    new = [t for t, _ in chunks]
    pools = [Pool(lengths, hkv, dh, block_size, device, seed=s) for s in (1, 2)]
    cu = torch.tensor([0, *torch.tensor(new).cumsum(0).tolist()], dtype=torch.int32, device=device)
    g = torch.Generator().manual_seed(3)
    queries = [torch.randn(sum(new), hq, dh, generator=g).bfloat16().to(device) for _ in range(2)]

    def both(pool, query):
        out = ops.paged_attention_prefill(
            query, pool.key, pool.value, pool.block_tables, pool.lens, cu, layer_index=0,
            max_query_len=max(new), max_seq_len=max(lengths), **pool.scales)
        last = ops.paged_attention_decode(
            query[:len(new)], pool.key, pool.value, pool.block_tables, pool.lens, layer_index=0,
            max_seq_len=max(lengths), pages_per_split=2, **pool.scales)
        return out, last

    want = [[both(pool, query) for query in queries] for pool in pools]
    torch.cuda.synchronize()
    graphs = []
    for pool in pools:
        static = queries[0].clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = both(pool, static)
        graphs.append((graph, static, out))
    for turn in range(4):
        for i, (graph, static, out) in enumerate(graphs):
            static.copy_(queries[turn % 2])
            graph.replay()
            eager = both(pools[1 - i], queries[turn % 2])
            torch.cuda.synchronize()
            for a, b in zip((*out, *eager), (*want[i][turn % 2], *want[1 - i][turn % 2])):
                assert torch.equal(a, b)
    streams = [torch.cuda.Stream() for _ in range(2)]
    results = []
    for turn in range(6):
        i = turn % 2
        streams[i].wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(streams[i]):
            results.append((i, both(pools[i], queries[i])))
    torch.cuda.synchronize()
    for i, got in results:
        for a, b in zip(got, want[i][i]):
            assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_cache_through_its_life(device, dtype) -> None:
    """Prefill in two chunks, then decode steps, through the storage: every step attends to
    what was appended before it, and the read-back agrees; replayed from graphs on another
    stream the decode gives the same."""

    hq, hkv, dh, block_size, prompt, steps = 8, 2, 64, 16, 45, 20
    storage = PagedKVStorage(num_layers=2, num_blocks=8, num_key_value_heads=hkv, device=device,
                             block_size=block_size, head_dim=dh, dtype=dtype, kv_dtype=CODES)
    table = ops.RotaryTable(dh, theta=1e4, max_position=128, dtype=dtype, device=device)
    blocks = torch.tensor([[5, 0, 7, 2, 6]], dtype=torch.int32)
    g = torch.Generator().manual_seed(1)
    total = prompt + steps
    query, key, value = (torch.randn(total, h, dh, generator=g).to(dtype) for h in (hq, hkv, hkv))
    positions = torch.arange(total)
    rq, rk = ops.rope(query.transpose(0, 1)[None].to(device), key.transpose(0, 1)[None].to(device),
                      positions.to(device), table)
    rq, rk = (x[0].transpose(0, 1).cpu() for x in (rq, rk))
    keys, vals = (mxfp4.values(*mxfp4.quantize(x)) for x in (rk, value))
    slots = blocks[0].long()[positions // block_size] * block_size + positions % block_size
    on = lambda x: x.to(device)  # noqa: E731
    for start, end in ((0, 30), (30, prompt)):
        q = ops.rope_kv_append(on(query[start:end]), on(key[start:end]), on(value[start:end]),
                               on(positions[start:end]), table, storage.key_storage,
                               storage.value_storage, on(slots[start:end]), 1, **storage.scales)
        out = ops.paged_attention_prefill(
            q, storage.key_storage, storage.value_storage, on(blocks),
            torch.tensor([end], dtype=torch.int32, device=device),
            torch.tensor([0, end - start], dtype=torch.int32, device=device), layer_index=1,
            max_query_len=end - start, max_seq_len=end, **storage.scales)
        _check_attention(out, rq[start:end], keys[:end].to(dtype).double(),
                         vals[:end].to(dtype).double())
    # One decode step as a graph: its inputs are static buffers.
    static = {n: on(x[:1].clone()) for n, x in (("q", query), ("k", key), ("v", value))}
    position, slot = on(positions[:1].clone()), on(slots[:1].clone())
    length = torch.ones(1, dtype=torch.int32, device=device)
    tables = on(blocks)

    def step():
        return ops.rope_append_paged_decode(
            static["q"], static["k"], static["v"], position, table, storage.key_storage,
            storage.value_storage, slot, tables, length, layer_index=1, max_seq_len=80,
            **storage.scales)

    slot.fill_(-1)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for p in range(prompt, total):
        for n, x in (("q", query), ("k", key), ("v", value)):
            static[n].copy_(x[p:p + 1])
        position.fill_(p)
        slot.copy_(slots[p:p + 1])
        length.fill_(p + 1)
        if p % 2:
            out = step()
        else:
            graph.replay()
            out = captured
        _check_attention(out, rq[p:p + 1], keys[:p + 1], vals[:p + 1])
    got = storage.gather(1, blocks[0].tolist(), total)
    assert torch.equal(got[0].cpu(), keys.to(dtype)) and torch.equal(got[1].cpu(), vals.to(dtype))
