"""paged_attention, qk_norm_rope and FP8Attention at unusual values and sizes.
Oracles are in 64 bits or follow from the definition alone."""

from __future__ import annotations

import math

import pytest
import torch

from tests.test_gpu_attention import DEV, U, Batch, gen, new_cache, randn

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------------------
# Rows that see a NaN score are NaN, all others keep their bits. Prefixes of 40
# and 1100 keys are one and several shares; 6 sequences of 8 query heads go
# through it in tiles of few rows (24 rows a key head), 16 query heads in tiles
# of many (48). 4000 keys are cut into chunks.
LENGTHS = [1, 16, 17, 48, 64, 4000]


def check_nan_rows(b, clean, rows):
    """rows [tokens] or [tokens, heads]: those that have to be NaN in every channel; the others are as in clean."""
    out = b.run()
    rows = rows if rows.dim() == 2 else rows[:, None].expand(out.shape[:2])
    assert out[rows].isnan().all(), (~out.isnan().all(-1) & rows).nonzero().tolist()
    assert torch.equal(out[~rows], clean[~rows])


@pytest.mark.parametrize("prefix", [0, 40, 1100])
@pytest.mark.parametrize("heads", [(8, 2), (16, 2)])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_a_nan_query_is_nan_at_every_length(prefix, heads, dim):
    b = Batch(40, LENGTHS, prefix=prefix, heads=heads, dim=dim)
    clean = b.check()
    for i in range(len(LENGTHS)):
        kept = b.q[i, 3].clone()
        b.q[i, 3, 7] = math.nan
        rows = torch.zeros(b.q.shape[:2], dtype=torch.bool, device=DEV)
        rows[i, 3] = True
        check_nan_rows(b, clean, rows)
        b.q[i, 3] = kept


# whole tiles; the keys of many-row tiles split; tiles of few rows, whole and cut
RAGGED = [([300, 500, 400], [300, 520, 400], 0, (64, 32)), ([64], [4000], 0, (8, 2)), ([64, 40], [3000, 900], 700, (8, 2)),
          ([3, 2, 4], [70, 3000, 9], 0, (8, 2)), ([3, 2, 4], [70, 3000, 9], 300, (8, 2))]


@pytest.mark.parametrize("queries,lengths,prefix,heads", RAGGED)
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_a_nan_query_of_many_is_nan(queries, lengths, prefix, heads, dim):
    b = Batch(41, lengths, queries, prefix=prefix, heads=heads, dim=dim)
    clean = b.check()
    for token in (0, queries[0] - 1, sum(queries) - 1):
        kept = b.q[token, 1].clone()
        b.q[token, 1, dim - 1] = math.nan
        rows = torch.zeros(b.q.shape[:2], dtype=torch.bool, device=DEV)
        rows[token, 1] = True
        check_nan_rows(b, clean, rows)
        b.q[token, 1] = kept


def sees_own(b, i, key):
    """[tokens]: the tokens that see own key `key` of sequence i."""
    at = sum(b.queries[:i])
    n, length = b.queries[i], b.lengths[i]
    rows = torch.zeros(b.q.shape[0], dtype=torch.bool, device=DEV)
    rows[at:at + n] = key <= length - n + torch.arange(n, device=DEV)
    return rows


@pytest.mark.parametrize("value", [math.nan, math.inf])
@pytest.mark.parametrize("queries,lengths,prefix,heads", [(None, [100, 64, 4000], 0, (8, 2)), (None, [100, 64, 4000], 40, (8, 2)),
                                                          (None, [100, 64, 4000], 1100, (16, 1)), *RAGGED])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_a_key_that_is_not_finite_reaches_every_row_that_sees_it(queries, lengths, prefix, heads, dim, value):
    """In the first, a middle and the last wave, chunk and prefix share. Queries are positive in the channel, so that an
    infinite key gives an infinite score, whose softmax is NaN."""
    b = Batch(42, lengths, queries, prefix=prefix, heads=heads, dim=dim)
    b.q[..., 3] = b.q[..., 3].abs() + 0.5
    clean = b.check()
    for i, length in enumerate(lengths):
        for key in sorted({0, min(17, length - 1), min(33, length - 1), length // 2, length - 1}):
            at = (int(b.table[i, key // b.page]), slice(None), key % b.page, 3)
            kept = b.cache.k[at].clone()
            b.cache.k[at] = value
            check_nan_rows(b, clean, sees_own(b, i, key))
            b.cache.k[at] = kept
    for key in sorted({0, prefix // 2, prefix - 1}) if prefix else []:
        at = (int(b.prefix_pages[key // b.page]), slice(None), key % b.page, 3)
        kept = b.cache.k[at].clone()
        b.cache.k[at] = value
        check_nan_rows(b, clean, torch.ones(b.q.shape[0], dtype=torch.bool, device=DEV))
        b.cache.k[at] = kept


@pytest.mark.parametrize("queries,lengths,prefix,low", [
    (None, [64, 64], 0, (0, 16)), (None, [64, 64], 0, (32, 48)), (None, [4000, 2500], 0, (0, 2000)), (None, [40, 40], 1100, (0, 608)),
    (None, [40, 40], 1100, (1008, 1088)), ([64], [4000], 0, (0, 2000)), ([64], [4000], 0, (2000, 3008))])
def test_a_nan_value_under_a_weight_of_zero(queries, lengths, prefix, low):
    """Keys whose weights are 0 in 32 bits, one of them with a NaN value: 0 * NaN, so the channel is NaN, also where these
    keys are all that a wave, a chunk or a share of the prefix has."""
    b = Batch(43, lengths, queries, prefix=prefix)
    b.q.fill_(4.0)
    b.cache.k.fill_(0.0)
    pages = (b.prefix_pages if prefix else b.table[0])[low[0] // 16:low[1] // 16].long()
    clean = b.run()
    b.cache.k[pages] = -8.0  # scores of -362: e^-362 is no number of 32 bits
    b.cache.v[pages[-1], :, 3, 5] = math.nan
    out = b.run()
    rows = torch.ones(b.q.shape[0], dtype=torch.bool, device=DEV) if prefix else sees_own(b, 0, low[1] - 13)
    assert out[rows][..., 5].isnan().all()
    others = [c for c in range(b.q.shape[2]) if c != 5]
    assert out[..., others].isfinite().all() and torch.equal(out[~rows], clean[~rows])


# ---------------------------------------------------------------------------
# weights
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("queries,lengths,prefix", [
    (None, [1, 2, 5, 17, 100, 1000, 5000], 0), (None, [1, 2, 5, 17, 100, 1000, 0], 50), (None, [1 + 9 * i for i in range(40)], 1100),
    ([3, 2, 4], [70, 3000, 9], 0), ([64, 90], [3000, 90], 0), ([700, 800], [700, 810], 90)])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_weights_add_to_one(queries, lengths, prefix, dim, dtype):
    """Values that are the same for all keys come out as they are: sum(w) v / sum(w), with both sums in 32 bits of the
    same weights, is v within 2^-14, which rounds to v, a number of the type."""
    b = Batch(44, lengths, queries, prefix=prefix, dim=dim, dtype=dtype)
    v = randn(gen(45), 1, b.cache.kv_heads, 1, dim, dtype=dtype)
    b.cache.v.copy_(v.expand_as(b.cache.v))
    out = b.run()
    want = v[0, :, 0].repeat_interleave(b.q.shape[1] // b.cache.kv_heads, 0).expand_as(out).clone()
    for i, length in enumerate(lengths):
        if length == 0 and prefix == 0:
            want[i] = 0
    assert torch.equal(out, want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("prefix", [0, 1, 9])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_weights_of_few_row_tiles_keep_more_than_16_bits(prefix, dim, dtype):
    """Weights that go into the product as the sum of two 16-bit numbers are off by 2 u^2 at most, so all but the output's
    rounding is that of the scores: 2 u |o| + (2^-14 + 4 u^2) m, m the softmax-weighted mean of |v|."""
    b = Batch(46, [1 + i for i in range(30)], prefix=prefix, heads=(4, 4), dim=dim, dtype=dtype)
    out = b.run().double()
    exact, mag = b.exact()
    u = U[dtype]
    bound = 2 * u * exact.abs() + (2.0 ** -14 + 4 * u * u) * mag + (2.0 ** -25 if dtype == torch.float16 else 0)
    assert ((out - exact).abs() <= bound).all(), ((out - exact).abs() / bound).max().item()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("queries,lengths,prefix", [(None, [600, 333, 4000, 7], 0), (None, [600, 333, 40, 7], 1100), ([2, 3], [600, 333], 0),
                                                    ([300, 400], [600, 433], 0), ([64], [4000], 100)])
@pytest.mark.parametrize("size", [2048.0, 8192.0])
def test_scores_past_32_bits_of_whole_numbers(queries, lengths, prefix, dtype, size):
    """Finite queries and keys whose scores reach 2^26 to 2^31: the largest takes all of the softmax, so its value comes
    out as it is. Rows whose two largest scores are closer than 32-bit sums tell apart (each is off by 2^-17 |q| |k| at
    most for 128 products) are left out."""
    b = Batch(47, lengths, queries, prefix=prefix, heads=(8, 2), dim=128, dtype=dtype)
    b.q.mul_(size)
    b.cache.k.mul_(size)
    assert b.q.isfinite().all() and b.cache.k.isfinite().all()
    out, at, left_out = b.run(scale=1.0), 0, 0
    for i, (n, length) in enumerate(zip(b.queries, lengths)):
        k, v = b.keys(i, b.cache.k), b.keys(i, b.cache.v)
        unseen = torch.arange(prefix + length, device=DEV)[None] > prefix + length - n + torch.arange(n, device=DEV)[:, None]
        for h in range(8):
            q = b.q[at:at + n, h].double()
            score = (q @ k[h // 4].t()).masked_fill(unseen, -math.inf)
            top = torch.cat([score, torch.full((n, 1), -math.inf, dtype=torch.float64, device=DEV)], 1).topk(2, 1)
            clear = top.values[:, 0] - top.values[:, 1] > 2.0 ** -14 * q.norm(dim=1) * k[h // 4].norm(dim=1).max() + 200
            got, want = out[at:at + n, h], v[h // 4][top.indices[:, 0]].to(dtype)
            assert torch.equal(got[clear], want[clear]), (i, h, (got != want).any(1).sum().item())
            left_out += int((~clear).sum())
        at += n
    assert left_out <= 0.05 * at * 8


# ---------------------------------------------------------------------------
# norm
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("exponent", [-62, -64, -66, -30, 30])
def test_norm_of_tiny_and_large_rows(dim, exponent):
    """Without eps, also where the mean square is below the normal numbers of 32 bits: rows of 2^-66 have squares of
    2^-132, on a grid of 2^-149, so the mean and its root are off by 2^-17 or less (2^-18 and a half below it)."""
    from jeeves_amd.attention import qk_norm_rope

    x = randn(gen(48), 33, 3, dim) * 2.0 ** exponent
    w = torch.ones(dim, device=DEV)
    y = x.double() / x.double().square().mean(-1, keepdim=True).sqrt()
    for out in qk_norm_rope(x, x, None, None, q_weight=w, k_weight=w, eps=0.0):
        assert ((out.double() - y).abs() <= (2 * U[x.dtype] + 2.0 ** -14) * y.abs() + 2.0 ** -20).all()


# ---------------------------------------------------------------------------
# index tensors
# ---------------------------------------------------------------------------
def test_wide_indices_are_held_in_range_before_they_are_narrowed():
    from jeeves_amd.attention import paged_attention

    b = Batch(49, [70, 5, 33], [4, 5, 6], heads=(8, 2))
    pages = b.cache.pages
    far = torch.tensor([[-2 ** 40, 2 ** 32 + 1, 0, 3], [1, 2 ** 62, 3, 2], [2 ** 31, -1, 2, -2 ** 32 + 1]], device=DEV)
    held = far.clamp(0, pages - 1).to(torch.int32)
    lengths = torch.tensor([2 ** 32 + 3, -2 ** 33 + 20, 40], device=DEV)
    starts = torch.tensor([0, 4, 9, 2 ** 32 + 3], device=DEV)
    out = paged_attention(b.q, b.cache, far, lengths, query_starts=starts)
    same = paged_attention(b.q, b.cache, held, torch.tensor([64, 0, 40], dtype=torch.int32, device=DEV), query_starts=b.starts)
    assert torch.equal(out, same)
    out = paged_attention(b.q, b.cache, b.table, b.device_lengths, query_starts=b.starts, prefix_pages=far[0], prefix_length=40)
    same = paged_attention(b.q, b.cache, b.table, b.device_lengths, query_starts=b.starts, prefix_pages=held[0], prefix_length=40)
    assert torch.equal(out, same)
    strided = torch.stack([far, far + 1], 2)[..., 0]
    lengths = torch.stack([b.device_lengths.long()] * 3, 1)[:, 1]
    assert not strided.is_contiguous() and not lengths.is_contiguous()
    assert torch.equal(paged_attention(b.q, b.cache, strided, lengths, query_starts=b.starts),
                       paged_attention(b.q, b.cache, held, b.device_lengths, query_starts=b.starts))


def test_a_long_prompt_under_a_wide_table():
    """32768 queries of 16 rows each in a table of 2^20 keys: 2^31 tiles times steps of 16 keys, of which none are added up."""
    from jeeves_amd.attention import paged_attention

    n, length, dim, page = 32768, 33000, 64, 16
    g = gen(54)
    cache = new_cache(g, 2100, 1, page, dim)
    q = randn(g, n, 16, dim)
    table = torch.zeros(1, 65536, dtype=torch.int32, device=DEV)
    table[0, :2063] = torch.randperm(2100, generator=g, device=DEV)[:2063]
    out = paged_attention(q, cache, table, torch.tensor([length], dtype=torch.int32, device=DEV),
                          query_starts=torch.tensor([0, n], dtype=torch.int32, device=DEV))
    ids = table[0, :2063].long()
    k, v = (x[ids, 0].flatten(0, 1)[:length].double() for x in (cache.k, cache.v))
    rows = torch.tensor([0, 1, 127, 128, 9999, 20000, 32000, n - 1], device=DEV)
    score = (q[rows].double() @ k.t()) * dim ** -0.5
    score.masked_fill_(torch.arange(length, device=DEV) > (length - n + rows)[:, None, None], -math.inf)
    p = torch.softmax(score, -1)
    exact, mag = p @ v, p @ v.abs()
    assert ((out[rows].double() - exact).abs() <= 2 * U[out.dtype] * (exact.abs() + mag) + 2.0 ** -14 * mag).all()


def test_rotation_needs_a_table():
    from jeeves_amd.attention import append_kv, qk_norm_rope, rope_table

    g = gen(50)
    q, k, pos = randn(g, 2, 4, 128), randn(g, 2, 2, 128), torch.zeros(2, dtype=torch.int32, device=DEV)
    cache = new_cache(g, 2, 2, 16, 128)
    for rope in (rope_table(8, 64)[:0], rope_table(0, 64)):
        with pytest.raises(ValueError):
            qk_norm_rope(q, k, rope, pos)
        with pytest.raises(ValueError):
            append_kv(cache, k, k, pos, rope=rope, positions=pos)


# ---------------------------------------------------------------------------
# tokens of no sequence
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("queries,heads,prefix", [([3, 4], (8, 2), 0), ([3, 4], (8, 2), 50), ([300, 500, 400], (64, 32), 0), ([64], (8, 2), 0)])
def test_tokens_before_the_first_sequence_are_zero(queries, heads, prefix):
    from jeeves_amd.attention import paged_attention

    b = Batch(51, [n + 900 for n in queries], queries, heads=heads, prefix=prefix)
    one = torch.ones(1, *b.q.shape[1:], dtype=b.dtype, device=DEV)
    padded = torch.cat([one.expand(5, -1, -1), b.q, one.expand(3, -1, -1)])
    dirty = [torch.full_like(padded, math.nan) for _ in range(8)]  # what the output's memory may have held before
    del dirty
    out = paged_attention(padded, b.cache, b.table, b.device_lengths, query_starts=b.starts + 5,
                          prefix_pages=b.prefix_pages if prefix else None, prefix_length=prefix)
    assert (out[:5] == 0).all() and (out[-3:] == 0).all()
    exact, mag = b.exact()
    assert ((out[5:-3].double() - exact).abs() <= 2 * U[b.dtype] * (exact.abs() + mag) + 2.0 ** -14 * mag).all()


def device_time(f):
    """Best time of a call in us on the device: ten runs of four in a graph."""
    s = torch.cuda.Stream()
    times = []
    with torch.cuda.stream(s):
        f()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            for _ in range(4):
                f()
        for _ in range(10):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record(s)
            graph.replay()
            b.record(s)
            torch.cuda.synchronize()
            times.append(a.elapsed_time(b) * 250)
    return min(times)


@pytest.mark.parametrize("queries,heads", [([100], (32, 8)), ([10] * 64, (8, 8)), ([1500, 600], (32, 8))])
def test_padding_costs_no_more_than_filling_the_output(queries, heads):
    """A batch padded to 16384 tokens: four times the call without the padding and the fill of the output, and 30 us, are
    margin enough for tokens cleared by all workgroups and not for tokens cleared by one a head, 1800 us."""
    from jeeves_amd.attention import paged_attention

    b = Batch(53, queries, queries, heads=heads)
    padded = torch.zeros(16384, *b.q.shape[1:], dtype=b.dtype, device=DEV)
    padded[:b.q.shape[0]] = b.q
    fill = torch.empty_like(padded)
    limit = 4 * (device_time(b.run) + device_time(fill.zero_)) + 30
    took = device_time(lambda: paged_attention(padded, b.cache, b.table, b.device_lengths, query_starts=b.starts))
    assert took <= limit, (took, limit)


# ---------------------------------------------------------------------------
# capture
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("queries,lengths,prefix,heads", [(None, [70, 5, 200], 100, (8, 2)), (None, [70] * 40, 1100, (8, 2)),
                                                          ([300, 500, 400], [300, 520, 400], 0, (64, 32))])
def test_what_counts_nothing_is_captured_on_a_new_stream(queries, lengths, prefix, heads):
    """Single tokens over a prefix, whose parts a launch of its own joins, and whole tiles: no counters to make first.
    Replayed between eager work, with other queries."""
    from jeeves_amd.fp8 import TILE_COUNTERS

    b = Batch(55, lengths, queries, prefix=prefix, heads=heads)
    b.run()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(64)]
    s = next((s for s in streams if (torch.device("cuda", s.device_index), s.cuda_stream) not in TILE_COUNTERS), streams[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        out = b.run()
    g = gen(56)
    for _ in range(4):
        b.q.copy_(randn(g, *b.q.shape))
        graph.replay()
        got = out.clone()
        assert torch.equal(got, b.run())
        torch.cuda.synchronize()


# ---------------------------------------------------------------------------
# the block
# ---------------------------------------------------------------------------
def block_of(g, hidden=1024, hq=8, hk=2, dim=128):
    from jeeves_amd import FP8Linear
    from jeeves_amd.attention import FP8Attention

    parts = [FP8Linear(hidden, n * dim, device=DEV) for n in (hq, hk, hk)]
    o = FP8Linear(hq * dim, hidden, device=DEV)
    for m in (*parts, o):
        m.load_weight(randn(g, m.out_features, m.in_features) * 0.03)
    return FP8Attention(FP8Linear.concatenated(parts), o, hq, hk)


def test_attention_block_of_no_tokens():
    from jeeves_amd.attention import PagedKVCache

    block = block_of(gen(52))
    cache = PagedKVCache.allocate(4, 2, 16, 128)
    none = torch.empty(0, dtype=torch.int32, device=DEV)
    x = torch.empty(0, 1024, dtype=torch.bfloat16, device=DEV)
    assert block(x, cache, none, none.view(0, 3), none).shape == (0, 1024)
    starts = torch.zeros(3, dtype=torch.int32, device=DEV)
    assert block(x, cache, none, torch.zeros(2, 3, dtype=torch.int32, device=DEV), starts[:2], query_starts=starts).shape == (0, 1024)


def test_warm_prepares_the_block_for_capture():
    """warm(block) on a stream, then a step of single tokens, whose keys are split, captured on it; no linear of these
    sizes counts."""
    from jeeves_amd import warm
    from jeeves_amd.attention import PagedKVCache
    from jeeves_amd.fp8 import TILE_COUNTERS

    g = gen(57)
    block = block_of(g, 6144, 32, 8)
    cache = PagedKVCache.allocate(12, 8, 16, 128)
    x = randn(g, 3, 6144)
    table = torch.arange(12, dtype=torch.int32, device=DEV).view(3, 4)
    lengths = torch.tensor([1, 17, 64], dtype=torch.int32, device=DEV)
    slots = table.gather(1, (lengths.long()[:, None] - 1) // 16)[:, 0] * 16 + (lengths - 1) % 16
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(64)]
    s = next((s for s in streams if (torch.device("cuda", s.device_index), s.cuda_stream) not in TILE_COUNTERS), streams[0])
    with torch.cuda.stream(s):
        assert warm(block) == 2
    torch.cuda.synchronize()
    assert (cache.k == 0).all()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        out = block(x, cache, slots, table, lengths)
    for _ in range(4):
        x.copy_(randn(g, 3, 6144))
        graph.replay()
        got = out.clone()
        assert torch.equal(got, block(x, cache, slots, table, lengths))
        torch.cuda.synchronize()


@pytest.mark.parametrize("hq,hk,dim", [(4, 4, 64), (32, 1, 64), (16, 4, 256)])
def test_warm_of_other_head_layouts(hq, hk, dim):
    block = block_of(gen(58), 256, hq, hk, dim)
    block.warm()
    torch.cuda.synchronize()
