"""qk_norm_rope, append_kv and paged_attention against their definitions in 64
bits, at the sizes, layouts and masks where such kernels go wrong.

Bounds, from the roundings that the kernels make (u = 2^-9 for bf16, 2^-12 for
fp16, half a unit in the last place relative to the next power of two, so at
most 2 u of the value):
* norm and rotation: fp32 with one rounding, 2 u |z| + 2^-20 (|y| + |y'|) for
  the pair y, y' that is turned;
* attention: each softmax weight is rounded once (2 u), the output once, and
  the scores carry fp32 rounding (of |s| < 64: 2^-18 and less per weight):
  2 u (|o| + m) + 2^-14 m with m the softmax-weighted mean of |v|.
fp16 adds 2^-25, half its smallest step."""

from __future__ import annotations

import math
import random

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"
U = {torch.bfloat16: 2.0 ** -9, torch.float16: 2.0 ** -12}


def gen(seed):
    return torch.Generator(DEV).manual_seed(seed)


def randn(g, *shape, dtype=torch.bfloat16):
    return torch.randn(*shape, generator=g, device=DEV).to(dtype)


# ---------------------------------------------------------------------------
# norm and rotation
# ---------------------------------------------------------------------------
def norm_rope_exact(x, weight, rope, pos, eps=1e-6):
    """(z, bound's magnitude) in 64 bits."""
    y = x.double()
    if weight is not None:
        y = y / (y.square().mean(-1, keepdim=True) + eps).sqrt() * weight.double()
    z, mag = y.clone(), y.abs()
    if rope is not None:
        half = rope.shape[1] // 2
        t = rope.double()[pos.long()][:, None]
        c, s = t[..., :half], t[..., half:]
        a, b = y[..., :half], y[..., half:2 * half]
        z[..., :half], z[..., half:2 * half] = a * c - b * s, b * c + a * s
        mag = mag.clone()
        mag[..., :half] = mag[..., half:2 * half] = a.abs() + b.abs()
    return z, mag


def check_norm_rope(out, x, weight, rope, pos):
    z, mag = norm_rope_exact(x, weight, rope, pos)
    bound = 2 * U[x.dtype] * z.abs() + 2.0 ** -20 * mag + (2.0 ** -25 if x.dtype == torch.float16 else 0)
    assert ((out.double() - z).abs() <= bound).all()


@pytest.mark.parametrize("dim,rotary", [(64, 64), (64, 16), (128, 128), (128, 96), (256, 64), (256, 256), (128, 0)])
@pytest.mark.parametrize("tokens", [1, 3, 67, 1031])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_norm_rope(dim, rotary, tokens, dtype):
    from jeeves_amd.attention import qk_norm_rope, rope_table

    g = gen(tokens * 7 + dim + rotary)
    hq, hk = 6, 3
    merged = randn(g, tokens, (hq + 2 * hk) * dim, dtype=dtype) * 3
    q, k, _ = merged.split([hq * dim, hk * dim, hk * dim], 1)
    q, k = q.view(tokens, hq, dim), k.view(tokens, hk, dim)
    rope = rope_table(500, rotary) if rotary else None
    pos = torch.randint(0, 500, (tokens,), generator=g, device=DEV, dtype=torch.int64 if tokens % 2 else torch.int32)
    qw, kw = 1 + torch.randn(dim, generator=g, device=DEV), torch.randn(dim, generator=g, device=DEV)
    before = merged.clone()
    for a, b in ((qw, kw), (qw, None), (None, None)):
        qo, ko = qk_norm_rope(q, k, rope, pos if rotary else None, q_weight=a, k_weight=b)
        check_norm_rope(qo, q, a, rope, pos)
        check_norm_rope(ko, k, b, rope, pos)
        again = qk_norm_rope(q, k, rope, pos if rotary else None, q_weight=a, k_weight=b)
        assert torch.equal(qo, again[0]) and torch.equal(ko, again[1])
    assert torch.equal(merged, before)


def test_norm_rope_many_heads_take_the_blocked_form():
    """Many rows, and odd head counts: a lane group takes two heads."""
    from jeeves_amd.attention import qk_norm_rope, rope_table

    g = gen(5)
    q, k = randn(g, 2003, 13, 128), randn(g, 2003, 5, 128)
    rope, pos = rope_table(64, 128), torch.randint(0, 64, (2003,), generator=g, device=DEV)
    w = torch.randn(128, generator=g, device=DEV)
    qo, ko = qk_norm_rope(q, k, rope, pos, q_weight=w, k_weight=w)
    check_norm_rope(qo, q, w, rope, pos)
    check_norm_rope(ko, k, w, rope, pos)


def test_norm_rope_strides_zero_rows_and_positions_outside_the_table():
    from jeeves_amd.attention import qk_norm_rope, rope_table

    g = gen(6)
    rope = rope_table(8, 64)
    base = randn(g, 4, 9, 128)
    q = base.transpose(0, 1)                      # heads apart further than tokens
    k = randn(g, 1, 1, 128).expand(9, 2, 128)     # one row for all
    w = torch.ones(128, device=DEV)
    pos = torch.tensor([0, 7, 8, -1, 3, 2 ** 31 - 1, 1, 2, 5], device=DEV)
    qo, ko = qk_norm_rope(q, k, rope, pos, q_weight=w, k_weight=w)
    inside = (pos >= 0) & (pos < 8)
    check_norm_rope(qo[inside], q[inside], w, rope, pos[inside])
    check_norm_rope(ko[inside], k[inside], w, rope, pos[inside])
    assert qo[~inside].isnan().all() and ko[~inside].isnan().all()
    odd = torch.empty(9 * 2 * 128 + 4, dtype=torch.bfloat16, device=DEV)[1:1 + 9 * 2 * 128].view(9, 2, 128).copy_(k)  # 2-byte aligned
    assert torch.equal(qk_norm_rope(q, odd, rope, pos.clamp(0, 7))[1], qk_norm_rope(q, k, rope, pos.clamp(0, 7))[1])
    zero = torch.zeros(2, 1, 128, dtype=torch.bfloat16, device=DEV)
    assert (qk_norm_rope(zero, zero, rope, pos[:2], q_weight=w, k_weight=w)[0] == 0).all()
    empty = torch.empty(0, 3, 64, dtype=torch.float16, device=DEV)
    assert qk_norm_rope(empty, empty, None, None)[0].shape == (0, 3, 64)


# ---------------------------------------------------------------------------
# append
# ---------------------------------------------------------------------------
def new_cache(g, pages, heads, page, dim, dtype=torch.bfloat16):
    from jeeves_amd.attention import PagedKVCache

    return PagedKVCache(randn(g, pages, heads, page, dim, dtype=dtype), randn(g, pages, heads, page, dim, dtype=dtype))


@pytest.mark.parametrize("dim,page,heads", [(64, 16, (5, 5)), (128, 32, (8, 2)), (256, 64, (4, 4)), (128, 1024, (3, 1))])
@pytest.mark.parametrize("tokens", [1, 5, 333])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_append(dim, page, heads, tokens, dtype):
    from jeeves_amd.attention import append_kv, rope_table

    g = gen(tokens + dim)
    hq, hk = heads
    pages = 340 // page + 2
    cache = new_cache(g, pages, hk, page, dim, dtype)
    k_before, v_before = cache.k.clone(), cache.v.clone()
    merged = randn(g, tokens, (hq + 2 * hk) * dim, dtype=dtype)
    q, k, v = (t.view(tokens, -1, dim) for t in merged.split([hq * dim, hk * dim, hk * dim], 1))
    slots = torch.randperm(pages * page, generator=g, device=DEV)[:tokens]
    slots[tokens // 2] = -1 if tokens % 2 else pages * page  # left out
    if tokens == 5:
        slots = slots.to(torch.int32)
    rope, pos = rope_table(100, dim // 2), torch.randint(0, 100, (tokens,), generator=g, device=DEV)
    w = torch.randn(dim, generator=g, device=DEV)
    qo = append_kv(cache, k, v, slots, rope=rope, positions=pos, k_weight=w, q=q, q_weight=w)
    check_norm_rope(qo, q, w, rope, pos)
    keep = (slots >= 0) & (slots < pages * page)
    s = slots[keep].long()
    check_norm_rope(cache.k[s // page, :, s % page], k[keep], w, rope, pos[keep])
    assert torch.equal(cache.v[s // page, :, s % page], v[keep])
    others = torch.ones(pages, page, dtype=torch.bool, device=DEV)
    others[s // page, s % page] = False
    assert torch.equal(cache.k.transpose(1, 2)[others], k_before.transpose(1, 2)[others])
    assert torch.equal(cache.v.transpose(1, 2)[others], v_before.transpose(1, 2)[others])
    k_after = cache.k.clone()
    assert append_kv(cache, k, v, slots, rope=rope, positions=pos, k_weight=w) is None
    assert torch.equal(cache.k, k_after)


def test_append_as_is_moves_bits():
    """Neither norm nor rotation: keys and values are copied, NaN and infinities with them."""
    from jeeves_amd.attention import append_kv

    g = gen(9)
    cache = new_cache(g, 4, 2, 16, 64)
    k, v = randn(g, 20, 2, 64), randn(g, 20, 2, 64)
    k[3, 1, 5], v[4, 0, 7], v[5, 1, 0] = math.inf, math.nan, -math.inf
    append_kv(cache, k, v, torch.arange(10, 30, device=DEV))
    rows = cache.k.transpose(1, 2).reshape(64, 2, 64)[10:30]
    assert torch.equal(rows.view(torch.int16), k.view(torch.int16))
    rows = cache.v.transpose(1, 2).reshape(64, 2, 64)[10:30]
    assert torch.equal(rows.view(torch.int16), v.view(torch.int16))


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------
class Batch:
    """A cache with shuffled pages and a batch over it."""

    def __init__(self, seed, lengths, queries=None, prefix=0, heads=(8, 2), dim=128, page=16, dtype=torch.bfloat16, spare=3):
        g = gen(seed)
        hq, hk = heads
        self.lengths, self.queries, self.prefix, self.page, self.dtype = lengths, queries or [1] * len(lengths), prefix, page, dtype
        need = [-(-l // page) for l in lengths]
        shared = -(-prefix // page)
        total = sum(need) + shared + spare
        order = torch.randperm(total, generator=g, device=DEV).to(torch.int32)
        self.cache = new_cache(g, total, hk, page, dim, dtype)
        self.prefix_pages = order[:shared].contiguous()
        self.table = torch.full((len(lengths), max(need + [0]) + 1), -1, dtype=torch.int32, device=DEV)
        at = shared
        for b, n in enumerate(need):
            self.table[b, :n] = order[at:at + n]
            at += n
        self.q = randn(g, sum(self.queries), hq, dim, dtype=dtype)
        self.device_lengths = torch.tensor(lengths, dtype=torch.int32, device=DEV)
        self.starts = None
        if queries is not None:
            self.starts = torch.tensor([sum(queries[:b]) for b in range(len(queries) + 1)], dtype=torch.int32, device=DEV)

    def run(self, **kw):
        from jeeves_amd.attention import paged_attention

        return paged_attention(self.q, self.cache, self.table, self.device_lengths, query_starts=self.starts,
                               prefix_pages=self.prefix_pages if self.prefix else None, prefix_length=self.prefix, **kw)

    def keys(self, b, pages):
        """Keys or values that sequence b can see, in order: [heads, prefix + length, dim]."""
        ids = self.table[b, :-(-self.lengths[b] // self.page)].long()
        own = pages[ids].transpose(0, 1).flatten(1, 2)[:, :self.lengths[b]]
        shared = pages[self.prefix_pages.long()].transpose(0, 1).flatten(1, 2)[:, :self.prefix]
        return torch.cat([shared, own], 1).double()

    def exact(self, scale=None):
        """(outputs, softmax-weighted means of |v|) in 64 bits, one query head at a time."""
        tokens, hq, dim = self.q.shape
        out = torch.zeros(tokens, hq, dim, dtype=torch.float64, device=DEV)
        mag = torch.zeros_like(out)
        scale = dim ** -0.5 if scale is None else scale
        group, at = hq // self.cache.kv_heads, 0
        for b, (n, length) in enumerate(zip(self.queries, self.lengths)):
            k, v = self.keys(b, self.cache.k), self.keys(b, self.cache.v)
            seen = torch.arange(self.prefix + length, device=DEV)[None] < \
                self.prefix + (length - n + 1 + torch.arange(n, device=DEV)).clamp(min=0)[:, None]
            for h in range(hq if k.shape[1] else 0):
                score = (self.q[at:at + n, h].double() @ k[h // group].t()) * scale
                score[~seen] = -math.inf
                p = torch.softmax(score, 1).nan_to_num(0.0) if not torch.isfinite(score[seen]).all() else \
                    torch.where(seen.any(1, keepdim=True), torch.softmax(score, 1), 0.0)
                out[at:at + n, h] = p @ v[h // group]
                mag[at:at + n, h] = p @ v[h // group].abs()
            at += n
        return out, mag

    def check(self, **kw):
        out = self.run(**kw)
        exact, mag = self.exact(**kw)
        u = U[self.dtype]
        bound = 2 * u * (exact.abs() + mag) + 2.0 ** -14 * mag + (2.0 ** -25 if self.dtype == torch.float16 else 0)
        err = (out.double() - exact).abs()
        assert (err <= bound).all(), (err - bound).max().item()
        assert torch.equal(out, self.run(**kw))  # the same bits again
        return out


@pytest.mark.parametrize("dim,heads", [(64, (4, 4)), (64, (14, 2)), (128, (8, 2)), (128, (5, 5)), (256, (4, 1)), (256, (8, 4))])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("page", [16, 64])
def test_decode_lengths(dim, heads, dtype, page):
    Batch(1, [1, 2, 15, 16, 17, 31, 32, 33, 64, 127, 128, 129, 255, 300, 511, 513, 1000], heads=heads, dim=dim, page=page,
          dtype=dtype).check()


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("batch", [1, 3])
@pytest.mark.parametrize("length", [4095, 20001])
def test_decode_long_keys_split_over_workgroups(dim, batch, length):
    Batch(2, [length - 100 * b for b in range(batch)], heads=(4, 2), dim=dim, page=32).check()


def test_decode_large_ragged_batch():
    rng = random.Random(3)
    Batch(3, [round(math.exp(rng.uniform(0, math.log(900)))) for _ in range(150)], heads=(4, 1), dim=64).check()


@pytest.mark.parametrize("ragged", [False, True])
@pytest.mark.parametrize("prefix", [0, 37])
def test_more_units_than_counters(ragged, prefix):
    """Twice the row tiles of all heads pass the stream's counters: no keys are
    split (with starts the tiles' bound is above their number, which must not
    leave room for a split either), unless a launch of its own joins them."""
    from jeeves_amd.attention import paged_attention

    g = gen(23)
    batch, heads, dim, page = 9001, 8, 64, 16
    cache = new_cache(g, 700, heads, page, dim)
    lengths = torch.randint(0, 49, (batch,), generator=g, device=DEV, dtype=torch.int32)
    lengths[::50] = 300
    table = torch.randint(0, 700, (batch, 19), generator=g, device=DEV, dtype=torch.int32)
    shared = torch.randint(0, 700, (3,), generator=g, device=DEV, dtype=torch.int32)
    q = randn(g, batch, heads, dim)
    starts = torch.arange(batch + 1, device=DEV, dtype=torch.int32) if ragged else None

    def run():
        return paged_attention(q, cache, table, lengths, query_starts=starts, prefix_pages=shared if prefix else None,
                               prefix_length=prefix)

    out = run()
    assert torch.equal(out, run())
    for first in range(0, batch, 500):
        ids = torch.cat([shared[None].expand(batch, -1), table], 1)[first:first + 500].long()
        at = torch.arange(ids.shape[1] * page, device=DEV)
        seen = (at[None] < prefix) | ((at[None] >= 48) & (at[None] - 48 < lengths[first:first + 500, None]))
        k, v = (x[ids].permute(0, 2, 1, 3, 4).reshape(ids.shape[0], heads, -1, dim).double() for x in (cache.k, cache.v))
        score = (k @ q[first:first + 500].double()[..., None])[..., 0] * dim ** -0.5
        p = torch.softmax(score.masked_fill(~seen[:, None], -math.inf), -1).nan_to_num(0.0)[..., None, :]
        exact, mag = (p @ v)[..., 0, :], (p @ v.abs())[..., 0, :]
        err = (out[first:first + 500].double() - exact).abs()
        assert (err <= 2 * 2.0 ** -9 * (exact.abs() + mag) + 2.0 ** -14 * mag).all()


@pytest.mark.parametrize("prefix", [0, 100])
@pytest.mark.parametrize("queries", [[1, 1, 1, 1], [200, 100, 300, 50]])
def test_starts_that_decrease_leave_later_calls_right(queries, prefix):
    """Outside the contract: whatever comes out, the next call's bits are the same."""
    b = Batch(25, [700, 800, 900, 600], queries, prefix=prefix)
    good, starts = b.check(), b.starts
    n = sum(queries)
    for bad in ([0, n, 0, n, n], [n, n - 1, 2, 1, 0], [-5, 2 ** 30, -7, n, 1], [0, n, n, 0, n]):
        b.starts = torch.tensor(bad, dtype=torch.int32, device=DEV)
        assert b.run().shape == b.q.shape
    b.starts = starts
    assert torch.equal(b.run(), good)


@pytest.mark.parametrize("heads", [(16, 1), (17, 1), (32, 1), (64, 2)])
def test_decode_wide_groups(heads):
    Batch(4, [5, 100, 333], heads=heads, dim=128, prefix=70).check()


@pytest.mark.parametrize("dim,heads", [(64, (4, 2)), (128, (8, 2)), (256, (4, 4))])
@pytest.mark.parametrize("prefix", [1, 16, 63, 64, 65, 1000, 5000])
@pytest.mark.parametrize("batch", [1, 2, 33])
def test_decode_with_prefix(dim, heads, prefix, batch):
    Batch(5, [(b * 37) % 200 for b in range(batch)], prefix=prefix, heads=heads, dim=dim, dtype=torch.float16 if prefix == 63 else
          torch.bfloat16).check()


@pytest.mark.parametrize("queries", [None, [1, 40, 3]])
@pytest.mark.parametrize("prefix", [0, 40])
def test_more_key_heads_than_workgroups_at_a_time(queries, prefix):
    Batch(27, [30, 100, 600], queries, prefix=prefix, heads=(600, 600), dim=64).check()


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("rows", [16, 17, 31, 32, 33])
def test_prefix_tiles_of_few_and_many_rows(dim, rows):
    """The rows of all heads of a group at and beside the tiles' sizes."""
    Batch(26, [(b * 53) % 700 for b in range(rows)], prefix=1100, heads=(2, 2), dim=dim).check()


@pytest.mark.parametrize("dim,heads", [(64, (6, 2)), (128, (8, 2)), (128, (3, 3)), (256, (8, 2))])
@pytest.mark.parametrize("prefix", [0, 47, 700])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_ragged_queries(dim, heads, prefix, dtype):
    """Sequences of one query and of many, some after keys of their own, some without."""
    queries = [1, 3, 200, 1, 32, 33, 64, 5]
    before = [0, 10, 0, 400, 31, 100, 1, 64]
    Batch(6, [n + m for n, m in zip(queries, before)], queries, prefix=prefix, heads=heads, dim=dim, page=32, dtype=dtype).check()


@pytest.mark.parametrize("dim,heads", [(64, (4, 1)), (128, (8, 8)), (256, (8, 2))])
def test_long_prompts_fill_the_device(dim, heads):
    """Enough row tiles that none splits its keys."""
    queries = [1500, 7, 2100, 900] if dim == 256 else [1800, 5, 3000, 1]
    b = Batch(7, queries, queries, prefix=100, heads=(heads[0] * 4, heads[1] * 4), dim=dim)
    b.check()


def test_short_speculative_blocks():
    """A few queries a sequence: rows still fit the decode kernel."""
    Batch(8, [100, 4, 260, 33], [4, 4, 2, 3], prefix=0, heads=(8, 2)).check()
    Batch(8, [100, 4, 260, 33], [4, 4, 2, 3], prefix=300, heads=(8, 2)).check()


def test_rows_that_see_nothing():
    # empty sequences, more queries than keys, and sequences without queries
    b = Batch(9, [0, 40, 0], heads=(8, 2))
    out = b.check()
    assert (out[0] == 0).all() and (out[2] == 0).all()
    b = Batch(9, [3, 0, 20, 9], [8, 2, 0, 9], heads=(8, 2))
    out = b.check()
    assert (out[:5] == 0).all() and (out[8:10] == 0).all()
    b = Batch(9, [0, 0, 0], [40, 1, 3], heads=(16, 2), dim=64)
    assert (b.check() == 0).all()
    b = Batch(9, [0, 0], heads=(4, 4))
    assert (b.check() == 0).all()


@pytest.mark.parametrize("heads,queries", [((8, 2), [3, 4]), ((16, 8), [900, 700])])
def test_tokens_of_no_sequence_are_zero(heads, queries):
    from jeeves_amd.attention import paged_attention

    b = Batch(10, [n + 5 for n in queries], queries, heads=heads)
    padded = torch.cat([b.q, torch.full((6, *b.q.shape[1:]), 1.0, dtype=b.dtype, device=DEV)])
    out = paged_attention(padded, b.cache, b.table, b.device_lengths, query_starts=b.starts)
    exact, mag = b.exact()
    assert ((out[:-6].double() - exact).abs() <= 2 * U[b.dtype] * (exact.abs() + mag) + 2.0 ** -14 * mag).all()
    assert (out[-6:] == 0).all()


@pytest.mark.parametrize("queries,lengths,prefix", [
    (None, [7, 90, 40, 200], 0), (None, [7, 90, 40, 200], 50), ([3, 2, 4, 1], [7, 90, 40, 200], 0),
    ([30, 90, 2, 60], [37, 90, 40, 61], 0), ([30, 90, 2, 60], [37, 90, 40, 61], 77), ([700, 800], [700, 810], 90)])
@pytest.mark.parametrize("value", [math.nan, math.inf])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_what_is_not_seen_has_no_effect(queries, lengths, prefix, value, dim):
    """Every page position that belongs to no key, and pages of no one, hold NaN or infinity; and the last own keys of
    a sequence hold them where earlier queries do not see them."""
    b = Batch(11, lengths, queries, prefix=prefix, heads=(16, 8) if max(lengths) > 500 else (8, 2), dim=dim, page=32)
    clean = b.check()
    used = torch.zeros(b.cache.pages, b.page, dtype=torch.bool, device=DEV)
    for i, l in enumerate(b.lengths):
        j = torch.arange(l, device=DEV)
        used[b.table[i].long()[j // b.page], j % b.page] = True
    j = torch.arange(prefix, device=DEV)
    used[b.prefix_pages.long()[j // b.page], j % b.page] = True
    unused = ~used[:, None, :, None]
    b.cache.k.masked_fill_(unused, value)
    b.cache.v.masked_fill_(unused, value)
    assert torch.equal(b.run(), clean)
    if queries is None:
        return
    # the last key of each sequence: only its last query sees it
    last = torch.tensor([sum(b.queries[:i + 1]) - 1 for i in range(len(lengths))], device=DEV)
    others = torch.ones(b.q.shape[0], dtype=torch.bool, device=DEV)
    others[last] = False
    at = [(int(b.table[i, (l - 1) // b.page]), (l - 1) % b.page) for i, l in enumerate(lengths)]
    for page, offset in at:
        b.cache.v[page, :, offset, 3] = value
    out = b.run()
    assert torch.equal(out[others], clean[others])
    bad = out[last][..., 3]
    assert bad.isnan().all() if math.isnan(value) else (bad == value).all()
    assert torch.equal(out[last][..., 4:], clean[last][..., 4:]) and torch.equal(out[last][..., :3], clean[last][..., :3])
    for page, offset in at:
        b.cache.k[page, :, offset, 3] = value
    assert torch.equal(b.run()[others], clean[others])


def test_infinities_of_both_signs_and_seen_ones():
    b = Batch(12, [40, 40], [40, 40], heads=(4, 4), dim=64)
    page, off = int(b.table[0, 2]), 5  # own key 37 of sequence 0
    b.cache.v[page, :, off, 0], b.cache.v[page, :, off, 1] = math.inf, -math.inf
    b.cache.v[page, :, off + 1, 0], b.cache.v[page, :, off + 1, 2] = -math.inf, math.nan
    out = b.run()
    assert out[:37].isfinite().all() and out[40:].isfinite().all()
    assert (out[37, :, 0] == math.inf).all() and (out[37:40, :, 1] == -math.inf).all()
    assert out[38:40, :, 0].isnan().all() and out[38:40, :, 2].isnan().all() and out[37, :, 2].isfinite().all()


@pytest.mark.parametrize("queries", [None, [2, 3], [300, 400]])
def test_large_scores(queries):
    """Scores of a few hundred with running maxima that keep growing, and a scale of the caller's."""
    lengths = [600, 333] if queries is None or queries[0] < 10 else [600, 433]
    b = Batch(13, lengths, queries, heads=(4, 2), dim=128)
    for i, l in enumerate(lengths):
        j = torch.arange(l, device=DEV)
        ids = b.table[i].long()[j // b.page]
        b.cache.k[ids, :, j % b.page] = (b.cache.k[ids, :, j % b.page].float() * (j[:, None, None] / l + 0.1)).to(b.dtype)
    b.check(scale=1.0)
    b.check(scale=0.01)


def test_a_nan_query_stays_its_own():
    b = Batch(14, [50, 60, 70], heads=(8, 2))
    clean = b.run()
    b.q[1, 3, 7] = math.nan
    out = b.run()
    assert out[1, 3].isnan().all()
    out[1, 3] = clean[1, 3]
    assert torch.equal(out, clean)


def test_strided_queries_and_wide_tables():
    from jeeves_amd.attention import paged_attention

    b = Batch(15, [70, 5, 200], heads=(8, 2))
    clean = b.run()
    merged = torch.zeros(3, 3, 8, 128, dtype=b.dtype, device=DEV)
    merged[:, 1] = b.q
    wide = torch.full((3, 64), 2 ** 30, dtype=torch.int64, device=DEV)
    wide[:, 8:8 + b.table.shape[1]] = b.table.clamp(min=0)
    out = paged_attention(merged[:, 1], b.cache, wide[:, 8:], b.device_lengths.long())
    assert torch.equal(out, clean)
    heads_first = b.q.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(paged_attention(heads_first, b.cache, b.table, b.device_lengths), clean)


def test_page_ids_and_lengths_outside_the_cache_are_held_in_range():
    """Ids of no page and lengths past the table read other keys than meant, but none outside the cache."""
    from jeeves_amd.attention import paged_attention

    b = Batch(16, [70, 5], heads=(8, 2))
    ids = torch.tensor([[-5, 2 ** 31 - 1, 0], [1, 2, 3]], dtype=torch.int32, device=DEV)
    out = paged_attention(b.q, b.cache, ids, torch.tensor([2 ** 31 - 1, -7], dtype=torch.int32, device=DEV))
    held = ids.clamp(0, b.cache.pages - 1)
    assert torch.equal(out, paged_attention(b.q, b.cache, held, torch.tensor([48, 0], dtype=torch.int32, device=DEV)))
    assert (out[1] == 0).all()


def test_cache_past_32_bit_offsets():
    """Pages past 2^32 bytes of a cache of 9 GiB."""
    from jeeves_amd.attention import PagedKVCache, append_kv, paged_attention

    heads, page, dim = 8, 64, 128
    pages = (9 << 30) // (2 * heads * page * dim * 2)
    assert (pages - 8) * heads * page * dim > 2 ** 31 and (pages - 8) * heads * page * dim * 2 > 2 ** 32
    cache = PagedKVCache(torch.zeros(pages, heads, page, dim, dtype=torch.bfloat16, device=DEV),
                         torch.zeros(pages, heads, page, dim, dtype=torch.bfloat16, device=DEV))
    g = gen(17)
    k, v, q = randn(g, 200, heads, dim), randn(g, 200, heads, dim), randn(g, 1, 16, dim)
    ids = torch.tensor([[pages - 1, pages - 3, pages - 2, pages - 7]], dtype=torch.int32, device=DEV)
    j = torch.arange(200, device=DEV)
    append_kv(cache, k, v, ids[0].long()[j // page] * page + j % page)
    out = paged_attention(q, cache, ids, torch.tensor([200], dtype=torch.int32, device=DEV))
    small = PagedKVCache(cache.k[-8:].clone(), cache.v[-8:].clone())
    assert torch.equal(out, paged_attention(q, small, ids - (pages - 8), torch.tensor([200], dtype=torch.int32, device=DEV)))
    assert torch.equal(small.k[7, :, 1], k[1]) and torch.equal(small.v[1, :, 199 - 192], v[199])


def test_another_stream_and_a_captured_graph():
    """The calls on a side stream, and in a graph replayed with new lengths and queries between eager work."""
    from jeeves_amd.attention import append_kv, paged_attention, rope_table

    b = Batch(18, [70, 5, 200], prefix=100, heads=(8, 2))
    g = gen(19)
    rope = rope_table(1000, 128)
    k, v = randn(g, 3, 2, 128), randn(g, 3, 2, 128)
    slots, pos = torch.full((3,), -1, device=DEV), torch.arange(3, device=DEV)

    def step():
        q = append_kv(b.cache, k, v, slots, rope=rope, positions=pos, q=b.q)
        return paged_attention(q, b.cache, b.table, b.device_lengths, prefix_pages=b.prefix_pages, prefix_length=100)

    want = step()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        assert torch.equal(step(), want)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            out = step()
    torch.cuda.current_stream().wait_stream(s)
    for i in range(4):
        b.q.copy_(randn(g, *b.q.shape))
        b.device_lengths.copy_(torch.tensor([70 - 20 * i, 5 * i, 200 - i], device=DEV))
        graph.replay()
        got = out.clone()
        assert torch.equal(got, step())
        torch.cuda.synchronize()


# ---------------------------------------------------------------------------
# the block
# ---------------------------------------------------------------------------
def test_attention_block_prompt_then_steps():
    """FP8Attention over a prompt, then token by token: its calls one by one give the same bits, and the cache holds
    what a step needs (the last token of a prompt of n + 1 is the step after a prompt of n)."""
    from jeeves_amd import FP8Linear
    from jeeves_amd.attention import FP8Attention, PagedKVCache, append_kv, paged_attention, rope_table

    g = gen(20)
    hidden, hq, hk, dim, page = 1024, 8, 2, 128, 16
    parts = [FP8Linear(hidden, n * dim, device=DEV) for n in (hq, hk, hk)]
    o = FP8Linear(hq * dim, hidden, device=DEV)
    for m in (*parts, o):
        m.load_weight(randn(g, m.out_features, m.in_features) * 0.03)
    w = 1 + 0.1 * torch.randn(dim, generator=g, device=DEV)
    block = FP8Attention(FP8Linear.concatenated(parts), o, hq, hk, w, w)
    rope = rope_table(256, dim)
    x = randn(g, 42, hidden)
    cache = PagedKVCache.allocate(8, hk, page, dim)
    table = torch.tensor([[5, 2, 7]], dtype=torch.int32, device=DEV)

    def slots(first, n):
        j = torch.arange(first, first + n, device=DEV)
        return table[0].long()[j // page] * page + j % page

    def run(first, n, cache):
        return block(x[first:first + n], cache, slots(first, n), table, torch.tensor([first + n], dtype=torch.int32, device=DEV),
                     rope=rope, positions=torch.arange(first, first + n, device=DEV),
                     query_starts=torch.tensor([0, n], dtype=torch.int32, device=DEV) if n > 1 else None)

    y = run(0, 40, cache)
    q, k, v = block.qkv(x[:40]).split([hq * dim, hk * dim, hk * dim], 1)
    again = PagedKVCache.allocate(8, hk, page, dim)
    q = append_kv(again, k.view(40, hk, dim), v.view(40, hk, dim), slots(0, 40), rope=rope, positions=torch.arange(40, device=DEV),
                  k_weight=w, q=q.view(40, hq, dim), q_weight=w)
    a = paged_attention(q, again, table, torch.tensor([40], device=DEV), query_starts=torch.tensor([0, 40], device=DEV))
    assert torch.equal(o(a.view(40, -1)), y) and torch.equal(again.k, cache.k) and torch.equal(again.v, cache.v)
    steps = [run(40 + i, 1, cache) for i in range(2)]
    whole = run(0, 42, PagedKVCache.allocate(8, hk, page, dim))
    for i in range(2):
        # other tiles round other sums: a step's attention output within one rounding of the prompt's, through o's codes
        diff = (steps[i][0].double() - whole[40 + i].double()).norm() / whole[40 + i].double().norm()
        assert diff < 0.05, diff


# ---------------------------------------------------------------------------
# refusals
# ---------------------------------------------------------------------------
def test_refusals():
    from jeeves_amd.attention import PagedKVCache, append_kv, paged_attention, qk_norm_rope, rope_table

    g = gen(21)
    b = Batch(21, [20, 30], heads=(8, 2))
    q, k = b.q, randn(g, 2, 2, 128)
    rope, pos = rope_table(8, 64), torch.zeros(2, dtype=torch.int32, device=DEV)
    slots = torch.zeros(2, dtype=torch.int64, device=DEV)
    table, lengths = b.table, b.device_lengths
    refused = [
        lambda: qk_norm_rope(q, k[:1], rope, pos),                                      # token counts
        lambda: qk_norm_rope(q, k.half(), rope, pos),                                   # types
        lambda: qk_norm_rope(q.float(), k.float(), rope, pos),
        lambda: qk_norm_rope(q[..., :96], k[..., :96], rope, pos),                      # head size
        lambda: qk_norm_rope(q, k, rope, None),                                         # no positions
        lambda: qk_norm_rope(q, k, rope, pos[:1]),
        lambda: qk_norm_rope(q, k, rope, pos.float()),
        lambda: qk_norm_rope(q, k, rope.cpu(), pos),                                    # devices
        lambda: qk_norm_rope(q.cpu(), k.cpu(), rope.cpu(), pos.cpu()),
        lambda: qk_norm_rope(q, k, rope[:, :24], pos),                                  # rotary size
        lambda: qk_norm_rope(q, k, rope_table(8, 256), pos),
        lambda: qk_norm_rope(q, k, rope, pos, q_weight=torch.ones(64, device=DEV)),
        lambda: append_kv(b.cache, k, k[:, :1], slots),                                 # heads
        lambda: append_kv(b.cache, k.half(), k.half(), slots),
        lambda: append_kv(b.cache, k, k, slots[:1]),
        lambda: append_kv(b.cache, k, k, slots.float()),
        lambda: append_kv(b.cache, k, k, slots.cpu()),
        lambda: append_kv(b.cache, k, k, slots, q=q[:1]),
        lambda: paged_attention(q[:, :7], b.cache, table, lengths),                     # 7 heads over 2
        lambda: paged_attention(q[:1], b.cache, table, lengths),                        # tokens without starts
        lambda: paged_attention(q, b.cache, table[:1], lengths),
        lambda: paged_attention(q, b.cache, table, lengths, query_starts=lengths),      # batch + 1
        lambda: paged_attention(q, b.cache, table, lengths.float()),
        lambda: paged_attention(q, b.cache, table.cpu(), lengths),
        lambda: paged_attention(q, b.cache, table, lengths, prefix_length=5),           # no pages
        lambda: paged_attention(q, b.cache, table, lengths, prefix_length=-1),
        lambda: paged_attention(q, b.cache, table, lengths, prefix_length=17, prefix_pages=table[0, :1]),
        lambda: paged_attention(q, b.cache, table, lengths, scale=0.0),
        lambda: paged_attention(q, b.cache, table, lengths, scale=math.nan),
        lambda: paged_attention(q.half(), b.cache, table, lengths),
        lambda: PagedKVCache(b.cache.k, b.cache.v[:1]),
        lambda: PagedKVCache(b.cache.k[:, :, :8].contiguous(), b.cache.v[:, :, :8].contiguous()),
        lambda: PagedKVCache(b.cache.k[:, :1], b.cache.v[:, :1]),                       # not contiguous
        lambda: PagedKVCache(b.cache.k.float(), b.cache.v.float()),
        lambda: rope_table(8, 40),
    ]
    for call in refused:
        with pytest.raises(ValueError):
            call()
    assert paged_attention(q[:0], b.cache, table[:0], lengths[:0]).shape == (0, 8, 128)
