"""What lies between the q/k/v projection and the o projection of a served
model, on MI355X: the norms and the rotation of queries and keys, the paged
key/value cache and the attention that reads it (C ABI
``include/jeeves_attention.h``).

* ``qk_norm_rope``: per-head RMS norms and the position rotation in one pass;
* ``PagedKVCache``, ``append_kv``: keys normed, rotated and written to their
  slots with the values, the queries in the same launch;
* ``paged_attention``: causal attention of a ragged batch over the cache, the
  keys of a prefix that the batch shares read once for all of it;
* ``FP8Attention``: the four FP8 projections of an attention block with these
  between them.

Tensors are bf16 or fp16. As in ``jeeves_amd.fp8``, everything is enqueued on
``torch.cuda.current_stream()`` without host synchronisation (so it may be
captured into a graph), outputs and workspaces come from torch's caching
allocator, and bad arguments raise ``ValueError``. No gradients: the framework
serves.
"""

from __future__ import annotations

from functools import lru_cache

import torch
import torch.nn as nn

from . import _lib
from .device import sm_count
from .fp8 import _CURRENT, TILE_COUNTER_SLOTS, FP8Linear, _stream_counters

HEAD_DIMS = (64, 128, 256)
_FP16 = {torch.bfloat16: 0, torch.float16: 1}
_WIDE = {torch.int32: 0, torch.int64: 1}


class PagedKVCache:
    """Keys and values of a served model's layer in pages: ``k`` and ``v``
    [pages, kv_heads, page_size, head_dim], bf16 or fp16, contiguous, the page
    size a power of two from 16 to 1024. Which pages a sequence has is the
    caller's to keep; token ``offset`` of page ``page`` is slot
    ``page * page_size + offset``."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor):
        if k.dim() != 4 or k.shape != v.shape or k.dtype != v.dtype or k.device != v.device:
            raise ValueError(f"k and v must be alike, [pages, kv_heads, page_size, head_dim], got {tuple(k.shape)} {k.dtype} and "
                             f"{tuple(v.shape)} {v.dtype}")
        if k.dtype not in _FP16:
            raise ValueError(f"the cache holds bfloat16 or float16, got {k.dtype}")
        page = k.shape[2]
        if page & (page - 1) or not 16 <= page <= 1024 or k.shape[3] not in HEAD_DIMS:
            raise ValueError(f"the page size is a power of two from 16 to 1024 and the head size one of {HEAD_DIMS}, got {page} and "
                             f"{k.shape[3]}")
        if not k.is_contiguous() or not v.is_contiguous() or k.data_ptr() % 16 or v.data_ptr() % 16:
            raise ValueError("the cache's pages must be contiguous and 16-byte aligned")
        self.k, self.v = k, v
        self.pages, self.kv_heads, self.page_size, self.head_dim = k.shape
        self._goes_with = (k.dtype, k.get_device(), self.head_dim)

    def check(self, dtype: torch.dtype, index: int, dim: int) -> None:
        """Refuses heads of another type, device (its index) or size than the cache's."""
        if (dtype, index, dim) != self._goes_with:
            raise ValueError(f"heads of {dim} channels of {dtype} on HIP device {index} do not go with a cache of "
                             f"{tuple(self.k.shape)} {self.k.dtype} on {self.k.device}")

    @classmethod
    def allocate(cls, pages: int, kv_heads: int, page_size: int, head_dim: int, dtype: torch.dtype = torch.bfloat16,
                 device: torch.device | str = "cuda") -> "PagedKVCache":
        shape = (pages, kv_heads, page_size, head_dim)
        return cls(torch.zeros(shape, dtype=dtype, device=device), torch.zeros(shape, dtype=dtype, device=device))


def rope_table(positions: int, rotary: int, base: float = 10000.0, device: torch.device | str = "cuda") -> torch.Tensor:
    """The angles of ``positions`` positions as the kernels read them: float32
    [positions, rotary], each position's ``rotary / 2`` cosines, then its sines,
    for the frequencies ``base ** (-2 i / rotary)``. Computed in 64 bits."""
    if rotary <= 0 or rotary % 16:
        raise ValueError(f"the rotation takes a multiple of 16 channels, got {rotary}")
    freq = base ** (-torch.arange(0, rotary, 2, dtype=torch.float64) / rotary)
    angle = torch.arange(positions, dtype=torch.float64)[:, None] * freq
    return torch.cat([angle.cos(), angle.sin()], 1).float().to(device)


# The calls below are a few microseconds of work on small batches, so their
# host path is kept short: sizes and devices are compared as they come from the
# tensors, once, and formatted only where they are refused.
def _refuse(name: str, t: torch.Tensor, wanted: str) -> None:
    raise ValueError(f"{name} must be {wanted}, got {tuple(t.shape)} {t.dtype} on {t.device}")


def _heads(name: str, t: torch.Tensor, dtype: torch.dtype, index: int, tokens: int, dim: int) -> tuple:
    """``t`` [tokens, heads, dim] with 16-byte aligned rows: (the tensor, its
    address, its token and head strides, its heads)."""
    shape = t.shape
    if len(shape) != 3 or shape[0] != tokens or shape[2] != dim or t.dtype is not dtype or t.get_device() != index:
        _refuse(name, t, f"{dtype} [{tokens}, heads, {dim}] on HIP device {index}")
    ts, hs, unit = t.stride()
    ptr = t.data_ptr()
    if unit != 1 or (ts | hs) & 7 or ptr & 15:
        t = t.clone(memory_format=torch.contiguous_format)
        (ts, hs, _), ptr = t.stride(), t.data_ptr()
    return t, ptr, ts, hs, shape[1]


def _first(name: str, t: torch.Tensor) -> tuple:
    """(dtype, device index, tokens, head size) that the other operands go by."""
    shape, dtype, index = t.shape, t.dtype, t.get_device()
    if len(shape) != 3 or shape[2] not in HEAD_DIMS or dtype not in _FP16 or index < 0:
        _refuse(name, t, f"bfloat16 or float16 [tokens, heads, head size of {HEAD_DIMS}] on a HIP device")
    return dtype, index, shape[0], shape[2]


def _indices(name: str, t: torch.Tensor, tokens: int, index: int) -> torch.Tensor:
    if t.dtype not in _WIDE or t.shape != (tokens,) or t.get_device() != index:
        _refuse(name, t, f"int32 or int64 [{tokens}] on HIP device {index}")
    return t if tokens < 2 or t.stride(0) == 1 else t.contiguous()


_NO_ROPE = (None, None, 0, 0, None, None, 0)


def _rope_operands(rope: torch.Tensor | None, positions: torch.Tensor | None, tokens: int, dim: int, index: int) -> tuple:
    """(table, its address, positions and channels; positions, their address, whether wide); the tensors to hold."""
    if rope is None:
        return _NO_ROPE
    shape = rope.shape
    # an empty table has no address, which would mean no rotation
    if (rope.dtype is not torch.float32 or len(shape) != 2 or rope.get_device() != index or not shape[0] or shape[1] & 15 or
            not 0 < shape[1] <= dim):
        _refuse("rope", rope, f"float32 [positions (1 at least), a multiple of 16 channels up to {dim}] on HIP device {index}")
    if positions is None:
        raise ValueError("the rotation needs the tokens' positions")
    if not rope.is_contiguous() or rope.data_ptr() & 15:
        rope = rope.clone(memory_format=torch.contiguous_format)
    positions = _indices("positions", positions, tokens, index)
    return rope, rope.data_ptr(), shape[0], shape[1], positions, positions.data_ptr(), _WIDE[positions.dtype]


def _head_weight(name: str, w: torch.Tensor, dim: int, index: int) -> torch.Tensor:
    if w.shape != (dim,) or w.get_device() != index:
        _refuse(name, w, f"[{dim}] on HIP device {index}")
    return w if w.dtype is torch.float32 and w.is_contiguous() else w.to(torch.float32).contiguous()


def _on(index: int):
    """``torch.cuda.device`` of a device index, which costs two switches even where it is current."""
    return _CURRENT if torch._C._cuda_getDevice() == index else torch.cuda.device(index)


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, rope: torch.Tensor | None, positions: torch.Tensor | None, *,
                 q_weight: torch.Tensor | None = None, k_weight: torch.Tensor | None = None,
                 eps: float = 1e-6) -> tuple[torch.Tensor, torch.Tensor]:
    """Queries [tokens, q_heads, head_dim] and keys [tokens, kv_heads,
    head_dim], normed and rotated, as new contiguous tensors.

    Each head row becomes ``x * weight / sqrt(mean(x^2) + eps)`` (a model whose
    norms scale by 1 + w passes 1 + w; None: no norm), then its channels i and
    ``i + rotary / 2`` are turned by the angle that ``rope`` (``rope_table``;
    None: no rotation) has for the token's position. In 32 bits, rounded once.
    The inputs may be views of a merged projection's output. A token whose
    position the table does not have comes out as NaN.
    """
    dtype, index, tokens, dim = _first("q", q)
    q, q_ptr, q_ts, q_hs, q_heads = _heads("q", q, dtype, index, tokens, dim)
    k, k_ptr, k_ts, k_hs, kv_heads = _heads("k", k, dtype, index, tokens, dim)
    rope, rope_ptr, n_pos, rotary, positions, pos_ptr, wide = _rope_operands(rope, positions, tokens, dim, index)
    if q_weight is not None:
        q_weight = _head_weight("q_weight", q_weight, dim, index)
    if k_weight is not None:
        k_weight = _head_weight("k_weight", k_weight, dim, index)
    q_out = torch.empty_like(q, memory_format=torch.contiguous_format)
    k_out = torch.empty_like(k, memory_format=torch.contiguous_format)
    if tokens:
        with _on(index):
            _lib.check(_lib.lib().jv_norm_rope(
                q_ptr, q_ts, q_hs, k_ptr, k_ts, k_hs, rope_ptr, n_pos, rotary, pos_ptr, wide,
                None if q_weight is None else q_weight.data_ptr(), None if k_weight is None else k_weight.data_ptr(), eps,
                q_out.data_ptr(), k_out.data_ptr(), tokens, q_heads, kv_heads, dim, _FP16[dtype],
                torch._C._cuda_getCurrentRawStream(index)))
    return q_out, k_out


def append_kv(cache: PagedKVCache, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, *, rope: torch.Tensor | None = None,
              positions: torch.Tensor | None = None, k_weight: torch.Tensor | None = None, q: torch.Tensor | None = None,
              q_weight: torch.Tensor | None = None, eps: float = 1e-6) -> torch.Tensor | None:
    """Writes keys [tokens, kv_heads, head_dim], normed and rotated as by
    ``qk_norm_rope``, and values into the cache's ``slots`` (int32 or int64
    [tokens]); a token whose slot is negative or past the cache is left out
    (padding). Slots are meant to differ: of two tokens with one slot either's
    row may stay. With ``q`` the same launch norms and rotates the queries,
    which are returned as a new contiguous tensor."""
    dtype, index, tokens, dim = _first("k", k)
    cache.check(dtype, index, dim)
    k, k_ptr, k_ts, k_hs, kv_heads = _heads("k", k, dtype, index, tokens, dim)
    v, v_ptr, v_ts, v_hs, v_heads = _heads("v", v, dtype, index, tokens, dim)
    if kv_heads != cache.kv_heads or v_heads != kv_heads:
        raise ValueError(f"the cache has {cache.kv_heads} heads, got {kv_heads} of k and {v_heads} of v")
    slots = _indices("slots", slots, tokens, index)
    rope, rope_ptr, n_pos, rotary, positions, pos_ptr, wide = _rope_operands(rope, positions, tokens, dim, index)
    if k_weight is not None:
        k_weight = _head_weight("k_weight", k_weight, dim, index)
    if q_weight is not None:
        q_weight = _head_weight("q_weight", q_weight, dim, index)
    q_out, q_ptr, q_ts, q_hs, q_heads = None, None, 0, 0, 0
    if q is not None:
        q, q_ptr, q_ts, q_hs, q_heads = _heads("q", q, dtype, index, tokens, dim)
        q_out = torch.empty_like(q, memory_format=torch.contiguous_format)
    if tokens:
        with _on(index):
            _lib.check(_lib.lib().jv_append_kv(
                k_ptr, k_ts, k_hs, v_ptr, v_ts, v_hs, slots.data_ptr(), _WIDE[slots.dtype], cache.k.data_ptr(), cache.v.data_ptr(),
                cache.pages, cache.page_size, rope_ptr, n_pos, rotary, pos_ptr, wide,
                None if k_weight is None else k_weight.data_ptr(), eps, q_ptr, q_ts, q_hs,
                None if q_weight is None else q_weight.data_ptr(), None if q is None else q_out.data_ptr(), q_heads, tokens,
                kv_heads, dim, _FP16[dtype], torch._C._cuda_getCurrentRawStream(index)))
    return q_out


@lru_cache(maxsize=4096)
def _plan(index: int, tokens: int, batch: int, q_heads: int, kv_heads: int, dim: int, prefix: int, ragged: bool) -> tuple[int, int]:
    """(workspace bytes, counters) for these sizes on a device, which is current."""
    L = _lib.lib()
    sizes = (L.jv_paged_attention_workspace_bytes(tokens, batch, q_heads, kv_heads, dim, prefix, ragged),
             L.jv_paged_attention_counters_needed(tokens, batch, q_heads, kv_heads, dim, prefix, ragged))
    if min(sizes) < 0:
        raise ValueError(f"the attention does not take {tokens} tokens of {batch} sequences, {q_heads} and {kv_heads} heads")
    return sizes


def _int32(name: str, t: torch.Tensor, shape: tuple, index: int) -> torch.Tensor:
    if t.dtype not in _WIDE or t.shape != shape or t.get_device() != index:
        _refuse(name, t, f"int32 or int64 {list(shape)} on HIP device {index}")
    if t.dtype is not torch.int32:
        rows, columns = shape if len(shape) == 2 else (1, shape[0])
        out = torch.empty(shape, dtype=torch.int32, device=t.device)
        with _on(index):
            _lib.check(_lib.lib().jv_narrow_indices(t.data_ptr(), rows, columns, t.stride(0), t.stride(-1), out.data_ptr(),
                                                    torch._C._cuda_getCurrentRawStream(index)))
        return out
    return t if t.stride(-1) == 1 or shape[-1] < 2 else t.contiguous()


def paged_attention(q: torch.Tensor, cache: PagedKVCache, page_table: torch.Tensor, lengths: torch.Tensor, *,
                    query_starts: torch.Tensor | None = None, prefix_pages: torch.Tensor | None = None, prefix_length: int = 0,
                    scale: float | None = None) -> torch.Tensor:
    """Attention of queries [tokens, q_heads, head_dim] over the cache; a new
    tensor of their shape.

    Sequence b of the batch owns the first ``lengths[b]`` keys of the pages
    ``page_table[b]`` ([batch, columns]); its queries are the tokens
    ``query_starts[b]`` to ``query_starts[b + 1] - 1`` ([batch + 1], not
    decreasing, from 0 to tokens; None: one token each), the last of them at
    its last key: query i of n sees the own keys up to ``lengths[b] - n + i``. With
    ``prefix_length`` all queries of the batch also see that many keys of
    ``prefix_pages``, which come before all own ones; where each sequence has
    few queries they are read once for the batch, not once for each sequence.
    Query head h reads key head ``h // (q_heads / kv_heads)``; ``scale``
    defaults to ``head_dim ** -0.5``.

    A token that sees no key, or that belongs to no sequence, comes out as 0.
    Keys that a token does not see have no effect on it, even infinite or NaN
    ones; nor has what the table holds past a sequence's length, nor the other
    sequences' keys (their lengths decide how keys are cut, which can change a
    token's last bits). A NaN that it sees stays NaN. The sums are in 32 bits; where many query rows go through the same
    keys (prompts, a prefix that many sequences share) the softmax's weights
    are rounded to the 16-bit type for the product with the values, and their
    sum is of the rounded ones.

    As a split-K GEMM of ``jeeves_amd.fp8`` does, a call whose keys are split
    over workgroups counts them in on the stream's tile counters, so run one on
    a stream before capturing a graph on it. (Single tokens over a prefix need
    none.)
    """
    dtype, index, tokens, dim = _first("q", q)
    cache.check(dtype, index, dim)
    q, q_ptr, q_ts, q_hs, q_heads = _heads("q", q, dtype, index, tokens, dim)
    kv_heads = cache.kv_heads
    if q_heads % kv_heads:
        raise ValueError(f"{q_heads} query heads are no multiple of the cache's {kv_heads}")
    if page_table.dim() != 2:
        _refuse("page_table", page_table, "int32 or int64 [batch, columns]")
    batch, columns = shape = page_table.shape
    page_table = _int32("page_table", page_table, shape, index)
    lengths = _int32("lengths", lengths, (batch,), index)
    starts_ptr = prefix_ptr = None
    if query_starts is not None:
        query_starts = _int32("query_starts", query_starts, (batch + 1,), index)
        starts_ptr = query_starts.data_ptr()
    elif tokens != batch:
        raise ValueError(f"without query_starts each of the {batch} sequences has one query, got {tokens}")
    if prefix_length:
        if prefix_length < 0 or prefix_pages is None or prefix_pages.dim() != 1:
            raise ValueError(f"a prefix of {prefix_length} keys needs its pages, int32 or int64 [n]")
        prefix_pages = _int32("prefix_pages", prefix_pages, prefix_pages.shape, index)
        if prefix_pages.shape[0] * cache.page_size < prefix_length:
            raise ValueError(f"{prefix_pages.shape[0]} pages of {cache.page_size} do not hold a prefix of {prefix_length} keys")
        prefix_ptr = prefix_pages.data_ptr()
    out = torch.empty_like(q, memory_format=torch.contiguous_format)
    if tokens:
        with _on(index):
            ws_bytes, counted = _plan(index, tokens, batch, q_heads, kv_heads, dim, prefix_length, query_starts is not None)
            ws_ptr, counters_ptr, n_counters = None, None, 0
            if ws_bytes:
                ws = torch.empty(ws_bytes, dtype=torch.uint8, device=q.device)
                ws_ptr = ws.data_ptr()
            if counted:
                counters_ptr, n_counters = _stream_counters(q.device).data_ptr(), TILE_COUNTER_SLOTS
            _lib.check(_lib.lib().jv_paged_attention(
                q_ptr, q_ts, q_hs, cache.k.data_ptr(), cache.v.data_ptr(), cache.pages, cache.page_size, page_table.data_ptr(),
                page_table.stride(0), columns, lengths.data_ptr(), starts_ptr, batch, prefix_ptr, prefix_length,
                dim ** -0.5 if scale is None else scale, out.data_ptr(), tokens, q_heads, kv_heads, dim, _FP16[dtype], ws_ptr,
                ws_bytes, counters_ptr, n_counters, torch._C._cuda_getCurrentRawStream(index)))
    return out


class FP8Attention(nn.Module):
    """An attention block over FP8 projections: the merged q/k/v projection
    (``FP8Linear.concatenated``, rows of all q heads, then k, then v), norms,
    rotation and append in one launch, the attention over the paged cache, and
    the o projection. A projection with other rows merged in, an output gate's
    say, is not for it: split those off around ``append_kv`` and
    ``paged_attention``."""

    def __init__(self, qkv: FP8Linear, o: FP8Linear, q_heads: int, kv_heads: int, q_weight: torch.Tensor | None = None,
                 k_weight: torch.Tensor | None = None, eps: float = 1e-6):
        super().__init__()
        if qkv.out_features % (q_heads + 2 * kv_heads):
            raise ValueError(f"{qkv.out_features} outputs are no whole heads of {q_heads} + 2 * {kv_heads}")
        self.qkv, self.o = qkv, o
        self.q_heads, self.kv_heads, self.head_dim = q_heads, kv_heads, qkv.out_features // (q_heads + 2 * kv_heads)
        if o.in_features != q_heads * self.head_dim or self.head_dim not in HEAD_DIMS or q_heads % kv_heads:
            raise ValueError(f"o takes {o.in_features} channels, q has {q_heads} heads of {self.head_dim}, k {kv_heads}")
        for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
            self.register_buffer(name, None if w is None else w.detach().to(torch.float32))
        self.eps = eps

    @torch.no_grad()
    def warm(self) -> None:
        """Runs the block's operators in each of their forms on empty sequences,
        as ``jeeves_amd.fp8.warm`` runs its linears: kernels load and the
        stream's counters exist before graph capture."""
        device, dim, group = self.qkv.weight.device, self.head_dim, self.q_heads // self.kv_heads
        cache = PagedKVCache.allocate(1, self.kv_heads, 16, dim, device=device)

        def batch(sequences: int, queries: int, prefix: int) -> None:
            tokens = sequences * queries
            q = torch.zeros(tokens, self.q_heads, dim, dtype=torch.bfloat16, device=device)
            none = torch.zeros(sequences, 1, dtype=torch.int32, device=device)
            starts = torch.arange(0, tokens + 1, queries, dtype=torch.int32, device=device) if queries > 1 else None
            paged_attention(q, cache, none, none[:, 0], query_starts=starts, prefix_pages=none[0] if prefix else None,
                            prefix_length=prefix)

        k = torch.zeros(1, self.kv_heads, dim, dtype=torch.bfloat16, device=device)
        append_kv(cache, k, k, torch.full((1,), -1, dtype=torch.int32, device=device),
                  q=torch.zeros(1, self.q_heads, dim, dtype=torch.bfloat16, device=device))
        many = 16 // group + 1  # queries of more than 16 rows
        batch(1, 1, 0)
        batch(1, 1, 16)
        batch(33, 1, 16)
        batch(1, max(many, 2), 0)
        batch(2 * sm_count(device) + 1, max(many, 2), 0)  # more row tiles than workgroups at a time: whole ones

    def forward(self, x: torch.Tensor, cache: PagedKVCache, slots: torch.Tensor, page_table: torch.Tensor, lengths: torch.Tensor, *,
                rope: torch.Tensor | None = None, positions: torch.Tensor | None = None, query_starts: torch.Tensor | None = None,
                prefix_pages: torch.Tensor | None = None, prefix_length: int = 0) -> torch.Tensor:
        """x [tokens, hidden] -> [tokens, hidden]. ``lengths`` count the keys
        that this call appends; the other arguments are ``append_kv``'s and
        ``paged_attention``'s."""
        tokens, q_size, kv_size = x.shape[0], self.q_heads * self.head_dim, self.kv_heads * self.head_dim
        q, k, v = self.qkv(x).split([q_size, kv_size, kv_size], 1)
        q = append_kv(cache, k.view(tokens, self.kv_heads, self.head_dim), v.view(tokens, self.kv_heads, self.head_dim), slots,
                      rope=rope, positions=positions, k_weight=self.k_weight, q=q.view(tokens, self.q_heads, self.head_dim),
                      q_weight=self.q_weight, eps=self.eps)
        y = paged_attention(q, cache, page_table, lengths, query_starts=query_starts, prefix_pages=prefix_pages,
                            prefix_length=prefix_length)
        return self.o(y.view(tokens, q_size))
