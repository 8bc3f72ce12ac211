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
from .fp8 import FP8Linear, _device_guard, _stream

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


def _heads(name: str, t: torch.Tensor, like: torch.Tensor | None = None) -> torch.Tensor:
    """``t`` as [tokens, heads, head_dim] with 16-byte aligned rows."""
    if t.dim() != 3 or t.dtype not in _FP16 or t.shape[2] not in HEAD_DIMS:
        raise ValueError(f"{name} must be bfloat16 or float16 [tokens, heads, head_dim] with a head size of {HEAD_DIMS}, got "
                         f"{tuple(t.shape)} {t.dtype}")
    if like is not None and (t.dtype != like.dtype or t.shape[0] != like.shape[0] or t.shape[2] != like.shape[2]
                             or t.device != like.device):
        raise ValueError(f"{name} {tuple(t.shape)} {t.dtype} on {t.device} does not go with {tuple(like.shape)} {like.dtype} on "
                         f"{like.device}")
    if not t.is_cuda:
        raise ValueError(f"the attention kernels run on a HIP device; {name} is on {t.device}")
    ts, hs, unit = t.stride()
    if unit != 1 or ts % 8 or hs % 8 or t.data_ptr() % 16:
        t = t.clone(memory_format=torch.contiguous_format)
    return t


def _indices(name: str, t: torch.Tensor, tokens: int, dev: torch.device) -> torch.Tensor:
    if t.dtype not in _WIDE or t.shape != (tokens,) or t.device != dev:
        raise ValueError(f"{name} must be int32 or int64 [{tokens}] on {dev}, got {tuple(t.shape)} {t.dtype} on {t.device}")
    return t if t.stride(0) == 1 or tokens < 2 else t.contiguous()


def _rope_operands(rope: torch.Tensor | None, positions: torch.Tensor | None, tokens: int, dim: int, dev: torch.device):
    if rope is None:
        return None, 0, 0, None, 0
    if rope.dtype != torch.float32 or rope.dim() != 2 or rope.device != dev or rope.shape[1] % 16 or not 0 < rope.shape[1] <= dim:
        raise ValueError(f"rope must be float32 [positions, rotary] on {dev} with rotary a multiple of 16 up to {dim}, got "
                         f"{tuple(rope.shape)} {rope.dtype} on {rope.device}")
    if positions is None:
        raise ValueError("the rotation needs the tokens' positions")
    if not rope.is_contiguous() or rope.data_ptr() % 16:
        rope = rope.clone(memory_format=torch.contiguous_format)
    positions = _indices("positions", positions, tokens, dev)
    return rope, rope.shape[0], rope.shape[1], positions, _WIDE[positions.dtype]


def _head_weight(name: str, w: torch.Tensor | None, dim: int, dev: torch.device) -> torch.Tensor | None:
    if w is None:
        return None
    if w.shape != (dim,) or w.device != dev:
        raise ValueError(f"{name} must be [{dim}] on {dev}, got {tuple(w.shape)} on {w.device}")
    return w if w.dtype == torch.float32 and w.is_contiguous() else w.to(torch.float32).contiguous()


def _ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


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
    q = _heads("q", q)
    k = _heads("k", k, q)
    tokens, q_heads, dim = q.shape
    dev = q.device
    rope, n_pos, rotary, positions, wide = _rope_operands(rope, positions, tokens, dim, dev)
    q_weight, k_weight = _head_weight("q_weight", q_weight, dim, dev), _head_weight("k_weight", k_weight, dim, dev)
    q_out = torch.empty(q.shape, dtype=q.dtype, device=dev)
    k_out = torch.empty(k.shape, dtype=q.dtype, device=dev)
    if tokens:
        with _device_guard(dev):
            _lib.check(_lib.lib().jv_norm_rope(q.data_ptr(), q.stride(0), q.stride(1), k.data_ptr(), k.stride(0), k.stride(1),
                                               _ptr(rope), n_pos, rotary, _ptr(positions), wide, _ptr(q_weight), _ptr(k_weight), eps,
                                               q_out.data_ptr(), k_out.data_ptr(), tokens, q_heads, k.shape[1], dim,
                                               _FP16[q.dtype], _stream(dev)))
    return q_out, k_out


def _check_cache(cache: PagedKVCache, t: torch.Tensor) -> None:
    if t.device != cache.k.device or t.dtype != cache.k.dtype or t.shape[2] != cache.head_dim:
        raise ValueError(f"{tuple(t.shape)} {t.dtype} on {t.device} does not go with a cache of {tuple(cache.k.shape)} {cache.k.dtype} "
                         f"on {cache.k.device}")


def append_kv(cache: PagedKVCache, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, *, rope: torch.Tensor | None = None,
              positions: torch.Tensor | None = None, k_weight: torch.Tensor | None = None, q: torch.Tensor | None = None,
              q_weight: torch.Tensor | None = None, eps: float = 1e-6) -> torch.Tensor | None:
    """Writes keys [tokens, kv_heads, head_dim], normed and rotated as by
    ``qk_norm_rope``, and values into the cache's ``slots`` (int32 or int64
    [tokens]); a token whose slot is negative or past the cache is left out
    (padding). Slots are meant to differ: of two tokens with one slot either's
    row may stay. With ``q`` the same launch norms and rotates the queries,
    which are returned as a new contiguous tensor."""
    k = _heads("k", k)
    v = _heads("v", v, k)
    tokens, kv_heads, dim = k.shape
    dev = k.device
    _check_cache(cache, k)
    if kv_heads != cache.kv_heads or v.shape[1] != kv_heads:
        raise ValueError(f"the cache has {cache.kv_heads} heads, got {kv_heads} of k and {v.shape[1]} of v")
    slots = _indices("slots", slots, tokens, dev)
    rope, n_pos, rotary, positions, wide = _rope_operands(rope, positions, tokens, dim, dev)
    k_weight, q_weight = _head_weight("k_weight", k_weight, dim, dev), _head_weight("q_weight", q_weight, dim, dev)
    q_out, q_heads, q_ts, q_hs = None, 0, 0, 0
    if q is not None:
        q = _heads("q", q, k)
        q_heads, (q_ts, q_hs, _) = q.shape[1], q.stride()
        q_out = torch.empty(q.shape, dtype=q.dtype, device=dev)
    if tokens:
        with _device_guard(dev):
            _lib.check(_lib.lib().jv_append_kv(k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(), v.stride(0), v.stride(1),
                                               slots.data_ptr(), _WIDE[slots.dtype], cache.k.data_ptr(), cache.v.data_ptr(),
                                               cache.pages, cache.page_size, _ptr(rope), n_pos, rotary, _ptr(positions), wide,
                                               _ptr(k_weight), eps, _ptr(q), q_ts, q_hs, _ptr(q_weight), _ptr(q_out), q_heads,
                                               tokens, kv_heads, dim, _FP16[k.dtype], _stream(dev)))
    return q_out


@lru_cache(maxsize=4096)
def _workspace(device: torch.device, tokens: int, batch: int, q_heads: int, kv_heads: int, dim: int, prefix: int,
               ragged: bool) -> int:
    """Workspace bytes for these sizes on ``device``, which is current."""
    n = _lib.lib().jv_paged_attention_workspace_bytes(tokens, batch, q_heads, kv_heads, dim, prefix, ragged)
    if n < 0:
        raise ValueError(f"the attention does not take {tokens} tokens of {batch} sequences, {q_heads} and {kv_heads} heads")
    return n


def _int32(name: str, t: torch.Tensor, dims: int, dev: torch.device) -> torch.Tensor:
    if t.dim() != dims or t.device != dev or t.dtype not in _WIDE:
        raise ValueError(f"{name} must be an int32 or int64 tensor of {dims} dimensions on {dev}, got {tuple(t.shape)} {t.dtype} on "
                         f"{t.device}")
    if t.dtype != torch.int32:
        t = t.to(torch.int32)
    return t if t.stride(-1) == 1 or t.shape[-1] < 2 else t.contiguous()


def paged_attention(q: torch.Tensor, cache: PagedKVCache, page_table: torch.Tensor, lengths: torch.Tensor, *,
                    query_starts: torch.Tensor | None = None, prefix_pages: torch.Tensor | None = None, prefix_length: int = 0,
                    scale: float | None = None) -> torch.Tensor:
    """Attention of queries [tokens, q_heads, head_dim] over the cache; a new
    tensor of their shape.

    Sequence b of the batch owns the first ``lengths[b]`` keys of the pages
    ``page_table[b]`` ([batch, columns]); its queries are the tokens
    ``query_starts[b]`` to ``query_starts[b + 1] - 1`` ([batch + 1], not
    decreasing from 0; None: one token each), the last of them at its last key: query i
    of n sees the own keys up to ``lengths[b] - n + i``. With
    ``prefix_length`` all queries of the batch also see that many keys of
    ``prefix_pages``, which come before all own ones; they are read once for
    the batch, not once for each sequence.
    Query head h reads key head ``h // (q_heads / kv_heads)``; ``scale``
    defaults to ``head_dim ** -0.5``.

    A token that sees no key, or that belongs to no sequence, comes out as 0.
    Keys that a token does not see have no effect on it, even infinite or NaN
    ones; nor has what the table holds past a sequence's length. The sums are
    in 32 bits; the softmax's weights are rounded to the 16-bit type for the
    product with the values.
    """
    q = _heads("q", q)
    tokens, q_heads, dim = q.shape
    dev = q.device
    _check_cache(cache, q)
    if q_heads % cache.kv_heads:
        raise ValueError(f"{q_heads} query heads are no multiple of the cache's {cache.kv_heads}")
    page_table = _int32("page_table", page_table, 2, dev)
    lengths = _int32("lengths", lengths, 1, dev)
    batch = lengths.shape[0]
    if page_table.shape[0] != batch:
        raise ValueError(f"page_table has {page_table.shape[0]} rows for {batch} lengths")
    if query_starts is None:
        if tokens != batch:
            raise ValueError(f"without query_starts each of the {batch} sequences has one query, got {tokens}")
    else:
        query_starts = _int32("query_starts", query_starts, 1, dev)
        if query_starts.shape[0] != batch + 1:
            raise ValueError(f"query_starts must have {batch + 1} values, got {query_starts.shape[0]}")
    if prefix_length < 0 or (prefix_length and prefix_pages is None):
        raise ValueError(f"a prefix of {prefix_length} keys needs its pages")
    if prefix_length:
        prefix_pages = _int32("prefix_pages", prefix_pages, 1, dev)
        if prefix_pages.shape[0] * cache.page_size < prefix_length:
            raise ValueError(f"{prefix_pages.shape[0]} pages of {cache.page_size} do not hold a prefix of {prefix_length} keys")
    out = torch.empty(q.shape, dtype=q.dtype, device=dev)
    if tokens:
        with _device_guard(dev):
            ws_bytes = _workspace(dev, tokens, batch, q_heads, cache.kv_heads, dim, prefix_length, query_starts is not None)
            ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev) if ws_bytes else None
            _lib.check(_lib.lib().jv_paged_attention(
                q.data_ptr(), q.stride(0), q.stride(1), cache.k.data_ptr(), cache.v.data_ptr(), cache.pages, cache.page_size,
                page_table.data_ptr(), page_table.stride(0), page_table.shape[1], lengths.data_ptr(), _ptr(query_starts), batch,
                _ptr(prefix_pages) if prefix_length else None, prefix_length, dim ** -0.5 if scale is None else scale,
                out.data_ptr(), tokens, q_heads, cache.kv_heads, dim, _FP16[q.dtype], _ptr(ws), ws_bytes, _stream(dev)))
    return out


class FP8Attention(nn.Module):
    """An attention block over FP8 projections: the merged q/k/v projection
    (``FP8Linear.concatenated``, rows of all q heads, then k, then v), norms,
    rotation and append in one launch, the attention over the paged cache, and
    the o projection."""

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

    def forward(self, x: torch.Tensor, cache: PagedKVCache, slots: torch.Tensor, page_table: torch.Tensor, lengths: torch.Tensor, *,
                rope: torch.Tensor | None = None, positions: torch.Tensor | None = None, query_starts: torch.Tensor | None = None,
                prefix_pages: torch.Tensor | None = None, prefix_length: int = 0) -> torch.Tensor:
        """x [tokens, hidden] -> [tokens, hidden]. ``lengths`` count the keys
        that this call appends; the other arguments are ``append_kv``'s and
        ``paged_attention``'s."""
        tokens, q_size, kv_size = x.shape[0], self.q_heads * self.head_dim, self.kv_heads * self.head_dim
        q, k, v = self.qkv(x).split([q_size, kv_size, kv_size], 1)
        q = append_kv(cache, k.view(tokens, self.kv_heads, -1), v.view(tokens, self.kv_heads, -1), slots, rope=rope,
                      positions=positions, k_weight=self.k_weight, q=q.view(tokens, self.q_heads, -1), q_weight=self.q_weight,
                      eps=self.eps)
        y = paged_attention(q, cache, page_table, lengths, query_starts=query_starts, prefix_pages=prefix_pages,
                            prefix_length=prefix_length)
        return self.o(y.view(tokens, q_size))
