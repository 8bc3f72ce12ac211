"""The attention's C entry points refuse bad arguments before they touch the
device, and count what they need on the host."""

from __future__ import annotations

import pytest

from jeeves_amd import _lib

P = 4096  # an aligned address that no refused call follows


def norm_rope(L, q=P, q_ts=1024, q_hs=128, k=P, rope=P, n_pos=8, rotary=64, pos=P, q_out=P, k_out=P, tokens=4, q_heads=8, kv_heads=2,
              dim=128):
    return L.jv_norm_rope(q, q_ts, q_hs, k, 256, 128, rope, n_pos, rotary, pos, 0, None, None, 1e-6, q_out, k_out, tokens, q_heads,
                          kv_heads, dim, 0, None)


def append(L, k=P, k_ts=256, v=P, slots=P, k_pages=P, v_pages=P, pages=4, page=16, rotary=64, q=None, q_out=None, tokens=4,
           kv_heads=2, dim=128):
    return L.jv_append_kv(k, k_ts, 128, v, 256, 128, slots, 1, k_pages, v_pages, pages, page, P, 8, rotary, P, 0, None, 1e-6, q, 1024,
                          128, None, q_out, 8, tokens, kv_heads, dim, 0, None)


def attention(L, q=P, q_ts=1024, k_pages=P, pages=4, page=16, table=P, stride=4, columns=4, lengths=P, starts=P, batch=2, prefix=None,
              prefix_len=0, scale=1.0, out=P, tokens=4, q_heads=8, kv_heads=2, dim=128):
    return L.jv_paged_attention(q, q_ts, 128, k_pages, P, pages, page, table, stride, columns, lengths, starts, batch, prefix,
                                prefix_len, scale, out, tokens, q_heads, kv_heads, dim, 0, P, 0, None, 0, None)


@pytest.mark.parametrize("bad", [
    dict(dim=96), dict(tokens=-1), dict(q_heads=0), dict(kv_heads=0), dict(q_heads=1 << 17), dict(tokens=1 << 28), dict(rotary=24),
    dict(rotary=256), dict(rotary=0), dict(n_pos=-1), dict(pos=None), dict(rope=P + 4), dict(q=None), dict(q=P + 2),
    dict(q_ts=1027), dict(q_hs=-4), dict(k=None), dict(q_out=None), dict(k_out=P + 8),
])
def test_norm_rope_refuses(product_lib, bad):
    assert norm_rope(product_lib, **bad) == _lib.JV_ERR_VALUE
    assert product_lib.jv_fp8_last_error()


@pytest.mark.parametrize("bad", [
    dict(dim=32), dict(tokens=-3), dict(kv_heads=-1), dict(k=None), dict(k=P + 8), dict(k_ts=4), dict(v=None), dict(slots=None),
    dict(k_pages=None), dict(v_pages=P + 2), dict(pages=0), dict(pages=1 << 31), dict(page=8), dict(page=24), dict(page=2048),
    dict(rotary=130), dict(q=P), dict(q=P + 2, q_out=P),
])
def test_append_refuses(product_lib, bad):
    assert append(product_lib, **bad) == _lib.JV_ERR_VALUE


@pytest.mark.parametrize("bad", [
    dict(dim=512), dict(tokens=-1), dict(q_heads=7), dict(kv_heads=3), dict(batch=-1), dict(batch=0), dict(batch=(1 << 20) + 1),
    dict(page=48), dict(k_pages=None), dict(pages=-1), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")),
    dict(scale=float("inf")), dict(starts=None), dict(columns=-1), dict(stride=-1), dict(columns=1 << 27), dict(lengths=None),
    dict(columns=(1 << 26) - 1, prefix=P, prefix_len=17),  # more keys than a query may see
    dict(table=None), dict(q=None), dict(q=P + 4), dict(q_ts=4), dict(out=None), dict(prefix_len=-1), dict(prefix_len=5),
    dict(prefix_len=(1 << 30) + 1), dict(tokens=1 << 27),
])
def test_attention_refuses(product_lib, bad):
    assert attention(product_lib, **bad) == _lib.JV_ERR_VALUE


def test_workspace_of_refused_and_empty_calls(product_lib):
    need = product_lib.jv_paged_attention_workspace_bytes
    assert need(0, 3, 8, 2, 128, 0, 1) == 0
    assert need(4, 0, 8, 2, 128, 0, 1) == 0
    for tokens, batch, q_heads, kv_heads, dim, prefix in ((4, 2, 7, 2, 128, 0), (4, 2, 8, 2, 96, 0), (-1, 2, 8, 2, 128, 0),
                                                          (4, 2, 8, 2, 128, -1), (4, -2, 8, 2, 128, 0)):
        assert need(tokens, batch, q_heads, kv_heads, dim, prefix, 1) == -1


def test_no_tokens_is_a_call_that_succeeds(product_lib):
    assert norm_rope(product_lib, tokens=0, q=None, k=None) == _lib.JV_OK
    assert append(product_lib, tokens=0, k=None, v=None, slots=None) == _lib.JV_OK
    assert attention(product_lib, tokens=0, q=None, out=None, batch=0) == _lib.JV_OK


@pytest.mark.parametrize("n_pos", [0, -7])
def test_rotation_needs_a_position(product_lib, n_pos):
    """A position outside the table reads the first one's angles, which there have to be."""
    assert norm_rope(product_lib, n_pos=n_pos, tokens=0) == _lib.JV_ERR_VALUE
    assert b"one position" in product_lib.jv_fp8_last_error()
    L = product_lib
    assert L.jv_append_kv(P, 256, 128, P, 256, 128, P, 1, P, P, 4, 16, P, n_pos, 64, P, 0, None, 1e-6, None, 0, 0, None, None, 8, 0, 2,
                          128, 0, None) == _lib.JV_ERR_VALUE


def test_narrowing_refuses(product_lib):
    narrow = product_lib.jv_narrow_indices
    for rows, cols, src, dst in ((-1, 3, P, P), (3, -1, P, P), (1 << 16, 1 << 15, P, P), (2, 3, None, P), (2, 3, P, None)):
        assert narrow(src, rows, cols, cols, 1, dst, None) == _lib.JV_ERR_VALUE
    assert narrow(None, 0, 3, 3, 1, None, None) == _lib.JV_OK
    assert narrow(None, 3, 0, 0, 1, None, None) == _lib.JV_OK


@pytest.mark.parametrize("tokens,columns", [(1 << 20, 1 << 16), (300000, 18750), (32768, 1 << 18)])
def test_long_prompts_are_not_refused_for_their_table(product_lib, tokens, columns):
    """Prompts whose row tiles stay whole add no keys up: such a call gets as far as the missing lengths."""
    assert attention(product_lib, tokens=tokens, batch=1, columns=columns, q_heads=32, kv_heads=4, lengths=None) == _lib.JV_ERR_VALUE
    assert b"lengths" in product_lib.jv_fp8_last_error()


def test_counters_of_refused_and_empty_calls(product_lib):
    need = product_lib.jv_paged_attention_counters_needed
    assert need(0, 3, 8, 2, 128, 0, 1) == 0 and need(4, 0, 8, 2, 128, 0, 1) == 0
    assert need(4, 2, 7, 2, 128, 0, 1) == -1 and need(4, 2, 8, 2, 96, 0, 1) == -1 and need(4, 2, 8, 2, 128, -1, 1) == -1
