"""The C entry points of the norms around a block, the short convolution and
the linear attention refuse bad arguments before they touch the device, and
their Python callers before they load the library's kernels."""

from __future__ import annotations

import shutil
import subprocess
from pathlib import Path

import pytest
import torch

from jeeves_amd import _lib, build

P = 4096  # an aligned address that no refused call follows


def norm(L, x=P, x_ts=1024, x_hs=128, residual=P, r_ts=1024, gate=P, g_ts=1024, g_hs=128, act=1, post=P, weight=P, eps=1e-6, h=P, y=P,
         codes=P, ldc=1024, scales=P, tokens=4, heads=8, dim=128):
    return L.jv_block_norm(x, x_ts, x_hs, residual, r_ts, gate, g_ts, g_hs, act, post, 1.0, weight, eps, h, y, codes, ldc, scales, tokens,
                           heads, dim, 0, None)


def conv(L, x=P, x_ts=512, weight=P, bias=P, width=4, act=1, states=P, n_slots=4, slots=P, starts=P, batch=2, out=P, tokens=4, channels=512):
    return L.jv_causal_conv(x, x_ts, weight, bias, width, act, states, n_slots, slots, None, starts, batch, out, tokens, channels, 0, None)


def linear(L, q=P, q_ts=1024, q_hs=128, k=P, v=P, decay=P, beta=P, rate=P, bias=P, norm_eps=1e-6, states=P, n_slots=4, slots=P, starts=P,
           batch=2, scale=1.0, out=P, tokens=4, k_heads=2, v_heads=4, k_dim=128, v_dim=128, ws=4096, ws_bytes=1 << 30):
    return L.jv_linear_attention(q, q_ts, q_hs, k, 256, 128, v, 512, 128, decay, 4, beta, 4, 0, rate, bias, norm_eps, states, n_slots, slots,
                                 None, starts, batch, scale, out, tokens, k_heads, v_heads, k_dim, v_dim, 0, ws, ws_bytes, None)


@pytest.mark.parametrize("bad", [
    dict(heads=0), dict(dim=0), dict(dim=132), dict(dim=96), dict(heads=1, dim=20), dict(heads=256), dict(heads=1, dim=16392),
    dict(tokens=-1), dict(tokens=1 << 22), dict(eps=-1e-6), dict(eps=float("nan")), dict(eps=float("inf")), dict(act=3), dict(act=-1),
    dict(codes=None), dict(scales=None), dict(ldc=1016), dict(ldc=1028), dict(heads=1, dim=264, ldc=0), dict(x=None), dict(x=P + 2),
    dict(x_ts=1020), dict(x_hs=4), dict(r_ts=4), dict(residual=P + 8), dict(gate=P + 8), dict(g_hs=-4), dict(post=P + 4),
    dict(weight=P + 8), dict(h=P + 8), dict(y=P + 8), dict(codes=P + 8),
])
def test_block_norm_refuses(product_lib, bad):
    assert norm(product_lib, **bad) == _lib.JV_ERR_VALUE
    assert product_lib.jv_fp8_last_error()


@pytest.mark.parametrize("bad", [
    dict(width=1), dict(width=5), dict(channels=0), dict(channels=516), dict(channels=65544), dict(act=2), dict(tokens=-1),
    dict(tokens=1 << 24), dict(batch=-1), dict(batch=0), dict(batch=(1 << 20) + 1), dict(starts=None), dict(slots=None), dict(n_slots=-1),
    dict(n_slots=1 << 31), dict(states=None), dict(states=P + 8), dict(x=None), dict(x=P + 8), dict(x_ts=508), dict(out=None),
    dict(out=P + 8), dict(weight=None), dict(weight=P + 4), dict(bias=P + 4), dict(tokens=(1 << 24) - 1, channels=65536),
])
def test_causal_conv_refuses(product_lib, bad):
    assert conv(product_lib, **bad) == _lib.JV_ERR_VALUE
    assert product_lib.jv_fp8_last_error()


@pytest.mark.parametrize("bad", [
    dict(k_dim=96), dict(v_dim=32), dict(k_heads=0), dict(v_heads=0), dict(v_heads=3), dict(v_heads=1 << 17), dict(tokens=-1),
    dict(tokens=1 << 24), dict(tokens=1 << 23, v_heads=64), dict(batch=-1), dict(batch=0), dict(batch=(1 << 20) + 1), dict(starts=None),
    dict(slots=None), dict(n_slots=-1), dict(states=None), dict(states=P + 8), dict(scale=float("nan")), dict(scale=float("inf")),
    dict(norm_eps=-1.0), dict(norm_eps=1e-40), dict(norm_eps=float("nan")), dict(rate=None), dict(q=None), dict(q=P + 2), dict(q_ts=4), dict(q_hs=2), dict(k=None),
    dict(v=None), dict(decay=None), dict(out=None), dict(out=P + 8), dict(ws=None), dict(ws=P + 16), dict(ws_bytes=64),
])
def test_linear_attention_refuses(product_lib, bad):
    assert linear(product_lib, **bad) == _lib.JV_ERR_VALUE
    assert product_lib.jv_fp8_last_error()


def test_empty_calls_need_no_device(product_lib):
    assert norm(product_lib, tokens=0, x=None) == _lib.JV_OK
    assert conv(product_lib, tokens=0, x=None) == _lib.JV_OK
    assert linear(product_lib, tokens=0, q=None) == _lib.JV_OK


def test_linear_attention_workspace_is_host_logic(product_lib):
    size = product_lib.jv_linear_attention_workspace_bytes
    assert size(64, 64, 16, 32, 128, 128, 0) == 0 and size(0, 3, 16, 32, 128, 128, 1) == 0
    one, two = size(1, 1, 16, 32, 128, 128, 1), size(64, 1, 16, 32, 128, 128, 1)
    assert 0 < one < two and size(640, 1, 16, 32, 128, 128, 1) - two == 9 * (two - one)
    assert size(1 << 23, 1, 16, 64, 128, 128, 1) == -1 and size(4, 1, 3, 4, 128, 128, 1) == -1
    assert size(4, 1, 4, 4, 100, 128, 1) == -1


def test_python_refuses_host_tensors_and_bad_names():
    from jeeves_amd import add_norm, causal_conv, gated_norm, linear_attention

    x = torch.zeros(4, 256, dtype=torch.bfloat16)
    heads = x.view(4, 2, 128)
    none = torch.zeros(4, dtype=torch.int32)
    with pytest.raises(ValueError, match="HIP device"):
        add_norm(x, None, torch.ones(256))
    with pytest.raises(ValueError, match="HIP device"):
        gated_norm(heads, heads, None)
    with pytest.raises(ValueError, match="HIP device"):
        causal_conv(x, torch.zeros(256, 4), torch.zeros(1, 3, 256, dtype=torch.bfloat16), none)
    with pytest.raises(ValueError, match="HIP device"):
        linear_attention(heads, heads, heads, torch.zeros(4, 2), torch.zeros(1, 2, 128, 128), none)


def test_forward_codes_needs_per_token_codes():
    from jeeves_amd import FP8Linear

    linear = FP8Linear(256, 64)
    codes, scales = torch.zeros(3, 256, dtype=torch.uint8), torch.ones(3)
    assert linear.takes_codes() and not FP8Linear(16512, 64).takes_codes()
    linear.set_activations("bf16")
    assert not linear.takes_codes()
    with pytest.raises(ValueError, match="codes"):
        linear.forward_codes(codes, scales)
    linear.set_activations("fp8")
    linear.set_lora(torch.zeros(16, 256), torch.zeros(64, 16), 2.0)
    assert not linear.takes_codes()
    with pytest.raises(ValueError, match="codes"):
        linear.forward_codes(codes, scales)


def test_linear_attention_block_checks_its_parts():
    from jeeves_amd import FP8Linear, FP8LinearAttention

    def block(outputs=512, inputs=128, gates=(4, 256), conv=(384, 4), k_heads=1, dims=(64, 64)):
        return FP8LinearAttention(FP8Linear(256, outputs), torch.zeros(gates), FP8Linear(inputs, 256), k_heads, 2, *dims, torch.zeros(conv),
                                  torch.ones(2), torch.zeros(2), torch.ones(64))

    with pytest.raises(ValueError, match="outputs"):
        block()
    block(outputs=384, conv=(256, 4))
    for bad in (dict(outputs=400), dict(outputs=384, conv=(384, 4)), dict(outputs=384, conv=(256, 4), gates=(2, 256)),
                dict(outputs=384, conv=(256, 4), inputs=256), dict(k_heads=3), dict(dims=(96, 64))):
        with pytest.raises(ValueError):
            block(**bad)


def test_linear_attention_block_refuses_what_a_call_would():
    """More output channels than a norm's row has, more than the convolution's, widths, weights' shapes and eps: when it is
    built, not at its first call."""
    from jeeves_amd import FP8Linear, FP8LinearAttention

    def block(k_heads=1, v_heads=2, k_dim=64, v_dim=64, width=4, rate=None, bias=None, norm=None, eps=1e-6):
        channels, outputs = 2 * k_heads * k_dim + v_heads * v_dim, v_heads * v_dim
        return FP8LinearAttention(FP8Linear(128, channels + outputs, device="meta"), torch.zeros(2 * v_heads, 128),
                                  FP8Linear(outputs, 128, device="meta"), k_heads, v_heads, k_dim, v_dim, torch.zeros(channels, width),
                                  torch.ones(v_heads if rate is None else rate), torch.zeros(v_heads if bias is None else bias),
                                  torch.ones(v_dim if norm is None else norm), eps)

    assert block(v_heads=64, v_dim=256).v_heads == 64
    for bad in (dict(v_heads=65, v_dim=256), dict(k_heads=128, v_heads=128, k_dim=256), dict(width=1), dict(width=5), dict(rate=1),
                dict(bias=3), dict(norm=128), dict(eps=0.0), dict(eps=-1.0), dict(eps=1e-40), dict(eps=float("nan")),
                dict(eps=float("inf")), dict(k_heads=0), dict(v_heads=0)):
        with pytest.raises(ValueError):
            block(**bad)


AMDCLANG = shutil.which("amdclang++") or "/opt/rocm/bin/amdclang++"


@pytest.fixture(scope="module")
def layer_rows(tmp_path_factory):
    if not Path(AMDCLANG).exists():
        pytest.skip("amdclang++ not found")
    exe = tmp_path_factory.mktemp("rows") / "layer_rows"
    subprocess.run([AMDCLANG, "-x", "hip", "--offload-host-only", "-O1", "-std=c++17", f"-I{build.CSRC}", f"-I{build.ROOT / 'include'}",
                    str(build.ROOT / "tests" / "csrc" / "layer_rows.cpp"), "-o", str(exe)], check=True, capture_output=True, timeout=600)
    return exe


@pytest.mark.parametrize("tokens,batch", [(1, 1), (64, 1), (65, 3), (64, 1 << 20), (200, 1 << 20), ((1 << 23) - 1, 7), ((1 << 20) - 5, (1 << 20) - 3)])
def test_places_share_the_tokens(product_lib, layer_rows, tokens, batch):
    """Each token is one place's to clear, and none is a place's that lies past the last one: sizes up to the largest that a
    call may have (one head of 256 channels), where an index over all places' rows would not fit 32 bits."""
    size = product_lib.jv_linear_attention_workspace_bytes(tokens, batch, 1, 1, 64, 256, 1)
    assert size > 0
    got = subprocess.run([str(layer_rows), str(tokens), str(batch)], capture_output=True, text=True, check=True, timeout=60).stdout.split()
    assert got == [str(tokens), str(min(tokens, 64)), "-1"]
