"""add_norm and gated_norm against their definitions in 64 bits.

Bounds, from the roundings that the kernel makes. u is half a step relative to
the value (2^-8 for bf16, 2^-11 for fp16, plus 2^-25, half of fp16's smallest
step). Everything else is fp32: a row's mean square is off by 2^-17 of itself
at most (16384 terms in chains of 32 and trees of at most 9 sums, so 45
roundings of 2^-24, and the products'), its root by half of that, and an
elementwise chain of less than 20 roundings by 2^-19. With b the block's output
after its norm and gate and m = |residual| + |scale b|:
  h  within u |h| + 2^-17 m
  y  within u |y| + 2^-16 |y| + 2^-17 m |weight| / root      (what m's error does to h, scaled as h is)
Codes stand for y / scale, each within half a step of it, which is 2^-4 of the
value or 2^-10 (e4m3's subnormals are 2^-9 apart), where y carries its own
error; scales within 2^-15 of theirs where that error is small."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"


def gen(seed):
    return torch.Generator(DEV).manual_seed(seed)


def randn(g, *shape, dtype=torch.bfloat16):
    return torch.randn(*shape, generator=g, device=DEV).to(dtype)


def rounding(t, dtype):
    return torch.finfo(dtype).eps / 2 * t.abs() + (2.0 ** -25 if dtype == torch.float16 else 0.0)


def act(z, name):
    return z if name is None else torch.sigmoid(z) * (z if name == "silu" else 1.0)


def rms(x, weight, eps):
    """(the norm, 1 / root)"""
    r = 1 / (x.square().mean(-1, keepdim=True) + eps).sqrt()
    return x * r * weight, r


def add_norm_exact(x, residual, weight, post_weight=None, gate=None, activation="sigmoid", scale=1.0, eps=1e-6):
    """(h, y, m, y's error before its rounding)"""
    b = x.double()
    if post_weight is not None:
        b = rms(b, post_weight.double(), eps)[0]
    if gate is not None:
        b = b * act(gate.double(), activation)
    res = torch.zeros_like(b) if residual is None else residual.double()
    h, m = res + scale * b, res.abs() + (scale * b).abs()
    if weight is None:
        return h, None, m, None
    y, r = rms(h, weight.double(), eps)
    return h, y, m, 2.0 ** -16 * y.abs() + 2.0 ** -17 * m * weight.double().abs() * r


def check_codes(codes, scales, y, error):
    top = y.abs().amax(-1)
    want = top.clamp(min=1e-12) / 448
    assert ((scales.double() - want).abs() <= 2.0 ** -15 * want + error.amax(-1) / 448).all()
    step = torch.maximum(2.0 ** -4 * y.abs(), 2.0 ** -10 * want[:, None])
    got = codes.double() * scales.double()[:, None]
    assert ((got - y).abs() <= 1.001 * step + 1.1 * error + 2.0 ** -15 * y.abs()).all()


def unpacked(packed, rows, cols):
    """Row-major codes of the packed order, its padding rows among them."""
    from jeeves_amd import FP8, untile_weight

    return untile_weight(packed.view((rows + 15) // 16 * 16, cols)).view(FP8)


@pytest.mark.parametrize("cols", [8, 64, 264, 1024, 4096, 4104, 5120, 8192, 12288, 16384])
@pytest.mark.parametrize("tokens", [1, 3, 130])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_add_norm(cols, tokens, dtype):
    from jeeves_amd import add_norm

    g = gen(cols + tokens)
    spread = randn(g, cols, dtype=torch.float32).exp()
    x, residual = (randn(g, tokens, cols, dtype=torch.float32) * spread).to(dtype), randn(g, tokens, cols, dtype=dtype) * 3
    gate = randn(g, tokens, cols, dtype=dtype) * 2
    w, pw = 1 + 0.3 * randn(g, cols, dtype=torch.float32), randn(g, cols, dtype=torch.float32)
    before = [t.clone() for t in (x, residual, gate)]
    for kw in (dict(), dict(post_weight=pw), dict(gate=gate), dict(post_weight=pw, gate=gate, activation="silu", scale=0.25),
               dict(gate=gate, activation=None, scale=-2.0)):
        for res, weight in ((residual, w), (None, w), (residual, None)):
            out = add_norm(x, res, weight, **kw)
            h, y, m, error = add_norm_exact(x, res, weight, **kw)
            assert ((out.h.double() - h).abs() <= rounding(h, dtype) + 2.0 ** -17 * m).all()
            assert out.codes is None and out.scales is None and (out.y is None) == (weight is None)
            if weight is None:
                continue
            assert ((out.y.double() - y).abs() <= rounding(y, dtype) + error).all()
            again = add_norm(x, res, weight, quantize="rows", **kw)
            assert torch.equal(again.h, out.h) and torch.equal(again.y, out.y)
            check_codes(again.codes, again.scales, y, error)
    assert all(torch.equal(a, b) for a, b in zip(before, (x, residual, gate)))


@pytest.mark.parametrize("heads,dim", [(1, 64), (1, 128), (3, 64), (2, 256), (32, 128), (40, 256), (128, 128), (16, 64)])
@pytest.mark.parametrize("tokens", [1, 5, 257])
@pytest.mark.parametrize("activation", ["silu", "sigmoid"])
def test_gated_norm(heads, dim, tokens, activation):
    from jeeves_amd import gated_norm

    for dtype in (torch.bfloat16, torch.float16):
        g = gen(heads * dim + tokens)
        merged = randn(g, tokens, 2 * heads * dim + 64, dtype=dtype)
        gate = merged[:, 64:64 + heads * dim].view(tokens, heads, dim)
        x = randn(g, heads, tokens, dim, dtype=dtype).transpose(0, 1) * 0.1
        for weight in (1 + 0.3 * randn(g, dim, dtype=torch.float32), None):
            b = x.double() if weight is None else rms(x.double(), weight.double(), 1e-6)[0]
            y = b * act(gate.double(), activation)
            out = gated_norm(x, gate, weight, activation=activation)
            assert out.shape == x.shape and out.is_contiguous()
            assert ((out.double() - y).abs() <= rounding(y, dtype) + 2.0 ** -16 * y.abs()).all()
            codes, scales = gated_norm(x, gate, weight, activation=activation, quantize="rows")
            check_codes(codes, scales, y.flatten(1), 2.0 ** -16 * y.flatten(1).abs())
            if heads * dim % 128 == 0:
                packed, pscales = gated_norm(x, gate, weight, activation=activation, quantize="packed")
                rows = unpacked(packed, tokens, heads * dim)
                assert torch.equal(pscales, scales) and torch.equal(rows[:tokens].view(torch.uint8), codes.view(torch.uint8))
                assert (rows[tokens:].view(torch.uint8) == 0).all()


@pytest.mark.parametrize("tokens", [1, 4, 16, 33, 300])
@pytest.mark.parametrize("cols", [128, 4096, 9088])
def test_codes_are_the_quantizers(tokens, cols):
    """A row that passes through unchanged has the bits of quantize_rows."""
    from jeeves_amd import gated_norm, quantize_rows

    x = randn(gen(cols), tokens, 1, cols)
    x[0, 0, 0] = 3e38
    if tokens > 3:
        x[1] = 0
        x[2, 0, 5] = float("inf")
        x[3, 0, 7] = float("nan")
    heads = x.view(tokens, cols // 64, 64) if cols % 64 == 0 else x
    codes, scales = gated_norm(heads, torch.ones_like(heads), None, activation=None, quantize="rows")
    want, want_scales = quantize_rows(x.view(tokens, cols).float())
    assert torch.equal(scales.view(torch.int32)[scales.isfinite()], want_scales.view(torch.int32)[scales.isfinite()])
    assert torch.equal(scales.isnan(), want_scales.isnan())
    a, b = codes.float(), want.float()
    assert torch.equal(a.isnan(), b.isnan()) and torch.equal(a[~a.isnan()], b[~b.isnan()])


@pytest.mark.parametrize("tokens", [1, 2, 5, 64, 200])
def test_codes_feed_the_next_projection(tokens):
    """The packed codes, the row-major ones and the linear on y differ by y's rounding alone."""
    from jeeves_amd import FP8Linear, add_norm

    g = gen(tokens)
    linear = FP8Linear(1024, 2048, bias=True, device=DEV)
    linear.load_weight(randn(g, 2048, 1024) * 0.02)
    linear.bias.data.copy_(randn(g, 2048))
    x, residual, w = randn(g, tokens, 1024), randn(g, tokens, 1024), 1 + 0.2 * randn(g, 1024, dtype=torch.float32)
    packed = add_norm(x, residual, w, quantize="packed", keep_y=False)
    rows = add_norm(x, residual, w, quantize="rows")
    assert packed.y is None and torch.equal(packed.h, rows.h) and torch.equal(packed.scales, rows.scales)
    out = linear.forward_codes(packed.codes, packed.scales, packed_rows=tokens)
    assert torch.equal(out, linear.forward_codes(rows.codes, rows.scales))
    far = (out.double() - linear(rows.y).double()).norm() / out.double().norm()
    assert far < 0.05  # codes on the other side of a border, a step of 2^-3 at most, one in 2^4 for a rounding of 2^-8


def test_rows_of_extremes():
    """A row is only its own: NaN and infinities stay in it; zeros come out as zeros, and as NaN without eps; squares past
    fp32 are infinite."""
    from jeeves_amd import add_norm

    x = randn(gen(3), 6, 512)
    clean = add_norm(x, None, torch.ones(512, device=DEV), quantize="rows")
    x[1], x[2, 3], x[3, 4] = 0, float("nan"), float("inf")
    out = add_norm(x, None, torch.ones(512, device=DEV), quantize="rows")
    for i in (0, 4, 5):
        assert torch.equal(out.y[i], clean.y[i]) and torch.equal(out.codes[i].view(torch.uint8), clean.codes[i].view(torch.uint8))
    assert (out.y[1] == 0).all() and (out.codes[1].float() == 0).all()
    assert out.y[2].isnan().all() and out.codes[2].float().isnan().all() and out.scales[2].isnan()
    assert out.y[3, 4].isnan() and (out.y[3, :4] == 0).all()
    assert add_norm(x[1:2], None, torch.ones(512, device=DEV), eps=0.0).y.isnan().all()
    assert (out.h[0] == x[0]).all()


@pytest.mark.parametrize("exponent", [-66, -30, 30])
def test_tiny_and_large_rows_without_eps(exponent):
    """Rows of 2^-66 have squares of 2^-132, on a grid of 2^-149: the mean is off by 2^-17 or less."""
    from jeeves_amd import add_norm

    x = randn(gen(5), 9, 256) * 2.0 ** exponent
    y = rms(x.double(), 1.0, 0.0)[0]
    out = add_norm(x, None, torch.ones(256, device=DEV), eps=0.0).y
    assert ((out.double() - y).abs() <= rounding(y, x.dtype) + 2.0 ** -14 * y.abs()).all()


def test_gates_of_extremes():
    from jeeves_amd import add_norm

    x = torch.ones(1, 16, dtype=torch.bfloat16, device=DEV)
    z = torch.tensor([-3e38, -200.0, -88.0, -20.0, -0.0, 0.0, 20.0, 88.0, 200.0, 3e38, float("inf"), -float("inf"), float("nan"), 1.0, -1.0, 5.0],
                     device=DEV).bfloat16()[None]
    for name in ("sigmoid", "silu"):
        got = add_norm(x, None, None, gate=z, activation=name).h.double()
        want = act(z.double(), name)
        want[(z == -float("inf")) | z.isnan()] = 0.0 if name == "sigmoid" else float("nan")
        want[z.isnan()] = float("nan")
        assert torch.equal(got.isnan(), want.isnan())
        fine = want.isfinite()
        assert torch.equal(got[~fine & ~want.isnan()], want[~fine & ~want.isnan()])
        # e^-z of a large -z is off by |z| 2^-24, and below 2^-126 it may be 0
        assert ((got - want)[fine].abs() <= 1.01 * rounding(want, x.dtype)[fine] + 2.0 ** -15 * want[fine].abs() + 2.0 ** -118).all()


def test_strides_broadcast_rows_and_no_tokens():
    from jeeves_amd import add_norm, gated_norm

    g = gen(9)
    big = randn(g, 7, 1000)
    x, w = big[:, 3:515], torch.ones(512, device=DEV)     # rows that are not 16-byte aligned
    gate = randn(g, 1, 512).expand(7, 512)                # one gate for all tokens
    out = add_norm(x, x, w.bfloat16(), gate=gate)
    want = add_norm(x.contiguous(), x.contiguous(), w, gate=gate.contiguous())
    assert torch.equal(out.y, want.y) and torch.equal(out.h, want.h)
    columns = randn(g, 512, 7).t()
    assert torch.equal(add_norm(columns, None, w).y, add_norm(columns.contiguous(), None, w).y)
    none = add_norm(x[:0], x[:0], w, quantize="packed")
    assert none.h.shape == none.y.shape == (0, 512) and none.codes.numel() == 0 and none.scales.shape == (0,)
    assert gated_norm(big[:0, :256].view(0, 2, 128), big[:0, :256].view(0, 2, 128), None).shape == (0, 2, 128)


def test_refusals():
    from jeeves_amd import add_norm, gated_norm

    x, w = torch.zeros(4, 256, dtype=torch.bfloat16, device=DEV), torch.ones(256, device=DEV)
    h = x.view(4, 2, 128)
    for bad in (lambda: add_norm(x.float(), None, w), lambda: add_norm(h, None, w), lambda: add_norm(x[:, :252], None, w[:252]),
                lambda: add_norm(x, x[:3], w), lambda: add_norm(x, x.half(), w), lambda: add_norm(x, None, w[:128]),
                lambda: add_norm(x, None, w.cpu()), lambda: add_norm(x, None, w, post_weight=w[:8]), lambda: add_norm(x, None, w, gate=x[:, :8]),
                lambda: add_norm(x, None, w, gate=x, activation="relu"), lambda: add_norm(x, None, w, quantize="e4m3"),
                lambda: add_norm(x, None, None, quantize="rows"), lambda: add_norm(x, None, w, eps=-1.0),
                lambda: add_norm(x[:, :192], None, w[:192], quantize="packed"), lambda: gated_norm(x, x, None), lambda: gated_norm(h, h[:3], None),
                lambda: gated_norm(h, x, None), lambda: gated_norm(h, h.half(), None), lambda: gated_norm(h, h, w),
                lambda: gated_norm(x.view(4, 8, 32), x.view(4, 8, 32), None),
                lambda: add_norm(torch.zeros(1, 16392, dtype=torch.bfloat16, device=DEV), None, torch.ones(16392, device=DEV))):
        with pytest.raises(ValueError):
            bad()


def test_captured_and_on_another_stream():
    from jeeves_amd import add_norm, gated_norm

    g = gen(11)
    x, residual, w = randn(g, 33, 1024), randn(g, 33, 1024), torch.ones(1024, device=DEV)
    heads = randn(g, 33, 8, 128)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        out = add_norm(x, residual, w, quantize="packed")
        codes, scales = gated_norm(out.h.view(33, 8, 128), heads, None, quantize="rows")
    for i in range(4):
        x.copy_(randn(g, 33, 1024))
        torch.cuda.synchronize()
        graph.replay()
        got = [t.clone() for t in (*out, codes.view(torch.uint8), scales)]
        want = add_norm(x, residual, w, quantize="packed")
        wc, ws = gated_norm(want.h.view(33, 8, 128), heads, None, quantize="rows")
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, (*want, wc.view(torch.uint8), ws)))
