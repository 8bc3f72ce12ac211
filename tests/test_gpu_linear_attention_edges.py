"""What the kernels between the projections of a linear attention layer keep of
their inputs' bits, and what they do with calls at the edge of what their
callers may ask."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

from jeeves_amd import causal_conv, linear_attention
from tests.test_gpu_linear_attention import DEV, SCANS, Case, gen, ints, randn, rounding, starts_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dims,empty", SCANS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("what,beta", [("state", True), ("state", False), ("products", True), ("products", False), ("updates", True)])
def test_outputs_keep_32_bits(what, beta, dims, empty, dtype):
    """Outputs that are the difference of two terms below 2 which agree to 12 bits or more: the terms come from the state, from
    the products q.k or from the updates beta v, each of 24 bits. Three parts keep a term to 2^-24 of it and sums of two such
    terms take 6 roundings of fp32 at most, so the difference is off by 8 x 2^-24 x 2 = 2^-20 and its own rounding; terms of
    16 bits would put it off by up to 2^-16."""
    (dk, dv), hk, hv = dims, 2, 4
    g = torch.Generator(DEV).manual_seed(dk + empty)
    lengths = [40, 150, 70] + [0] * empty
    starts, n = starts_of(lengths), len(lengths)
    tokens = starts[-1]
    q, k = torch.zeros(tokens, hk, dk, device=DEV), torch.zeros(tokens, hk, dk, device=DEV)
    v, betas = torch.zeros(tokens, hv, dv, device=DEV), torch.ones(tokens, hv, device=DEV)
    states = torch.zeros(n, hv, dk, dv, device=DEV)
    near = torch.zeros(tokens, hv, dv, dtype=torch.float64, device=DEV)
    for b, length in enumerate(lengths):
        at, end = starts[b], starts[b + 1]
        if not length:
            continue
        if what == "state":
            q[at:end, :, :2] = 1
            states[b, :, 0] = 1 + torch.rand(hv, dv, generator=g, device=DEV)
            states[b, :, 1] = -states[b, :, 0] + torch.rand(hv, dv, generator=g, device=DEV) * 2.0 ** -13
            near[at:end] = states[b, :, 0].double() + states[b, :, 1].double()
            continue
        v[at], v[at + 1] = 1, -1
        if what == "products":
            # 1 + 2^-9 (1 + m / 128) + n 2^-23 of the first two tokens' keys, which have no channel in common
            q[at:end, :, :6] = 1
            for h in range(hk):
                m, low = 17 + 31 * b + h, (100 - h, 60 + b)
                for t in range(2):
                    k[at + t, h, 3 * t:3 * t + 3] = torch.tensor([1, 2.0 ** -9 * (1 + m / 128), low[t] * 2.0 ** -23], device=DEV)
                first = 1 + 2.0 ** -9 * (1 + m / 128) + low[0] * 2.0 ** -23
                near[at, 2 * h:2 * h + 2], near[at + 1:end, 2 * h:2 * h + 2] = first, (low[0] - low[1]) * 2.0 ** -23
        else:
            q[at:end, :, :2] = 1
            k[at, :, 0] = k[at + 1, :, 1] = 1
            betas[at] = 0.5 + 0.5 * torch.rand(hv, generator=g, device=DEV)
            betas[at + 1] = betas[at] - torch.rand(hv, generator=g, device=DEV) * 2.0 ** -13
            near[at], near[at + 1:end] = betas[at, :, None].double(), (betas[at] - betas[at + 1])[:, None].double()
    out = linear_attention(q.to(dtype), k.to(dtype), v.to(dtype), torch.zeros(tokens, hv, device=DEV), states, ints(list(range(n))),
                           beta=betas if beta else None, query_starts=ints(starts), scale=1.0)
    assert ((out.double() - near).abs() <= rounding(near, dtype) + 2.0 ** -20).all(), (out.double() - near).abs().max().item()


def test_as_many_sequences_as_a_call_may_have():
    """2^20 sequences, two of them with tokens, and tokens behind the last: places past the last token clear nothing."""
    c = Case(60, [70, 110], heads=(1, 1), dims=(64, 256), raw=True, behind=20)
    n, tokens = 1 << 20, c.v.shape[0]
    if torch.cuda.mem_get_info()[0] < 80 << 30:
        pytest.skip("the workspace takes 50 GB")
    starts = torch.zeros(n + 1, dtype=torch.int32, device=DEV)
    starts[6:], starts[n - 1:] = 70, 180
    slots, source = torch.full((n,), -1, dtype=torch.int32, device=DEV), torch.full((n,), -1, dtype=torch.int32, device=DEV)
    for b, seq in enumerate((5, n - 2)):
        slots[seq], source[seq] = c.to[b], c.source[b]
    states = c.states.clone()
    out = linear_attention(c.q, c.k, c.v, c.decay, states, slots, beta=c.beta, rate=c.rate, decay_bias=c.bias, from_slots=source,
                           query_starts=starts, norm_eps=c.norm_eps)
    exact, mag, far, want, spread = c.exact()
    assert out.shape[0] == tokens and (out[180:] == 0).all()
    assert ((out.double() - exact).abs() <= rounding(exact, out.dtype) + 2.0 ** -14 * mag + 2.0 ** -17 * far).all()
    assert ((states.double() - want).norm(dim=2) <= 2.0 ** -17 * spread).all()
    torch.cuda.empty_cache()


@pytest.mark.parametrize("single", [True, False])
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("what,beta", [("v", True), ("v", False), ("k", True), ("decay", True), ("beta", True)])
@pytest.mark.parametrize("dims,empty", SCANS)
def test_an_update_that_is_not_finite_leaves_nan(what, beta, value, dims, empty, single):
    """The same for single tokens and for prompts: the value channels of such an update are NaN from its token on, and in the
    state; what does not see it keeps its bits."""
    if what == "decay" and value < 0:
        return  # a state dropped whole
    c = Case(61, [1, 1, 1] if single else [40, 150, 70] + [0] * empty, dims=dims, beta=beta, single=single)
    at, end = (1, 2) if single else (40 + 64 + 21, 190)
    clean, clean_states = c.run()
    heads, channels = slice(0, 2) if what == "k" else slice(1, 2), 17 if what == "v" else slice(None)
    t = getattr(c, what).clone()
    if what in ("v", "k"):
        t[at, 0 if what == "k" else 1, channels if what == "v" else 9] = value
    else:
        t[at, 1] = value
    setattr(c, what, t)
    out, states = c.run()
    hit, left = torch.zeros(out.shape, dtype=torch.bool, device=DEV), torch.zeros(states.shape, dtype=torch.bool, device=DEV)
    hit[at:end, heads, channels], left[c.to[1], heads, :, channels] = True, True
    assert out[hit].isnan().all() and states[left].isnan().all()
    assert torch.equal(out[~hit], clean[~hit]) and torch.equal(states[~left], clean_states[~left])


def test_reciprocal_rounds_as_the_division_does(hooks_lib):
    """Every float from 1 to infinity."""
    hooks_lib.th_inverse_sweep.argtypes = [ctypes.c_uint32, ctypes.c_uint32, ctypes.c_void_p, ctypes.c_void_p]
    count = torch.zeros(1, dtype=torch.int64, device=DEV)
    assert hooks_lib.th_inverse_sweep(0x3F800000, 0x7F800001 - 0x3F800000, count.data_ptr(), torch.cuda.current_stream().cuda_stream) == 0
    assert count.item() == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("width,bias", [(2, True), (3, False), (4, True), (4, False)])
@pytest.mark.parametrize("single", [True, False])
def test_conv_has_the_bits_of_the_elementary_operations(single, width, bias, dtype):
    """Products, sums in the inputs' order, exponential, sum, quotient and product, each rounded to 32 bits."""
    g = gen(62 + width)
    tokens, channels = (300, 1024)
    x, weight = randn(g, tokens, channels, dtype=dtype) * 3, randn(g, channels, width, dtype=torch.float32)
    b = randn(g, channels, dtype=torch.float32) if bias else None
    n = tokens if single else 1
    states = randn(g, n, width - 1, channels, dtype=dtype)
    before = states.clone()
    out = causal_conv(x, weight, states, ints(list(range(n))), bias=b, query_starts=None if single else ints([0, tokens]))
    if single:
        rows = torch.cat([before, x[:, None]], 1).float()
        taps = [rows[:, j] for j in range(width)]
    else:
        rows = torch.cat([before[0], x]).float()
        taps = [rows[j:j + tokens] for j in range(width)]
    y = torch.zeros(tokens, channels, device=DEV) if b is None else b.expand(tokens, channels)
    for j in range(width):
        y = y + taps[j] * weight[:, j]
    assert torch.equal(out, (y * (1 / (1 + torch.exp(-y)))).to(dtype))


@pytest.mark.parametrize("single", [True, False])
def test_decays_of_raw_gates_keep_32_bits(single):
    """States of 1 that nothing is added to, so that they become the decays, for gates down to -85 with rates that bring g to
    -1. softplus takes at most 8 roundings of 2^-24 (the exponential two), the rate one, so e^g is off by 9 x 2^-24 |g|; its
    own exponential and the product add 4: below 2^-20 of the state."""
    n, hv, d = 86, 2, 64
    z = -torch.arange(n, dtype=torch.float32, device=DEV)[:, None].expand(n, hv) - torch.tensor([0.0, 0.37], device=DEV)
    zeros = torch.zeros(n, hv, d, dtype=torch.bfloat16, device=DEV)
    for at in range(n):
        rate = (1 / torch.logaddexp(z[at].double(), torch.zeros(hv, dtype=torch.float64, device=DEV))).float()
        states = torch.ones(1, hv, d, d, device=DEV)
        linear_attention(zeros[:1], zeros[:1], zeros[:1], z[at:at + 1], states, ints([0]), rate=rate,
                         query_starts=None if single else ints([0, 1]))
        want = (-rate.double() * torch.logaddexp(z[at].double(), torch.zeros(hv, dtype=torch.float64, device=DEV))).exp()
        assert ((states.double() / want[None, :, None, None] - 1).abs() <= 2.0 ** -20).all(), at
