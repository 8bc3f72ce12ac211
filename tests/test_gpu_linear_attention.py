"""causal_conv and linear_attention against their definitions, token by token in
64 bits, at the lengths, slots and values where such kernels go wrong.

Bounds, from the roundings that the kernels make; u is half a step relative to
the value (2^-8 for bf16, 2^-11 for fp16, plus 2^-25, half of fp16's smallest
step).
* convolution: at most 10 roundings of fp32 over a, the sum of the products'
  magnitudes; silu's slope is below 1.1: u |y| + 2^-20 a.
* linear attention: what goes into a product towards an output is kept to 2^-16
  (two bf16 values), so products of two such are off by 2^-16 + 2^-16 and the
  one that is left out by 2^-16: within 2^-14 of the sum of their magnitudes,
  which is at most |q|^T B with B = e^g B + |k| |u|^T. Towards the state it is
  kept to 2^-24 and sums of 3 x 256 terms at most are off by 2^-14 of their
  magnitudes in the worst case and by sqrt(768) 2^-24 = 2^-19.2 where errors
  are of both signs. With keys no longer than 1 and betas in [0, 1] a step never
  lengthens an error of a state's column, so it is below the sum E of what the
  steps add, E = e^g E + |k| mu with mu = beta (|v| + |k|^T B), times 2^-17, four
  times the estimate. Outputs within u |o| + 2^-14 scale |q|^T B +
  2^-17 scale |q| E, a state's column within 2^-17 E in its 2-norm."""

from __future__ import annotations

import math

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


def ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device=DEV)


def starts_of(lengths, before=0):
    out = [before]
    for n in lengths:
        out.append(out[-1] + n)
    return out


# ---------------------------------------------------------------------------
# convolution
# ---------------------------------------------------------------------------
def conv_exact(x, weight, bias, states, slots, from_slots, starts, activation):
    """(y, the products' magnitudes, states)"""
    width, n_slots = weight.shape[1], states.shape[0]
    y, mag, new = torch.zeros(x.shape, dtype=torch.float64, device=DEV), torch.zeros(x.shape, dtype=torch.float64, device=DEV), states.clone()
    for b, (slot, source) in enumerate(zip(slots, from_slots)):
        lo, hi = starts[b], starts[b + 1]
        if hi == lo:
            continue
        old = states[source] if 0 <= source < n_slots else torch.zeros_like(states[0])
        rows = torch.cat([old, x[lo:hi]])
        taps = [rows[j:j + hi - lo].double() * weight[:, j].double() for j in range(width)] + ([] if bias is None else [bias.double()])
        y[lo:hi], mag[lo:hi] = sum(taps), sum(t.abs() for t in taps)
        if 0 <= slot < n_slots:
            new[slot] = rows[hi - lo:]
    return y * torch.sigmoid(y) if activation == "silu" else y, mag, new


@pytest.mark.parametrize("width", [2, 3, 4])
@pytest.mark.parametrize("channels", [8, 520, 2048])
@pytest.mark.parametrize("lengths", [None, [1], [7], [8], [9, 1, 2, 3, 0, 5, 8, 16, 7], [0, 0, 1, 0], [6, 1, 1, 1, 1, 40], [3, 200, 65]])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_causal_conv(width, channels, lengths, dtype):
    from jeeves_amd import causal_conv

    g = gen(width * channels + len(lengths or [7]))
    batch = len(lengths) if lengths else 7
    before = 3 if lengths and len(lengths) > 2 else 0
    starts = starts_of(lengths, before) if lengths else list(range(batch + 1))
    tokens = starts[-1] + (5 if before else 0)
    merged = randn(g, tokens, channels + 24, dtype=dtype)
    x = merged[:, 8:8 + channels]
    weight, bias = randn(g, channels, width, dtype=torch.float32), randn(g, channels, dtype=torch.float32)
    order = torch.randperm(2 * batch, generator=g, device=DEV).tolist()
    to, source = order[:batch], order[batch:]
    if batch > 4:
        to[1], to[2], source[3], source[4] = -1, 1000, -1, 2 ** 31 - 1
    for b, activation, same in ((bias, "silu", False), (None, None, True)):
        states = randn(g, 2 * batch, width - 1, channels, dtype=dtype)
        y, mag, new = conv_exact(x, weight, b, states, to, to if same else source, starts, activation)
        out = causal_conv(x, weight, states, ints(to), bias=b, from_slots=None if same else ints(source, torch.int64),
                          query_starts=ints(starts, torch.int64) if lengths else None, activation=activation)
        assert out.is_contiguous() and ((out.double() - y).abs() <= rounding(y, dtype) + 2.0 ** -20 * mag).all()
        assert torch.equal(states, new)


def test_conv_of_pieces_is_that_of_the_whole():
    from jeeves_amd import causal_conv

    g = gen(2)
    x, weight = randn(g, 100, 64), randn(g, 64, 4, dtype=torch.float32)
    states = torch.zeros(2, 3, 64, dtype=torch.bfloat16, device=DEV)
    whole = causal_conv(x, weight, states, ints([0]), from_slots=ints([-1]), query_starts=ints([0, 100]))
    parts, at = [], 0
    for n in (1, 1, 2, 5, 8, 3, 80):
        starts = ints([0, n]) if n > 1 else None
        parts.append(causal_conv(x[at:at + n], weight, states, ints([1]), from_slots=ints([-1]) if at == 0 else None, query_starts=starts))
        at += n
    assert torch.equal(torch.cat(parts), whole) and torch.equal(states[0], states[1])


def test_conv_values_that_are_not_finite_stay_in_their_window():
    from jeeves_amd import causal_conv

    g = gen(3)
    x, weight = randn(g, 40, 32), 0.5 + randn(g, 32, 4, dtype=torch.float32).abs()
    states = torch.zeros(4, 3, 32, dtype=torch.bfloat16, device=DEV)
    states[0] = float("nan")  # a slot that no one starts from
    args = (weight, states, ints([1, 2]))
    kw = dict(from_slots=ints([-1, -1]), query_starts=ints([0, 17, 40]), activation=None)
    clean = causal_conv(x, *args, **kw)
    x[9, 5], x[16, 6], x[20, 7] = float("nan"), float("inf"), -float("inf")
    out = causal_conv(x, *args, **kw)
    hit = torch.zeros(40, 32, dtype=torch.bool, device=DEV)
    hit[9:13, 5], hit[16, 6], hit[20:24, 7] = True, True, True
    assert torch.equal(out[~hit], clean[~hit]) and not out[hit].isfinite().any()


# ---------------------------------------------------------------------------
# linear attention
# ---------------------------------------------------------------------------
class Case:
    """A batch of sequences with states, and the recurrence on it in 64 bits."""

    def __init__(self, seed, lengths, heads=(2, 4), dims=(128, 128), dtype=torch.bfloat16, beta=True, raw=False, norm=True, single=False,
                 before=0, behind=0):
        g = self.g = gen(seed)
        (hk, hv), (dk, dv) = heads, dims
        self.lengths, self.norm_eps = lengths, 1e-6 if norm else None
        self.starts = starts_of(lengths, before)
        tokens = self.starts[-1] + behind
        merged = randn(g, tokens, 2 * hk * dk + hv * dv + 8, dtype=dtype)
        q, k, v, _ = merged.split([hk * dk, hk * dk, hv * dv, 8], 1)
        self.q, self.k, self.v = q.view(tokens, hk, dk), k.view(tokens, hk, dk), v.view(tokens, hv, dv)
        if not norm:
            self.q, self.k = self.q * dk ** -0.5, self.k * dk ** -0.5 * 0.5
        self.rate = self.bias = None
        if raw:
            gates = randn(g, tokens, 2 * hv, dtype=dtype)
            self.decay, self.beta = gates[:, :hv], gates[:, hv:] if beta else None
            self.rate, self.bias = 0.2 + torch.rand(hv, generator=g, device=DEV) * 8, randn(g, hv, dtype=torch.float32) - 3
        else:
            self.decay = -torch.exp(randn(g, tokens, hv, dtype=torch.float32) * 2 - 2)
            self.beta = torch.rand(tokens, hv, generator=g, device=DEV) if beta else None
        n = len(lengths)
        self.states = randn(g, 2 * n + 1, hv, dk, dv, dtype=torch.float32)
        order = torch.randperm(2 * n + 1, generator=g, device=DEV).tolist()
        self.to, self.source = order[:n], order[n:2 * n]
        self.single = single

    def run(self, states=None, **kw):
        from jeeves_amd import linear_attention

        args = dict(beta=self.beta, rate=self.rate, decay_bias=self.bias, from_slots=ints(self.source),
                    query_starts=None if self.single else ints(self.starts), norm_eps=self.norm_eps) | kw
        states = self.states.clone() if states is None else states
        return linear_attention(self.q, self.k, self.v, self.decay, states, ints(self.to), **args), states

    def exact(self):
        """(outputs, B's bound on their sums, E's on the states' part; states, E)"""
        hk, hv, dk, dv = self.q.shape[1], self.v.shape[1], self.q.shape[2], self.v.shape[2]
        q, k, v = self.q.double(), self.k.double(), self.v.double()
        if self.norm_eps:
            q, k = (t / (t.square().sum(-1, keepdim=True) + self.norm_eps).sqrt() for t in (q, k))
        q, k = (t.repeat_interleave(hv // hk, 1) for t in (q * dk ** -0.5, k))
        g, beta = self.decay.double(), None if self.beta is None else self.beta.double()
        if self.rate is not None:
            z = g if self.bias is None else g + self.bias.double()
            g = -self.rate.double() * torch.logaddexp(z, torch.zeros_like(z))
            beta = None if beta is None else 1 / (1 + torch.exp(-beta))
        out, mag, far = (torch.zeros(*v.shape, dtype=torch.float64, device=DEV) for _ in range(3))
        states, spread = self.states.double(), torch.zeros(self.states.shape[0], hv, dv, dtype=torch.float64, device=DEV)
        olds = self.states.double()
        for b, n in enumerate(self.lengths):
            if n == 0:
                continue
            old = 0 <= self.source[b] < len(olds)
            S = olds[self.source[b]].clone() if old else torch.zeros(hv, dk, dv, dtype=torch.float64, device=DEV)
            B, E = S.abs(), S.norm(dim=1) * 2.0 ** -4
            for t in range(self.starts[b], self.starts[b] + n):
                d = g[t].exp()
                S, B, E = d[:, None, None] * S, d[:, None, None] * B, d[:, None] * E
                kt = k[t][..., None]
                u, mu = v[t], v[t].abs() + (kt.abs() * B).sum(1)
                if beta is not None:
                    u, mu = beta[t][:, None] * (u - (kt * S).sum(1)), beta[t][:, None].abs() * mu
                S, B, E = S + kt * u[:, None], B + kt.abs() * u[:, None].abs(), E + k[t].norm(dim=-1, keepdim=True) * mu
                out[t] = (q[t][..., None] * S).sum(1)
                mag[t], far[t] = (q[t][..., None].abs() * B).sum(1), q[t].norm(dim=-1, keepdim=True) * E
            if 0 <= self.to[b] < len(olds):
                states[self.to[b]], spread[self.to[b]] = S, E
        return out, mag, far, states, spread

    def check(self, **kw):
        got, states = self.run(**kw)
        out, mag, far, want, spread = self.exact()
        bound = rounding(out, self.q.dtype) + 2.0 ** -14 * mag + 2.0 ** -17 * far
        assert got.is_contiguous() and ((got.double() - out).abs() <= bound).all(), ((got.double() - out).abs() / bound).max().item()
        assert ((states.double() - want).norm(dim=2) <= 2.0 ** -17 * spread).all()
        again, same = self.run(**kw)
        assert torch.equal(again, got) and torch.equal(same, states)
        return got, states


LAYOUTS = [((2, 4), (128, 128)), ((3, 3), (64, 64)), ((1, 3), (128, 64)), ((2, 2), (64, 256)), ((1, 2), (256, 256)), ((2, 2), (256, 128))]


@pytest.mark.parametrize("heads,dims", LAYOUTS)
@pytest.mark.parametrize("beta", [True, False])
@pytest.mark.parametrize("raw", [True, False])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_single_tokens(heads, dims, beta, raw, dtype):
    Case(1, [1] * 5, heads, dims, dtype, beta, raw, single=True).check()


@pytest.mark.parametrize("heads,dims", LAYOUTS)
@pytest.mark.parametrize("beta", [True, False])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_prompts_of_every_layout(heads, dims, beta, dtype):
    Case(2, [70, 3, 128], heads, dims, dtype, beta, raw=beta).check()
    Case(3, [65, 130], heads, dims, dtype, beta, raw=not beta, norm=False).check()


# Sequences without tokens that bring a batch of four value heads to each of the scans: 16 and 32 columns a workgroup, 64 and 128.
SCANS = [((64, 64), 0), ((128, 128), 9), ((64, 64), 45), ((128, 128), 20)]


@pytest.mark.parametrize("heads,dims", LAYOUTS + [((2, 4), (64, 128))])
@pytest.mark.parametrize("beta", [True, False])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("columns", [300, 700])
def test_prompts_of_every_layout_in_large_batches(heads, dims, beta, dtype, columns):
    """As above in the scans for more than 256 and 512 times 16 state columns, which batches of empty sequences reach too."""
    empty = columns * 16 // (heads[1] * dims[1]) + 1
    Case(5, [0] * (empty // 2) + [70, 3, 128, 65, 1] + [0] * (empty // 2), heads, dims, dtype, beta, raw=beta).check()


@pytest.mark.parametrize("lengths", [[1], [2], [63], [64], [65], [0], [0, 0, 5, 0, 64, 0], [127, 128, 129], [1] * 70, [3, 61, 64, 0, 1, 191, 16]])
@pytest.mark.parametrize("beta", [True, False])
def test_prompt_lengths(lengths, beta):
    Case(4 + len(lengths), lengths, beta=beta, dims=(64, 64), raw=True, before=5, behind=9).check()


def test_tokens_of_no_sequence_are_zero():
    c = Case(20, [30, 0, 70], dims=(64, 64), before=7, behind=66)
    out, _ = c.check()
    assert (out[:7] == 0).all() and (out[107:] == 0).all()
    # a batch of empty sequences: no state is touched
    c = Case(21, [0, 0], before=0, behind=3)
    out, states = c.run()
    assert (out == 0).all() and torch.equal(states, c.states)


@pytest.mark.parametrize("single", [True, False])
def test_slots(single):
    """New sequences, padding, one slot that several start from, slots in place, wide indices."""
    c = Case(22, [1] * 6 if single else [5, 70, 1, 64, 3, 9], dims=(64, 128), raw=True, single=single)
    c.source[0], c.source[1], c.source[2], c.source[3] = -1, 10 ** 6, c.source[4], c.source[4]
    c.to[4], c.to[5] = -1, len(c.states)
    c.check()
    got, states = c.run()
    wide, same = c.run(from_slots=ints(c.source, torch.int64), query_starts=None if single else ints(c.starts, torch.int64))
    assert torch.equal(got, wide) and torch.equal(states, same)
    c.source = c.to = list(range(6))
    c.check(from_slots=None)


def test_no_slots_at_all():
    for single in (True, False):
        c = Case(23, [1, 1] if single else [3, 66], dims=(64, 64), single=single)
        c.source = c.to = [0, 1]
        c.states = c.states[:0]
        c.check()


def test_pieces_are_near_the_whole():
    """A prompt whole, in pieces, and token by token."""
    whole = Case(24, [200], raw=True)
    out, mag, far, want, spread = whole.exact()
    states = whole.states.clone()
    from jeeves_amd import linear_attention

    at, slot = 0, ints(whole.to)
    for n in (64, 1, 1, 30, 103, 1):
        s = slice(at, at + n)
        got = linear_attention(whole.q[s], whole.k[s], whole.v[s], whole.decay[s], states, slot, beta=whole.beta[s], rate=whole.rate,
                               decay_bias=whole.bias, from_slots=ints(whole.source) if at == 0 else None, norm_eps=1e-6,
                               query_starts=ints([0, n]) if n > 1 else None)
        assert ((got.double() - out[s]).abs() <= rounding(out[s], got.dtype) + 2.0 ** -14 * mag[s] + 2.0 ** -17 * far[s]).all()
        at += n
    assert ((states.double() - want).norm(dim=2) <= 2.0 ** -17 * spread).all()


def test_states_keep_32_bits():
    """Errors of both signs: the relative 2-norm of a state's error is that of sums of a few hundred fp32 roundings, at
    most sqrt(768) 2^-24 for a chunk and less for what decays; a product of 16 bits would be off by 2^-17."""
    for dtype in (torch.bfloat16, torch.float16):
        c = Case(25, [500], raw=True, dtype=dtype)
        _, states = c.run()
        want = c.exact()[3]
        slot = c.to[0]
        assert (states[slot].double() - want[slot]).norm() / want[slot].norm() < 2.0 ** -19


@pytest.mark.parametrize("single", [True, False])
def test_decays_of_extremes(single):
    """Decays of 0 (log -inf, or far below) drop the state whole, decays of 1 keep it; a chunk's later tokens keep their
    own decays' bits behind one."""
    for beta in (True, False):
        c = Case(26, [1] * 40 if single else [150, 64], dims=(64, 64), beta=beta, single=single)
        c.decay[::7] = 0.0
        c.decay[3::11] = -float("inf")
        c.decay[5::13] = -1e30
        c.decay[6::17] = -300.0
        c.check()


def test_keys_that_are_the_same():
    """The triangular system at its largest: keys of one direction, betas of 1."""
    c = Case(27, [256, 100], dims=(128, 64))
    c.k = c.k[:1].expand(c.k.shape)
    c.beta = torch.ones_like(c.beta)
    c.decay = torch.zeros_like(c.decay)
    c.check()
    c.beta = c.beta * 0
    c.check()


def test_strides_and_scale():
    c = Case(28, [66, 5], heads=(2, 2), dims=(64, 64))
    c.q = c.q.transpose(0, 1).contiguous().transpose(0, 1)
    c.k = randn(c.g, 1, 1, 64).expand(c.k.shape)
    c.decay = c.decay.t().contiguous().t()
    c.check()
    got, states = c.run()
    twice, same = c.run(scale=2 * 64 ** -0.5)
    assert torch.equal(twice, 2 * got) and torch.equal(states, same)
    odd = torch.zeros(c.v.numel() + 3, dtype=c.v.dtype, device=DEV)[3:].view(c.v.shape)
    odd.copy_(c.v)
    c.v = odd
    again, same = c.run()
    assert torch.equal(again, got) and torch.equal(states, same)


@pytest.mark.parametrize("beta", [True, False])
@pytest.mark.parametrize("what", ["v", "k", "q", "decay", "beta"])
@pytest.mark.parametrize("value", [math.nan, math.inf])
@pytest.mark.parametrize("dims,empty", SCANS)
def test_what_is_not_finite_reaches_later_tokens_alone(what, value, beta, dims, empty):
    """Of a token in the middle of a chunk: the tokens before it, and the other sequences, heads and (for a value) channels
    keep their bits; what sees it is not finite."""
    if what == "beta" and not beta:
        return
    c = Case(29, [40, 150, 70] + [0] * empty, dims=dims, beta=beta)
    clean, clean_states = c.run()
    at = 40 + 64 + 21
    if what == "v":
        c.v = c.v.clone()
        c.v[at, 1, 17] = value
    elif what in ("k", "q"):
        t = getattr(c, what).clone()
        t[at, 0, 9] = value
        setattr(c, what, t)
    else:
        getattr(c, what)[at, 1] = value
    out, states = c.run()
    hit = torch.zeros(out.shape, dtype=torch.bool, device=DEV)
    heads = slice(0, 2) if what in ("k", "q") else slice(1, 2)  # heads 0 and 1 read key head 0
    hit[at:at + 1 if what == "q" else 190, heads, 17 if what == "v" else slice(None)] = True
    assert torch.equal(out[~hit], clean[~hit])
    assert not out[hit].isfinite().any()
    if what != "q":
        assert not states[c.to[1], heads][..., 17 if what == "v" else slice(None)].isfinite().all()
    same = torch.ones(states.shape, dtype=torch.bool, device=DEV)
    same[c.to[1], heads, :, 17 if what == "v" else slice(None)] = what == "q"
    assert torch.equal(states[same], clean_states[same])


@pytest.mark.parametrize("dims,empty", SCANS)
def test_a_state_that_is_not_finite_stays_in_its_column(dims, empty):
    for single in (True, False):
        c = Case(30, [1, 1, 1] if single else [10, 130, 5] + [0] * empty, dims=dims, single=single)
        clean, clean_states = c.run()
        c.states[c.source[1], 2, 5, 33] = math.nan
        c.states[c.source[2]] = math.inf
        c.source[2] = -1  # no one's
        out, states = c.run()
        rows = slice(c.starts[1], c.starts[2])
        assert out[rows, 2, 33].isnan().all() and states[c.to[1], 2, :, 33].isnan().any()
        out[rows, 2, 33] = clean[rows, 2, 33]
        assert torch.equal(out[:c.starts[2]], clean[:c.starts[2]])


def test_slots_past_32_bit_offsets():
    """States of more than 2^31 values."""
    for single in (True, False):
        c = Case(31, [1, 1] if single else [70, 2], heads=(4, 8), dims=(256, 256), single=single)
        small = c.states
        n = (1 << 31) // small[0].numel() + 40
        states = torch.zeros(n, *small.shape[1:], device=DEV)
        far = [n - 1, n - 2, n - 3, n - 4, n - 5]
        for i, s in enumerate(far):
            states[s] = small[i]
        want, want_states = c.run()
        c.to, c.source = [far[i] for i in c.to], [far[i] for i in c.source]
        got, states = c.run(states)
        assert torch.equal(got, want) and all(torch.equal(states[s], want_states[i]) for i, s in enumerate(far))
        assert (states[:n - 5].view(-1)[::1009] == 0).all()
        del states


def test_long_prompt():
    c = Case(32, [3000], heads=(1, 1), dims=(64, 64), raw=True)
    c.check()


def test_many_sequences():
    c = Case(33, [i % 4 for i in range(150)], heads=(1, 1), dims=(64, 64), raw=True, before=2)
    c.check()
    c = Case(37, [i % 7 == 3 for i in range(1500)], heads=(1, 1), dims=(64, 64), raw=True, behind=1)  # too many to be ranked by length
    c.check()


@pytest.mark.parametrize("single", [True, False])
def test_captured_with_other_slots_and_starts(single):
    """Two graphs and eager calls by turns, each replay with other inputs, slots and starts."""
    from jeeves_amd import causal_conv, linear_attention

    g = gen(34)
    batch, hk, hv, d = 4, 2, 4, 64
    tokens, channels = (batch if single else 150), 2 * hk * d + hv * d
    x, weight = randn(g, tokens, channels), randn(g, channels, 4, dtype=torch.float32)
    gates, rate = randn(g, tokens, 2 * hv), torch.ones(hv, device=DEV)
    slots, source, starts = ints([0, 1, 2, 3]), ints([4, 5, 6, 7]), ints([0, 20, 20, 90, 150])

    def step(conv_states, states):
        mixed = causal_conv(x, weight, conv_states, slots, from_slots=source, query_starts=None if single else starts)
        q, k, v = mixed.split([hk * d, hk * d, hv * d], 1)
        return mixed, linear_attention(q.view(tokens, hk, d), k.view(tokens, hk, d), v.view(tokens, hv, d), gates[:, :hv], states, slots,
                                       beta=gates[:, hv:], rate=rate, from_slots=source, query_starts=None if single else starts,
                                       norm_eps=1e-6)

    def fresh():
        return randn(gen(35), 8, 3, channels), randn(gen(36), 8, hv, d, d, dtype=torch.float32)

    held = [fresh(), fresh()]
    eager = fresh()
    torch.cuda.synchronize()
    graphs, outs = [], []
    s = torch.cuda.Stream()
    for states in held:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            outs.append(step(*states))
        graphs.append(graph)
    for i in range(4):
        x.copy_(randn(g, tokens, channels))
        gates.copy_(randn(g, tokens, 2 * hv))
        order = torch.randperm(8, generator=g, device=DEV).int()
        slots.copy_(order[:4])
        source.copy_(order[4:] if i % 2 else order[:4])
        if i == 2:
            source[1] = -1
        starts.copy_(ints([[0, 20, 20, 90, 150], [3, 3, 4, 70, 148], [0, 64, 128, 129, 150], [0, 0, 0, 0, 150]][i]))
        torch.cuda.synchronize()
        for graph in graphs:
            graph.replay()
        want = step(*eager)
        torch.cuda.synchronize()
        for out, states in zip(outs, held):
            assert all(torch.equal(a, b) for a, b in zip((*out, *states), (*want, *eager)))


def test_refusals():
    from jeeves_amd import causal_conv, linear_attention

    x = torch.zeros(4, 256, dtype=torch.bfloat16, device=DEV)
    h, f32 = x.view(4, 2, 128), torch.zeros(4, 2, device=DEV)
    w, cs, slots = torch.zeros(256, 4, device=DEV), torch.zeros(2, 3, 256, dtype=torch.bfloat16, device=DEV), ints([0, 1, 0, 1])
    states = torch.zeros(2, 2, 128, 128, device=DEV)
    for bad in (lambda: causal_conv(x.float(), w, cs, slots), lambda: causal_conv(x[:, :252], w[:252], cs, slots), lambda: causal_conv(h, w, cs, slots),
                lambda: causal_conv(x, w[:128], cs, slots), lambda: causal_conv(x, w[:, :1], cs, slots), lambda: causal_conv(x, w, cs.half(), slots),
                lambda: causal_conv(x, w, cs[:, :2], slots), lambda: causal_conv(x, w, cs, slots[:3]), lambda: causal_conv(x, w, cs, slots.float()),
                lambda: causal_conv(x, w, cs, slots.cpu()), lambda: causal_conv(x, w, cs, slots, from_slots=slots[:2]),
                lambda: causal_conv(x, w, cs, slots, query_starts=slots), lambda: causal_conv(x, w, cs, slots, bias=w[:8, 0]),
                lambda: causal_conv(x, w, cs, slots, activation="relu"), lambda: causal_conv(x, w, cs[:, :, ::2], slots)):
        with pytest.raises(ValueError):
            bad()
    ok = linear_attention
    for bad in (lambda: ok(h.float(), h, h, f32, states, slots), lambda: ok(h, h[:3], h, f32, states, slots), lambda: ok(h, h[:, :1], h, f32, states, slots),
                lambda: ok(h, h, h.half(), f32, states, slots), lambda: ok(h, h, h[..., :32], f32, states, slots),
                lambda: ok(h, h, h, f32[:, :1], states, slots), lambda: ok(h, h, h, f32.half(), states, slots), lambda: ok(h, h, h, f32.cpu(), states, slots),
                lambda: ok(h, h, h, f32, states.bfloat16(), slots), lambda: ok(h, h, h, f32, states[:, :1], slots),
                lambda: ok(h, h, h, f32, states.transpose(2, 3), slots), lambda: ok(h, h, h, f32, states, slots[:2]),
                lambda: ok(h, h, h, f32, states, slots, beta=f32.bfloat16()), lambda: ok(h, h, h, f32, states, slots, beta=f32[:3]),
                lambda: ok(h, h, h, f32, states, slots, decay_bias=f32[0]), lambda: ok(h, h, h, f32, states, slots, rate=f32[:, 0]),
                lambda: ok(h, h, h, f32, states, slots, norm_eps=0.0), lambda: ok(h, h, h, f32, states, slots, norm_eps=1e-60), lambda: ok(h, h, h, f32, states, slots, scale=math.inf),
                lambda: ok(h, h, h, f32, states, slots, query_starts=ints([0, 4])), lambda: ok(x.view(4, 8, 32), h, h, f32, states, slots)):
        with pytest.raises(ValueError):
            bad()
    none = torch.empty(0, 2, 128, dtype=torch.bfloat16, device=DEV)
    assert ok(none, none, none, f32[:0], states, slots[:0]).shape == (0, 2, 128)
    assert causal_conv(x[:0], w, cs, slots[:0]).shape == (0, 256)


# ---------------------------------------------------------------------------
# a run of them, as a layer has them
# ---------------------------------------------------------------------------
def block_of(g, hidden=256, hk=2, hv=4, d=64):
    from jeeves_amd import FP8Linear, FP8LinearAttention

    channels = 2 * hk * d + hv * d
    qkvz, out = FP8Linear(hidden, channels + hv * d, device=DEV), FP8Linear(hv * d, hidden, device=DEV)
    qkvz.load_weight(randn(g, channels + hv * d, hidden) * hidden ** -0.5)
    out.load_weight(randn(g, hidden, hv * d) * (hv * d) ** -0.5)
    return FP8LinearAttention(qkvz, randn(g, 2 * hv, hidden) * hidden ** -0.5, out, hk, hv, d, d, randn(g, channels, 4) * 0.5,
                              torch.rand(hv, generator=g, device=DEV) * 4, randn(g, hv) - 2, 1 + 0.2 * randn(g, d))


def layer(block, mlp, norms, x, conv_states, states, slots, quantize, **kw):
    """A decoder layer between two residual sums: norm, block, sum and norm, FP8 linear, sum."""
    from jeeves_amd import add_norm

    first = add_norm(torch.zeros_like(x), x, norms[0])
    second = add_norm(block(first.y, conv_states, states, slots, **kw), first.h, norms[1], quantize=quantize)
    y = mlp.forward_codes(second.codes, second.scales, packed_rows=x.shape[0]) if quantize else mlp(second.y)
    return add_norm(y, second.h, None).h


@pytest.mark.parametrize("lengths", [None, [5, 90, 1]])
def test_layer(lengths):
    """The operators in a row give what the same steps in float64 give, but for the two FP8 projections' codes: a
    perturbation of 2^-8 (an intermediate's rounding) turns at most one code in 16 by a step of 2^-3, and each e4m3 code
    is off by 2^-4 at most, 0.027 of the value in the 2-norm; three projections one after the other and the sums between
    them leave the layer's update within 0.15."""
    from jeeves_amd import FP8Linear

    g = gen(40)
    block, mlp = block_of(g), FP8Linear(256, 256, device=DEV)
    mlp.load_weight(randn(g, 256, 256) * 256 ** -0.5)
    batch = len(lengths) if lengths else 3
    starts = starts_of(lengths) if lengths else list(range(batch + 1))
    tokens = starts[-1]
    x, norms = randn(g, tokens, 256), [1 + 0.2 * randn(g, 256, dtype=torch.float32) for _ in range(2)]
    conv_states, states = block.allocate(batch)
    conv_states.copy_(randn(g, *conv_states.shape))
    states.copy_(randn(g, *states.shape, dtype=torch.float32) * 0.1)
    kw = dict(query_starts=ints(starts)) if lengths else {}
    runs = []
    for quantize in ("packed", None):
        cs, st = conv_states.clone(), states.clone()
        runs.append((layer(block, mlp, norms, x, cs, st, ints(list(range(batch))), quantize, **kw), cs, st))

    def project(linear, t):
        return t @ (linear.weight.double() * linear.scale.double()[:, None]).t()

    def normed(t, w):
        return rms(t) * w.double()

    def rms(t):
        return t / (t.square().mean(-1, keepdim=True) + 1e-6).sqrt()

    h = normed(x.double(), norms[0])
    proj, gates = project(block.qkvz, h), h @ block.gates.double().t()
    hk, hv, d = block.k_heads, block.v_heads, block.k_dim
    rows = []
    for b in range(batch):
        lo, hi = starts[b], starts[b + 1]
        inputs = torch.cat([conv_states[b].double(), proj[lo:hi, :block.channels]])
        mixed = sum(inputs[j:j + hi - lo] * block.conv_weight[:, j].double() for j in range(4))
        mixed = mixed * torch.sigmoid(mixed)
        q, k, v = mixed.split([hk * d, hk * d, hv * d], 1)
        q, k = (t.view(-1, hk, d).repeat_interleave(hv // hk, 1) for t in (q, k))
        q, k = (t / (t.square().sum(-1, keepdim=True) + 1e-6).sqrt() for t in (q, k))
        v, S = v.view(-1, hv, d), states[b].double()
        for i in range(hi - lo):
            a, be = gates[lo + i, :hv], torch.sigmoid(gates[lo + i, hv:])
            S = S * torch.exp(-block.rate.double() * torch.nn.functional.softplus(a + block.decay_bias.double()))[:, None, None]
            u = be[:, None] * (v[i] - (k[i][..., None] * S).sum(1))
            S = S + k[i][..., None] * u[:, None]
            rows.append((q[i][..., None] * S).sum(1) * d ** -0.5)
        for _, cs, st in runs:
            assert (st[b].double() - S).norm() / S.norm() < 0.15
            assert (cs[b].double() - inputs[hi - lo:]).norm() / inputs[hi - lo:].norm() < 0.1
    z = proj[:, block.channels:].view(tokens, hv, d)
    y = rms(torch.stack(rows)) * block.norm_weight.double() * z * torch.sigmoid(z)
    h = x.double() + project(block.out, y.flatten(1))
    want = h + project(mlp, normed(h, norms[1]))
    for got, _, _ in runs:
        assert (got.double() - want).norm() / (want - x.double()).norm() < 0.15


def test_block_takes_codes_or_not():
    """With a LoRA adapter on the out projection its input stays 16-bit; a zero adapter changes the codes' source alone."""
    g = gen(41)
    block = block_of(g)
    x = randn(g, 6, 256)
    slots = ints(list(range(6)))
    with_codes = block(x, *block.allocate(6), slots)
    block.out.set_lora(torch.zeros(16, 256, device=DEV), torch.zeros(256, 16, device=DEV), 1.0)
    plain = block(x, *block.allocate(6), slots)
    assert (with_codes.double() - plain.double()).norm() / plain.double().norm() < 0.05
    none = torch.empty(0, 256, dtype=torch.bfloat16, device=DEV)
    assert block(none, *block.allocate(1), slots[:0]).shape == (0, 256)


def test_warm_prepares_the_block_for_capture():
    from jeeves_amd import warm

    g = gen(42)
    block = block_of(g)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        assert warm(block) == 2
    torch.cuda.synchronize()
    for starts in (None, ints([0, 1, 1, 6])):
        x, slots = randn(g, 3 if starts is None else 6, 256), ints([0, 1, 2])
        held, eager = block.allocate(3), block.allocate(3)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            out = block(x, *held, slots, query_starts=starts)
        for _ in range(4):
            x.copy_(randn(g, *x.shape))
            graph.replay()
            want = block(x, *eager, slots, query_starts=starts)
            torch.cuda.synchronize()
            assert torch.equal(out, want) and all(torch.equal(a, b) for a, b in zip(held, eager))
