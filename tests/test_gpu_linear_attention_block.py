"""``FP8LinearAttention`` as a module: what prepares it for capture, its hooks,
and its output against the steps in 64 bits."""

from __future__ import annotations

import pytest
import torch

from tests.test_gpu_linear_attention import DEV, Case, block_of, gen, ints, randn, rounding, starts_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d", [64, 128])
def test_warm_reaches_every_form(monkeypatch, d):
    """Batches on both sides of each bound between the scans, both forms of the norm, the small projection and the out projection
    of codes; then a batch of the wide scan is captured."""
    from jeeves_amd import recurrent, sm_count, warm

    seen = {"columns": set(), "quantize": set(), "gates": set(), "codes": set()}
    attention, norm, linear, forward_codes = recurrent.linear_attention, recurrent.gated_norm, torch.nn.functional.linear, recurrent.FP8Linear.forward_codes
    block = block_of(gen(70), d=d)

    def counted(q, k, v, decay, states, slots, **kw):
        seen["columns"].add((kw["query_starts"] is not None) * slots.shape[0] * v.shape[1] * v.shape[2] // 16)
        return attention(q, k, v, decay, states, slots, **kw)

    monkeypatch.setattr(recurrent, "linear_attention", counted)
    monkeypatch.setattr(recurrent, "gated_norm", lambda *a, **kw: (seen["quantize"].add(kw.get("quantize")), norm(*a, **kw))[1])
    monkeypatch.setattr(torch.nn.functional, "linear", lambda x, w, b=None: (seen["gates"].add(x.shape[0]), linear(x, w, b))[1])
    monkeypatch.setattr(recurrent.FP8Linear, "forward_codes",
                        lambda self, *a, **kw: (seen["codes"].add(kw["packed_rows"]), forward_codes(self, *a, **kw))[1])
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        assert warm(block) == 2
    torch.cuda.synchronize()
    monkeypatch.undo()
    units = sm_count(block.gates.device)
    assert 0 in seen["columns"] and seen["quantize"] == {None, "packed"}
    for lo, hi in ((1, units), (units + 1, 2 * units), (2 * units + 1, 1 << 20)):
        assert any(lo <= c <= hi for c in seen["columns"]), (lo, hi, seen["columns"])
    assert seen["gates"] == seen["codes"] == set(recurrent.WARM_ROWS)

    n = 2 * units * 16 // (4 * d) + 3
    x, starts = randn(gen(71), 90, 256), torch.full((n + 1,), 90, dtype=torch.int32, device=DEV)
    starts[0], starts[1] = 0, 70
    slots, held, eager = ints(list(range(n))), block.allocate(n), block.allocate(n)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        out = block(x, *held, slots, query_starts=starts)
    for i in range(3):
        x.copy_(randn(gen(72 + i), *x.shape))
        graph.replay()
        want = block(x, *eager, slots, query_starts=starts)
        torch.cuda.synchronize()
        assert torch.equal(out, want) and all(torch.equal(a, b) for a, b in zip(held, eager))


def test_hooks_of_the_projections_run():
    """Those of the out projection too, which then takes the 16-bit input that they see."""
    block = block_of(gen(75))
    x, slots, seen = randn(gen(76), 6, 256), ints(list(range(6))), []
    plain = block(x, *block.allocate(6), slots)
    block.out.set_lora(torch.zeros(16, 256, device=DEV), torch.zeros(256, 16, device=DEV), 1.0)
    sixteen = block(x, *block.allocate(6), slots)  # from 16-bit input, by an adapter that adds nothing
    block.out.lora = None
    handles = [block.qkvz.register_forward_hook(lambda m, a, y: seen.append("qkvz")),
               block.out.register_forward_pre_hook(lambda m, a: seen.append(a[0].shape)),
               block.out.register_forward_hook(lambda m, a, y: y + 1)]
    hooked = block(x, *block.allocate(6), slots)
    assert seen == ["qkvz", (6, 256)] and torch.equal(hooked, sixteen + 1)
    for h in handles:
        h.remove()
    assert torch.equal(block(x, *block.allocate(6), slots), plain)
    handle = torch.nn.modules.module.register_module_forward_pre_hook(lambda m, a: seen.append(m))
    try:
        block(x, *block.allocate(6), slots)
    finally:
        handle.remove()
    assert block.out in seen

    class Doubled(type(block.out)):
        def forward(self, x):
            return 2 * super().forward(x)

    block.out.__class__ = Doubled
    assert torch.equal(block(x, *block.allocate(6), slots), 2 * sixteen)


@pytest.mark.parametrize("lengths", [None, [5, 90, 1]])
def test_block_against_its_steps_in_64_bits(monkeypatch, lengths):
    """From the FP8 projection's own output on: the convolution has the bits of the elementary operations, the linear attention
    is within its bound d of the recurrence in 64 bits, and the norm of what it stored is off by that and its own rounding: with
    r the root mean square of a head, |w act(z)| / r (d + |y| |d| / |y|) in the 2-norms over the head, and u of the result. The
    16-bit input of the out projection is compared, and the block's output is that projection of its codes, bit for bit."""
    from jeeves_amd import gated_norm, recurrent

    g = gen(80)
    block = block_of(g)
    n = len(lengths) if lengths else 3
    starts = starts_of(lengths) if lengths else list(range(n + 1))
    tokens, hk, hv, d = starts[-1], block.k_heads, block.v_heads, block.k_dim
    x, (conv_states, states) = randn(g, tokens, 256), block.allocate(2 * n)
    conv_states.copy_(randn(g, *conv_states.shape))
    states.copy_(randn(g, *states.shape, dtype=torch.float32) * 0.3)
    c = Case.__new__(Case)
    c.lengths, c.starts, c.single = lengths or [1] * n, starts, lengths is None
    c.to, c.source, c.norm_eps, c.rate, c.bias = list(range(n)), list(range(n, 2 * n)), block.eps, block.rate, block.decay_bias
    c.states = states.clone()

    proj, gates = block.qkvz(x), torch.nn.functional.linear(x, block.gates)
    rows = torch.zeros(tokens, block.channels, device=DEV)
    for b in range(n):
        inputs = torch.cat([conv_states[n + b], proj[starts[b]:starts[b + 1], :block.channels]]).float()
        for j in range(4):
            rows[starts[b]:starts[b + 1]] += inputs[j:j + c.lengths[b]] * block.conv_weight[:, j]
    mixed = (rows * (1 / (1 + torch.exp(-rows)))).bfloat16()
    q, k, v = mixed.split([hk * d, hk * d, hv * d], 1)
    c.q, c.k, c.v, c.decay, c.beta = q.view(tokens, hk, d), k.view(tokens, hk, d), v.view(tokens, hv, d), gates[:, :hv], gates[:, hv:]
    y, mag, far, want, spread = c.exact()
    off = rounding(y, torch.bfloat16) + 2.0 ** -14 * mag + 2.0 ** -17 * far

    stored = []
    monkeypatch.setattr(recurrent, "gated_norm", lambda y, *a, **kw: (stored.append(y), gated_norm(y, *a, **kw))[1])
    out = block(x, conv_states, states, ints(c.to), from_slots=ints(c.source), query_starts=ints(starts) if lengths else None)
    (y_stored,) = stored
    z = proj[:, block.channels:].view(tokens, hv, d)
    assert ((y_stored.double() - y).abs() <= off).all()
    assert ((states.double() - want).norm(dim=2) <= 2.0 ** -17 * spread).all()
    root = (y.square().mean(-1, keepdim=True) + block.eps).sqrt()
    factor = block.norm_weight.double() * z.double() * torch.sigmoid(z.double())
    normed = gated_norm(y_stored, z, block.norm_weight, eps=block.eps)
    exact = y / root * factor
    bound = factor.abs() / root * (off + y.abs() * off.norm(dim=-1, keepdim=True) / y.norm(dim=-1, keepdim=True)) * (1 + 2.0 ** -6)
    assert ((normed.double() - exact).abs() <= bound + rounding(exact, torch.bfloat16) * (1 + 2.0 ** -6) + 2.0 ** -18 * exact.abs()).all()
    codes = gated_norm(y_stored, z, block.norm_weight, eps=block.eps, quantize="packed")
    assert torch.equal(out, block.out.forward_codes(*codes, packed_rows=tokens))
