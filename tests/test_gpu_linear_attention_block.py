"""``FP8LinearAttention`` as a module: what prepares it for capture, its hooks,
and its output against the steps in 64 bits."""

from __future__ import annotations

import pytest
import torch

from tests.test_gpu_linear_attention import DEV, block_of, gen, ints, randn

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
