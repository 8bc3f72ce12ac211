"""What lies between the projections of a layer whose attention is linear, on
MI355X (C ABI ``include/jeeves_linear_attention.h``):

* ``causal_conv``: the short depthwise convolution that q, k and v go through,
  each sequence's last inputs kept in a slot;
* ``linear_attention``: attention with a state and a decay for each head, with
  the delta rule's correction or without: chunked for prompts, one read and
  write of the states for single tokens;
* ``FP8LinearAttention``: the FP8 projections of such a layer with these and
  ``gated_norm`` between them.

A sequence carries its state in a slot: it is read from ``from_slots[b]`` and
written to ``slots[b]``. ``from_slots`` defaults to ``slots``; a negative one
starts a sequence from zeros, one slot may start several sequences (a shared
prompt), and a negative entry of ``slots`` keeps nothing (padding). Slots
written by one call are meant to differ, and not to be others' ``from_slots``:
each value of one that two write is either's.

Tensors are bf16 or fp16, states of the linear attention float32. As in
``jeeves_amd.attention``, everything is enqueued on
``torch.cuda.current_stream()`` without host synchronisation (so it may be
captured into a graph, for other slots and starts on replay), outputs and
workspaces come from torch's caching allocator, and bad arguments raise
``ValueError``. No gradients: the framework serves.
"""

from __future__ import annotations

from functools import lru_cache

import torch
import torch.nn as nn

from . import _lib
from .attention import _FP16, HEAD_DIMS, _first, _heads, _int32, _on, _refuse
from .device import sm_count
from .fp8 import QUANT_MAX_PACKED_COLS, WARM_ROWS, FP8Linear
from .norms import _ptr, _weight, gated_norm

CONV_WIDTHS = (2, 3, 4)
CONV_MAX_CHANNELS = 65536
_CONV_ACTIVATIONS = {None: 0, "silu": 1}
_TINY = torch.finfo(torch.float32).tiny


def _batch(slots: torch.Tensor, from_slots: torch.Tensor | None, query_starts: torch.Tensor | None, tokens: int, index: int) -> tuple:
    """(sequences; slots, from_slots, query_starts as the kernels read them)."""
    if slots.dim() != 1:
        _refuse("slots", slots, "int32 or int64 [batch]")
    batch = slots.shape[0]
    slots = _int32("slots", slots, (batch,), index)
    if from_slots is not None:
        from_slots = _int32("from_slots", from_slots, (batch,), index)
    if query_starts is not None:
        query_starts = _int32("query_starts", query_starts, (batch + 1,), index)
    elif tokens != batch:
        raise ValueError(f"without query_starts each of the {batch} sequences has one token, got {tokens}")
    return batch, slots, from_slots, query_starts


def causal_conv(x: torch.Tensor, weight: torch.Tensor, states: torch.Tensor, slots: torch.Tensor, *, bias: torch.Tensor | None = None,
                from_slots: torch.Tensor | None = None, query_starts: torch.Tensor | None = None,
                activation: str | None = "silu") -> torch.Tensor:
    """Depthwise causal convolution of tokens ``x`` [tokens, channels] (channels
    a multiple of 8; a view of a merged projection's output will do) with
    ``weight`` [channels, width] (width 2 to 4, the last column the token's
    own) and ``bias`` [channels], in 32 bits, through ``activation``
    (``"silu"`` or None) and rounded once; a new tensor.

    Sequence b of the batch has the tokens ``query_starts[b]`` to
    ``query_starts[b + 1] - 1`` ([batch + 1], not decreasing, from 0 to tokens;
    None: one token each), behind the last ``width - 1`` inputs of the slot
    ``from_slots[b]`` of ``states`` [slots, width - 1, channels] (x's type,
    contiguous, oldest first), whose last inputs go to ``slots[b]``. A sequence
    without tokens changes nothing; tokens of no sequence come out as 0.
    """
    dtype, index, shape = x.dtype, x.get_device(), x.shape
    if len(shape) != 2 or dtype not in _FP16 or index < 0 or shape[1] % 8 or not 0 < shape[1] <= CONV_MAX_CHANNELS:
        _refuse("x", x, f"bfloat16 or float16 [tokens, a multiple of 8 channels up to {CONV_MAX_CHANNELS}] on a HIP device")
    tokens, channels = shape
    if activation not in _CONV_ACTIVATIONS:
        raise ValueError(f"activation must be one of {tuple(_CONV_ACTIVATIONS)}, got {activation!r}")
    if weight.dim() != 2 or weight.shape[0] != channels or weight.shape[1] not in CONV_WIDTHS or weight.get_device() != index:
        _refuse("weight", weight, f"[{channels}, a width of {CONV_WIDTHS}] on HIP device {index}")
    width = weight.shape[1]
    if (states.dtype is not dtype or states.dim() != 3 or states.shape[1:] != (width - 1, channels) or states.get_device() != index
            or not states.is_contiguous() or states.data_ptr() & 15):
        _refuse("states", states, f"contiguous 16-byte aligned {dtype} [slots, {width - 1}, {channels}] on HIP device {index}")
    if weight.dtype is not torch.float32 or not weight.is_contiguous() or weight.data_ptr() & 15:
        weight = weight.to(torch.float32, memory_format=torch.contiguous_format, copy=True)
    bias = _weight("bias", bias, channels, index)
    ts, unit = x.stride()
    if unit != 1 or ts & 7 or x.data_ptr() & 15:
        x = x.clone(memory_format=torch.contiguous_format)
        ts = x.stride(0)
    batch, slots, from_slots, query_starts = _batch(slots, from_slots, query_starts, tokens, index)
    out = torch.empty(shape, dtype=dtype, device=x.device)
    if tokens:
        with _on(index):
            _lib.check(_lib.lib().jv_causal_conv(
                x.data_ptr(), ts, weight.data_ptr(), _ptr(bias), width, _CONV_ACTIVATIONS[activation], states.data_ptr(), states.shape[0],
                slots.data_ptr(), _ptr(from_slots), _ptr(query_starts), batch, out.data_ptr(), tokens, channels, _FP16[dtype],
                torch._C._cuda_getCurrentRawStream(index)))
    return out


def _gate(name: str, t: torch.Tensor, dtype: torch.dtype, tokens: int, heads: int, index: int) -> tuple:
    """``t`` [tokens, heads] of ``dtype``: (the tensor, its address and row stride)."""
    if t.dtype is not dtype or t.shape != (tokens, heads) or t.get_device() != index:
        _refuse(name, t, f"{dtype} [{tokens}, {heads}] on HIP device {index}")
    if heads > 1 and t.stride(1) != 1:
        t = t.contiguous()
    return t, t.data_ptr(), t.stride(0)


@lru_cache(maxsize=4096)
def _workspace(tokens: int, batch: int, k_heads: int, v_heads: int, k_dim: int, v_dim: int, ragged: bool) -> int:
    size = _lib.lib().jv_linear_attention_workspace_bytes(tokens, batch, k_heads, v_heads, k_dim, v_dim, ragged)
    if size < 0:
        _lib.check(_lib.JV_ERR_VALUE)
    return size


def linear_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, decay: torch.Tensor, states: torch.Tensor, slots: torch.Tensor, *,
                     beta: torch.Tensor | None = None, rate: torch.Tensor | None = None, decay_bias: torch.Tensor | None = None,
                     from_slots: torch.Tensor | None = None, query_starts: torch.Tensor | None = None, scale: float | None = None,
                     norm_eps: float | None = None) -> torch.Tensor:
    """Linear attention of queries and keys [tokens, k_heads, k_dim] and values
    [tokens, v_heads, v_dim] (head sizes 64, 128 or 256) with a state [k_dim,
    v_dim] for each value head; a new tensor [tokens, v_heads, v_dim]. Token by
    token of a sequence, value head h with query and key head ``h // (v_heads /
    k_heads)``:

        S = exp(g) S
        u = beta (v - S^T k)        (``beta`` None: u = v)
        S = S + k u^T
        out = scale S^T q           (``scale`` defaults to k_dim ** -0.5)

    ``norm_eps``: q and k are divided by ``sqrt(sum(x^2) + norm_eps)`` first
    (the delta rule wants keys of length 1). ``decay`` and ``beta`` [tokens,
    v_heads] (both float32 or both q's type; views will do) are the log decays g
    and the betas; with ``rate`` [v_heads] they are a projection's outputs, and
    g = -rate softplus(decay + decay_bias), beta = sigmoid(beta).

    Sequence b has the tokens ``query_starts[b]`` to ``query_starts[b + 1] - 1``
    ([batch + 1], not decreasing, from 0 to tokens; None: one token each); its
    state comes from slot ``from_slots[b]`` of ``states`` (float32 [slots,
    v_heads, k_dim, v_dim], contiguous) and goes to ``slots[b]``. A sequence
    without tokens changes nothing; tokens of no sequence come out as 0.

    States, sums and norms are in 32 bits, the output is rounded once; prompts
    go in chunks of 64 tokens, so a prompt's last bits differ from those of its
    tokens one at a time, and take a workspace of 38 KB a value head and 128
    k_dim bytes a key head for each 64 tokens and each sequence. A token has no effect on those before it, whatever its
    values; an update that is not finite makes its value channel NaN from that
    token on, and in the state.
    """
    dtype, index, tokens, k_dim = _first("q", q)
    q, q_ptr, q_ts, q_hs, k_heads = _heads("q", q, dtype, index, tokens, k_dim)
    k, k_ptr, k_ts, k_hs, heads = _heads("k", k, dtype, index, tokens, k_dim)
    if v.dim() != 3 or v.shape[2] not in HEAD_DIMS:
        _refuse("v", v, f"{dtype} [{tokens}, heads, head size of {HEAD_DIMS}] on HIP device {index}")
    v_dim = v.shape[2]
    v, v_ptr, v_ts, v_hs, v_heads = _heads("v", v, dtype, index, tokens, v_dim)
    if heads != k_heads or not k_heads or not v_heads or v_heads % k_heads:
        raise ValueError(f"q and k have as many heads and v a multiple of them, got {k_heads}, {heads} and {v_heads}")
    if (states.dtype is not torch.float32 or states.dim() != 4 or states.shape[1:] != (v_heads, k_dim, v_dim)
            or states.get_device() != index or not states.is_contiguous() or states.data_ptr() & 15):
        _refuse("states", states, f"contiguous 16-byte aligned float32 [slots, {v_heads}, {k_dim}, {v_dim}] on HIP device {index}")
    gate_type = decay.dtype
    if gate_type is not torch.float32 and gate_type is not dtype:
        _refuse("decay", decay, f"float32 or {dtype} [{tokens}, {v_heads}] on HIP device {index}")
    decay, d_ptr, d_ts = _gate("decay", decay, gate_type, tokens, v_heads, index)
    b_ptr, b_ts = None, 0
    if beta is not None:
        beta, b_ptr, b_ts = _gate("beta", beta, gate_type, tokens, v_heads, index)
    if rate is None and decay_bias is not None:
        raise ValueError("a decay bias goes with the heads' rates")
    rate, decay_bias = _weight("rate", rate, v_heads, index), _weight("decay_bias", decay_bias, v_heads, index)
    if norm_eps is not None and not norm_eps >= _TINY:  # a smaller one would be none in 32 bits
        raise ValueError(f"norm_eps is at least {_TINY}, got {norm_eps}")
    batch, slots, from_slots, query_starts = _batch(slots, from_slots, query_starts, tokens, index)
    out = torch.empty(tokens, v_heads, v_dim, dtype=dtype, device=q.device)
    if tokens:
        size = _workspace(tokens, batch, k_heads, v_heads, k_dim, v_dim, query_starts is not None)
        ws = torch.empty(size, dtype=torch.uint8, device=q.device) if size else None
        with _on(index):
            _lib.check(_lib.lib().jv_linear_attention(
                q_ptr, q_ts, q_hs, k_ptr, k_ts, k_hs, v_ptr, v_ts, v_hs, d_ptr, d_ts, b_ptr, b_ts, gate_type is not torch.float32,
                _ptr(rate), _ptr(decay_bias), norm_eps or 0.0, states.data_ptr(), states.shape[0], slots.data_ptr(), _ptr(from_slots),
                _ptr(query_starts), batch, k_dim ** -0.5 if scale is None else scale, out.data_ptr(), tokens, k_heads, v_heads, k_dim,
                v_dim, _FP16[dtype], _ptr(ws), size, torch._C._cuda_getCurrentRawStream(index)))
    return out


class FP8LinearAttention(nn.Module):
    """A layer's linear attention block over FP8 projections, as the reference's
    ``GatedDeltaNet`` has it (``model/model.py:442-517``): the merged q/k/v/z
    projection (``FP8Linear.concatenated``, rows of all query heads, then keys,
    values, gates z), the small 16-bit projection of decays and betas
    (``gates`` [2 v_heads, hidden]: decay rows, then beta rows), the convolution
    of q, k and v, the linear attention with keys of length 1, the gated norm
    straight to the out projection's codes, and the out projection (called as a
    module, with 16-bit input, where it has hooks)."""

    def __init__(self, qkvz: FP8Linear, gates: torch.Tensor, out: FP8Linear, k_heads: int, v_heads: int, k_dim: int, v_dim: int,
                 conv_weight: torch.Tensor, rate: torch.Tensor, decay_bias: torch.Tensor, norm_weight: torch.Tensor, eps: float = 1e-6):
        super().__init__()
        channels = 2 * k_heads * k_dim + v_heads * v_dim
        # what a call would refuse is refused here
        if k_heads < 1 or v_heads < 1 or v_heads % k_heads or k_dim not in HEAD_DIMS or v_dim not in HEAD_DIMS:
            raise ValueError(f"{v_heads} value heads of {v_dim} do not go with {k_heads} key heads of {k_dim}")
        if qkvz.out_features != channels + v_heads * v_dim or out.in_features != v_heads * v_dim:
            raise ValueError(f"the projections have {qkvz.out_features} outputs and {out.in_features} inputs, the heads "
                             f"{channels + v_heads * v_dim} and {v_heads * v_dim}")
        if gates.shape != (2 * v_heads, qkvz.in_features) or conv_weight.dim() != 2 or conv_weight.shape[0] != channels \
                or conv_weight.shape[1] not in CONV_WIDTHS:
            raise ValueError(f"gates must be [{2 * v_heads}, {qkvz.in_features}] and conv_weight [{channels}, a width of {CONV_WIDTHS}], "
                             f"got {tuple(gates.shape)} and {tuple(conv_weight.shape)}")
        if channels > CONV_MAX_CHANNELS or v_heads * v_dim > QUANT_MAX_PACKED_COLS:
            raise ValueError(f"q, k and v may have {CONV_MAX_CHANNELS} channels and the output {QUANT_MAX_PACKED_COLS}, got {channels} "
                             f"and {v_heads * v_dim}")
        for name, w, n in (("rate", rate, v_heads), ("decay_bias", decay_bias, v_heads), ("norm_weight", norm_weight, v_dim)):
            if w.shape != (n,):
                raise ValueError(f"{name} must be [{n}], got {tuple(w.shape)}")
        if not _TINY <= eps < float("inf"):
            raise ValueError(f"eps is at least {_TINY}, got {eps}")
        self.qkvz, self.out = qkvz, out
        self.k_heads, self.v_heads, self.k_dim, self.v_dim, self.channels, self.eps = k_heads, v_heads, k_dim, v_dim, channels, eps
        self.register_buffer("gates", gates.detach().to(torch.bfloat16))
        for name, w in (("conv_weight", conv_weight), ("rate", rate), ("decay_bias", decay_bias), ("norm_weight", norm_weight)):
            self.register_buffer(name, w.detach().to(torch.float32))

    def allocate(self, slots: int) -> tuple[torch.Tensor, torch.Tensor]:
        """(conv_states, states) of ``slots`` slots for this layer, zeros."""
        device = self.qkvz.weight.device
        return (torch.zeros(slots, self.conv_weight.shape[1] - 1, self.channels, dtype=torch.bfloat16, device=device),
                torch.zeros(slots, self.v_heads, self.k_dim, self.v_dim, dtype=torch.float32, device=device))

    @torch.no_grad()
    def warm(self) -> None:
        """Runs what the block does around its FP8 linears, keeping nothing, so
        that kernels load and the library of the small projection is set up
        before graph capture: that projection and the out projection of codes
        at ``WARM_ROWS``, single tokens, and prompts in batches that reach
        each form of the linear attention, with the norm's codes and without."""
        device, columns = self.qkvz.weight.device, self.v_heads * self.v_dim // 16
        conv_states, states = self.allocate(1)
        for rows in WARM_ROWS:
            nn.functional.linear(torch.zeros(rows, self.qkvz.in_features, dtype=torch.bfloat16, device=device), self.gates)
            if self.out.takes_codes():
                z = torch.zeros(rows, self.v_heads, self.v_dim, dtype=torch.bfloat16, device=device)
                self.out.forward_codes(*gated_norm(z, z, self.norm_weight, eps=self.eps, quantize="packed"), packed_rows=rows)
        # the form goes by the state columns of a batch, 16 a workgroup, to the compute units
        units = sm_count(device)
        for sequences in (0, 1, units // columns + 1, 2 * units // columns + 1):
            tokens, starts = 1, None
            if sequences:
                tokens, starts = 2, torch.full((sequences + 1,), 2, dtype=torch.int32, device=device)
                starts[0] = 0
            none = torch.full((max(sequences, 1),), -1, dtype=torch.int32, device=device)
            proj = torch.zeros(tokens, self.qkvz.out_features, dtype=torch.bfloat16, device=device)
            gates = torch.zeros(tokens, 2 * self.v_heads, dtype=torch.bfloat16, device=device)
            for codes in {False, self.out.takes_codes()}:
                self._between(proj, gates, conv_states, states, none, none, starts, codes)

    def _codes(self) -> bool:
        """Whether the out projection is given codes: not where its call is more than
        its forward, as with hooks, which see its 16-bit input."""
        out, every = self.out, nn.modules.module
        return out.takes_codes() and not (
            out._forward_pre_hooks or out._forward_hooks or out._backward_pre_hooks or out._backward_hooks or every._global_forward_pre_hooks
            or every._global_forward_hooks or every._global_backward_pre_hooks or every._global_backward_hooks
            or getattr(out.forward, "__func__", None) is not FP8Linear.forward)

    def _between(self, proj: torch.Tensor, gates: torch.Tensor, conv_states: torch.Tensor, states: torch.Tensor, slots: torch.Tensor,
                 from_slots: torch.Tensor | None, query_starts: torch.Tensor | None,
                 codes: bool) -> tuple[torch.Tensor | None, tuple | None]:
        """(the out projection's input, None), or (None, its packed codes and scales)."""
        tokens, hk, hv, dk, dv = proj.shape[0], self.k_heads, self.v_heads, self.k_dim, self.v_dim
        mixed = causal_conv(proj[:, :self.channels], self.conv_weight, conv_states, slots, from_slots=from_slots, query_starts=query_starts)
        q, k, v = mixed.split([hk * dk, hk * dk, hv * dv], 1)
        y = linear_attention(q.view(tokens, hk, dk), k.view(tokens, hk, dk), v.view(tokens, hv, dv), gates[:, :hv], states, slots,
                             beta=gates[:, hv:], rate=self.rate, decay_bias=self.decay_bias, from_slots=from_slots,
                             query_starts=query_starts, norm_eps=self.eps)
        z = proj[:, self.channels:].view(tokens, hv, dv)
        if codes:
            return None, gated_norm(y, z, self.norm_weight, eps=self.eps, quantize="packed")
        return gated_norm(y, z, self.norm_weight, eps=self.eps).view(tokens, hv * dv), None

    def forward(self, x: torch.Tensor, conv_states: torch.Tensor, states: torch.Tensor, slots: torch.Tensor, *,
                from_slots: torch.Tensor | None = None, query_starts: torch.Tensor | None = None) -> torch.Tensor:
        """x [tokens, hidden] -> [tokens, hidden]; ``conv_states`` and
        ``states`` (``allocate``) are updated in place. The other arguments are
        ``linear_attention``'s."""
        if not x.shape[0]:
            return self.out(x.new_zeros(0, self.out.in_features))
        gates = nn.functional.linear(x.to(torch.bfloat16), self.gates)
        y, codes = self._between(self.qkvz(x), gates, conv_states, states, slots, from_slots, query_starts, self._codes())
        return self.out(y) if codes is None else self.out.forward_codes(*codes, packed_rows=x.shape[0])
