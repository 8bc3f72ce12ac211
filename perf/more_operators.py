"""What lies between the FP8 projections of a layer whose attention is linear, as measurable cases: the short causal
convolution of q, k and v, the linear attention with a decay for each head (with the delta rule's correction and without),
its gated norm, and the residual add with the norms around a block, whose output the next FP8 projection takes as codes.

Head layouts follow the projections of the 9B shapes (8192 channels of q, k and v: 16 key heads and 32 value heads of 128;
hidden size 4096); batch sizes and ragged lengths are bench.py's (decode 1-64 rows, prompts of 64-2048 tokens); the
longer prompts and the other layouts are generic.

A case is one of these kinds:

conv        causal_conv over a batch of sequences whose last inputs are kept in slots
linear      linear_attention: prompts, or one token for each sequence ("len_hi" 1), from one set of state slots into another
add_norm    add_norm: residual + scale * act(gate) * norm(x), and the norm of that, with "codes" as e4m3 codes too
gated_norm  gated_norm: per-head norm times act(gate), with "codes" as the e4m3 codes of the token's row
layer_step  causal_conv, linear_attention and gated_norm one after the other: what a decode step runs in such a layer

Lengths of a batch are drawn from the case's own "mix", evenly over their logarithm, so that a case is the same batch
whatever the seed of its values.
"""

import math
import random

import torch

own = False

EPS = 1e-6
FP8 = torch.float8_e4m3fn
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
CHUNK = 64


def listed():
    heads = {"k_heads": 16, "v_heads": 32, "k_dim": 128, "v_dim": 128}
    return [
        # one new token of every sequence of a decode batch, its oldest inputs in the state
        {"name": "conv_step_b48", "kind": "conv", "batch": 48, "len_lo": 1, "len_hi": 1, "channels": 8192, "width": 4, "bias": False,
         "act": "silu", "fresh": 0, "dtype": "bf16", "mix": 1},
        # packed prompts of uneven lengths, some of them new, some going on from a state
        {"name": "conv_prompts_b16", "kind": "conv", "batch": 16, "len_lo": 64, "len_hi": 2048, "channels": 8192, "width": 4,
         "bias": False, "act": "silu", "fresh": 2, "dtype": "bf16", "mix": 2},
        # the next token of one sequence: the smallest call
        {"name": "step_b1", "kind": "linear", "batch": 1, "len_lo": 1, "len_hi": 1, **heads, "beta": True, "raw": True, "fresh": 0,
         "dtype": "bf16", "mix": 3},
        # a full decode batch: every sequence's state read and written
        {"name": "step_b64", "kind": "linear", "batch": 64, "len_lo": 1, "len_hi": 1, **heads, "beta": True, "raw": True, "fresh": 0,
         "dtype": "bf16", "mix": 4},
        # one short question, its state new
        {"name": "prompt_301", "kind": "linear", "batch": 1, "len_lo": 301, "len_hi": 301, **heads, "beta": True, "raw": True,
         "fresh": 1, "dtype": "bf16", "mix": 5},
        # packed prompts of uneven lengths, every other one behind a prefix whose state is there
        {"name": "prompts_b16", "kind": "linear", "batch": 16, "len_lo": 64, "len_hi": 2048, **heads, "beta": True, "raw": True,
         "fresh": 2, "dtype": "bf16", "mix": 6},
        # one long document: the largest call
        {"name": "prompt_16384", "kind": "linear", "batch": 1, "len_lo": 16384, "len_hi": 16384, **heads, "beta": True, "raw": True,
         "fresh": 1, "dtype": "bf16", "mix": 7},
        # decays given as they are, no correction, small heads, the other 16-bit type
        {"name": "decay_b7_d64_fp16", "kind": "linear", "batch": 7, "len_lo": 5, "len_hi": 999, "k_heads": 8, "v_heads": 16,
         "k_dim": 64, "v_dim": 64, "beta": False, "raw": False, "fresh": 3, "dtype": "fp16", "mix": 8},
        # around a block of a one-token step: the next projection's codes in the same call
        {"name": "add_norm_t1_codes", "kind": "add_norm", "tokens": 1, "cols": 4096, "post": False, "gate": "", "scale": 1.0,
         "codes": True, "dtype": "bf16"},
        # a long prompt, norms on both sides of the block, a gate and a residual scale
        {"name": "add_norm_t8192_post_gate", "kind": "add_norm", "tokens": 8192, "cols": 4096, "post": True, "gate": "sigmoid",
         "scale": 0.5, "codes": False, "dtype": "bf16"},
        # the linear attention's output norm over packed prompts, straight to the out projection's codes
        {"name": "gated_norm_t4099_codes", "kind": "gated_norm", "tokens": 4099, "heads": 32, "dim": 128, "act": "silu", "norm": True,
         "codes": True, "dtype": "bf16"},
        # a layer's share of a decode step
        {"name": "layer_step_b32", "kind": "layer_step", "batch": 32, "len_lo": 1, "len_hi": 1, **heads, "width": 4, "beta": True,
         "raw": True, "fresh": 0, "dtype": "bf16", "mix": 9},
    ]


def _between(rng, lo, hi):
    """A whole number from lo to hi, even over its logarithm."""
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choice(["conv", "linear", "linear", "linear", "linear", "add_norm", "add_norm", "gated_norm", "layer_step"])
    case = {"kind": kind, "dtype": rng.choice(["bf16", "bf16", "bf16", "fp16"])}
    if kind in ("conv", "linear", "layer_step"):
        case["mix"] = rng.randrange(1 << 30)
        case["fresh"] = rng.choice([0, 1, 2, 3])
        if kind == "layer_step" or rng.random() < 0.4:
            case.update(batch=_between(rng, 1, 128), len_lo=1, len_hi=1)
        else:
            batch = _between(rng, 1, 48)
            len_hi = _between(rng, 2, max(3, 16384 // batch))
            case.update(batch=batch, len_lo=max(1, len_hi // rng.choice([1, 4, 32])), len_hi=len_hi)
    if kind in ("linear", "layer_step"):
        k_heads, v_heads, k_dim, v_dim = rng.choice([(16, 32, 128, 128), (16, 32, 128, 128), (16, 16, 128, 128), (10, 20, 64, 128),
                                                     (5, 5, 256, 256), (5, 10, 128, 64), (14, 14, 64, 64), (7, 7, 128, 256)])
        case.update(k_heads=k_heads, v_heads=v_heads, k_dim=k_dim, v_dim=v_dim, beta=rng.random() < 0.75, raw=rng.random() < 0.75)
    if kind == "conv":
        case.update(channels=8 * _between(rng, 8, 1536), width=rng.choice([2, 3, 4, 4]), bias=rng.random() < 0.5,
                    act=rng.choice(["silu", "silu", ""]))
    elif kind == "layer_step":
        case["width"] = rng.choice([3, 4, 4])
    elif kind == "add_norm":
        case.update(tokens=_between(rng, 1, 8192), cols=128 * _between(rng, 1, 64), post=rng.random() < 0.5,
                    gate=rng.choice(["", "", "sigmoid", "silu"]), scale=rng.choice([1.0, 1.0, 0.25]), codes=rng.random() < 0.5)
    elif kind == "gated_norm":
        case.update(tokens=_between(rng, 1, 8192), heads=rng.choice([4, 16, 32, 32, 40]), dim=rng.choice([64, 128, 128, 256]),
                    act=rng.choice(["silu", "silu", "sigmoid"]), norm=rng.random() < 0.8, codes=rng.random() < 0.5)
    return case


def _lengths(case):
    rng = random.Random(case["mix"])
    return [_between(rng, case["len_lo"], case["len_hi"]) for _ in range(case["batch"])]


def _inputs(case, seed):
    """The tensors of a case, from the seed alone."""
    g = torch.Generator("cuda").manual_seed(seed)
    dtype, kind = DTYPES[case["dtype"]], case["kind"]
    s = {}

    def randn(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    if kind == "add_norm":
        tokens, cols = case["tokens"], case["cols"]
        spread = randn(cols).mul_(0.7).exp_()  # some channels run larger than others, as a trained model's do
        s["x"] = (randn(tokens, cols) * spread).to(dtype)
        s["residual"] = (randn(tokens, cols) * 3 * spread).to(dtype)
        s["weight"] = 1 + 0.2 * randn(cols)
        s["post_weight"] = 1 + 0.2 * randn(cols) if case["post"] else None
        s["gate"] = randn(tokens, cols).to(dtype) if case["gate"] else None
        return s
    if kind == "gated_norm":
        tokens, heads, dim = case["tokens"], case["heads"], case["dim"]
        s["x"] = (randn(tokens, heads, dim) * 0.1).to(dtype)
        # the gate is part of a merged projection's output
        s["gate"] = randn(tokens, 2 * heads * dim).to(dtype)[:, heads * dim:].view(tokens, heads, dim)
        s["norm_weight"] = 1 + 0.2 * randn(dim) if case["norm"] else None
        return s
    lengths = _lengths(case)
    batch, tokens = len(lengths), sum(lengths)
    s["query_starts"] = None
    if case["len_hi"] > 1:
        starts = [0]
        for n in lengths:
            starts.append(starts[-1] + n)
        s["query_starts"] = torch.tensor(starts, dtype=torch.int32, device="cuda")
    # the slots that states come from and go to: every "fresh"-th sequence is new and starts from nothing
    order = torch.randperm(2 * batch + 1, generator=g, device="cuda").to(torch.int32)
    s["slots"], s["from_slots"] = order[:batch].contiguous(), order[batch:2 * batch].contiguous()
    if case["fresh"]:
        s["from_slots"][::case["fresh"]] = -1
    if kind != "conv":
        hk, hv, dk, dv = case["k_heads"], case["v_heads"], case["k_dim"], case["v_dim"]
        channels, gate = 2 * hk * dk + hv * dv, hv * dv
        s["states"] = randn(2 * batch + 1, hv, dk, dv) * (0.3 if case["raw"] else 3.0)
        if case["raw"]:
            # decay and beta as a small projection gives them, side by side
            ab = randn(tokens, 2 * hv).to(dtype)
            s["decay"] = ab[:, :hv]
            s["beta"] = ab[:, hv:] if case["beta"] else None
            s["rate"] = 1 + 15 * torch.rand(hv, generator=g, device="cuda")
            s["decay_bias"] = torch.rand(hv, generator=g, device="cuda") * 4 - 6.5
        else:
            # one rate a head, from long memories to short ones
            rates = 2.0 ** -torch.linspace(1, 9, hv, device="cuda")
            s["decay"] = (-rates).expand(tokens, hv).contiguous()
            s["beta"] = torch.rand(tokens, hv, generator=g, device="cuda") if case["beta"] else None
            s["rate"] = s["decay_bias"] = None
    else:
        channels, gate = case["channels"], 0
    if kind != "linear":
        width = case["width"]
        s["conv_states"] = randn(2 * batch + 1, width - 1, channels).to(dtype)
        s["conv_weight"] = randn(channels, width) * 0.5
        s["conv_bias"] = randn(channels) * 0.1 if case.get("bias") else None
    # what the convolution takes is a part of a merged projection's output, what the linear attention takes is the convolution's
    if kind == "linear":
        mixed = torch.nn.functional.silu(randn(tokens, channels)).to(dtype)
    else:
        merged = randn(tokens, channels + max(gate, 64)).to(dtype)
        mixed = s["x"] = merged[:, :channels]
        if gate:
            s["gate"] = merged[:, channels:].view(tokens, hv, dv)
            s["norm_weight"] = 1 + 0.2 * randn(dv)
    if kind != "conv":
        s["mixed"] = mixed
    return s


@torch.no_grad()
def prepare(case, seed):
    state = _inputs(case, seed)
    state["case"] = case
    return state


def _heads_of(mixed, case):
    """q, k and v of the convolution's output."""
    hk, hv, dk, dv = case["k_heads"], case["v_heads"], case["k_dim"], case["v_dim"]
    q, k, v = mixed.split([hk * dk, hk * dk, hv * dv], 1)
    return q.unflatten(1, (hk, dk)), k.unflatten(1, (hk, dk)), v.unflatten(1, (hv, dv))


def _norm_eps(case):
    """q and k are divided by their lengths where a correction is, or the decays come from the tokens."""
    return EPS if case["beta"] or case["raw"] else None


def _run_own(s):
    from jeeves_amd import add_norm, causal_conv, gated_norm, linear_attention

    case, kind = s["case"], s["case"]["kind"]
    if kind == "add_norm":
        out = add_norm(s["x"], s["residual"], s["weight"], post_weight=s["post_weight"], gate=s["gate"], activation=case["gate"] or None,
                       scale=case["scale"], eps=EPS, quantize="rows" if case["codes"] else None)
        return [t for t in out if t is not None]
    if kind == "gated_norm":
        out = gated_norm(s["x"], s["gate"], s["norm_weight"], activation=case["act"], eps=EPS, quantize="rows" if case["codes"] else None)
        return list(out) if case["codes"] else [out]
    outs = []
    if kind != "linear":
        mixed = causal_conv(s["x"], s["conv_weight"], s["conv_states"], s["slots"], bias=s["conv_bias"], from_slots=s["from_slots"],
                            query_starts=s["query_starts"], activation=case.get("act", "silu") or None)
        outs = [mixed, s["conv_states"]]
        if kind == "conv":
            return outs
    else:
        mixed = s["mixed"]
    q, k, v = _heads_of(mixed, case)
    y = linear_attention(q, k, v, s["decay"], s["states"], s["slots"], beta=s["beta"], rate=s["rate"], decay_bias=s["decay_bias"],
                         from_slots=s["from_slots"], query_starts=s["query_starts"], norm_eps=_norm_eps(case))
    outs += [y, s["states"]]
    if kind == "layer_step":
        outs.append(gated_norm(y, s["gate"], s["norm_weight"], activation="silu", eps=EPS))
    return outs


def _act(x, name):
    return x * torch.sigmoid(x) if name == "silu" else torch.sigmoid(x) if name == "sigmoid" else x


def _rms(x, weight):
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * weight


def _codes(y):
    """e4m3 codes of the rows and their scales."""
    scale = y.abs().amax(-1).clamp(min=1e-12) * (1 / 448)
    return (y / scale[:, None]).to(FP8), scale


def _plain_norm(s):
    case, x = s["case"], s["x"].float()
    if case["kind"] == "add_norm":
        if case["post"]:
            x = _rms(x, s["post_weight"])
        if case["gate"]:
            x = x * _act(s["gate"].float(), case["gate"])
        h = s["residual"].float() + case["scale"] * x
        y = _rms(h, s["weight"])
        outs = [h, y]
    else:
        y = _rms(x, s["norm_weight"]) if s["norm_weight"] is not None else x
        y = y * _act(s["gate"].float(), case.get("act", "silu"))
        outs = [] if case.get("codes") else [y]
    outs = [t.to(s["x"].dtype) for t in outs]
    return outs + list(_codes(y.flatten(1))) if case.get("codes") else outs


def _spans(s, tokens):
    """Each token's sequence, each sequence's first token and length."""
    starts = s["query_starts"]
    if starts is None:
        at = torch.arange(tokens, device="cuda")
        return at, at, torch.ones_like(at)
    starts = starts.long()
    lengths = starts[1:] - starts[:-1]
    return torch.repeat_interleave(torch.arange(len(lengths), device="cuda"), lengths, output_size=tokens), starts[:-1], lengths


def _old_states(states, from_slots):
    """The states that the sequences start from, 0 for the new ones."""
    old = states[from_slots.clamp(min=0).long()].float()
    return old.masked_fill((from_slots < 0).view(-1, *[1] * (old.dim() - 1)), 0.0)


def _plain_conv(s):
    case, x, weight = s["case"], s["x"], s["conv_weight"]
    tokens, width = x.shape[0], case["width"]
    seq, first, lengths = _spans(s, tokens)
    old = _old_states(s["conv_states"], s["from_slots"])
    place = torch.arange(tokens, device="cuda") - first[seq]
    y = torch.zeros(x.shape, device="cuda") if s["conv_bias"] is None else s["conv_bias"].expand(x.shape)
    for j in range(width):
        back = width - 1 - j
        tap = x[(torch.arange(tokens, device="cuda") - back).clamp(min=0)].float()
        before = (place < back).nonzero()[:, 0]
        tap[before] = old[seq[before], (place + j)[before]]
        y = y + tap * weight[:, j]
    last = (lengths[:, None] + torch.arange(width - 1, device="cuda")) - (width - 1)
    inputs = x[(first[:, None] + last).clamp(min=0)].float()
    kept = old.gather(1, (last + width - 1).clamp(max=width - 2)[:, :, None].expand(old.shape))
    s["conv_states"][s["slots"].long()] = torch.where(last[:, :, None] < 0, kept, inputs).to(x.dtype)
    return _act(y, case.get("act", "silu")).to(x.dtype)


def _unit(x, eps):
    return x if eps is None else x * torch.rsqrt((x * x).sum(-1, keepdim=True) + eps)


def _gates(s):
    """Log decays and betas in 32 bits."""
    decay, beta = s["decay"].float(), s["beta"]
    if s["rate"] is not None:
        z = decay + s["decay_bias"]
        decay = -s["rate"] * (z.clamp(min=0) + torch.log1p(torch.exp(-z.abs())))
        beta = None if beta is None else torch.sigmoid(beta.float())
    return decay, beta


def _plain_linear(s, mixed):
    """Chunks of up to 64 tokens, all sequences and heads at a time, the sequences padded to the longest."""
    case = s["case"]
    hk, hv, dk, dv = case["k_heads"], case["v_heads"], case["k_dim"], case["v_dim"]
    tokens = mixed.shape[0]
    seq, first, lengths = _spans(s, tokens)
    batch, longest = len(lengths), case["len_hi"]
    size = min(CHUNK, longest)
    chunks = -(-longest // size)
    place = torch.arange(chunks * size, device="cuda")
    token = (first[:, None] + place).clamp(max=tokens - 1)
    real = place < lengths[:, None]

    def laid_out(x):
        """[tokens, heads, ...] -> [batch, value heads, chunks, size, ...], 0 behind a sequence's end"""
        x = x[token].masked_fill(~real.view(*real.shape, *[1] * (x.dim() - 1)), 0.0)
        x = x.transpose(1, 2).unflatten(2, (chunks, size))
        return x.repeat_interleave(hv // x.shape[1], 1) if x.shape[1] != hv else x

    q, k, v = _heads_of(mixed, case)
    eps = _norm_eps(case)
    q, k, v = laid_out(_unit(q.float(), eps) * dk ** -0.5), laid_out(_unit(k.float(), eps)), laid_out(v.float())
    decay, beta = _gates(s)
    # sums of decays lose their small ones in 32 bits
    total = laid_out(decay.double()).cumsum(-1)
    lower = torch.ones(size, size, dtype=torch.bool, device="cuda").tril()
    between = (total[..., :, None] - total[..., None, :]).masked_fill(~lower, -math.inf).exp().float()
    to_end, total = (total[..., -1:] - total).exp().float(), total.exp().float()
    within = (q @ k.transpose(-1, -2)) * between
    if beta is not None:
        beta = laid_out(beta)
        pull = (beta[..., None] * between * (k @ k.transpose(-1, -2))).tril(-1)
        solve = torch.eye(size, device="cuda").expand(pull.shape).clone()
        for i in range(1, size):
            solve[..., i, :i] = -(pull[..., i, :i, None] * solve[..., :i, :i]).sum(-2)
    state = _old_states(s["states"], s["from_slots"])
    out = torch.empty(batch, hv, chunks, size, dv, device="cuda")
    for n in range(chunks):
        new = v[:, :, n]
        grown = total[:, :, n, :, None]
        if beta is not None:
            new = solve[:, :, n] @ (beta[:, :, n, :, None] * (new - (k[:, :, n] * grown) @ state))
        out[:, :, n] = (q[:, :, n] * grown) @ state + within[:, :, n] @ new
        state = state * total[:, :, n, -1, None, None] + (k[:, :, n] * to_end[:, :, n, :, None]).transpose(-1, -2) @ new
    s["states"][s["slots"].long()] = state
    return out.flatten(2, 3).transpose(1, 2)[real].to(mixed.dtype)


def _run_plain(s):
    kind = s["case"]["kind"]
    if kind in ("add_norm", "gated_norm"):
        return _plain_norm(s)
    outs = []
    if kind != "linear":
        mixed = _plain_conv(s)
        outs = [mixed, s["conv_states"]]
        if kind == "conv":
            return outs
    else:
        mixed = s["mixed"]
    y = _plain_linear(s, mixed)
    outs += [y, s["states"]]
    if kind == "layer_step":
        outs += _plain_norm({**s, "x": y})
    return outs


@torch.no_grad()
def run(state):
    return _run_own(state) if own else _run_plain(state)


def work(case):
    """Inputs read once and outputs written once, states that a sequence starts from and ends with among them; the products
    with the state, token by token, as the recurrence has them."""
    kind = case["kind"]
    total = flops = 0
    if kind == "add_norm":
        n = case["tokens"] * case["cols"]
        total = 2 * n * (4 + bool(case["gate"])) + (n + 4 * case["tokens"] if case["codes"] else 0)
        flops = 10 * n
    elif kind == "gated_norm":
        n = case["tokens"] * case["heads"] * case["dim"]
        total = 2 * n * 2 + (n + 4 * case["tokens"] if case["codes"] else 2 * n)
        flops = 8 * n
    if kind in ("add_norm", "gated_norm"):
        return {"bytes": total, "flops": flops}
    lengths = _lengths(case)
    tokens, batch = sum(lengths), len(lengths)
    old = batch - (-(-batch // case["fresh"]) if case["fresh"] else 0)
    if kind != "linear":
        channels = case["channels"] if kind == "conv" else 2 * case["k_heads"] * case["k_dim"] + case["v_heads"] * case["v_dim"]
        total += 4 * tokens * channels + 2 * (batch + old) * (case["width"] - 1) * channels + 4 * channels * case["width"]
        flops += 2 * tokens * channels * case["width"]
    if kind != "conv":
        hk, hv, dk, dv = case["k_heads"], case["v_heads"], case["k_dim"], case["v_dim"]
        total += 2 * tokens * (2 * hk * dk + 2 * hv * dv) + (2 if case["raw"] else 4) * tokens * hv * (1 + case["beta"])
        total += 4 * (batch + old) * hv * dk * dv
        flops += (6 if case["beta"] else 4) * tokens * hv * dk * dv
    if kind == "layer_step":
        total += 2 * 3 * tokens * hv * dv
        flops += 8 * tokens * hv * dv
    return {"bytes": total, "flops": flops}


def _exact_norm(s, case, x):
    def normed(t, w):
        return t / (t.square().sum(-1, keepdim=True) / t.shape[-1] + EPS).sqrt() * w.double()

    def gated(t, name):
        z = s["gate"].double()
        return t / (1 + torch.exp(-z)) * (z if name == "silu" else 1.0)

    if case["kind"] == "add_norm":
        b = normed(x, s["post_weight"]) if case["post"] else x
        h = s["residual"].double() + case["scale"] * (gated(b, case["gate"]) if case["gate"] else b)
        y = normed(h, s["weight"])
        outs = [h, y]
    else:
        y = gated(x if s["norm_weight"] is None else normed(x, s["norm_weight"]), case.get("act", "silu"))
        outs = [] if case.get("codes") else [y]
    if case.get("codes"):
        # codes stand for what their rounding takes in
        rows = y.flatten(1)
        scale = rows.abs().amax(1) / 448
        outs += [rows / scale[:, None], scale]
    return outs


def _exact_conv(s, case, lengths):
    """One sequence after the other, behind the inputs that its state holds."""
    width, states, ys, at = case["width"], s["conv_states"].double(), [], 0
    for n, slot, source in zip(lengths, s["slots"].tolist(), s["from_slots"].tolist()):
        before = s["conv_states"][source].double() if source >= 0 else torch.zeros_like(states[0])
        row = torch.cat([before, s["x"][at:at + n].double()])
        y = sum(row[j:j + n] * s["conv_weight"][:, j].double() for j in range(width))
        if s["conv_bias"] is not None:
            y = y + s["conv_bias"].double()
        ys.append(y / (1 + torch.exp(-y)) if case.get("act", "silu") else y)
        states[slot] = row[n:]
        at += n
    return torch.cat(ys), states


def _exact_linear(s, case, lengths, mixed):
    """The recurrence, token by token, all sequences that still have one at a time, the longest first."""
    hk, hv, dk, dv = case["k_heads"], case["v_heads"], case["k_dim"], case["v_dim"]
    q, k, v = (t.double() for t in _heads_of(mixed, case))
    if _norm_eps(case) is not None:
        q, k = (t / (t.square().sum(-1, keepdim=True) + EPS).sqrt() for t in (q, k))
    q, k = (t.repeat_interleave(hv // hk, 1) for t in (q / math.sqrt(dk), k))
    decay, beta = s["decay"].double(), None if s["beta"] is None else s["beta"].double()
    if s["rate"] is not None:
        z = decay + s["decay_bias"].double()
        decay = -s["rate"].double() * torch.logaddexp(z, torch.zeros_like(z))
        beta = None if beta is None else 1 / (1 + torch.exp(-beta))
    keep = decay.exp()
    order = sorted(range(len(lengths)), key=lambda b: -lengths[b])
    firsts = [0]
    for n in lengths:
        firsts.append(firsts[-1] + n)
    first = torch.tensor([firsts[b] for b in order], device="cuda")
    source = s["from_slots"].long()[torch.tensor(order, device="cuda")]
    S = s["states"][source.clamp(min=0)].double() * (source >= 0)[:, None, None, None]
    out, states = torch.empty(mixed.shape[0], hv, dv, dtype=torch.float64, device="cuda"), s["states"].double()
    live = len(order)
    for i in range(max(lengths)):
        while lengths[order[live - 1]] <= i:
            live -= 1
        t = first[:live] + i
        now = S[:live]
        now *= keep[t][:, :, None, None]
        value = v[t]
        if beta is not None:
            value = beta[t][:, :, None] * (value - (now * k[t][..., None]).sum(2))
        now += k[t][..., None] * value[:, :, None]
        out[t] = (now * q[t][..., None]).sum(2)
    states[s["slots"].long()[torch.tensor(order, device="cuda")]] = S
    return out, states


@torch.no_grad()
def exact(case, seed):
    s = _inputs(case, seed)
    kind = case["kind"]
    if kind in ("add_norm", "gated_norm"):
        return _exact_norm(s, case, s["x"].double())
    lengths, outs = _lengths(case), []
    dtype = DTYPES[case["dtype"]]
    if kind != "linear":
        mixed, states = _exact_conv(s, case, lengths)
        outs = [mixed, states]
        if kind == "conv":
            return outs
        # each operator's inputs are what the one before it stored: 16-bit values
        mixed = mixed.to(dtype)
    else:
        mixed = s["mixed"]
    y, states = _exact_linear(s, case, lengths, mixed)
    outs += [y, states]
    if kind == "layer_step":
        outs += _exact_norm(s, case, y.to(dtype).double())
    return outs
