"""What lies between the merged q/k/v projection and the o projection of a served model, as measurable cases: the norms
and the rotation of queries and keys, the append to a paged cache, and the attention that reads the cache for a batch
whose sequences may share a prefix.

Head layouts are those of the 9B projections of jeeves_amd/synthetic.py (q 4096 and k/v 1024 channels: 32 and 8 heads of
128, or 16 and 4 heads of 256); the batch sizes and the ragged lengths are bench.py's (decode 1-64 rows, prompts of
64-2048 tokens); the longer caches, pages and prefixes are generic.

A case is one of these kinds:

norm_rope  qk_norm_rope: per-head RMS norms and the rotation of q and k, both views of one merged projection
append     append_kv: keys normed, rotated and written to their pages with the values; with "with_q" the queries are
           normed and rotated by the same call
attention  paged_attention over a batch of sequences with their own pages and, with "prefix", a prefix that all share
step       append_kv with the queries, then paged_attention: what a decode step runs in every layer

Lengths of a batch are drawn from the case's own "mix", evenly over their logarithm, so that a case is the same batch
whatever the seed of its values.
"""

import math
import random

import torch

own = False

EPS = 1e-6
ROPE_BASE = 10000.0
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def listed():
    return [
        # one new token of one sequence: the smallest call
        {"name": "norm_rope_t1", "kind": "norm_rope", "tokens": 1, "q_heads": 32, "kv_heads": 8, "dim": 128, "rotary": 128,
         "norm": True, "dtype": "bf16"},
        # packed prompts of uneven lengths
        {"name": "norm_rope_t7921", "kind": "norm_rope", "tokens": 7921, "q_heads": 32, "kv_heads": 8, "dim": 128, "rotary": 128,
         "norm": True, "dtype": "bf16"},
        # wide heads, a quarter of the channels rotated, the other 16-bit type
        {"name": "norm_rope_t777_d256_fp16", "kind": "norm_rope", "tokens": 777, "q_heads": 16, "kv_heads": 4, "dim": 256,
         "rotary": 64, "norm": True, "dtype": "fp16"},
        # a full decode batch, all that lies between projection and attention in one call
        {"name": "append_t64", "kind": "append", "tokens": 64, "q_heads": 32, "kv_heads": 8, "dim": 128, "rotary": 128,
         "norm": True, "with_q": True, "page": 16, "pages": 1024, "padded": 3, "dtype": "bf16"},
        # a prompt taken into the cache
        {"name": "append_t4096_d256", "kind": "append", "tokens": 4096, "q_heads": 16, "kv_heads": 4, "dim": 256, "rotary": 64,
         "norm": True, "with_q": False, "page": 64, "pages": 256, "padded": 0, "dtype": "bf16"},
        # the next token of one short sequence
        {"name": "decode_b1", "kind": "attention", "batch": 1, "q_lo": 1, "q_hi": 1, "own_lo": 517, "own_hi": 517, "prefix": 0,
         "q_heads": 32, "kv_heads": 8, "dim": 128, "page": 16, "dtype": "bf16", "mix": 6},
        # bench.py's ragged sequences, one new token each
        {"name": "decode_b64_ragged", "kind": "attention", "batch": 64, "q_lo": 1, "q_hi": 1, "own_lo": 64, "own_hi": 2048,
         "prefix": 0, "q_heads": 32, "kv_heads": 8, "dim": 128, "page": 16, "dtype": "bf16", "mix": 7},
        # many questions on one long document
        {"name": "decode_b64_prefix8192", "kind": "attention", "batch": 64, "q_lo": 1, "q_hi": 1, "own_lo": 1, "own_hi": 300,
         "prefix": 8192, "q_heads": 32, "kv_heads": 8, "dim": 128, "page": 16, "dtype": "bf16", "mix": 8},
        # a few very long sequences
        {"name": "decode_b4_long_d256", "kind": "attention", "batch": 4, "q_lo": 1, "q_hi": 1, "own_lo": 30000, "own_hi": 65536,
         "prefix": 0, "q_heads": 16, "kv_heads": 4, "dim": 256, "page": 64, "dtype": "bf16", "mix": 9},
        # the questions themselves, taken in after the document
        {"name": "extend_b16_prefix2000_d256", "kind": "attention", "batch": 16, "q_lo": 5, "q_hi": 200, "own_lo": 0, "own_hi": 100,
         "prefix": 2000, "q_heads": 16, "kv_heads": 4, "dim": 256, "page": 32, "dtype": "bf16", "mix": 10},
        # a long prompt: the largest call
        {"name": "prompt_8192", "kind": "attention", "batch": 1, "q_lo": 8192, "q_hi": 8192, "own_lo": 0, "own_hi": 0, "prefix": 0,
         "q_heads": 32, "kv_heads": 8, "dim": 128, "page": 16, "dtype": "bf16", "mix": 11},
        # a layer's share of a decode step
        {"name": "step_b32_prefix4096", "kind": "step", "batch": 32, "q_lo": 1, "q_hi": 1, "own_lo": 1, "own_hi": 1000, "prefix": 4096,
         "q_heads": 32, "kv_heads": 8, "dim": 128, "rotary": 128, "norm": True, "page": 16, "dtype": "bf16", "mix": 12},
    ]


def _between(rng, lo, hi):
    """A whole number from lo to hi, even over its logarithm."""
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choice(["norm_rope", "append", "attention", "attention", "attention", "step"])
    q_heads, kv_heads, dim = rng.choice([(32, 8, 128), (16, 4, 256), (32, 8, 128), (16, 4, 256), (16, 16, 64), (24, 8, 128),
                                         (14, 2, 64), (20, 4, 256)])
    case = {"kind": kind, "q_heads": q_heads, "kv_heads": kv_heads, "dim": dim, "dtype": rng.choice(["bf16", "bf16", "bf16", "fp16"])}
    if kind in ("attention", "step"):
        case["mix"] = rng.randrange(1 << 30)
    if kind != "attention":
        case["rotary"] = rng.choice([dim, dim, dim // 2, dim // 4])
        case["norm"] = rng.random() < 0.75
    if kind != "norm_rope":
        case["page"] = rng.choice([16, 16, 32, 64, 128])
    if kind == "norm_rope":
        case["tokens"] = _between(rng, 1, 16384)
    elif kind == "append":
        tokens = _between(rng, 1, 8192)
        case.update(tokens=tokens, with_q=rng.random() < 0.6, padded=rng.choice([0, 0, tokens // 5]),
                    pages=max(4, 2 * tokens // case["page"]))
    elif kind == "step" or rng.random() < 0.6:
        # one new token for each sequence of a batch
        batch = _between(rng, 1, 128)
        own_hi = _between(rng, 1, max(16, min(65536, 200000 // batch)))
        case.update(batch=batch, q_lo=1, q_hi=1, own_lo=rng.choice([1, max(1, own_hi // 8)]), own_hi=own_hi,
                    prefix=rng.choice([0, _between(rng, 32, 32768)]))
    else:
        # prompts, or questions after a prefix: work of at most the longest listed prompt's
        batch = _between(rng, 1, 32)
        q_hi = _between(rng, 1, max(2, min(6000, 16000 // batch)))
        prefix = rng.choice([0, _between(rng, 32, 8192)])
        own_hi = rng.choice([0, _between(rng, 1, 4096)])
        while batch * q_hi * (prefix + own_hi + q_hi / 2) > 2.4e7:
            q_hi, prefix, own_hi = q_hi * 3 // 4 + 1, prefix * 3 // 4, own_hi * 3 // 4
        case.update(batch=batch, q_lo=max(1, q_hi // 16), q_hi=q_hi, own_lo=0, own_hi=own_hi, prefix=prefix)
    return case


def _batch(case):
    """(queries, own keys) of each sequence; own keys hold the queries' own, which come last. Every eleventh sequence of a
    decode batch without a prefix is a padding one: a query with no key at all."""
    rng = random.Random(case["mix"])
    queries, lengths = [], []
    for b in range(case["batch"]):
        n = _between(rng, case["q_lo"], case["q_hi"])
        before = _between(rng, max(1, case["own_lo"]), max(1, case["own_hi"])) if case["own_hi"] else 0
        if case["q_hi"] == 1:
            # own keys of a decode step count the new token's
            length = 0 if case["kind"] == "attention" and not case["prefix"] and b % 11 == 10 else max(1, before)
        else:
            length = before + n
        queries.append(n)
        lengths.append(length)
    return queries, lengths


def _visible(case):
    queries, lengths = _batch(case)
    return sum(n * case["prefix"] + sum(max(0, l - n + i + 1) for i in range(n)) for n, l in zip(queries, lengths))


def _rope_table(positions, rotary):
    """float32 [positions, rotary]: each position's cosines, then its sines."""
    freq = ROPE_BASE ** (-torch.arange(0, rotary, 2, dtype=torch.float64) / rotary)
    angle = torch.arange(positions, dtype=torch.float64)[:, None] * freq
    return torch.cat([angle.cos(), angle.sin()], 1).float().cuda()


def _inputs(case, seed):
    """The tensors of a case, from the seed alone."""
    g = torch.Generator("cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    hq, hk, d, kind = case["q_heads"], case["kv_heads"], case["dim"], case["kind"]
    s = {}

    def normal(*shape, std=1.0):
        return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype)

    def pages(n):
        # written in pieces of 2^28 values: a randn of a whole long cache would need twice its memory in 32 bits
        t = torch.empty(n, hk, case["page"], d, dtype=dtype, device="cuda")
        flat = t.view(-1)
        for i in range(0, flat.numel(), 1 << 28):
            flat[i:i + (1 << 28)] = torch.randn(min(1 << 28, flat.numel() - i), generator=g, device="cuda").to(dtype)
        return t

    if kind in ("attention", "step"):
        queries, lengths = _batch(case)
        tokens, page = sum(queries), case["page"]
        need = [(l + page - 1) // page for l in lengths]
        shared = (case["prefix"] + page - 1) // page
        total = sum(need) + shared + 3
        order = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
        s["k_pages"], s["v_pages"] = pages(total), pages(total)
        table = torch.zeros(len(need), max(max(need), 1), dtype=torch.int32, device="cuda")
        at = shared
        for b, n in enumerate(need):
            table[b, :n] = order[at:at + n]
            at += n
        s["page_table"] = table
        s["lengths"] = torch.tensor(lengths, dtype=torch.int32, device="cuda")
        s["prefix_pages"] = order[:shared].contiguous() if shared else None
        s["query_starts"] = None
        if case["q_hi"] > 1:
            starts = [0]
            for n in queries:
                starts.append(starts[-1] + n)
            s["query_starts"] = torch.tensor(starts, dtype=torch.int32, device="cuda")
        if kind == "step":
            last = [max(l - 1, 0) for l in lengths]
            at = torch.tensor(last, device="cuda")
            s["slots"] = table.gather(1, (at // page)[:, None])[:, 0].long() * page + at % page
            s["positions"] = (at + case["prefix"]).to(torch.int32)
    else:
        tokens = case["tokens"]
        s["positions"] = torch.randint(0, 8192, (tokens,), generator=g, device="cuda", dtype=torch.int32)
    if kind == "append":
        s["k_pages"], s["v_pages"] = pages(case["pages"]), pages(case["pages"])
        s["slots"] = torch.randperm(case["pages"] * case["page"], generator=g, device="cuda")[:tokens].contiguous()
        # a batch padded to a fixed size: its last tokens are no one's
        s["slots"][tokens - case["padded"]:] = -1
    # q, k and v are views of one merged projection's output; some channels run larger than others, as a trained model's do
    merged = torch.randn(tokens, (hq + 2 * hk) * d, generator=g, device="cuda")
    if kind != "attention":
        merged *= torch.randn(merged.shape[1], generator=g, device="cuda").exp_()
    merged = merged.to(dtype)
    q, k, v = merged.split([hq * d, hk * d, hk * d], 1)
    s["q"], s["k"], s["v"] = q.view(tokens, hq, d), k.view(tokens, hk, d), v.view(tokens, hk, d)
    if kind != "attention":
        longest = 8192 if kind != "step" else case["prefix"] + max(lengths) + 1
        s["rope"] = _rope_table(longest, case["rotary"])
        s["q_weight"] = (1 + 0.2 * torch.randn(d, generator=g, device="cuda")) if case["norm"] else None
        s["k_weight"] = (1 + 0.2 * torch.randn(d, generator=g, device="cuda")) if case["norm"] else None
    return s


@torch.no_grad()
def prepare(case, seed):
    state = _inputs(case, seed)
    state["case"] = case
    if own and case["kind"] != "norm_rope":
        from jeeves_amd.attention import PagedKVCache

        state["cache"] = PagedKVCache(state["k_pages"], state["v_pages"])
    return state


def _run_own(s):
    from jeeves_amd.attention import append_kv, paged_attention, qk_norm_rope

    case, kind = s["case"], s["case"]["kind"]
    if kind == "norm_rope":
        return list(qk_norm_rope(s["q"], s["k"], s["rope"], s["positions"], q_weight=s["q_weight"], k_weight=s["k_weight"], eps=EPS))
    q = s["q"]
    outs = []
    if kind in ("append", "step"):
        with_q = kind == "step" or case["with_q"]
        q = append_kv(s["cache"], s["k"], s["v"], s["slots"], rope=s["rope"], positions=s["positions"], k_weight=s["k_weight"],
                      q=q if with_q else None, q_weight=s["q_weight"], eps=EPS)
        outs = [s["cache"].k, s["cache"].v] + ([q] if with_q else [])
    if kind in ("attention", "step"):
        outs.append(paged_attention(q, s["cache"], s["page_table"], s["lengths"], query_starts=s["query_starts"],
                                    prefix_pages=s["prefix_pages"], prefix_length=case["prefix"]))
    return outs


def _norm_rope(x, weight, rope, positions):
    """x [tokens, heads, dim] normed and rotated, in 32 bits."""
    x = x.float()
    if weight is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * weight
    half = rope.shape[1] // 2
    c, s = rope[positions.long()][:, None].split(half, -1)
    a, b, rest = x[..., :half], x[..., half:2 * half], x[..., 2 * half:]
    return torch.cat([a * c - b * s, b * c + a * s, rest], -1)


def _gather(pages, ids):
    """Pages [n, heads, page, dim] by ids [..., m] -> float32 [..., heads, m * page, dim]."""
    picked = pages[ids.long()].float().transpose(-4, -3)
    return picked.reshape(*picked.shape[:-3], -1, picked.shape[-1])


def _softmax_sum(scores, values, seen):
    """Weighted sums of the values under the softmax of the scores over all their parts; rows that see no key are 0."""
    scores = [x if m is None else x.masked_fill(~m, -math.inf) for x, m in zip(scores, seen)]
    top = torch.stack([x.amax(-1) for x in scores]).amax(0)[..., None]
    top = torch.where(top == -math.inf, 0.0, top)
    weights = [(x - top).exp() for x in scores]
    total = sum(w.sum(-1, keepdim=True) for w in weights)
    return sum(w @ v for w, v in zip(weights, values)) / torch.where(total == 0, 1.0, total)


def _attend(q, k_pages, v_pages, s):
    """The attention in 32 bits: a decode batch padded to its longest sequence, or one sequence after the other."""
    case = s["case"]
    hq, hk, d, prefix = case["q_heads"], case["kv_heads"], case["dim"], case["prefix"]
    groups, scale = hq // hk, d ** -0.5
    q = q.float() * scale
    tokens = q.shape[0]
    kp = vp = None
    if prefix:
        kp, vp = (_gather(p, s["prefix_pages"])[:, :prefix] for p in (k_pages, v_pages))
    if s["query_starts"] is None:
        ko, vo = _gather(k_pages, s["page_table"]), _gather(v_pages, s["page_table"])
        seen = torch.arange(ko.shape[2], device=q.device)[None, None, None] < s["lengths"].view(-1, 1, 1, 1)
        qh = q.view(tokens, hk, groups, d)
        # what lies past a sequence's end is another's data and must not count
        vo = vo.masked_fill(~seen.view(tokens, 1, -1, 1), 0.0)
        scores, values, masks = [qh @ ko.transpose(2, 3)], [vo], [seen]
        if prefix:
            scores.append(qh @ kp.transpose(1, 2))
            values.append(vp)
            masks.append(None)
        return _softmax_sum(scores, values, masks).reshape(tokens, hq, d)
    queries, lengths = _batch(case)
    out = torch.empty(tokens, hq, d, device=q.device)
    at = 0
    for b, (n, length) in enumerate(zip(queries, lengths)):
        need = (length + case["page"] - 1) // case["page"]
        ko, vo = (_gather(p, s["page_table"][b, :need])[:, :length] for p in (k_pages, v_pages))
        seen = torch.arange(length, device=q.device)[None] <= length - n + torch.arange(n, device=q.device)[:, None]
        for h in range(hk):
            qh = q[at:at + n, h * groups:(h + 1) * groups].transpose(0, 1)
            scores, values, masks = [qh @ ko[h].t()], [vo[h]], [seen]
            if prefix:
                scores.append(qh @ kp[h].t())
                values.append(vp[h])
                masks.append(None)
            out[at:at + n, h * groups:(h + 1) * groups] = _softmax_sum(scores, values, masks).transpose(0, 1)
        at += n
    return out


def _write(pages, rows, slots):
    """The rows into their slots, in place; slots below zero are left out."""
    keep = slots >= 0
    slots, page = slots[keep], pages.shape[2]
    pages[slots // page, :, slots % page] = rows[keep]


def _run_plain(s):
    case, kind = s["case"], s["case"]["kind"]
    dtype = DTYPES[case["dtype"]]
    q = s["q"]
    outs = []
    if kind != "attention":
        k = _norm_rope(s["k"], s["k_weight"], s["rope"], s["positions"]).to(dtype)
        if kind in ("norm_rope", "step") or case["with_q"]:
            q = _norm_rope(q, s["q_weight"], s["rope"], s["positions"]).to(dtype)
        if kind == "norm_rope":
            return [q, k]
        _write(s["k_pages"], k, s["slots"])
        _write(s["v_pages"], s["v"], s["slots"])
        outs = [s["k_pages"], s["v_pages"]] + ([q] if kind == "step" or case["with_q"] else [])
    if kind != "append":
        outs.append(_attend(q, s["k_pages"], s["v_pages"], s).to(dtype))
    return outs


@torch.no_grad()
def run(state):
    return _run_own(state) if own else _run_plain(state)


def work(case):
    """Inputs read once and outputs written once, the prefix's keys and values once for the whole batch; the products of
    the scores and of the weighted sums over the visible keys."""
    hq, hk, d, kind = case["q_heads"], case["kv_heads"], case["dim"], case["kind"]
    total = flops = 0
    if kind in ("attention", "step"):
        queries, lengths = _batch(case)
        tokens = sum(queries)
        total += 2 * 2 * tokens * hq * d + 2 * 2 * hk * d * (case["prefix"] + sum(lengths)) + 4 * len(lengths)
        flops += 4 * d * hq * _visible(case)
    else:
        tokens = case["tokens"]
    if kind != "attention":
        kept = tokens - case.get("padded", 0)
        total += 4 * tokens * case["rotary"] + 4 * tokens
        if kind in ("norm_rope", "step") or case["with_q"]:
            total += 2 * 2 * tokens * hq * d
            flops += 8 * tokens * hq * d
        total += 2 * 2 * hk * d * (tokens if kind == "norm_rope" else 2 * kept) + (0 if kind == "norm_rope" else 8 * tokens)
        flops += 8 * tokens * hk * d
    return {"bytes": total, "flops": flops}


def _exact_head(x, weight, rope, positions):
    """z of a head by complex products: pair (i, i + rotary/2) turned by its angle."""
    x = x.double()
    if weight is not None:
        x = x / (x.square().sum(-1, keepdim=True) / x.shape[-1] + EPS).sqrt() * weight.double()
    half = rope.shape[1] // 2
    turn = torch.complex(rope[:, :half].double(), rope[:, half:].double())[positions.long()].unsqueeze(1)
    turned = torch.complex(x[..., :half], x[..., half:2 * half]) * turn
    z = x.clone()
    z[..., :half], z[..., half:2 * half] = turned.real, turned.imag
    return z


def _exact_attention(q, k_pages, v_pages, s, case):
    """Each sequence's keys laid out in order (prefix, then its own), softmax by log-sum-exp, in 64 bits."""
    hq, hk, d, prefix, page = case["q_heads"], case["kv_heads"], case["dim"], case["prefix"], case["page"]
    queries, lengths = _batch(case)
    out = torch.zeros(q.shape[0], hq, d, dtype=torch.float64, device=q.device)
    at = 0
    for b, (n, length) in enumerate(zip(queries, lengths)):
        j = torch.arange(prefix + length, device=q.device)
        ids = s["page_table"][b, ((j - prefix).clamp(min=0) // page)].long()
        offset = (j - prefix) % page
        if prefix:
            shared = s["prefix_pages"][(j.clamp(max=prefix - 1) // page)].long()
            ids, offset = torch.where(j < prefix, shared, ids), torch.where(j < prefix, j % page, offset)
        last = prefix + length - n + torch.arange(n, device=q.device)
        if prefix + length:
            for h in range(hk):
                keys, values = k_pages[ids, h, offset].double(), v_pages[ids, h, offset].double()
                for head in range(h * hq // hk, (h + 1) * hq // hk):
                    score = torch.mm(q[at:at + n, head].double(), keys.t().contiguous()) / math.sqrt(d)
                    hidden = j[None] > torch.maximum(last[:, None], torch.full_like(last[:, None], prefix - 1))
                    score[hidden] = -math.inf
                    weight = torch.exp(score - torch.logsumexp(score, 1, keepdim=True)).nan_to_num_(0.0)
                    out[at:at + n, head] = torch.mm(weight, values)
        at += n
    return out


@torch.no_grad()
def exact(case, seed):
    s = _inputs(case, seed)
    kind = case["kind"]
    q, outs = s["q"].double(), []
    if kind != "attention":
        k = _exact_head(s["k"], s["k_weight"], s["rope"], s["positions"])
        q = _exact_head(q, s["q_weight"], s["rope"], s["positions"])
        if kind == "norm_rope":
            return [q, k]
        k_pages, v_pages = s["k_pages"].double(), s["v_pages"].double()
        for t, slot in enumerate(s["slots"].tolist()):
            if slot >= 0:
                k_pages[slot // case["page"], :, slot % case["page"]] = k[t]
                v_pages[slot // case["page"], :, slot % case["page"]] = s["v"][t].double()
        outs = [k_pages, v_pages] + ([q] if kind == "step" or case["with_q"] else [])
        if kind == "append":
            return outs
        # the attention's operands are what the call before it stored: 16-bit values
        q, k_pages, v_pages = (x.to(DTYPES[case["dtype"]]) for x in (q, k_pages, v_pages))
        return outs + [_exact_attention(q, k_pages, v_pages, s, case)]
    return [_exact_attention(q, s["k_pages"], s["v_pages"], s, case)]
