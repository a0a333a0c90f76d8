"""The generation and scoring operators around the W4A4 linears, as measured workloads: appending keys and
values to a 4-bit paged cache (with the position rotation of queries and keys), attention over that cache, and
log probabilities of given tokens with entropy and the top alternatives.

A batch of sequences is described the same way for every cache operator: `q_start` [B + 1] gives each
sequence's rows in the ragged token axis, `lengths` [B] its cached tokens once those rows are in, `page_table`
[B, P] its pages. Row i of a sequence with n rows stands at position lengths - n + i.
"""
import math
import random

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


# ---------------------------------------------------------------------------------------------- cases
def listed():
    llama7b = {"heads": 32, "kv_heads": 32, "dim": 128}
    llama70b = {"heads": 64, "kv_heads": 8, "dim": 128}
    return [
        # one user's next token: the smallest call, its latency counts
        {"name": "append-one", "op": "append", "seqs": 1, "least_new": 1, "most_new": 1,
         "least_past": 700, "most_past": 700, **llama7b, "page": 64, "type": "bf16", "pad": 0, "mix": 1},
        # one step of a serving batch of grouped heads, padded as a captured graph pads it
        {"name": "append-batch", "op": "append", "seqs": 64, "least_new": 1, "most_new": 1,
         "least_past": 0, "most_past": 4000, **llama70b, "page": 16, "type": "f16", "pad": 8, "mix": 2},
        # prompts of mixed lengths entering the cache together
        {"name": "append-prompts", "op": "append", "seqs": 6, "least_new": 1, "most_new": 2600,
         "least_past": 0, "most_past": 900, **llama7b, "page": 64, "type": "bf16", "pad": 0, "mix": 3},
        # one user's next token over a short context
        {"name": "attend-one", "op": "attend", "seqs": 1, "least_new": 1, "most_new": 1,
         "least_past": 700, "most_past": 700, **llama7b, "page": 64, "type": "bf16", "pad": 0, "mix": 4},
        # a serving batch of grouped heads with ragged contexts
        {"name": "attend-batch", "op": "attend", "seqs": 64, "least_new": 1, "most_new": 1,
         "least_past": 0, "most_past": 8191, **llama70b, "page": 64, "type": "bf16", "pad": 8, "mix": 5},
        # few users with very long contexts: the keys have to be split
        {"name": "attend-long", "op": "attend", "seqs": 3, "least_new": 1, "most_new": 1,
         "least_past": 50000, "most_past": 65000, **llama70b, "page": 64, "type": "bf16", "pad": 0, "mix": 6},
        # drafted tokens being verified, small heads and pages
        {"name": "attend-drafts", "op": "attend", "seqs": 24, "least_new": 1, "most_new": 6,
         "least_past": 60, "most_past": 2500, "heads": 16, "kv_heads": 4, "dim": 64,
         "page": 16, "type": "f16", "pad": 3, "mix": 7},
        # whole prompts, one head per key head
        {"name": "attend-prompts", "op": "attend", "seqs": 3, "least_new": 900, "most_new": 2048,
         "least_past": 0, "most_past": 0, **llama7b, "page": 64, "type": "bf16", "pad": 0, "mix": 8},
        # the next chunk of long prompts, grouped heads
        {"name": "attend-chunk", "op": "attend", "seqs": 2, "least_new": 1000, "most_new": 1500,
         "least_past": 7000, "most_past": 10000, **llama70b, "page": 64, "type": "f16", "pad": 0, "mix": 9},
        # a decode step that reports its token and five alternatives
        {"name": "score-one", "op": "score", "rows": 1, "vocab": 32000, "top": 5, "type": "bf16", "mix": 10},
        # a small evaluation batch in 32 bits with a ragged vocabulary
        {"name": "score-odd", "op": "score", "rows": 77, "vocab": 50001, "top": 3, "type": "f32", "mix": 11},
        # two prompts of 2048 tokens scored with twenty alternatives each
        {"name": "score-prompts", "op": "score", "rows": 4096, "vocab": 32000, "top": 20, "type": "bf16", "mix": 12},
    ]


def _spread(rng, lo, hi):
    """A whole number from lo to hi, over the logarithm where the range spans more than a factor of ten."""
    if hi > 10 * max(1, lo):
        return min(hi, max(lo, int(math.exp(rng.uniform(math.log(max(1, lo)), math.log(hi + 1))))))
    return rng.randint(lo, hi)


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "score"])
    mix = rng.randrange(1 << 30)
    if op == "score":
        vocab = _spread(rng, 500, 130000)
        rows = _spread(rng, 1, max(1, min(4096, 131072000 // vocab)))
        return {"op": op, "rows": rows, "vocab": vocab, "top": rng.choice([0, 1, 5, 20, 32]),
                "type": rng.choice(["bf16", "f16", "f32"] if rows * vocab < 60000000 else ["bf16", "f16"]), "mix": mix}
    kv_heads = rng.choice([1, 2, 4, 8, 32])
    group = rng.choice([1, 1, 2, 4, 7, 8]) if kv_heads <= 8 else 1
    case = {"op": op, "heads": kv_heads * group, "kv_heads": kv_heads, "dim": rng.choice([64, 128, 128]),
            "page": rng.choice([16, 32, 64, 128]), "type": rng.choice(["bf16", "f16"]), "pad": rng.choice([0, 0, 5]),
            "mix": mix}
    if op == "append":
        seqs = _spread(rng, 1, 100)
        return {**case, "seqs": seqs, "least_new": 1, "most_new": _spread(rng, 1, max(1, 8000 // seqs)),
                "least_past": 0, "most_past": _spread(rng, 1, 4000)}
    if rng.random() < 0.6:  # single tokens and drafts
        seqs = _spread(rng, 1, 100)
        return {**case, "seqs": seqs, "least_new": 1, "most_new": rng.choice([1, 1, 1, 4]), "least_past": 0,
                "most_past": _spread(rng, 30, min(65000, 1500000 // (seqs * kv_heads)))}
    seqs = rng.choice([1, 1, 2, 3])
    new = _spread(rng, 20, 2048)
    past = _spread(rng, 1, max(1, min(10000, 1000000000 // (case["heads"] * new * seqs))))
    return {**case, "seqs": seqs, "least_new": max(1, new // 2), "most_new": new, "least_past": 0, "most_past": past}


def _shape(case):
    """(rows, cached tokens) of each sequence: fixed by the case."""
    rng = random.Random(case["mix"])
    new = [rng.randint(case["least_new"], case["most_new"]) for _ in range(case["seqs"])]
    return new, [n + rng.randint(case["least_past"], case["most_past"]) for n in new]


def _visible(case):
    """Query-key pairs that the causal mask leaves, over one head."""
    return sum(n * (length - n) + n * (n + 1) // 2 for n, length in zip(*_shape(case)))


# ---------------------------------------------------------------------------------------------- inputs
def _quantised(y, dtype):
    """4-bit rows: codes (whole numbers 0..15), and step and low of `dtype`, along the last axis of y."""
    low = y.amin(-1, keepdim=True).to(dtype).to(y.dtype)
    step = ((y.amax(-1, keepdim=True) - low) / 15).to(dtype).to(y.dtype)
    bad = ~(torch.isfinite(low) & torch.isfinite(step))
    code = torch.where((step == 0) | bad, torch.zeros_like(y), ((y - low) / step).round().clamp(0, 15))
    return code, torch.where(bad, math.nan, step), torch.where(bad, math.nan, low)


def _noise(shape, gen, scale=1.0):
    return torch.randn(shape, generator=gen, device="cuda") * scale


def _pool(pages, case, gen, outliers):
    """Cached rows as generation leaves them: normal values, for keys a few channels far larger; packed two
    codes a byte, the even channel low."""
    h, ps, d, dtype = case["kv_heads"], case["page"], case["dim"], TYPES[case["type"]]
    codes = torch.empty((pages, h, ps, d // 2), dtype=torch.uint8, device="cuda")
    affine = torch.empty((pages, h, ps, 2), dtype=dtype, device="cuda")
    per = max(1, (1 << 26) // (h * ps * d))
    for at in range(0, pages, per):
        y = _noise((min(per, pages - at), h, ps, d), gen) * outliers
        code, step, low = _quantised(y, dtype)
        code = code.to(torch.uint8)
        codes[at:at + per] = code[..., 0::2] | (code[..., 1::2] << 4)
        affine[at:at + per] = torch.cat((step, low), -1).to(dtype)
    return codes, affine


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    dtype = TYPES[case["type"]]
    if case["op"] == "score":
        rows, vocab = case["rows"], case["vocab"]
        logits = _noise((rows, vocab), gen, 2.5)
        logits += _noise((1, vocab), gen)  # some tokens are likelier everywhere
        logits[:, -2:] = -math.inf         # a vocabulary padded to its width
        targets = torch.multinomial(logits[:, :4096].softmax(-1), 1, generator=gen)[:, 0]
        targets[torch.rand(rows, generator=gen, device="cuda") < 0.02] = -1  # padding: no token
        return {"case": case, "logits": logits.to(dtype), "targets": targets}
    new, length = _shape(case)
    heads, kv_heads, d, ps = case["heads"], case["kv_heads"], case["dim"], case["page"]
    used = [-(-n // ps) for n in length]
    pages, wide = sum(used) + 2, max(used) + 1
    order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
    row = torch.tensor([b for b, n in enumerate(used) for _ in range(n)], device="cuda")
    column = torch.tensor([i for n in used for i in range(n)], device="cuda")
    table = torch.full((len(new), wide), -1, dtype=torch.int32, device="cuda")
    table[row, column] = order[:sum(used)]
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    total = starts[-1] + case["pad"]
    outliers = 1 + 6 * (torch.rand(kv_heads, 1, d, generator=gen, device="cuda") < 0.03)
    k_codes, k_affine = _pool(pages, case, gen, outliers)
    v_codes, v_affine = _pool(pages, case, gen, 1.0)
    state = {"case": case, "cache": (k_codes, k_affine, v_codes, v_affine), "page_table": table,
             "q_start": torch.tensor(starts, dtype=torch.int32, device="cuda"),
             "lengths": torch.tensor(length, dtype=torch.int32, device="cuda"),
             "q": _noise((total, heads, d), gen).to(dtype)}
    if case["op"] == "append":
        state["k"] = (_noise((total, kv_heads, d), gen) * outliers[:, 0]).to(dtype)
        state["v"] = _noise((total, kv_heads, d), gen).to(dtype)
        rate = 10000.0 ** -(torch.arange(0, d, 2, dtype=torch.float64, device="cuda") / d)
        angle = torch.outer(torch.arange(max(length) + 7, dtype=torch.float64, device="cuda"), rate).repeat(1, 2)
        state["cos"], state["sin"] = angle.cos().to(dtype), angle.sin().to(dtype)
    return state


# ---------------------------------------------------------------------------------------------- one pass
def run(state):
    case = state["case"]
    if own:
        return _own(state)
    return {"append": _append, "attend": _attend, "score": _score}[case["op"]](state)


def _own(state):
    from dscquant_b200 import PagedKV4, ops

    case = state["case"]
    if case["op"] == "score":
        r = ops.token_logprobs(state["logits"], state["targets"], top_k=case["top"])
        return _scored(r.logprobs, r.entropy, r.top_logprobs, r.top_ids)
    cache = PagedKV4(*state["cache"])
    where = state["page_table"], state["q_start"], state["lengths"]
    if case["op"] == "append":
        q = ops.kv4_append(cache, state["q"], state["k"], state["v"], state["cos"], state["sin"], *where)
        k, v = ops.kv4_read(cache, *where, rows=q.shape[0])
        return {"q": q, "k": k, "v": v}
    return {"out": ops.kv4_attention(cache, state["q"], *where, max_q=case["most_new"])}


def _scored(logprobs, entropy, top, ids):
    out = {"logprobs": logprobs, "entropy": entropy}
    return out if not ids.shape[1] else {**out, "top_logprobs": top, "top_ids": ids}


def _rows(state, total):
    """Of every row of the token axis: whether a sequence has it, the sequence, and its position."""
    start, t = state["q_start"].long(), torch.arange(total, device="cuda")
    b = (torch.searchsorted(start, t, right=True) - 1).clamp(0, start.numel() - 2)
    return t < start[-1], b, state["lengths"].long()[b] - start[b + 1] + t


def _append(state):
    """Rotation, 4-bit rows and the scatter into the pages, then the values that the pages hold. In 64 bits:
    a value next to the border of two codes goes to the right one."""
    dtype, d = state["q"].dtype, state["case"]["dim"]
    total, ps = state["q"].shape[0], state["case"]["page"]
    real, b, position = _rows(state, total)
    position = torch.where(real, position, 0)
    cos, sin = state["cos"][position].double()[:, None], state["sin"][position].double()[:, None]

    def rotated(x):
        x = x.double()
        return x * cos + torch.cat((-x[..., d // 2:], x[..., :d // 2]), -1) * sin

    keep = real[:, None, None]
    q = torch.where(keep, rotated(state["q"]), 0).to(dtype)
    rows = torch.nonzero(real)[:, 0]
    page, slot = state["page_table"][b, position // ps].long()[rows], (position % ps)[rows]
    held = []
    for y, codes, affine in ((rotated(state["k"]), *state["cache"][:2]), (state["v"].double(), *state["cache"][2:])):
        code, step, low = _quantised(y, dtype)
        whole = code.to(torch.uint8)
        codes[page, :, slot] = (whole[..., 0::2] | (whole[..., 1::2] << 4))[rows]
        affine[page, :, slot] = torch.cat((step, low), -1).to(dtype)[rows]
        held.append(torch.where(keep, code * step + low, 0).to(dtype))
    return {"q": q, "k": held[0], "v": held[1]}


def _values(codes, affine, table):
    """The cached rows of every sequence in 32 bits, [sequences, heads, tokens, dim]; unmapped pages repeat page 0."""
    pages = table.clamp_min(0).long()
    packed, affine = codes[pages], affine[pages].float()
    code = torch.stack((packed & 15, packed >> 4), -1).flatten(-2).float()
    return (code * affine[..., :1] + affine[..., 1:]).transpose(1, 2).flatten(2, 3)


def _attend(state):
    case, q = state["case"], state["q"]
    total, heads, d = q.shape
    kv_heads, most = case["kv_heads"], max(_shape(case)[0])
    start, length = state["q_start"].long(), state["lengths"].long()
    count = start[1:] - start[:-1]
    i = torch.arange(most, device="cuda")
    there = i < count[:, None]
    at = torch.where(there, start[:-1, None] + i, 0)
    x = q[at].float().view(len(count), most, kv_heads, heads // kv_heads, d).permute(0, 2, 3, 1, 4).flatten(2, 3)
    keys = _values(*state["cache"][:2], state["page_table"])
    s = (x @ keys.transpose(2, 3)) * d ** -0.5
    del keys
    position = (length - count)[:, None] + i
    seen = torch.arange(s.shape[3], device="cuda") <= position[..., None]
    s = s.view(len(count), heads, most, -1).masked_fill_(~seen[:, None], -math.inf)
    s = (s - s.amax(-1, keepdim=True)).exp_()
    s /= s.sum(-1, keepdim=True)
    y = s.view(len(count), kv_heads, -1, s.shape[3]) @ _values(*state["cache"][2:], state["page_table"])
    y = y.view(len(count), heads, most, d).transpose(1, 2)
    out = torch.zeros_like(q)
    out[at[there]] = y[there].to(q.dtype)
    return {"out": out}


def _score(state):
    x, target, top = state["logits"].float(), state["targets"], state["case"]["top"]
    most = x.amax(-1, keepdim=True)
    e = (x - most).exp()
    total = e.sum(-1, keepdim=True)
    logs = x - most - total.log()
    p = e / total
    entropy = -torch.where(p > 0, p * logs, 0).sum(-1)
    logprobs = torch.where(target < 0, 0.0, logs.gather(-1, target.clamp_min(0)[:, None])[:, 0])
    if not top:
        return {"logprobs": logprobs, "entropy": entropy}
    ids = x.sort(dim=-1, descending=True, stable=True)[1][:, :top].contiguous()
    return _scored(logprobs, entropy, logs.gather(-1, ids), ids)


# ---------------------------------------------------------------------------------------------- what it takes
def work(case):
    if case["op"] == "score":
        rows, vocab = case["rows"], case["vocab"]
        size = 4 if case["type"] == "f32" else 2
        return {"bytes": rows * (vocab * size + 16 + 12 * case["top"]), "flops": 5 * rows * vocab}
    new, length = _shape(case)
    t, heads, kv_heads, d = sum(new), case["heads"], case["kv_heads"], case["dim"]
    row = kv_heads * 2 * (d // 2 + 4)  # a cached token, keys and values
    if case["op"] == "append":
        # q in and out, k and v in, the angles, the cached rows out, and their values out
        return {"bytes": t * (2 * heads * d * 2 + 2 * kv_heads * d * 2 + 4 * d + row + 2 * kv_heads * d * 2),
                "flops": t * (3 * (heads + kv_heads) * d + 8 * 2 * kv_heads * d)}
    return {"bytes": sum(length) * row + 2 * t * heads * d * 2, "flops": 4 * d * heads * _visible(case)}


# ---------------------------------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "score":
        x = state["logits"].double()
        logs = x - torch.logsumexp(x, -1, keepdim=True)
        entropy = torch.special.entr(logs.exp()).sum(-1)
        targets = state["targets"].tolist()
        picked = torch.stack([logs[r, t] if t >= 0 else logs.new_zeros(()) for r, t in enumerate(targets)])
        if not case["top"]:
            return {"logprobs": picked, "entropy": entropy}
        ids = torch.argsort(-x, dim=-1, stable=True)[:, :case["top"]]
        return {"logprobs": picked, "entropy": entropy, "top_logprobs": torch.take_along_dim(logs, ids, -1),
                "top_ids": ids}
    if case["op"] == "append":
        return _exact_append(state)
    if 4 * case["dim"] * case["heads"] * _visible(case) > 2e12:
        return None
    return _exact_attend(state)


def _exact_append(state):
    case, dtype = state["case"], TYPES[state["case"]["type"]]
    half = case["dim"] // 2
    out = {n: torch.zeros(state[n].shape, dtype=torch.float64, device="cuda") for n in ("q", "k", "v")}
    starts = state["q_start"].tolist()
    for b, length in enumerate(state["lengths"].tolist()):
        rows = slice(starts[b], starts[b + 1])
        where = slice(length - (starts[b + 1] - starts[b]), length)
        cos, sin = (state[n][where].double().unsqueeze(1) for n in ("cos", "sin"))
        for n in ("q", "k", "v"):
            y = state[n][rows].double()
            if n != "v":
                a, c = y[..., :half], y[..., half:]
                y = torch.cat((a * cos[..., :half] - c * sin[..., :half],
                               c * cos[..., half:] + a * sin[..., half:]), -1)
            if n != "q":
                low = y.min(-1, True)[0].to(dtype).double()
                step = ((y.max(-1, True)[0] - low) / 15).to(dtype).double()
                y = low + step * torch.clamp(torch.round((y - low) / step), 0, 15)
            out[n][rows] = y
    return out


def _exact_attend(state):
    case = state["case"]
    group, d, ps = case["heads"] // case["kv_heads"], case["dim"], case["page"]
    k_codes, k_affine, v_codes, v_affine = state["cache"]
    out = torch.zeros(state["q"].shape, dtype=torch.float64, device="cuda")
    starts = state["q_start"].tolist()
    for b, length in enumerate(state["lengths"].tolist()):
        pages = state["page_table"][b, :-(-length // ps)].long()
        rows = slice(starts[b], starts[b + 1])
        n = starts[b + 1] - starts[b]
        hidden = torch.ones((n, length), dtype=torch.bool, device="cuda").triu(length - n + 1)
        for h in range(case["kv_heads"]):
            held = []
            for codes, affine in ((k_codes, k_affine), (v_codes, v_affine)):
                packed = codes[pages, h].reshape(-1, d // 2)[:length]
                both = affine[pages, h].reshape(-1, 2)[:length].double()
                y = torch.empty((length, d), dtype=torch.float64, device="cuda")
                y[:, 0::2], y[:, 1::2] = packed % 16, packed // 16
                held.append(y * both[:, :1] + both[:, 1:])
            for g in range(h * group, (h + 1) * group):
                s = state["q"][rows, g].double() @ held[0].T / math.sqrt(d)
                out[rows, g] = torch.softmax(s.masked_fill(hidden, -math.inf), -1) @ held[1]
    return {"out": out}
