"""Serving a decoder: the operators of one step, as cases that can be timed and
checked. The norm in front of a product with the residual's addition and an
8-bit output, attention over a window with a few first tokens that stay
visible, the 8-bit key and value cache that a step appends to and reads, and
the log probabilities of the tokens that come out.

A case is a dict of plain values. `listed` names twelve; `draw` gives more of
the same ranges. `prepare` makes what a program holds before the call. `run`
makes one call: of the framework's operators where `own` is true, else of their
plain forms in torch. `exact` computes the results in 64 bits from the
definitions, `work` the bytes and operations that a call cannot do without.
"""

import torch

own = False

DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16,
          "e4m3": torch.float8_e4m3fn}
SIZE = {"fp32": 4, "fp16": 2, "bf16": 2, "e4m3": 1}
E4M3_MAX = 448.0
TINY = 2.0 ** -126


def listed():
    return [
        # one token of one sequence between two layers: the call is the cost
        {"name": "rmsnorm_bf16_1x4096", "kind": "rmsnorm", "dtype": "bf16", "rows": 1,
         "cols": 4096, "residual": True, "out": "bf16", "group": 0},
        # a long prompt's tokens in front of an 8-bit product, a scale for each
        # 128 columns
        {"name": "rmsnorm_bf16_4096x8192_e4m3", "kind": "rmsnorm", "dtype": "bf16", "rows": 4096,
         "cols": 8192, "residual": True, "out": "e4m3", "group": 128},
        # prompts of the attention benchmark's size, four query heads to a KV
        # head, in a window of 1024 tokens
        {"name": "window_bf16_4x32x4096x128", "kind": "window", "dtype": "bf16", "B": 4, "H": 32,
         "KV": 8, "Sq": 4096, "Sk": 4096, "D": 128, "window": 1024, "sinks": 4, "ragged": False},
        # a ragged chunk of prompts whose first tokens are there already
        {"name": "window_fp16_3x16x333of1999x64", "kind": "window", "dtype": "fp16", "B": 3,
         "H": 16, "KV": 16, "Sq": 333, "Sk": 1999, "D": 64, "window": 500, "sinks": 16,
         "ragged": True},
        # single tokens of 16 sequences over keys that are not compressed
        {"name": "window_bf16_16x32x1of8192x128", "kind": "window", "dtype": "bf16", "B": 16,
         "H": 32, "KV": 8, "Sq": 1, "Sk": 8192, "D": 128, "window": 4096, "sinks": 4,
         "ragged": True},
        # one step's tokens of 64 sequences go into their caches
        {"name": "append_bf16_64x1", "kind": "append", "dtype": "bf16", "B": 64, "KV": 8, "S": 1,
         "D": 128, "block": 64, "L": 4096},
        # ragged prompts go into their caches behind a shared beginning
        {"name": "append_bf16_8x2048", "kind": "append", "dtype": "bf16", "B": 8, "KV": 8,
         "S": 2048, "D": 128, "block": 64, "L": 4096},
        # a step of one sequence with 8 thousand tokens behind it
        {"name": "cached_bf16_1x32x8191x128", "kind": "cached", "dtype": "bf16", "B": 1, "H": 32,
         "KV": 8, "Sq": 1, "L": 8191, "D": 128, "block": 64, "window": 0, "sinks": 0},
        # a step of 64 sequences of up to 8 thousand tokens
        {"name": "cached_bf16_64x32x8192x128", "kind": "cached", "dtype": "bf16", "B": 64,
         "H": 32, "KV": 8, "Sq": 1, "L": 8192, "D": 128, "block": 64, "window": 0, "sinks": 0},
        # five drafted tokens to be checked at once, small blocks, in a window
        {"name": "cached_fp16_24x16x5of6000x64", "kind": "cached", "dtype": "fp16", "B": 24,
         "H": 16, "KV": 4, "Sq": 5, "L": 6000, "D": 64, "block": 16, "window": 2048, "sinks": 4},
        # the next token of one sequence with its alternatives
        {"name": "logprobs_bf16_1x128000", "kind": "logprobs", "dtype": "bf16", "rows": 1,
         "vocab": 128000, "top": 20, "temperature": 1.0},
        # the tokens of prompts and answers, an odd vocabulary
        {"name": "logprobs_bf16_2048x100003", "kind": "logprobs", "dtype": "bf16", "rows": 2048,
         "vocab": 100003, "top": 5, "temperature": 0.7},
    ]


def _log_int(rng, lo, hi):
    """A whole number spread evenly over the logarithm of [lo, hi]."""
    return max(lo, min(hi, round(lo * (hi / lo) ** rng.random())))


def _size(rng, lo, hi):
    """Sizes as they come: half of them multiples of 64, a quarter multiples
    of 8, the rest any whole number."""
    step = rng.choice((64, 64, 8, 1))
    return max(lo, min(hi, -(-_log_int(rng, lo, hi) // step) * step))


def draw(rng):
    kind = rng.choice(("rmsnorm", "window", "window", "append", "cached", "cached", "logprobs"))
    dtype = rng.choice(("bf16", "bf16", "fp16"))
    if kind == "rmsnorm":
        cols = _size(rng, 64, 16384)
        out = rng.choice(("same", "e4m3"))
        dtype = rng.choice((dtype, dtype, "fp32"))
        return {"kind": kind, "dtype": dtype, "rows": _log_int(rng, 1, (1 << 25) // cols),
                "cols": cols, "residual": rng.random() < 0.7,
                "out": dtype if out == "same" else out,
                "group": rng.choice((0, 128)) if out == "e4m3" and cols % 128 == 0 else 0}
    if kind == "logprobs":
        vocab = _log_int(rng, 1000, 200000)
        return {"kind": kind, "dtype": rng.choice((dtype, "fp32")),
                "rows": _log_int(rng, 1, min(4096, (1 << 27) // vocab)), "vocab": vocab,
                "top": rng.choice((0, 1, 5, 20)), "temperature": rng.choice((1.0, 1.0, 0.7))}
    KV, D = rng.choice((1, 2, 4, 8, 16)), rng.choice((64, 128, 128))
    if kind == "append":
        S = 1 if rng.random() < 0.4 else _log_int(rng, 2, 4096)
        L = S + _log_int(rng, 1, 4096)
        return {"kind": kind, "dtype": dtype, "B": _log_int(rng, 1, max(1, min(64, (1 << 18) // L))),
                "KV": min(KV, 8), "S": S, "D": D, "block": rng.choice((16, 32, 64, 128)), "L": L}
    H = KV * rng.choice((1, 2, 4, 8))
    window = rng.choice((0, 1, 1, 1)) and _log_int(rng, 16, 4096)
    sinks = rng.choice((0, 1, 4, 64)) if window else 0
    if kind == "cached":
        L = _log_int(rng, 1, 16384)
        return {"kind": kind, "dtype": dtype, "B": _log_int(rng, 1, max(1, min(64, (1 << 18) // L))),
                "H": H, "KV": KV, "Sq": rng.choice((1, 1, 1, 2, 5, 16)), "L": L, "D": D,
                "block": rng.choice((16, 32, 64, 128)), "window": window, "sinks": sinks}
    Sk = _size(rng, 1, 8192)
    Sq = rng.choice((1, Sk, Sk, _log_int(rng, 1, Sk)))
    B = max(1, min(_log_int(rng, 1, 16), (1 << 29) // (H * Sq * Sk), (1 << 25) // (KV * Sk * D)))
    while B * H * Sq * Sk > 1 << 31:
        H //= 2
    return {"kind": kind, "dtype": dtype, "B": B, "H": H, "KV": min(KV, H), "Sq": Sq, "Sk": Sk,
            "D": D, "window": window, "sinks": sinks, "ragged": rng.random() < 0.5}


def _spread(n, lo, hi):
    """n whole numbers over [lo, hi] in no order, the largest among them, the
    same ones for every seed: lengths decide a call's work."""
    return [hi if i == n // 2 else lo + int((hi - lo + 1) * ((0.618034 * (i + 1)) % 1.0))
            for i in range(n)]


def _starts(case):
    """window: the position of each sequence's first query."""
    last = case["Sk"] - case["Sq"]
    return _spread(case["B"], last // 2, last) if case["ragged"] else [last] * case["B"]


def _appends(case):
    """append: each sequence's length before the call and its new tokens."""
    S, most = case["S"], case["L"] - case["S"]
    return _spread(case["B"], most // 2, most), _spread(case["B"], max(1, S // 2), S)


def _lens(case):
    """cached: each sequence's length with the queries' own tokens."""
    return _spread(case["B"], max(1, case["L"] // 4), case["L"])


def _blocks(case):
    return -(-case["L"] // case["block"])


def _pairs(case, first):
    """How many (query, key) pairs a sequence's queries from position `first`
    on see, and how many keys at least one of them sees."""
    n = seen = 0
    Sk = case["Sk"] if case["kind"] == "window" else case["L"]
    low = Sk
    for p in range(max(first, 0), first + case["Sq"]):
        lo = max(0, p + 1 - case["window"]) if case["window"] else 0
        n += max(0, min(p + 1, Sk) - lo) + min(case["sinks"], lo)
        low = min(low, lo)
    if first + case["Sq"] > 0:
        seen = min(first + case["Sq"], Sk) - low + min(case["sinks"], low)
    return n, seen


def work(case):
    kind, size = case["kind"], SIZE[case["dtype"]]
    if kind == "rmsnorm":
        n = case["rows"] * case["cols"]
        scales = 0 if case["out"] != "e4m3" else n // (case["group"] or case["cols"]) * 4
        return {"bytes": n * (size * (3 if case["residual"] else 1) + SIZE[case["out"]]) + scales
                + case["cols"] * size, "flops": 0}
    if kind == "logprobs":
        return {"bytes": case["rows"] * (case["vocab"] * size + 16 + 12 * case["top"]), "flops": 0}
    KV, D = case["KV"], case["D"]
    if kind == "append":
        starts, counts = _appends(case)
        touched = sum((s + c - 1) // case["block"] - s // case["block"] + 1
                      for s, c in zip(starts, counts))
        return {"bytes": 2 * KV * (sum(counts) * D * (size + 1) + touched * 8), "flops": 0}
    each = 1 if kind == "cached" else size
    firsts = _starts(case) if kind == "window" else [n - case["Sq"] for n in _lens(case)]
    pairs, seen = (sum(v) for v in zip(*(_pairs(case, f) for f in firsts)))
    return {"bytes": 2 * case["B"] * case["H"] * case["Sq"] * D * size + 2 * KV * seen * D * each,
            "flops": 4 * case["H"] * D * pairs}


def _cache(g, case):
    """A cache whose blocks lie in any order, each with scales of its own, and
    the table of every sequence's blocks. Values as keys and values have them:
    normal, with a scale that fits the block."""
    B, KV, D, block = case["B"], case["KV"], case["D"], case["block"]
    per = _blocks(case)
    n = B * per + 3
    at = {"generator": g, "device": "cuda"}
    k = (torch.randn(n, KV, block, D, **at) * 100).clamp(-E4M3_MAX, E4M3_MAX)
    v = (torch.randn(n, KV, D, block, **at) * 100).clamp(-E4M3_MAX, E4M3_MAX)
    scales = [torch.exp2(torch.randint(-8, -5, (n, KV), **at).float()) for _ in range(2)]
    table = torch.randperm(n, **at)[:B * per].view(B, per).to(torch.int32)
    return [k.to(DTYPES["e4m3"]), v.to(DTYPES["e4m3"]), *scales], table


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    kind, t = case["kind"], DTYPES[case["dtype"]]

    def randn(*shape):
        return torch.randn(*shape, generator=g, device="cuda").to(t)

    def ints(values):
        return torch.tensor(values, dtype=torch.int32, device="cuda")

    s = {"case": case}
    if kind == "rmsnorm":
        shape = (case["rows"], case["cols"])
        s["x"] = randn(*shape)
        s["residual"] = randn(*shape) * 3 if case["residual"] else None
        s["w"] = (randn(case["cols"]) * 0.2 + 1.0).to(t)
    elif kind == "window":
        s["q"] = randn(case["B"], case["H"], case["Sq"], case["D"])
        s["k"], s["v"] = (randn(case["B"], case["KV"], case["Sk"], case["D"]) for _ in range(2))
        s["start"] = ints(_starts(case))
    elif kind == "append":
        s["cache"], s["table"] = _cache(g, case)
        shape = (case["B"], case["KV"], case["S"], case["D"])
        s["k"], s["v"] = randn(*shape), randn(*shape)
        starts, counts = _appends(case)
        s["start"], s["count"] = ints(starts), ints(counts)
    elif kind == "cached":
        s["cache"], s["table"] = _cache(g, case)
        s["q"] = randn(case["B"], case["H"], case["Sq"], case["D"])
        s["lens"] = ints(_lens(case))
    else:
        x = randn(case["rows"], case["vocab"]) * 2.5
        # tokens that may not come next, as constrained decoding masks them
        x[:, torch.randint(case["vocab"], (case["vocab"] // 100,), generator=g,
                           device="cuda")] = float("-inf")
        s["logits"] = x
        s["tokens"] = torch.randint(case["vocab"], (case["rows"],), generator=g, device="cuda")
    return s


def run(state):
    case = state["case"]
    kind, window = case["kind"], case.get("window") or None
    if own:
        from newt_amd import workloads as W
        if kind == "rmsnorm":
            out = W.rmsnorm(state["x"], state["w"], eps=1e-6, residual=state["residual"],
                            out_dtype=DTYPES[case["out"]], group=case["group"] or None)
        elif kind == "window":
            return W.window_attention(state["q"], state["k"], state["v"], window,
                                      sinks=case["sinks"], q_start=state["start"])
        elif kind == "append":
            W.kv_append(W.KVCache(*state["cache"]), state["k"], state["v"], state["table"],
                        state["start"], count=state["count"])
            return state["cache"]
        elif kind == "cached":
            return W.cached_attention(state["q"], W.KVCache(*state["cache"]), state["table"],
                                      state["lens"], window=window, sinks=case["sinks"])
        else:
            out = W.token_logprobs(state["logits"], state["tokens"], top=case["top"],
                                   temperature=case["temperature"])
    elif kind == "rmsnorm":
        out = _rmsnorm(state["x"], state["w"], state["residual"], case)
    elif kind == "window":
        at = state["start"][:, None] + torch.arange(case["Sq"], device="cuda")
        return _attention(state["q"], state["k"].float(), state["v"].float(), at, case)
    elif kind == "append":
        return _append(state)
    elif kind == "cached":
        k, v, ks, vs = state["cache"]
        rows = state["table"].long()
        B, KV, D = case["B"], case["KV"], case["D"]
        k = k[rows].float() * ks[rows][..., None, None]  # [B, blocks, KV, block, D]
        v = v[rows].float() * vs[rows][..., None, None]  # [B, blocks, KV, D, block]
        at = state["lens"][:, None] - case["Sq"] + torch.arange(case["Sq"], device="cuda")
        return _attention(state["q"], k.transpose(1, 2).reshape(B, KV, -1, D),
                          v.permute(0, 2, 1, 4, 3).reshape(B, KV, -1, D), at, case)
    else:
        out = _logprobs(state["logits"], state["tokens"], case)
    return [x for x in out if x is not None]


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------
def _rmsnorm(x, w, residual, case):
    hidden = None
    if residual is not None:
        hidden = x = (x.float() + residual.float()).to(x.dtype)
    y = x.float()
    y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + 1e-6) * w.float()
    if case["out"] != "e4m3":
        return y.to(x.dtype), None, hidden
    groups = y.view(y.shape[0], -1, case["group"] or y.shape[1])
    scale = (groups.abs().amax(-1) / E4M3_MAX).clamp_min(TINY)
    q = (groups / scale[..., None]).clamp(-E4M3_MAX, E4M3_MAX).to(DTYPES["e4m3"])
    return q.view(y.shape), scale, hidden


def _attention(q, k, v, at, case):
    """q [B, H, Sq, D] at positions at [B, Sq] over k, v [B, KV, Sk, D] fp32."""
    B, H, Sq, D = q.shape
    KV, Sk = k.shape[1], k.shape[2]
    j = torch.arange(Sk, device="cuda")
    seen = j <= at[..., None]
    if case["window"]:
        seen &= (at[..., None] - j < case["window"]) | (j < case["sinks"])
    seen = seen[:, None, None]
    s = torch.matmul((q.float() * D ** -0.5).view(B, KV, -1, D),
                     k.transpose(-1, -2).contiguous()).view(B, KV, H // KV, Sq, Sk)
    s = s.masked_fill(~seen, float("-inf"))
    top = s.amax(-1, keepdim=True).clamp_min(-1e30)
    p = torch.exp(s - top)
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(B, KV, -1, Sk), v).view(B, KV, H // KV, Sq, D)
    return torch.where(total > 0, o / total, 0.0).view(B, H, Sq, D).to(q.dtype)


def _power_of_two(top):
    """The smallest power of two s with top <= 448 s, from 2^-100 on."""
    m, e = torch.frexp(top)  # top = m 2^e, m in [0.5, 1); 448 = 0.875 * 2^9
    e = torch.where(m > 0.875, e - 8, e - 9)
    return torch.where(top > 0, torch.exp2(e.clamp_min(-100).float()), 2.0 ** -100)


def _append(state):
    case, table, start, count = state["case"], state["table"], state["start"], state["count"]
    block, B = case["block"], case["B"]
    # the blocks that a sequence's new tokens reach, the last one repeated
    first, last = start // block, (start + count - 1) // block
    b = torch.arange(B, device="cuda")[:, None]
    slot = torch.minimum(first[:, None] + torch.arange(
        (case["S"] + block - 2) // block + 1, device="cuda"), last[:, None])
    page = table[b, slot].long()  # [B, n]
    token = slot[..., None] * block + torch.arange(block, device="cuda") - start[:, None, None]
    old = (token < 0)[:, :, None, None]
    new = ((token >= 0) & (token < count[:, None, None]))[:, :, None, None]
    token = token.clamp(0, case["S"] - 1)  # [B, n, block]
    for_v = (state["v"], state["cache"][1].transpose(-1, -2), state["cache"][3])
    for_k = (state["k"], state["cache"][0], state["cache"][2])
    _append_one(*for_k, b, page, token, old, new)
    _append_one(*for_v, b, page, token, old, new)
    return state["cache"]


def _append_one(x, pages, scales, b, page, token, old, new):
    """pages: [blocks, KV, block, D], a view of the cache."""
    x = x.transpose(1, 2)[b[..., None], token].float().permute(0, 1, 3, 4, 2)
    had = scales[page]
    need = _power_of_two(torch.where(new, x, 0.0).abs().amax((-1, -2)))
    scale = torch.where(old.any(-1)[..., 0], torch.maximum(had, need), need)
    values = pages[page].transpose(-1, -2)  # [B, n, KV, D, block]
    was = values.float() * (had / scale)[..., None, None]
    x = torch.where(new, x / scale[..., None, None], was)
    x = torch.where(old | new, x.to(DTYPES["e4m3"]).float(), values.float())
    pages[page] = x.transpose(-1, -2).to(DTYPES["e4m3"])
    scales[page] = scale


def _logprobs(logits, tokens, case):
    x = logits.float() / case["temperature"]
    top = x.amax(-1, keepdim=True)
    e = torch.exp(x - top)
    total = e.sum(-1, keepdim=True)
    lse = top + torch.log(total)
    spread = torch.where(e > 0, e * (x - top), 0.0).sum(-1, keepdim=True)
    entropy = (torch.log(total) - spread / total)[:, 0]
    logp = (torch.gather(x, 1, tokens[:, None]) - lse)[:, 0]
    if not case["top"]:
        return logp, entropy, None, None
    values, ids = torch.sort(logits, dim=-1, descending=True, stable=True)
    values, ids = values[:, :case["top"]], ids[:, :case["top"]].contiguous()
    return logp, entropy, values.float() / case["temperature"] - lse, ids


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------
def _e4m3(x):
    """x to the nearest number of 4 significant bits from 2^-6 on, a multiple
    of 2^-9 below, ties to even."""
    most = x.abs().clamp_min(2.0 ** -6)
    step = most / torch.frexp(most)[0] / 16  # a power of two, exactly
    return (x / step).round() * step


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "rmsnorm":
        x, hidden = s["x"].double(), None
        if case["residual"]:
            hidden = (x + s["residual"].double()).to(s["x"].dtype)
            x = hidden.double()
        y = x / (x.pow(2).sum(-1, keepdim=True) / case["cols"] + 1e-6).sqrt() * s["w"].double()
        scale = None
        if case["out"] == "e4m3":
            parts = y.unflatten(1, (-1, case["group"] or case["cols"]))
            scale = torch.clamp(parts.abs().amax(-1) / E4M3_MAX, min=TINY)
            y = _e4m3(parts / scale[..., None]).flatten(1)
        return [v.double() for v in (y, scale, hidden) if v is not None]
    if kind == "logprobs":
        x = s["logits"].double() / case["temperature"]
        logp = x - torch.logsumexp(x, -1, keepdim=True)
        entropy = -torch.nansum(logp.exp() * logp, -1)
        out = [torch.gather(logp, 1, s["tokens"][:, None])[:, 0], entropy]
        if case["top"]:
            out += [torch.sort(logp, -1, descending=True).values[:, :case["top"]], None]
        return out
    if kind == "append":
        return _exact_append(case, s)
    B, H, KV, Sq = case["B"], case["H"], case["KV"], case["Sq"]
    out = torch.zeros(B, H, Sq, case["D"], dtype=torch.float64, device="cuda")
    firsts = _starts(case) if kind == "window" else [n - Sq for n in _lens(case)]
    for b in range(B):
        for kv in range(KV):
            if kind == "window":
                k, v = s["k"][b, kv].double(), s["v"][b, kv].double()
            else:
                pages = s["table"][b].long()
                ks, vs = (c[pages, kv].double()[:, None, None] for c in s["cache"][2:])
                k = (s["cache"][0][pages, kv].double() * ks).flatten(0, 1)
                v = (s["cache"][1][pages, kv].double() * vs).transpose(1, 2).flatten(0, 1)
            p = torch.arange(firsts[b], firsts[b] + Sq, device="cuda")[:, None]
            j = torch.arange(len(k), device="cuda")[None]
            hidden = j > p
            if case["window"]:
                hidden = hidden | ((j <= p - case["window"]) & (j >= case["sinks"]))
            none = hidden.all(-1)[:, None]
            for h in range(kv * (H // KV), (kv + 1) * (H // KV)):
                score = s["q"][b, h].double() @ k.T / case["D"] ** 0.5
                weight = torch.softmax(score.masked_fill(hidden, -1e300), -1)
                out[b, h] = (weight @ v).masked_fill(none, 0.0)
    return out


def _exact_append(case, s):
    block = case["block"]
    out = [c.double() for c in s["cache"]]
    for b, (start, count) in enumerate(zip(*_appends(case))):
        for slot in range(start // block, (start + count - 1) // block + 1):
            page = int(s["table"][b, slot])
            lo, hi = max(start, slot * block), min(start + count, (slot + 1) * block)
            held = slice(0, lo - slot * block)
            put = slice(lo - slot * block, hi - slot * block)
            for x, pages, scales in ((s["k"], out[0], out[2]),
                                     (s["v"], out[1].transpose(-1, -2), out[3])):
                x = x[b, :, lo - start:hi - start].double()  # [KV, tokens, D]
                need = torch.exp2(torch.ceil(torch.log2(x.abs().amax((1, 2)) / E4M3_MAX)))
                had = scales[page].clone()
                scale = torch.maximum(had, need) if lo > slot * block else need
                pages[page][:, held] = _e4m3(pages[page][:, held] * (had / scale)[:, None, None])
                pages[page][:, put] = _e4m3(x / scale[:, None, None])
                scales[page] = scale
    return out
