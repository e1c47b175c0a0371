"""The serving operators from their definitions, in 64 bits and plain torch, a
row, a block or a head at a time. No counterpart in the reference.

Functions take tensors on any device and return float64 there (ids int64).
"""

import torch

E4M3_MAX = 448.0
LOWEST_SCALE = 2.0 ** -100


def round_e4m3(x):
    """x, |x| <= 464, to the nearest e4m3 number: 4 significant bits from 2^-6
    on, multiples of 2^-9 below, ties to even; not finite: NaN."""
    x = x.double()
    most = torch.where(x.isfinite(), x.abs(), 1.0).clamp_min(2.0 ** -6)
    step = most / torch.frexp(most)[0] / 16.0  # a power of two, exactly
    return torch.where(x.isfinite(), (x / step).round() * step, float("nan"))


def rmsnorm(x, w, eps, residual=None):
    """(y, hidden): hidden is rounded as the operator rounds it, x + residual
    in fp32 (exact or itself rounded once) and then to x's dtype."""
    hidden = None
    if residual is not None:
        hidden = x = (x.float() + residual.float()).to(x.dtype)
    x = x.double()
    return x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * w.double(), hidden


def scales(y, group=None):
    """[M, groups] scales of rows y in 8 bits; NaN does not count."""
    parts = y.view(y.shape[0], -1, group or y.shape[1]).abs().nan_to_num(nan=0.0, posinf=float("inf"))
    return (parts.amax(-1) / E4M3_MAX).clamp_min(2.0 ** -126)


def logprobs(logits, tokens, top=0, temperature=1.0):
    """(logp, entropy, top_logp, top_ids)"""
    x = logits.double() / temperature
    bad = (x.isnan() | (x == float("inf"))).any(-1) | (x == float("-inf")).all(-1)
    x = torch.where(bad[:, None], float("nan"), x)
    logs = torch.log_softmax(x, -1)
    p = logs.exp()
    entropy = -torch.where(p == 0, 0.0, p * logs).sum(-1)
    V = logits.shape[1]
    inside = (tokens >= 0) & (tokens < V)
    logp = logs.gather(1, tokens.clamp(0, V - 1)[:, None])[:, 0]
    logp = torch.where(tokens == -1, 0.0, torch.where(inside, logp, float("nan")))
    if not top:
        return logp, entropy, None, None
    order = torch.where(logits.isnan(), float("-inf"), logits.double())
    ids = torch.sort(order, dim=-1, descending=True, stable=True).indices
    # NaN behind everything else, -inf too
    ids = torch.stack([torch.cat([r[~logits[i, r].isnan()], r[logits[i, r].isnan()]])
                       for i, r in enumerate(ids)])[:, :top]
    none = logits.gather(1, ids).isnan()
    return logp, entropy, logs.gather(1, ids), torch.where(none, -1, ids)


def power_of_two(top):
    """The smallest power of two s >= LOWEST_SCALE with top <= 448 s."""
    s = LOWEST_SCALE
    while top > E4M3_MAX * s:
        s *= 2.0
    return s


def append(cache, k, v, table, start, count=None):
    """The cache (k, v, k_scale, v_scale) after the call, as float64 numbers of
    its bytes, and its scales."""
    out = [c.double().clone() for c in cache]
    size = cache[0].shape[2]
    B, heads, S, _ = k.shape
    for b in range(B):
        first, n = int(start[b]), S if count is None else min(int(count[b]), S)
        if first < 0 or n <= 0:
            continue
        for slot in range(first // size, (first + n - 1) // size + 1):
            if slot >= table.shape[1] or not 0 <= int(table[b, slot]) < len(out[0]):
                continue
            page = int(table[b, slot])
            lo, hi = max(first, slot * size), min(first + n, (slot + 1) * size)
            held, end = lo - slot * size, hi - slot * size
            for x, pages, scale in ((k, out[0], out[2]), (v, out[1].transpose(-1, -2), out[3])):
                for h in range(heads):
                    new = x[b, h, lo - first:hi - first].double()
                    top = float(torch.where(new.isfinite(), new.abs(), 0.0).max())
                    s, had = power_of_two(top), float(scale[page, h])
                    if held and had > s:
                        s = had
                    pages[page, h, :held] = round_e4m3(pages[page, h, :held] * (had / s))
                    pages[page, h, held:end] = round_e4m3(new / s)
                    scale[page, h] = s
    return out


def cached(cache, table, b, n):
    """Keys and values [kv_heads, n, D] of sequence b's first n positions, and
    which of them the cache has."""
    k, v, ks, vs = cache
    blocks, heads, size, D = k.shape
    keys, values = (torch.zeros(heads, n, D, dtype=torch.float64, device=k.device) for _ in range(2))
    has = torch.zeros(n, dtype=torch.bool, device=k.device)
    for slot in range(min(-(-n // size), table.shape[1])):
        page, m = int(table[b, slot]), min(size, n - slot * size)
        if not 0 <= page < blocks:
            continue
        at = slice(slot * size, slot * size + m)
        keys[:, at] = k[page, :, :m].double() * ks[page].double()[:, None, None]
        values[:, at] = (v[page].double() * vs[page].double()[:, None, None]).transpose(1, 2)[:, :m]
        has[at] = True
    return keys, values, has


def attention(q, k, v, positions, window=None, sinks=0, scale=None, has=None):
    """(o, a): outputs of q [H, S, D] at positions [S] over k and v [kv_heads,
    n, D], and sum p |v| beside them, what roundings of the weights p are
    relative to. `has` [n]: the keys that there are."""
    H, S, D = q.shape
    heads, n = k.shape[0], k.shape[1]
    scale = D ** -0.5 if scale is None else scale
    o = torch.zeros(H, S, D, dtype=torch.float64, device=q.device)
    a = torch.zeros_like(o)
    for i in range(S):
        p = int(positions[i])
        j = torch.arange(n, device=q.device)
        seen = j <= p
        if window is not None:
            seen &= (p - j < window) | (j < sinks)
        if has is not None:
            seen &= has
        j = j[seen]
        if len(j) == 0:
            continue
        for h in range(heads):
            at = slice(h * (H // heads), (h + 1) * (H // heads))
            w = torch.softmax(q[at, i].double() @ k[h, j].double().T * scale, -1)
            o[at, i] = w @ v[h, j].double()
            a[at, i] = w @ v[h, j].double().abs()
    return o, a
