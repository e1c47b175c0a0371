"""The operators of newt_amd/serving.py that turn, project and choose, in 64 bits
from their definitions: rotary positions, products with 4-bit weights, sampling."""

import math

import torch


def frequencies(dim, base=10000.0, factor=1.0, ramp=None, given=None):
    """Radians a position, one a pair."""
    out = []
    for i in range(dim // 2):
        f = float(base) ** (-2.0 * i / dim) if given is None else float(given[i])
        share = 0.0
        if ramp is not None:
            original, low, high = ramp
            share = min(1.0, max(0.0, (original * abs(f) / (2 * math.pi) - low) / (high - low)))
        out.append(f * share + f / factor * (1.0 - share))
    return torch.tensor(out, dtype=torch.float64)


def rotate(x, freqs, positions, interleaved=False, amplitude=1.0, transposed=False):
    """x [B, H, S, D] on the CPU; positions [B, S] of whole numbers."""
    x = x.double()
    n = len(freqs)
    angle = positions.double()[:, None, :, None] * freqs
    cos, sin = torch.cos(angle) * amplitude, torch.sin(angle) * amplitude
    if transposed:
        sin = -sin
    ia = torch.arange(n) * 2 if interleaved else torch.arange(n)
    ib = ia + 1 if interleaved else ia + n
    y = x.clone()
    y[..., ia] = x[..., ia] * cos - x[..., ib] * sin
    y[..., ib] = x[..., ib] * cos + x[..., ia] * sin
    return y


def q4(x, q, scales, zeros=None):
    """(x times the transposed weights, the sum of the products' absolute values)."""
    numbers = torch.stack((q & 15, q >> 4), -1).flatten(1).double()
    group = numbers.shape[1] // scales.shape[1]
    z = 8.0 if zeros is None else zeros.double().repeat_interleave(group, 1)
    w = (numbers - z) * scales.double().repeat_interleave(group, 1)
    return x.double() @ w.T, x.double().abs() @ w.abs().T


def activate(v, act):
    if act == "silu":
        return v * torch.sigmoid(v)
    return v * 0.5 * (1.0 + torch.erf(v / math.sqrt(2.0)))


def kept_weights(x, temperature, top_k=0, top_p=1.0, min_p=0.0):
    """The weights of one row of logits (64 bits) after the filters, 0 elsewhere."""
    V = len(x)
    order = torch.sort(x, descending=True, stable=True).indices
    w = torch.exp((x - x.max()) / temperature)
    ranked = w[order]
    n = min(top_k, V) if top_k > 0 else V
    if top_p < 1.0:
        run = ranked[:n].cumsum(0)
        before = torch.cat((run.new_zeros(1), run[:-1]))
        n = max(1, int((before < top_p * run[-1]).sum()))
    n = max(1, min(n, int((ranked >= min(min_p, 1.0)).sum())))
    out = torch.zeros_like(w)
    out[order[:n]] = ranked[:n]
    return out


def sample(x, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """The chosen id of one row, or -1."""
    x = x.double().cpu()
    settings = (u, temperature, top_p, min_p)
    if (bool(x.isnan().any()) or not math.isfinite(float(x.max())) or any(v != v for v in settings)
            or not 0 <= temperature < math.inf):
        return -1
    if temperature == 0:
        return int(torch.argmax((x == x.max()).int()))
    mass = kept_weights(x, temperature, top_k, top_p, min_p).cumsum(0)
    u = min(max(u, 0.0), 1.0 - 2.0 ** -53)
    return int((mass <= u * mass[-1]).sum())
