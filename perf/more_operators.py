"""The rest of a decoder's step, as cases that can be timed and checked: products
with 4-bit weights, alone and as the gated half of a feed-forward block, rotary
positions of queries and keys, and the choice of the next tokens from their
logits.

A case is a dict of plain values. `listed` names twelve; `draw` gives more of
the same ranges. `prepare` makes what a program holds before the call. `run`
makes one call: of the framework's operators where `own` is true, else of their
plain forms in torch. `exact` computes the results in 64 bits from the
definitions, `work` the bytes and operations that a call cannot do without.
"""

import math

import numpy
import torch

own = False

DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"fp32": 4, "fp16": 2, "bf16": 2}


def listed():
    return [
        # the query, key and value products of one token: nothing but the
        # weights' bytes
        {"name": "q4_bf16_1x4096x6144", "kind": "q4", "dtype": "bf16", "rows": 1, "K": 4096,
         "N": 6144, "group": 128, "zeros": True, "bias": True, "out": "bf16"},
        # the logits of four sequences over a vocabulary, to be sampled in fp32
        {"name": "q4_bf16_4x4096x128000_fp32", "kind": "q4", "dtype": "bf16", "rows": 4, "K": 4096,
         "N": 128000, "group": 128, "zeros": False, "bias": False, "out": "fp32"},
        # a ragged chunk of a prompt, small groups, an odd number of outputs
        {"name": "q4_fp16_333x8192x2003", "kind": "q4", "dtype": "fp16", "rows": 333, "K": 8192,
         "N": 2003, "group": 32, "zeros": True, "bias": False, "out": "fp16"},
        # a feed-forward block's first half for one token
        {"name": "gated_bf16_1x4096x12288", "kind": "gated", "dtype": "bf16", "rows": 1, "K": 4096,
         "F": 12288, "group": 128, "zeros": True, "act": "silu"},
        # ... for one step of 48 sequences
        {"name": "gated_fp16_48x2048x5504", "kind": "gated", "dtype": "fp16", "rows": 48, "K": 2048,
         "F": 5504, "group": 64, "zeros": False, "act": "gelu"},
        # ... for a chunk of prompts, where the products take longer than the bytes
        {"name": "gated_bf16_512x4096x12288", "kind": "gated", "dtype": "bf16", "rows": 512,
         "K": 4096, "F": 12288, "group": 128, "zeros": True, "act": "silu"},
        # one token's queries and keys: the call is the cost
        {"name": "rotate_bf16_1x32+8x1x128", "kind": "rotate", "dtype": "bf16", "B": 1, "H": 32,
         "KV": 8, "S": 1, "D": 128, "rot": 128, "interleaved": False, "scaled": "none",
         "far": 8191, "each": False, "fused": True},
        # a ragged batch, half of each head turned, every token with a position
        # of its own in a context that is stretched 32 times
        {"name": "rotate_fp16_3x16+16x333x64", "kind": "rotate", "dtype": "fp16", "B": 3, "H": 16,
         "KV": 16, "S": 333, "D": 64, "rot": 32, "interleaved": True, "scaled": "ramp",
         "far": 131072, "each": True, "fused": False},
        # prompts of the attention benchmark's size, as slices of one product
        {"name": "rotate_bf16_4x32+8x4096x128", "kind": "rotate", "dtype": "bf16", "B": 4, "H": 32,
         "KV": 8, "S": 4096, "D": 128, "rot": 128, "interleaved": False, "scaled": "all",
         "far": 4096, "each": False, "fused": True},
        # the next token of one sequence
        {"name": "sample_bf16_1x128000", "kind": "sample", "dtype": "bf16", "rows": 1,
         "vocab": 128000, "filters": "all"},
        # 64 sequences, each with settings of its own
        {"name": "sample_fp32_64x32000", "kind": "sample", "dtype": "fp32", "rows": 64,
         "vocab": 32000, "filters": "mixed"},
        # many sequences by mass alone, an odd vocabulary
        {"name": "sample_bf16_256x100003", "kind": "sample", "dtype": "bf16", "rows": 256,
         "vocab": 100003, "filters": "p"},
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
    kind = rng.choice(("q4", "q4", "gated", "gated", "rotate", "rotate", "sample", "sample"))
    dtype = rng.choice(("bf16", "bf16", "fp16"))
    if kind == "sample":
        vocab = _log_int(rng, 1000, 200000)
        return {"kind": kind, "dtype": rng.choice((dtype, "fp32")),
                "rows": _log_int(rng, 1, min(512, 25600000 // vocab)), "vocab": vocab,
                "filters": rng.choice(("none", "k", "p", "min", "all", "mixed"))}
    if kind == "rotate":
        D = rng.choice((64, 80, 128, 128, 256))
        KV = rng.choice((1, 2, 4, 8, 16))
        H = KV * rng.choice((1, 2, 4, 8))
        S = 1 if rng.random() < 0.4 else _log_int(rng, 2, 8192)
        return {"kind": kind, "dtype": rng.choice((dtype, dtype, "fp32")),
                "B": _log_int(rng, 1, max(1, min(64, (1 << 26) // (S * (H + KV) * D)))), "H": H,
                "KV": KV, "S": S, "D": D, "rot": rng.choice((D, D, D // 2)),
                "interleaved": rng.random() < 0.4, "scaled": rng.choice(("none", "all", "ramp")),
                "far": _log_int(rng, S, 1 << 20), "each": rng.random() < 0.3,
                "fused": rng.random() < 0.5}
    rows = 1 if rng.random() < 0.3 else _log_int(rng, 2, 512)
    group = rng.choice((32, 64, 128, 128))
    K = max(group, -(-_log_int(rng, 256, 16384) // group) * group)
    each = {"kind": kind, "dtype": dtype, "rows": rows, "K": K}
    rest = {"group": group, "zeros": rng.random() < 0.5}
    most = min(1 << 29, (1 << 35) // rows) // K
    if kind == "q4":
        return {**each, "N": _size(rng, 16, min(131072, most)), **rest, "bias": rng.random() < 0.3,
                "out": rng.choice((dtype, dtype, "fp32"))}
    return {**each, "F": _size(rng, 16, min(32768, most // 2)), **rest,
            "act": rng.choice(("silu", "gelu"))}


def _outputs(case):
    """How many rows the 4-bit weights have: a gated product's are those of the
    gate, then those of what is gated."""
    return case["N"] if case["kind"] == "q4" else 2 * case["F"]


def work(case):
    kind, size = case["kind"], SIZE[case["dtype"]]
    if kind == "sample":
        return {"bytes": case["rows"] * (case["vocab"] * size + 4 + 16 + 8), "flops": 0}
    if kind == "rotate":
        n = case["B"] * case["S"] * (case["H"] + case["KV"]) * case["D"]
        return {"bytes": 2 * n * size + 4 * case["B"] * (case["S"] if case["each"] else 1),
                "flops": 0}
    N, K, M = _outputs(case), case["K"], case["rows"]
    y = M * case["N"] * SIZE[case["out"]] if kind == "q4" else M * case["F"] * size
    bias = N * size if case.get("bias") else 0
    return {"bytes": N * K // 2 + N * (K // case["group"]) * (size + case["zeros"]) + M * K * size
            + y + bias, "flops": 2 * M * N * K}


# how far a context is stretched: (factor, (original length, low, high))
SCALED = {"none": (1.0, None), "all": (4.0, None), "ramp": (32.0, (4096, 1.0, 4.0))}
BASE = 500000.0


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    at = {"generator": g, "device": "cuda"}
    kind, t = case["kind"], DTYPES[case["dtype"]]
    s = {"case": case}
    if kind == "sample":
        T, V = case["rows"], case["vocab"]
        x = torch.randn(T, V, **at) * 2.5
        # half of the rows are sure of what comes next, and no row has some tokens
        x[::2] *= 1.6
        x.scatter_add_(1, torch.randint(V, (T, 8), **at), torch.rand(T, 8, **at) * 12.0)
        x[:, torch.randint(V, (V // 100,), **at)] = float("-inf")
        s["logits"], s["u"] = x.to(t), torch.rand(T, **at)
        s.update(_settings(case, g))
    elif kind == "rotate":
        B, H, KV, S, D = (case[k] for k in ("B", "H", "KV", "S", "D"))
        if case["fused"]:  # slices of one product's rows
            x = torch.randn(B, S, H + 2 * KV, D, **at).to(t).transpose(1, 2)
            s["q"], s["k"] = x[:, :H], x[:, H:H + KV]
        else:
            s["q"], s["k"] = (torch.randn(B, n, S, D, **at).to(t) for n in (H, KV))
        # the first tokens' positions, or those of several texts in a row
        start = torch.randint(max(1, case["far"] - S), (B,), **at)
        at_least = torch.randint(0, 3, (B, S), **at).cumsum(-1) % max(1, S)
        s["positions"] = (start[:, None] + at_least if case["each"] else start).to(torch.int32)
        if own:
            from newt_amd import workloads as W
            factor, ramp = SCALED[case["scaled"]]
            s["rotary"] = W.rotary(case["rot"], base=BASE, factor=factor, ramp=ramp,
                                   interleaved=case["interleaved"])
    else:
        N, K, M = _outputs(case), case["K"], case["rows"]
        # activations with some channels that are larger than the others
        s["x"] = (torch.randn(M, K, **at) * torch.exp(torch.randn(K, **at) * 0.7)).to(t)
        q = torch.empty(N, K // 2, dtype=torch.uint8, device="cuda")  # the low half first
        for i in range(0, N, 16384):
            n = min(16384, N - i)
            v = (torch.randn(n, K, **at) * 2.7 + 8.0).round_().clamp_(0, 15).to(torch.uint8)
            q[i:i + n] = v[:, ::2] | v[:, 1::2] << 4
        scales = (torch.exp(torch.randn(N, K // case["group"], **at) * 0.3) * 0.4 / K ** 0.5).to(t)
        zeros = None
        if case["zeros"]:
            zeros = torch.randint(6, 11, scales.shape, **at).to(torch.uint8)
        s["w"] = (q, scales, zeros)
        s["bias"] = torch.randn(N, **at).to(t) if case.get("bias") else None
        if own:
            from newt_amd import workloads as W
            s["laid_out"] = W.q4_weights(q, scales, zeros, gated=kind == "gated")
    return s


def _settings(case, g):
    """Temperature, top_k, top_p and min_p: the same for all rows, or one each
    where requests come with their own (some of them greedy)."""
    T, filters = case["rows"], case["filters"]
    same = {"none": (1.0, 0, 1.0, 0.0), "k": (0.8, 50, 1.0, 0.0), "p": (1.0, 0, 0.9, 0.0),
            "min": (1.25, 0, 1.0, 0.05), "all": (0.75, 64, 0.95, 0.015625)}
    names = ("temperature", "top_k", "top_p", "min_p")
    if filters != "mixed":
        return dict(zip(names, same[filters]))
    at = {"generator": g, "device": "cuda"}

    def pick(values, dtype=torch.float32):
        return torch.tensor(values, device="cuda")[torch.randint(len(values), (T,), **at)].to(dtype)

    return dict(zip(names, (pick([0.0, 0.7, 1.0, 1.5]), pick([0, 0, 1, 40, 1000], torch.int32),
                            pick([1.0, 0.5, 0.9, 0.99]), pick([0.0, 0.0, 0.02, 0.1]))))


def run(state):
    case = state["case"]
    kind = case["kind"]
    if own:
        from newt_amd import workloads as W
        if kind == "sample":
            return W.sample(state["logits"], state["u"], state["temperature"], state["top_k"],
                            state["top_p"], state["min_p"])
        if kind == "rotate":
            return list(W.rotate(state["q"], state["k"], state["rotary"], state["positions"]))
        if kind == "gated":
            return W.q4_gated(state["x"], state["laid_out"], act=case["act"])
        return W.q4_matmul(state["x"], state["laid_out"], bias=state["bias"],
                           out_dtype=DTYPES[case["out"]])
    if kind == "sample":
        return _sample(state)
    if kind == "rotate":
        return _rotate(state)
    y = torch.matmul(state["x"].float(), _weights(state["w"], case).t())
    if kind == "q4":
        if case["bias"]:
            y = y + state["bias"].float()
        return y.to(DTYPES[case["out"]])
    gate, up = y[:, :case["F"]], y[:, case["F"]:]
    if case["act"] == "silu":
        gate = gate / (1.0 + torch.exp(-gate))
    else:
        gate = gate * 0.5 * (1.0 + torch.erf(gate * 0.5 ** 0.5))
    return (gate * up).to(state["x"].dtype)


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------
def _weights(w, case):
    """[N, K] fp32: (q - zero) * scale, zero 8 where there are none."""
    q, scales, zeros = w
    v = torch.stack((q & 15, q >> 4), -1).view(q.shape[0], -1, case["group"]).float()
    v = v - (8.0 if zeros is None else zeros.float()[..., None])
    return (v * scales.float()[..., None]).flatten(1)


def _frequencies(case):
    """Radians a position of each pair, in 64 bits."""
    rot = case["rot"]
    f = BASE ** (-torch.arange(0, rot, 2, dtype=torch.float64, device="cuda") / rot)
    factor, ramp = SCALED[case["scaled"]]
    if ramp is None:
        return f / factor
    # what turns less than `low` times over the original length is stretched,
    # what turns `high` times is not
    original, low, high = ramp
    keep = ((original * f / (2 * math.pi) - low) / (high - low)).clamp(0.0, 1.0)
    return f * keep + f / factor * (1.0 - keep)


def _rotate(state):
    case, positions = state["case"], state["positions"]
    if not case["each"]:
        positions = positions[:, None] + torch.arange(case["S"], device="cuda")
    angle = positions.double()[:, None, :, None] * _frequencies(case)
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    rot, out = case["rot"], []
    for x in (state["q"], state["k"]):
        y = x.contiguous()
        turned = y[..., :rot].float()
        if case["interleaved"]:
            a, b = turned[..., ::2], turned[..., 1::2]
            turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
        else:
            a, b = turned.chunk(2, -1)
            turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
        out.append(torch.cat((turned.to(x.dtype), y[..., rot:]), -1))
    return out


def _sample(state):
    logits, u = state["logits"], state["u"].double()[:, None]
    T, V = logits.shape

    def column(name):
        v = state[name]
        if not isinstance(v, torch.Tensor):
            v = torch.full((T,), v, dtype=torch.int32 if name == "top_k" else torch.float32,
                           device="cuda")
        return v[:, None]

    t, k = column("temperature").double(), column("top_k").long()
    p, least = column("top_p").double(), column("min_p").double()
    order = torch.sort(logits, dim=-1, descending=True, stable=True).indices
    x = logits.double()
    w = torch.exp((x - x.amax(-1, keepdim=True)) / torch.where(t > 0, t, 1.0))
    w = torch.gather(w, 1, order)  # the largest first, the lowest index among equal ones
    rank = torch.arange(V, device="cuda")
    kept = torch.where(rank < torch.where(k > 0, k, V), w, 0.0)
    mass = kept.cumsum(-1)
    # a token stays while those before it are less than top_p of the mass
    stays = ((mass - kept < p * mass[:, -1:]) | (p >= 1.0)) & (kept >= least) | (rank == 0)
    kept = torch.zeros_like(w).scatter_(1, order, torch.where(stays, kept, 0.0))
    mass = kept.cumsum(-1)  # in the order of the vocabulary
    ids = (mass <= u * mass[:, -1:]).sum(-1)
    return torch.where(t[:, 0] > 0, ids, order[:, 0])


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "sample":
        return _exact_sample(case, s)
    if kind == "rotate":
        return [_exact_rotate(case, x, s["positions"]) for x in (s["q"], s["k"])]
    x = s["x"].double()
    q, scales, zeros = s["w"]
    y = torch.empty(len(x), len(q), dtype=torch.float64, device="cuda")
    for i in range(0, len(q), 4096):
        rows = slice(i, i + 4096)
        w = torch.empty(len(q[rows]), case["K"], dtype=torch.float64, device="cuda")
        w[:, 0::2], w[:, 1::2] = q[rows] % 16, q[rows] // 16
        less = 8 if zeros is None else torch.repeat_interleave(zeros[rows].double(), case["group"], 1)
        w -= less
        w *= torch.repeat_interleave(scales[rows].double(), case["group"], 1)
        y[:, rows] = x @ w.T
    if kind == "q4":
        return y + s["bias"].double() if case["bias"] else y
    gate = y[:, :case["F"]]
    if case["act"] == "silu":
        gate = gate * torch.sigmoid(gate)
    else:
        gate = gate * 0.5 * torch.special.erfc(-gate / math.sqrt(2.0))
    return gate * y[:, case["F"]:]


def _exact_rotate(case, x, positions):
    """Pairs as complex numbers times e^(i position frequency)."""
    rot, S = case["rot"], case["S"]
    factor, ramp = SCALED[case["scaled"]]
    turns = []
    for i in range(rot // 2):
        f = math.exp(-2.0 * i / rot * math.log(BASE))
        share = 0.0  # of the frequency as it is
        if ramp is not None:
            share = min(1.0, max(0.0, (ramp[0] * f / math.tau - ramp[1]) / (ramp[2] - ramp[1])))
        turns.append(f * share + (1.0 - share) * f / factor)
    at = positions.double()
    if not case["each"]:
        at = at[:, None] + torch.arange(S, dtype=torch.float64, device="cuda")
    angle = at[..., None] * torch.tensor(turns, dtype=torch.float64, device="cuda")
    by = torch.polar(torch.ones_like(angle), angle)[:, None]
    y = x.double()
    if case["interleaved"]:
        pairs = torch.view_as_complex(y[..., :rot].unflatten(-1, (-1, 2)).contiguous())
        out = torch.view_as_real(pairs * by).flatten(-2)
    else:
        z = torch.complex(y[..., :rot // 2], y[..., rot // 2:rot]) * by
        out = torch.cat((z.real, z.imag), -1)
    return torch.cat((out, y[..., rot:]), -1)


def _exact_sample(case, s):
    """A row at a time: the smallest logit that stays and how many of those
    equal to it do, then the first token whose running weight passes u's."""
    T, V = case["rows"], case["vocab"]
    if T * V > 1 << 26:
        return None
    logits, u = s["logits"].float().cpu().numpy().astype(numpy.float64), s["u"].cpu().numpy()
    settings = []
    for name in ("temperature", "top_k", "top_p", "min_p"):
        v = s[name]
        v = v.cpu().numpy() if isinstance(v, torch.Tensor) else numpy.full(T, v, numpy.float32)
        settings.append(v.astype(numpy.float64))
    ids = numpy.empty(T, numpy.int64)
    for r, (t, k, p, least) in enumerate(zip(*settings)):
        x = logits[r]
        if t == 0:
            ids[r] = x.argmax()
            continue
        w = numpy.exp((x - x.max()) / t)
        down = numpy.sort(x)[::-1]
        n = min(int(k), V) if k > 0 else V
        run = numpy.cumsum(numpy.exp((down[:n] - x.max()) / t))
        if p < 1.0:
            n = min(n, 1 + int(numpy.searchsorted(run, p * run[-1])))
        n = max(1, min(n, int((w >= least).sum())))
        stays = x > down[n - 1]
        ties = numpy.flatnonzero(x == down[n - 1])
        stays[ties[:n - int(stays.sum())]] = True
        mass = numpy.cumsum(numpy.where(stays, w, 0.0))
        ids[r] = numpy.searchsorted(mass, float(u[r]) * mass[-1], side="right")
    return torch.from_numpy(ids)
