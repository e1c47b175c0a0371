"""The operators of a decoder's serving step, as hand-written gfx950 kernels.

They stand beside the kernels of `newt_amd.workloads`, which re-exports them:
`rmsnorm` beside `layernorm`, `window_attention` and `cached_attention` beside
`attention`, `token_logprobs` and `sample` beside `softmax`, `q4_matmul` and
`q4_gated` beside `matmul`, `rotate` in front of `kv_append`. All are forward
only, as the others are (`rotate` transposed is its own gradient). The kernels
are in csrc/ops, behind the C ABI of include/newt_ops.h; they are compiled ahead
of time, so a first call costs no compilation.

As everywhere in newt, tensors have to be on the current GPU, a call launches
on torch's current stream, synchronizes nothing and can be captured into a
graph. Outputs that are not given are new tensors. Wrong arguments raise
TypeError (kind of argument, device, dtype) or ValueError (shape, stride,
range) before anything is launched.

One step of a decoder layer over the 8-bit cache:

    x, _, hidden = rmsnorm(x, w_norm, residual=hidden)
    q, k, v = ...                      # slices of q4_matmul(x, w_qkv), [B, heads, S, D]
    q, k = rotate(q, k, turns, lens - S)             # turns = rotary(D), once
    kv_append(cache, k, v, block_table, lens - S)
    o = cached_attention(q, cache, block_table, lens)
    o = o.transpose(1, 2).reshape(B * S, -1)         # a row a token again
    x, _, hidden = rmsnorm(q4_matmul(o, w_out), w_norm2, residual=hidden)
    x = q4_matmul(q4_gated(x, w_gate_up), w_down)

and after the last one ids = sample(q4_matmul(x, w_vocab), u, top_p=0.9).
"""

import ctypes
import decimal
import functools
import math
import os
import struct
from typing import NamedTuple

import torch

from .runtime import hip as _hip
from .runtime.jit import _Dev

LIB_PATH = os.path.join(os.path.dirname(os.path.abspath(__file__)), "csrc", "libnewt_ops.so")

E4M3 = torch.float8_e4m3fn
_DTYPE = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2, E4M3: 3}
_HEAD_DIMS = (64, 128, 256)
_BLOCK_SIZES = (16, 32, 64, 128, 256)

# the structs of include/newt_ops.h, field by field
_RMSNORM = struct.Struct("=6Q6qf5i")
_LOGPROBS = struct.Struct("=7Q3qf3i")
_CACHE = "4Qq4i"
_APPEND = struct.Struct("=" + _CACHE + "5Q10q2i")
_CACHED = struct.Struct("=" + _CACHE + "5Q12qf3i")
_WINDOW = struct.Struct("=6Q17qf5i")
_ROTATE = struct.Struct("=6Q20qf5i")
_Q4 = struct.Struct("=7Q5q6i")
_SAMPLE = struct.Struct("=8Q3q3f3i")


@functools.cache
def lib():
    _hip.lib()  # torch's HIP runtime first, then ours binds to the same
    if not os.path.exists(LIB_PATH):
        raise RuntimeError(
            f"newt: the operator library {LIB_PATH} is not built; run "
            f"`python -c 'import __graft_entry__ as g; g.build()'` or "
            f"`python -m newt_amd.build`")
    L = ctypes.CDLL(LIB_PATH)
    for name in ("newt_rmsnorm", "newt_token_logprobs", "newt_kv_append", "newt_cached_attention",
                 "newt_window_attention", "newt_rotate", "newt_q4_matmul", "newt_sample"):
        f = getattr(L, name)
        f.restype, f.argtypes = ctypes.c_int, [ctypes.c_char_p, ctypes.c_void_p]
    for name in ("newt_cached_attention_workspace", "newt_window_attention_workspace",
                 "newt_q4_matmul_workspace"):
        f = getattr(L, name)
        f.restype, f.argtypes = ctypes.c_size_t, [ctypes.c_char_p]
    L.newt_token_logprobs_workspace.restype = ctypes.c_size_t
    L.newt_token_logprobs_workspace.argtypes = [ctypes.c_int64, ctypes.c_int64, ctypes.c_int32,
                                                ctypes.c_int32]
    L.newt_sample_workspace.restype = ctypes.c_size_t
    L.newt_sample_workspace.argtypes = [ctypes.c_int64, ctypes.c_int64, ctypes.c_int32]
    L.newt_ops_last_error.restype = ctypes.c_char_p
    if L.newt_ops_abi_version() != 1:
        raise RuntimeError("newt: libnewt_ops.so ABI mismatch; rebuild it")
    return L


class _Fast:
    """The operators' ordinary calls in C++ (csrc/newt_pyops.cpp, the _newt_ops
    extension): each returns None for what is not plainly right, which the
    Python of this file then looks into. Where the extension is not built, all
    calls go through Python."""

    module = None

    @classmethod
    def load(cls):
        lib()
        try:
            import importlib.util
            import sysconfig
            path = os.path.join(os.path.dirname(LIB_PATH),
                                "_newt_ops" + sysconfig.get_config_var("EXT_SUFFIX"))
            spec = importlib.util.spec_from_file_location("_newt_ops", path)
            module = importlib.util.module_from_spec(spec)
            spec.loader.exec_module(module)
        except (ImportError, OSError):
            module = False
        cls.module = module
        return module


def _fast(name, *args):
    module = _Fast.module
    if module is None:
        module = _Fast.load()
    if not module:
        return None
    device = _Dev.device()
    return getattr(module, name)(*args, device, _Dev.stream(device))


def _call(entry, what, params, device):
    status = entry(params, _Dev.stream(device))
    if status:
        detail = (lib().newt_ops_last_error() or b"").decode(errors="replace")
        raise (ValueError if status >= 10000 else _hip.HIPError)(f"{what}: {detail}")


def _tensors(what, device, optional=None, **tensors):
    """All are tensors on the current GPU; `optional` ones may be None."""
    tensors.update((name, t) for name, t in (optional or {}).items() if t is not None)
    for name, t in tensors.items():
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{what}: {name} must be a tensor")
    for name, t in tensors.items():
        if not t.is_cuda or t.device.index != device:
            raise TypeError(f"{what}: {name} must be on the current GPU")


def _shape(what, name, t, shape, dtype=None):
    if t.shape != shape:
        raise ValueError(f"{what}: {name} has shape {tuple(t.shape)}, not {tuple(shape)}")
    if dtype is not None and t.dtype != dtype:
        raise TypeError(f"{what}: {name} is {t.dtype}, not {dtype}")


def _whole(what, name, value, least):
    if isinstance(value, bool) or not isinstance(value, int):
        raise TypeError(f"{what}: {name} must be an int")
    if not least <= value < 2 ** 30:
        raise ValueError(f"{what}: {name}={value} is out of range")


def _fp32(value):
    """A number as fp32 holds it, infinite beyond its range, as a cast in C++."""
    try:
        return ctypes.c_float(float(value)).value
    except OverflowError:  # an int that no double holds
        return math.inf if value > 0 else -math.inf


def _ptr(t):
    return 0 if t is None else t.data_ptr()


# ---------------------------------------------------------------------------
# root-mean-square norm
# ---------------------------------------------------------------------------
def rmsnorm(x, w, eps=1e-6, residual=None, out_dtype=None, group=None, out=None, hidden=None):
    """(out, scale, hidden) of the root-mean-square norm of x [M, N] fp32, fp16
    or bf16, whose rows may be strided:

        hidden = x + residual              (rounded to x's dtype; None without)
        y = hidden * rsqrt(mean(hidden^2) + eps) * w

    computed in fp32 (the squares' sum too: rows of numbers around 1e19 give 0).
    w [N] is of x's dtype or fp32, residual [M, N] of x's.
    `out` is y in x's dtype (scale None), or with out_dtype=float8_e4m3fn y /
    scale in 8 bits, with fp32 scales [M, 1] of whole rows, or [M, N / group] of
    `group` (32, 64, 128, 256) columns each: scale = max(amax |y| / 448, 2^-126),
    NaN not counted; under an infinity all numbers become 0. newt has no product
    of 8-bit operands: this output is for ones outside of it. `out` and `hidden`
    given may be x or residual itself, and overlap nothing else."""
    r = _fast("rmsnorm", x, w, eps, residual, -1 if out_dtype is None else
              _DTYPE.get(out_dtype, -2), group, out, hidden)
    if r is not None:
        return r
    device = _Dev.device()
    _tensors("rmsnorm", device, {"residual": residual, "out": out, "hidden": hidden}, x=x, w=w)
    if x.dim() != 2 or x.shape[1] == 0:
        raise ValueError(f"rmsnorm: x has shape {tuple(x.shape)}, not [M, N]")
    dtype = x.dtype
    if dtype not in _DTYPE or dtype == E4M3:
        raise TypeError(f"rmsnorm: x is {dtype}")
    M, N = x.shape
    if w.dtype != dtype and w.dtype != torch.float32:
        raise TypeError(f"rmsnorm: w is {w.dtype}, not {dtype} or float32")
    _shape("rmsnorm", "w", w, (N,))
    out_dtype = dtype if out_dtype is None else out_dtype
    if out_dtype != dtype and out_dtype != E4M3:
        raise TypeError(f"rmsnorm: no {out_dtype} output of {dtype}")
    scale = None
    if group is not None:
        if out_dtype != E4M3:
            raise ValueError("rmsnorm: a group needs an 8-bit output")
        if group not in (32, 64, 128, 256) or N % group:
            raise ValueError(f"rmsnorm: no groups of {group} in {N} columns")
    if out is None:
        out = torch.empty((M, N), dtype=out_dtype, device=x.device)
    else:
        _shape("rmsnorm", "out", out, (M, N), out_dtype)
    if out_dtype == E4M3:
        scale = torch.empty((M, N // group if group else 1), dtype=torch.float32, device=x.device)
    if residual is not None:
        _shape("rmsnorm", "residual", residual, (M, N), dtype)
        if hidden is None:
            hidden = torch.empty((M, N), dtype=dtype, device=x.device)
        else:
            _shape("rmsnorm", "hidden", hidden, (M, N), dtype)
    elif hidden is not None:
        raise ValueError("rmsnorm: hidden is an output of the residual's addition")
    sx, so = x.stride(), out.stride()
    sr = (0, 1) if residual is None else residual.stride()
    sh = (0, 1) if hidden is None else hidden.stride()
    if N > 1 and not sx[1] == so[1] == sr[1] == sh[1] == w.stride(0) == 1:
        raise ValueError("rmsnorm: rows and w need unit stride")
    if M > 1 and (so[0] < N or (hidden is not None and sh[0] < N)):
        raise ValueError("rmsnorm: rows of an output overlap")
    _call(lib().newt_rmsnorm, "rmsnorm", _RMSNORM.pack(
        x.data_ptr(), _ptr(residual), w.data_ptr(), out.data_ptr(), _ptr(hidden), _ptr(scale),
        M, N, sx[0], sr[0], so[0], sh[0], _fp32(eps), _DTYPE[dtype], _DTYPE[w.dtype],
        _DTYPE[out_dtype], group or 0, 0), device)
    return out, scale, hidden


# ---------------------------------------------------------------------------
# log probabilities
# ---------------------------------------------------------------------------
def token_logprobs(logits, tokens, top=0, temperature=1.0):
    """(logp, entropy, top_logp, top_ids) of the distributions softmax(logits /
    temperature), logits [T, V] fp32, fp16 or bf16 with rows of any stride.

    logp [T] fp32: of tokens [T] int64. A token of -1 stands for none and gets
    0, another outside of the vocabulary NaN. entropy [T] fp32, in nats.
    top_logp [T, top] fp32 and top_ids [T, top] int64: the `top` (at most 64)
    largest, the lowest id first among equal logits; None for top=0. Logits of
    -inf have probability 0. A row that holds nothing else, a NaN or +inf gets
    NaN for all its values; NaN logits are not among its top_ids (-1 where
    there are too few others)."""
    r = _fast("token_logprobs", logits, tokens, top, temperature)
    if r is not None:
        return r
    device = _Dev.device()
    _tensors("token_logprobs", device, logits=logits, tokens=tokens)
    if logits.dim() != 2 or logits.shape[1] == 0:
        raise ValueError(f"token_logprobs: logits have shape {tuple(logits.shape)}, not [T, V]")
    if logits.dtype not in _DTYPE or logits.dtype == E4M3:
        raise TypeError(f"token_logprobs: logits are {logits.dtype}")
    T, V = logits.shape
    _shape("token_logprobs", "tokens", tokens, (T,), torch.int64)
    _whole("token_logprobs", "top", top, 0)
    if top > min(V, 64):
        raise ValueError(f"token_logprobs: no {top} alternatives of {V} (at most 64)")
    if not (temperature > 0 and 2.0 ** -100 < temperature < 2.0 ** 100):
        raise ValueError(f"token_logprobs: temperature {temperature}")
    if (V > 1 and logits.stride(1) != 1) or (T > 1 and tokens.stride(0) != 1):
        raise ValueError("token_logprobs: rows of logits and tokens need unit stride")
    f32 = {"dtype": torch.float32, "device": logits.device}
    # the logprobs, the entropies and, in rows, the alternatives
    values = torch.empty(T * (2 + top), **f32)
    logp, entropy, top_logp, top_ids = values[:T], values[T:2 * T], None, None
    if top:
        top_logp = values[2 * T:].view(T, top)
        top_ids = torch.empty((T, top), dtype=torch.int64, device=logits.device)
    L = lib()
    code = _DTYPE[logits.dtype]
    need = L.newt_token_logprobs_workspace(T, V, top, code)
    workspace = torch.empty(need, dtype=torch.uint8, device=logits.device) if need else None
    _call(L.newt_token_logprobs, "token_logprobs", _LOGPROBS.pack(
        logits.data_ptr(), tokens.data_ptr(), logp.data_ptr(), entropy.data_ptr(), _ptr(top_logp),
        _ptr(top_ids), _ptr(workspace), T, V, logits.stride(0), 1.0 / temperature, code, top, 0),
        device)
    return logp, entropy, top_logp, top_ids


# ---------------------------------------------------------------------------
# the 8-bit cache
# ---------------------------------------------------------------------------
class KVCache(NamedTuple):
    """Keys and values in 8 bits (float8_e4m3fn), in blocks of tokens with one
    fp32 scale, not negative, for each block and head; an element is its 8-bit
    number times its scale. A block's values lie transposed."""
    k: torch.Tensor        # [blocks, kv_heads, block_size, head_dim]
    v: torch.Tensor        # [blocks, kv_heads, head_dim, block_size]
    k_scale: torch.Tensor  # [blocks, kv_heads]
    v_scale: torch.Tensor  # [blocks, kv_heads]


def kv_cache(blocks, kv_heads, head_dim, block_size=64, device=None):
    """An empty KVCache. block_size is 16, 32, 64, 128 or 256 tokens, head_dim
    64, 128 or 256."""
    for name, value in (("blocks", blocks), ("kv_heads", kv_heads)):
        _whole("kv_cache", name, value, 1)
    if block_size not in _BLOCK_SIZES:
        raise ValueError(f"kv_cache: no blocks of {block_size} tokens {_BLOCK_SIZES}")
    if head_dim not in _HEAD_DIMS:
        raise ValueError(f"kv_cache: head_dim {head_dim} is not one of {_HEAD_DIMS}")
    device = torch.device("cuda", _Dev.device()) if device is None else device

    def zeros(*shape):
        return torch.zeros(shape, dtype=torch.uint8, device=device).view(E4M3)

    scales = [torch.zeros(blocks, kv_heads, dtype=torch.float32, device=device) for _ in range(2)]
    return KVCache(zeros(blocks, kv_heads, block_size, head_dim),
                   zeros(blocks, kv_heads, head_dim, block_size), *scales)


def _cache_tensors(what, cache, block_table):
    """What _tensors looks at of a cache and its table."""
    if not isinstance(cache, (tuple, list)):
        raise TypeError(f"{what}: cache must be a KVCache")
    if len(cache) != 4:
        raise ValueError(f"{what}: a cache has 4 tensors, not {len(cache)}")
    return dict(zip(("k_cache", "v_cache", "k_scale", "v_scale"), cache), block_table=block_table)


def _pages(what, cache, block_table, batch):
    """The checked cache as packed fields, the table's width and stride."""
    k, v, ks, vs = cache
    if k.dim() != 4:
        raise ValueError(f"{what}: the cache's keys have shape {tuple(k.shape)}, not [blocks, "
                         f"kv_heads, block_size, head_dim]")
    blocks, heads, size, dim = k.shape
    if size not in _BLOCK_SIZES or dim not in _HEAD_DIMS:
        raise ValueError(f"{what}: no cache with blocks of {size} tokens and head_dim {dim}")
    _shape(what, "v_cache", v, (blocks, heads, dim, size), E4M3)
    _shape(what, "k_scale", ks, (blocks, heads), torch.float32)
    _shape(what, "v_scale", vs, (blocks, heads), torch.float32)
    if k.dtype != E4M3:
        raise TypeError(f"{what}: k_cache is {k.dtype}, not {E4M3}")
    if not (k.is_contiguous() and v.is_contiguous() and ks.is_contiguous() and vs.is_contiguous()):
        raise ValueError(f"{what}: the cache has to be contiguous")
    kp, vp = k.data_ptr(), v.data_ptr()
    if (kp | vp) & 15:
        raise ValueError(f"{what}: keys and values of the cache have to be aligned to 16 bytes")
    if block_table.dtype != torch.int32:
        raise TypeError(f"{what}: block_table is {block_table.dtype}, not int32")
    if block_table.dim() != 2 or block_table.shape[0] != batch:
        raise ValueError(f"{what}: block_table has shape {tuple(block_table.shape)}, not "
                         f"[{batch}, blocks of a sequence]")
    width = block_table.shape[1]
    if width > 1 and block_table.stride(1) != 1:
        raise ValueError(f"{what}: rows of block_table need unit stride")
    if width * size >= 2 ** 30:
        raise ValueError(f"{what}: sequences of {width} blocks are too long")
    fields = (kp, vp, ks.data_ptr(), vs.data_ptr(), blocks, heads, size, dim, 0)
    return fields, heads, size, dim, width, block_table.stride(0)


def _per_sequence(what, name, t, batch):
    _shape(what, name, t, (batch,), torch.int32)
    if batch > 1 and t.stride(0) != 1:
        raise ValueError(f"{what}: {name} needs unit stride")


def kv_append(cache, k, v, block_table, start, count=None):
    """Writes new tokens' keys and values, k and v [B, kv_heads, S, head_dim]
    fp32, fp16 or bf16 (any strides but along head_dim), into the cache: of
    sequence b the first count[b] (all S without count, none below 1) to its
    positions start[b] on. block_table [B, n] int32 names the blocks that hold
    a sequence's positions, block_size each; start and count are [B] int32.

    A block's scale is the smallest power of two under which all that it holds
    fits, from 2^-100 on: set anew by the call that writes its first token,
    raised where a later token needs it (older ones are rounded to the new
    scale). Infinities and NaN are kept as NaN and do not count for the scale.
    Positions behind the last new token keep their bytes. Tokens whose
    position lies behind the table, or in a block that is not in the cache,
    are dropped, and all of a sequence with a negative start. No block may be
    written at two places by one call, neither of two sequences nor of one."""
    if _fast("kv_append", cache, k, v, block_table, start, count):
        return
    device = _Dev.device()
    _tensors("kv_append", device, {"count": count}, k=k, v=v, start=start,
             **_cache_tensors("kv_append", cache, block_table))
    if k.dim() != 4:
        raise ValueError(f"kv_append: k has shape {tuple(k.shape)}, not [B, kv_heads, S, head_dim]")
    B, _, S, _ = k.shape
    fields, heads, size, dim, width, table_stride = _pages("kv_append", cache, block_table, B)
    if k.dtype not in _DTYPE or k.dtype == E4M3:
        raise TypeError(f"kv_append: k is {k.dtype}")
    _shape("kv_append", "k", k, (B, heads, S, dim))
    _shape("kv_append", "v", v, (B, heads, S, dim), k.dtype)
    _per_sequence("kv_append", "start", start, B)
    if count is not None:
        _per_sequence("kv_append", "count", count, B)
    sk, sv = k.stride(), v.stride()
    if not sk[3] == sv[3] == 1:
        raise ValueError("kv_append: k and v need unit stride along head_dim")
    _call(lib().newt_kv_append, "kv_append", _APPEND.pack(
        *fields, k.data_ptr(), v.data_ptr(), block_table.data_ptr(), start.data_ptr(), _ptr(count),
        B, S, width, table_stride, *sk[:3], *sv[:3], _DTYPE[k.dtype], 0), device)


def _queries(what, q, out, window, sinks, scale):
    """The checked output, window (0: none) and scale of an attention."""
    if q.dim() != 4:
        raise ValueError(f"{what}: q has shape {tuple(q.shape)}, not [B, H, S, head_dim]")
    if q.dtype != torch.bfloat16 and q.dtype != torch.float16:
        raise TypeError(f"{what}: q is {q.dtype}, not float16 or bfloat16")
    if window is not None:
        _whole(what, "window", window, 1)
    _whole(what, "sinks", sinks, 0)
    if sinks and window is None:
        raise ValueError(f"{what}: sinks stay visible behind a window, and there is none")
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    else:
        _shape(what, "out", out, q.shape, q.dtype)
    if q.stride(3) != 1 or out.stride(3) != 1:
        raise ValueError(f"{what}: q and out need unit stride along head_dim")
    return out, window or 0, q.shape[3] ** -0.5 if scale is None else _fp32(scale)


def cached_attention(q, cache, block_table, lens, window=None, sinks=0, scale=None, out=None):
    """Attention of the last S tokens of each sequence, q [B, H, S, head_dim]
    fp16 or bf16, over the cache, which holds them already (kv_append).

    lens [B] int32 counts each sequence's tokens, so query i is at position p =
    lens[b] - S + i. It sees the tokens at positions j <= p, and with a window
    those with p - j < window or j < sinks. block_table [B, n] int32 is as in
    kv_append. H is a multiple of the cache's heads, each shared by H / kv_heads
    neighbouring query heads. A query that sees nothing (its position is
    negative) gets zeros. Tokens behind the table, and those of blocks that are
    not in the cache, are not seen; blocks that hold no visible token are not
    read, and their table entries may be anything. scale (finite) defaults to
    head_dim^-0.5. Rows of an `out` given must not overlap each other, not
    even in part: each of its strides steps over what the smaller ones reach."""
    r = _fast("cached_attention", q, cache, block_table, lens, window, sinks, scale, out)
    if r is not None:
        return r
    device = _Dev.device()
    _tensors("cached_attention", device, {"out": out}, q=q, lens=lens,
             **_cache_tensors("cached_attention", cache, block_table))
    out, window, scale = _queries("cached_attention", q, out, window, sinks, scale)
    B, H, S, D = q.shape
    fields, heads, size, dim, width, table_stride = _pages("cached_attention", cache, block_table,
                                                           B)
    if D != dim or heads == 0 or H == 0 or H % heads:
        raise ValueError(f"cached_attention: {H} heads of {D} dims over a cache of {heads} of {dim}")
    if S * H >= 2 ** 30:
        raise ValueError("cached_attention: too many queries")
    _per_sequence("cached_attention", "lens", lens, B)
    if fields[4] == 0 and width:
        raise ValueError("cached_attention: the cache has no blocks")
    L = lib()
    rest = (B, S, width, table_stride, *q.stride()[:3], *out.stride()[:3], window, sinks, scale, H,
            _DTYPE[q.dtype], 0)
    pointers = (q.data_ptr(), out.data_ptr(), block_table.data_ptr(), lens.data_ptr())
    params = _CACHED.pack(*fields, *pointers, 0, *rest)
    need = L.newt_cached_attention_workspace(params)
    if need:
        workspace = torch.empty(need, dtype=torch.uint8, device=q.device)
        params = _CACHED.pack(*fields, *pointers, workspace.data_ptr(), *rest)
    _call(L.newt_cached_attention, "cached_attention", params, device)
    return out


# ---------------------------------------------------------------------------
# attention in a window
# ---------------------------------------------------------------------------
def window_attention(q, k, v, window=None, sinks=0, scale=None, q_start=None, out=None):
    """Causal attention of q [B, H, S, head_dim] over k and v [B, kv_heads, Sk,
    head_dim], fp16 or bf16, head_dim 64, 128 or 256, any strides but along
    head_dim.

    Query i of sequence b is at position p = q_start[b] + i (q_start [B] int32;
    by default the queries are the last of the keys' positions, p = Sk - S + i).
    It sees the keys at positions j <= p, and with a window those with p - j <
    window or j < sinks. A query that sees nothing gets zeros. Keys that no
    query sees are not read where a whole tile of 64 of them is unseen, and
    never matter: what k and v hold behind the last query's position, or before
    every window, may be anything. Query heads share KV heads as in
    cached_attention; scale and `out` are as there. A weight is rounded to q's
    dtype before the product with the values; one below 2^-21 (fp16) of its row's
    largest is off by up to 2^-32 of that. cached_attention rounds fp16 weights
    to 16 bits, bf16 ones as here."""
    r = _fast("window_attention", q, k, v, window, sinks, scale, q_start, out)
    if r is not None:
        return r
    device = _Dev.device()
    _tensors("window_attention", device, {"q_start": q_start, "out": out}, q=q, k=k, v=v)
    out, window, scale = _queries("window_attention", q, out, window, sinks, scale)
    B, H, S, D = q.shape
    if D not in _HEAD_DIMS:
        raise ValueError(f"window_attention: head_dim {D} is not one of {_HEAD_DIMS}")
    if k.dim() != 4:
        raise ValueError(f"window_attention: k has shape {tuple(k.shape)}, not [B, kv_heads, Sk, "
                         f"head_dim]")
    heads, Sk = k.shape[1], k.shape[2]
    _shape("window_attention", "k", k, (B, heads, Sk, D), q.dtype)
    _shape("window_attention", "v", v, (B, heads, Sk, D), q.dtype)
    if heads == 0 or H == 0 or H % heads:
        raise ValueError(f"window_attention: {H} query heads over {heads}")
    if Sk >= 2 ** 30 or S * H >= 2 ** 30:
        raise ValueError("window_attention: sequences are too long")
    if q_start is not None:
        _per_sequence("window_attention", "q_start", q_start, B)
    sk, sv = k.stride(), v.stride()
    if not sk[3] == sv[3] == 1:
        raise ValueError("window_attention: k and v need unit stride along head_dim")
    L = lib()
    rest = (B, S, Sk, *q.stride()[:3], *sk[:3], *sv[:3], *out.stride()[:3], window, sinks, scale, H,
            heads, D, _DTYPE[q.dtype], 0)
    pointers = (q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), _ptr(q_start))
    params = _WINDOW.pack(*pointers, 0, *rest)
    need = L.newt_window_attention_workspace(params)
    if need:
        workspace = torch.empty(need, dtype=torch.uint8, device=q.device)
        params = _WINDOW.pack(*pointers, workspace.data_ptr(), *rest)
    _call(L.newt_window_attention, "window_attention", params, device)
    return out


# ---------------------------------------------------------------------------
# rotary positions
# ---------------------------------------------------------------------------
class Rotary(NamedTuple):
    """How pairs of a head turn with the position, made by `rotary`."""
    turns: torch.Tensor  # [dim / 2] int64: 2^64 of a full turn a position
    amplitude: float
    interleaved: bool


_PI = decimal.Decimal("3.14159265358979323846264338327950288419716939937510")
_MOST_TURNS = 10 ** 30  # of which 50 digits of pi give 2^-64


def rotary(dim, base=10000.0, factor=1.0, ramp=None, amplitude=1.0, interleaved=False,
           frequencies=None, device=None):
    """The Rotary of heads whose first `dim` dimensions turn: pair i by base^(-2 i /
    dim) radians a position, or by frequencies[i], 1e30 turns at most. Pairs are (i, i
    + dim / 2), or (2 i, 2 i + 1) where interleaved.

    For contexts longer than a model was trained on, frequencies are divided by
    `factor`; with ramp=(original, low, high) only those that turn less than `low`
    times over `original` positions, not those that turn at least `high` times,
    and in between a share that falls evenly with the number of turns. The turned
    dimensions come out `amplitude` times as large."""
    _whole("rotary", "dim", dim, 2)
    if dim % 2:
        raise ValueError(f"rotary: dim={dim} is odd")
    if not isinstance(interleaved, bool):
        raise TypeError("rotary: interleaved must be a bool")
    for name, value in (("base", base), ("factor", factor)):
        if not 0.0 < value < math.inf:
            raise ValueError(f"rotary: {name}={value} has to be positive and finite")
    amplitude = _fp32(amplitude)
    if not math.isfinite(amplitude):
        raise ValueError("rotary: amplitude has to be finite")
    if ramp is not None:
        original, low, high = ramp
        if not (0.0 < original < math.inf and 0.0 <= low < high < math.inf):
            raise ValueError(f"rotary: ramp={ramp} is not (original, low, high), low < high")
    number = decimal.Decimal
    # a fraction of a turn to 64 bits, whatever its size, needs more than fp64
    with decimal.localcontext(decimal.Context(prec=60)):
        if frequencies is None:
            step, frequencies = number(base) ** (number(-2) / dim), [number(1)]
            while len(frequencies) < dim // 2:
                frequencies.append(frequencies[-1] * step)
        else:
            frequencies = [float(f) for f in frequencies]
            if len(frequencies) != dim // 2 or not all(math.isfinite(f) for f in frequencies):
                raise ValueError(f"rotary: {dim // 2} finite frequencies are needed")
        turns = []
        for f in frequencies:
            f = number(f) / (2 * _PI)
            share = number(0)  # of the frequency as it is
            if ramp is not None:
                share = (abs(f) * number(original) - number(low)) / (number(high) - number(low))
                share = min(max(share, number(0)), number(1))
            f = f * share + f / number(factor) * (1 - share)
            if abs(f) > _MOST_TURNS:
                raise ValueError("rotary: a frequency is above 1e30 turns a position")
            t = int((f * 2 ** 64).to_integral_value()) % 2 ** 64
            turns.append(t - 2 ** 64 if t >= 2 ** 63 else t)
    device = torch.device("cuda", _Dev.device()) if device is None else device
    return Rotary(torch.tensor(turns, dtype=torch.int64, device=device), amplitude, interleaved)


def rotate(q, k, rotary, positions, transposed=False, q_out=None, k_out=None):
    """(q_out, k_out): q [B, H, S, head_dim] and k [B, kv_heads, S, head_dim], fp32,
    fp16 or bf16 (any strides but along head_dim), turned as `rotary` says by
    their tokens' positions; k may be None. positions are int32, [B, S], or [B]: the
    first token's, the others follow it. They may be any, negative ones too: the
    angle is right to 2^-29 of a radian everywhere.

    (a, b) -> amplitude (a cos - b sin, b cos + a sin) in fp32, rounded once;
    dimensions from the rotary's on are copied. Transposed, the angle's sign is
    changed: the map that takes the outputs' gradients to the inputs'. Outputs
    given may be q and k themselves, and overlap nothing else."""
    r = _fast("rotate", q, k, rotary, positions, transposed, q_out, k_out)
    if r is not None:
        return r
    device = _Dev.device()
    if not isinstance(rotary, (tuple, list)) or len(rotary) != 3:
        raise TypeError("rotate: rotary must be a Rotary")
    turns, amplitude, interleaved = rotary
    _tensors("rotate", device, {"k": k, "q_out": q_out, "k_out": k_out}, q=q, turns=turns,
             positions=positions)
    if q.dim() != 4:
        raise ValueError(f"rotate: q has shape {tuple(q.shape)}, not [B, H, S, head_dim]")
    if q.dtype not in _DTYPE or q.dtype == E4M3:
        raise TypeError(f"rotate: q is {q.dtype}")
    B, H, S, D = q.shape
    KV = 0
    if k is not None:
        if k.dim() != 4:
            raise ValueError(f"rotate: k has shape {tuple(k.shape)}, not [B, kv_heads, S, head_dim]")
        KV = k.shape[1]
        _shape("rotate", "k", k, (B, KV, S, D), q.dtype)
    elif k_out is not None:
        raise ValueError("rotate: k_out is an output of k")
    if turns.dim() != 1 or turns.dtype != torch.int64 or not turns.is_contiguous():
        raise TypeError("rotate: rotary must be a Rotary")
    rot = 2 * turns.shape[0]
    if not 2 <= rot <= D:
        raise ValueError(f"rotate: a rotary of {rot} dimensions for heads of {D}")
    if positions.dtype != torch.int32:
        raise TypeError(f"rotate: positions are {positions.dtype}, not int32")
    if positions.shape != (B,) and positions.shape != (B, S):
        raise ValueError(f"rotate: positions have shape {tuple(positions.shape)}, not {(B,)} or "
                         f"{(B, S)}")
    each = positions.dim() == 2
    outs = []
    for name, x, out in (("q_out", q, q_out), ("k_out", k, k_out)):
        if x is not None and out is None:
            out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        elif x is not None:
            _shape("rotate", name, out, x.shape, x.dtype)
        outs.append(out)
    if any(t is not None and t.stride(3) != 1 and D > 1 for t in (q, k, *outs)):
        raise ValueError("rotate: tensors need unit stride along head_dim")
    strides = [s for t in (q, outs[0], k, outs[1]) for s in ((0, 0, 0) if t is None
                                                           else t.stride()[:3])]
    _call(lib().newt_rotate, "rotate", _ROTATE.pack(
        q.data_ptr(), outs[0].data_ptr(), _ptr(k), _ptr(outs[1]), turns.data_ptr(),
        positions.data_ptr(), B, H, KV, S, D, rot, *strides, positions.stride(0),
        positions.stride(1) if each else 0, _fp32(amplitude), _DTYPE[q.dtype], bool(interleaved),
        bool(transposed), each, 0), device)
    return tuple(outs)


# ---------------------------------------------------------------------------
# products with 4-bit weights
# ---------------------------------------------------------------------------
class Q4Weights(NamedTuple):
    """4-bit weights laid out for the kernels by `q4_weights`."""
    q: torch.Tensor       # [tiles, ceil(cols / 128), 64, 4] int32
    scales: torch.Tensor  # [tiles, groups, 16]
    zeros: torch.Tensor   # as scales, uint8, or None
    outputs: int          # rows of weights; of a gated pair those of one
    cols: int
    group: int
    gated: bool


def q4_weights(q, scales, zeros=None, gated=False):
    """Weights [N, K] of 4 bits, laid out once for q4_matmul or, gated, for q4_gated:
    (number - zero) * scale. q [N, K / 2] uint8 holds two neighbouring columns'
    numbers a byte, the first one's in the lower half. scales [N, K / group] fp16
    or bf16 and zeros, any uint8 as scales (8 without), are for groups of 32, 64 or
    128 columns. Of gated weights the first N / 2 rows are the gate's."""
    for name, t in (("q", q), ("scales", scales)) + ((("zeros", zeros),) if zeros is not None else ()):
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"q4_weights: {name} must be a tensor")
        if t.dim() != 2:
            raise ValueError(f"q4_weights: {name} has shape {tuple(t.shape)}, not two dimensions")
        if t.device != q.device:
            raise TypeError(f"q4_weights: {name} is not on q's device")
    if not isinstance(gated, bool):
        raise TypeError("q4_weights: gated must be a bool")
    if q.dtype != torch.uint8:
        raise TypeError(f"q4_weights: q is {q.dtype}, not uint8")
    if scales.dtype != torch.float16 and scales.dtype != torch.bfloat16:
        raise TypeError(f"q4_weights: scales are {scales.dtype}, not float16 or bfloat16")
    N, K = q.shape[0], 2 * q.shape[1]
    groups = scales.shape[1]
    if scales.shape[0] != N or groups == 0 or K % groups or K // groups not in (32, 64, 128):
        raise ValueError(f"q4_weights: scales of shape {tuple(scales.shape)} are not those of [{N}, "
                         f"{K}] in groups of 32, 64 or 128 columns")
    group = K // groups
    if zeros is not None:
        _shape("q4_weights", "zeros", zeros, scales.shape, torch.uint8)
    if N == 0:
        raise ValueError("q4_weights: no rows")
    if gated and N % 2:
        raise ValueError(f"q4_weights: {N} rows are not a gate's and what it gates")
    if N >= 2 ** 30 or K >= 2 ** 30:
        raise ValueError("q4_weights: sizes stay below 2^30")
    halves = 2 if gated else 1
    outputs, blocks = N // halves, -(-K // 128)
    tiles = -(-outputs // 16)

    def tiled(t, cols, fill):
        """[halves * tiles, 16, cols], the halves' tiles in turn, `fill` around."""
        r = t.new_full((halves, tiles * 16, cols), fill)
        r[:, :outputs, :t.shape[1]] = t.view(halves, outputs, -1)
        return r.view(halves, tiles, 16, cols).transpose(0, 1).reshape(halves * tiles, 16, cols)

    words = torch.empty(halves * tiles, blocks, 64, 4, dtype=torch.int32, device=q.device)
    packed = tiled(q.contiguous(), blocks * 64, 0x88)
    step = max(1, (1 << 26) // (blocks * 1024))  # tiles at a time
    for i in range(0, len(words), step):
        # [tiles, row, block, j, part, pair] -> [tiles, block, part, row, j, pair]
        b = packed[i:i + step].view(-1, 16, blocks, 4, 4, 4).permute(0, 2, 4, 1, 3, 5).int()
        w = torch.zeros(b.shape[:-1], dtype=torch.int32, device=q.device)
        for pair in range(4):
            w |= (b[..., pair] & 15) << (4 * pair) | (b[..., pair] >> 4) << (16 + 4 * pair)
        w = w << 3 | (w >> 29) & 7
        words[i:i + step] = w.view(-1, blocks, 64, 4)
    per = blocks * (128 // group)
    laid_out = [None if t is None else tiled(t.contiguous(), per, fill).transpose(1, 2).contiguous()
                for t, fill in ((scales, 0.0), (zeros, 8))]
    return Q4Weights(words, *laid_out, outputs, K, group, gated)


def _q4(what, x, w, gated, optional):
    """Checked sizes, x's type and the weights' packed fields."""
    if not isinstance(w, Q4Weights):
        raise TypeError(f"{what}: w must be Q4Weights")
    device = _Dev.device()
    _tensors(what, device, {"zeros": w.zeros, **optional}, x=x, q=w.q, scales=w.scales)
    if x.dim() != 2:
        raise ValueError(f"{what}: x has shape {tuple(x.shape)}, not [M, K]")
    if x.dtype != torch.float16 and x.dtype != torch.bfloat16:
        raise TypeError(f"{what}: x is {x.dtype}, not float16 or bfloat16")
    if w.gated != gated:
        raise ValueError(f"{what}: weights are {'' if w.gated else 'not '}laid out gated")
    M, K = x.shape
    if K != w.cols:
        raise ValueError(f"{what}: x has {K} columns, the weights {w.cols}")
    if K > 1 and x.stride(1) != 1:
        raise ValueError(f"{what}: rows of x need unit stride")
    if w.group not in (32, 64, 128):
        raise ValueError(f"{what}: no groups of {w.group} columns")
    tiles, blocks = -(-w.outputs // 16) * (2 if gated else 1), -(-K // 128)
    _shape(what, "q", w.q, (tiles, blocks, 64, 4), torch.int32)
    _shape(what, "scales", w.scales, (tiles, blocks * (128 // w.group), 16))
    if w.scales.dtype != torch.float16 and w.scales.dtype != torch.bfloat16:
        raise TypeError(f"{what}: scales are {w.scales.dtype}, not float16 or bfloat16")
    if w.zeros is not None:
        _shape(what, "zeros", w.zeros, w.scales.shape, torch.uint8)
    if not all(t is None or t.is_contiguous() for t in w[:3]):
        raise ValueError(f"{what}: weights have to be contiguous")
    return device, M


def _q4_call(what, x, w, bias, out, act, device):
    M, N = x.shape[0], w.outputs
    if N > 1 and out.stride(1) != 1:
        raise ValueError(f"{what}: rows of out need unit stride")
    if M > 1 and out.stride(0) < N:
        raise ValueError(f"{what}: rows of out overlap")
    L = lib()
    pointers = (x.data_ptr(), w.q.data_ptr(), w.scales.data_ptr(), _ptr(w.zeros), _ptr(bias),
                out.data_ptr())
    rest = (M, w.cols, N, x.stride(0), out.stride(0), w.group, _DTYPE[x.dtype],
            _DTYPE[w.scales.dtype], _DTYPE[out.dtype], act, 0)
    params = _Q4.pack(*pointers, 0, *rest)
    need = L.newt_q4_matmul_workspace(params)
    if need:
        workspace = torch.empty(need, dtype=torch.uint8, device=x.device)
        params = _Q4.pack(*pointers, workspace.data_ptr(), *rest)
    _call(L.newt_q4_matmul, what, params, device)
    return out


def q4_matmul(x, w, bias=None, out_dtype=None, out=None):
    """x [M, K] fp16 or bf16, rows of any stride, times the transposed 4-bit
    weights (q4_weights): [M, N] of x's dtype or, with out_dtype=float32, fp32. bias
    [N] is of x's dtype. Products are summed in fp32 and multiplied there by their
    group's scale; the result is rounded once. The sums hold x (16 + number) and x
    (16 + zero), so their roundings count against the sum of |x| (32 + number + zero)
    |scale|, not against the result: a large x whose weights are all 0 still costs the
    others precision. For few rows the weights are read once; for hundreds, matmul is
    faster where a program has the weights in 16 bits too. A row of x that holds an
    infinity or NaN gives no numbers. An `out` given shares no memory with x or bias."""
    r = _fast("q4_matmul", x, w, bias, -1 if out_dtype is None else _DTYPE.get(out_dtype, -2), out)
    if r is not None:
        return r
    device, M = _q4("q4_matmul", x, w, False, {"bias": bias, "out": out})
    N = w.outputs
    if bias is not None:
        _shape("q4_matmul", "bias", bias, (N,), x.dtype)
        if N > 1 and bias.stride(0) != 1:
            raise ValueError("q4_matmul: bias needs unit stride")
    out_dtype = x.dtype if out_dtype is None else out_dtype
    if out_dtype != x.dtype and out_dtype != torch.float32:
        raise TypeError(f"q4_matmul: no {out_dtype} output of {x.dtype}")
    if out is None:
        out = torch.empty((M, N), dtype=out_dtype, device=x.device)
    else:
        _shape("q4_matmul", "out", out, (M, N), out_dtype)
    return _q4_call("q4_matmul", x, w, bias, out, 0, device)


_ACTS = {"silu": 1, "gelu": 2}


def q4_gated(x, w, act="silu", out=None):
    """act(x Wg) * (x Wu) [M, F] in x's dtype, the first half of a gated feed-forward
    block: x [M, K] fp16 or bf16, w of q4_weights(..., gated=True) with the 2 F rows
    of Wg and Wu transposed. act is silu, v / (1 + e^-v), or gelu, v (1 + erf(v / sqrt
    2)) / 2. Both products stay in fp32 until the result is rounded; x and `out`
    as in q4_matmul."""
    r = _fast("q4_gated", x, w, act, out)
    if r is not None:
        return r
    device, M = _q4("q4_gated", x, w, True, {"out": out})
    if act not in _ACTS:
        raise ValueError(f"q4_gated: act={act!r} is not one of {tuple(_ACTS)}")
    if out is None:
        out = torch.empty((M, w.outputs), dtype=x.dtype, device=x.device)
    else:
        _shape("q4_gated", "out", out, (M, w.outputs), x.dtype)
    return _q4_call("q4_gated", x, w, None, out, _ACTS[act], device)


# ---------------------------------------------------------------------------
# the next token
# ---------------------------------------------------------------------------
def sample(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """ids [T] int64: of each row of logits [T, V] fp32, fp16 or bf16 (rows of any
    stride) a token, chosen by u [T] fp32, random numbers in [0, 1) that the caller
    draws.

    A token's weight is e^((logit - largest) / temperature). Kept are the top_k
    largest (0: all); of these the first, from the largest on, until they have
    top_p of the weight that top_k leaves (1: all; the first one always); of these
    the ones of weight min_p or more. Equal logits go by the lowest id. The choice
    is the first id, in the vocabulary's order, whose running sum of kept weights
    exceeds u times their sum; with a temperature of 0 the largest logit's. Weights
    below 2^-46 (for more than 2^17 tokens 2^(bits of V - 63)) count as 0.

    temperature, top_p and min_p are numbers, taken as fp32, or fp32 [T], top_k an
    int or int32 [T]: settings of each row's own. -1 stands for no token: a row
    that holds a NaN or +inf or nothing but -inf, or whose u or setting is NaN, or
    its temperature negative or infinite."""
    r = _fast("sample", logits, u, temperature, top_k, top_p, min_p)
    if r is not None:
        return r
    device = _Dev.device()
    settings = {"temperature": temperature, "top_k": top_k, "top_p": top_p, "min_p": min_p}
    rows = {name: v for name, v in settings.items() if isinstance(v, torch.Tensor)}
    _tensors("sample", device, logits=logits, u=u, **rows)
    if logits.dim() != 2 or not 0 < logits.shape[1] < 2 ** 30:
        raise ValueError(f"sample: logits have shape {tuple(logits.shape)}, not [T, V]")
    if logits.dtype not in _DTYPE or logits.dtype == E4M3:
        raise TypeError(f"sample: logits are {logits.dtype}")
    T, V = logits.shape
    _shape("sample", "u", u, (T,), torch.float32)
    for name, v in rows.items():
        _shape("sample", name, v, (T,), torch.int32 if name == "top_k" else torch.float32)
    if T > 1 and any(t.stride(0) != 1 for t in (u, *rows.values())):
        raise ValueError("sample: u and the rows' settings need unit stride")
    if V > 1 and logits.stride(1) != 1:
        raise ValueError("sample: rows of logits need unit stride")
    if "top_k" not in rows:
        _whole("sample", "top_k", top_k, 0)
    for name, most in (("temperature", math.inf), ("top_p", math.inf), ("min_p", 1.0)):
        if name not in rows:
            if isinstance(settings[name], bool) or not isinstance(settings[name], (int, float)):
                raise TypeError(f"sample: {name} must be a number or a tensor")
            v = settings[name] = _fp32(settings[name])
            if not 0.0 <= v <= most or (name == "temperature" and v == math.inf):
                raise ValueError(f"sample: {name}={v} is out of range")
    ids = torch.empty(T, dtype=torch.int64, device=logits.device)
    L = lib()
    code = _DTYPE[logits.dtype]
    need = L.newt_sample_workspace(T, V, code)
    workspace = torch.empty(need, dtype=torch.uint8, device=logits.device) if need else None
    scalar = {name: 0 if name in rows else v for name, v in settings.items()}
    _call(L.newt_sample, "sample", _SAMPLE.pack(
        logits.data_ptr(), u.data_ptr(), ids.data_ptr(), *(_ptr(rows.get(n)) for n in settings),
        _ptr(workspace), T, V, logits.stride(0), scalar["temperature"], scalar["top_p"],
        scalar["min_p"], scalar["top_k"], code, 0), device)
    return ids
