"""The operators of a decoder's serving step, as hand-written gfx950 kernels.

They stand beside the kernels of `newt_amd.workloads`, which re-exports them:
`rmsnorm` beside `layernorm`, `window_attention` and `cached_attention` beside
`attention`, `token_logprobs` beside `softmax`. All are forward only, as the
others are. The kernels are in csrc/ops, behind the C ABI of
include/newt_ops.h; they are compiled ahead of time, so a first call costs no
compilation.

As everywhere in newt, tensors have to be on the current GPU, a call launches
on torch's current stream, synchronizes nothing and can be captured into a
graph. Outputs that are not given are new tensors. Wrong arguments raise
TypeError (kind of argument, device, dtype) or ValueError (shape, stride,
range) before anything is launched.

One step of a decoder layer over the 8-bit cache:

    x, _, hidden = rmsnorm(x, w_norm, residual=hidden)
    q, k, v = ...                      # matmul(x, ...), rotated
    kv_append(cache, k, v, block_table, lens - k.shape[2])
    o = cached_attention(q, cache, block_table, lens)
"""

import ctypes
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
                 "newt_window_attention"):
        f = getattr(L, name)
        f.restype, f.argtypes = ctypes.c_int, [ctypes.c_char_p, ctypes.c_void_p]
    for name in ("newt_cached_attention_workspace", "newt_window_attention_workspace"):
        f = getattr(L, name)
        f.restype, f.argtypes = ctypes.c_size_t, [ctypes.c_char_p]
    L.newt_token_logprobs_workspace.restype = ctypes.c_size_t
    L.newt_token_logprobs_workspace.argtypes = [ctypes.c_int64, ctypes.c_int64, ctypes.c_int32,
                                                ctypes.c_int32]
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
