"""The serving operators without a GPU: what the Python entry points refuse
before a launch, what the C entries refuse, the C structs against the packed
fields, and the 64-bit definitions that the GPU tests compare with."""

import ctypes
import os
import re
import subprocess

import pytest
import torch

from newt_amd import serving, workloads
from oracle import serving as orc

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "newt_ops.h")
BF16, E4M3 = torch.bfloat16, torch.float8_e4m3fn


class Launched(Exception):
    pass


@pytest.fixture
def calls(monkeypatch):
    """Entry points on CPU tensors, up to the launch."""
    def call(entry, what, params, device):
        raise Launched(what)
    monkeypatch.setattr(serving, "_tensors", lambda *a, **k: None)
    monkeypatch.setattr(serving, "_call", call)
    monkeypatch.setattr(serving, "_fast", lambda *a: None)
    monkeypatch.setattr(serving._Dev, "device", classmethod(lambda cls: 0))
    return None


def refused(kind, match, f, *args, **kw):
    with pytest.raises(kind, match=match):
        f(*args, **kw)


def test_tensors_have_to_be_on_the_gpu(monkeypatch):
    """Through the C++ calls too, which leave such tensors to Python."""
    monkeypatch.setattr(serving._Dev, "device", classmethod(lambda cls: 0))
    monkeypatch.setattr(serving._Dev, "stream", staticmethod(lambda device: 0))
    assert serving._Fast.load()
    x, t = torch.zeros(2, 64), torch.zeros(2, dtype=torch.int64)
    refused(TypeError, "current GPU", workloads.rmsnorm, x, x[0])
    refused(TypeError, "must be a tensor", workloads.rmsnorm, [1.0], x[0])
    refused(TypeError, "current GPU", workloads.token_logprobs, x, t)
    q = torch.zeros(1, 2, 3, 64, dtype=BF16)
    refused(TypeError, "current GPU", workloads.window_attention, q, q, q)
    cache = workloads.kv_cache(2, 2, 64, device="cpu")
    refused(TypeError, "current GPU", workloads.cached_attention, q, cache, t, t)
    refused(TypeError, "current GPU", workloads.kv_append, cache, q, q, t, t)


def test_rmsnorm_refusals(calls):
    f = workloads.rmsnorm
    x, w = torch.zeros(4, 256, dtype=BF16), torch.zeros(256, dtype=BF16)
    refused(Launched, "rmsnorm", f, x, w)
    refused(Launched, "rmsnorm", f, x, w.float(), residual=x, out_dtype=E4M3, group=128)
    refused(ValueError, "shape", f, x[0], w)
    refused(ValueError, "shape", f, x[:, :0], w[:0])
    refused(ValueError, "w has shape", f, x, w[1:])
    refused(TypeError, "x is", f, x.double(), w)
    refused(TypeError, "x is", f, x.to(E4M3), w)
    refused(TypeError, "w is", f, x, w.half())
    refused(TypeError, "output", f, x, w, out_dtype=torch.float32)
    refused(TypeError, "output", f, x, w, out_dtype=torch.int8)
    refused(ValueError, "8-bit", f, x, w, group=128)
    for group in (0, 16, 96, 512, True):
        refused(ValueError, "groups", f, x, w, out_dtype=E4M3, group=group)
    refused(ValueError, "groups", f, x[:, :192], w[:192], out_dtype=E4M3, group=128)
    refused(ValueError, "residual has shape", f, x, w, residual=x[:2])
    refused(TypeError, "residual is", f, x, w, residual=x.float())
    refused(TypeError, "hidden is", f, x, w, residual=x, hidden=x.float())
    refused(ValueError, "hidden", f, x, w, hidden=x)
    refused(TypeError, "out is", f, x, w, out=x.float())
    refused(ValueError, "unit stride", f, x.t()[:, :4], w[:4])
    refused(ValueError, "unit stride", f, x[:, ::2], w[:128])
    refused(ValueError, "unit stride", f, x[:, :128], w[::2])
    refused(ValueError, "overlap", f, x, w, out=x[:1].expand(4, 256))
    refused(ValueError, "overlap", f, x, w, residual=x, hidden=x[:1].expand(4, 256))


def test_logprobs_refusals(calls):
    f = workloads.token_logprobs
    x, t = torch.zeros(3, 100), torch.zeros(3, dtype=torch.int64)
    refused(Launched, "token_logprobs", f, x, t, top=64)
    refused(ValueError, "shape", f, x[0], t)
    refused(ValueError, "shape", f, x[:, :0], t)
    refused(TypeError, "logits are", f, x.double(), t)
    refused(TypeError, "tokens is", f, x, t.int())
    refused(ValueError, "tokens has shape", f, x, t[:2])
    refused(ValueError, "alternatives", f, x, t, top=65)
    refused(ValueError, "alternatives", f, x[:, :5], t, top=6)
    refused(ValueError, "out of range", f, x, t, top=-1)
    refused(TypeError, "int", f, x, t, top=2.0)
    refused(TypeError, "int", f, x, t, top=True)
    for temperature in (0.0, -1.0, float("nan"), float("inf"), 1e-40):
        refused(ValueError, "temperature", f, x, t, temperature=temperature)
    refused(ValueError, "unit stride", f, x[:, ::2], t)
    refused(ValueError, "unit stride", f, x, torch.zeros(6, dtype=torch.int64)[::2])


def test_cache_refusals(calls):
    make = workloads.kv_cache
    refused(ValueError, "blocks", make, 0, 1, 64, device="cpu")
    refused(ValueError, "kv_heads", make, 1, 0, 64, device="cpu")
    refused(ValueError, "tokens", make, 1, 1, 64, block_size=48, device="cpu")
    refused(ValueError, "head_dim", make, 1, 1, 96, device="cpu")
    cache = make(4, 2, 64, block_size=16, device="cpu")
    assert cache.k.shape == (4, 2, 16, 64) and cache.v.shape == (4, 2, 64, 16)
    table, lens = torch.zeros(3, 2, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    k = torch.zeros(3, 2, 5, 64, dtype=BF16)
    q = torch.zeros(3, 6, 5, 64, dtype=BF16)

    def append(cache=cache, k=k, v=k, table=table, start=lens, count=None):
        workloads.kv_append(cache, k, v, table, start, count=count)

    def attend(cache=cache, q=q, table=table, lens=lens, **kw):
        workloads.cached_attention(q, cache, table, lens, **kw)

    refused(Launched, "kv_append", append, count=lens)
    refused(Launched, "cached_attention", attend, window=3, sinks=2)
    for f in (append, attend):
        refused(TypeError, "not int32", f, table=table.long())
        refused(ValueError, "block_table", f, table=table[:2])
        refused(ValueError, "block_table", f, table=table[0])
        refused(ValueError, "unit stride", f, table=torch.zeros(2, 3, dtype=torch.int32).t())
        refused(ValueError, "too long", f, table=torch.empty(1, 2 ** 27, dtype=torch.int32).expand(3, -1))
        refused(TypeError, "not torch.float8", f, cache=cache._replace(k=cache.k.to(BF16)))
        refused(TypeError, "not torch.float8", f, cache=cache._replace(v=cache.v.to(BF16)))
        refused(ValueError, "v_cache has shape", f, cache=cache._replace(v=cache.k))
        refused(ValueError, "k_scale has shape", f, cache=cache._replace(k_scale=cache.k_scale[:2]))
        refused(TypeError, "v_scale is", f, cache=cache._replace(v_scale=cache.v_scale.half()))
        refused(ValueError, "shape", f, cache=cache._replace(k=cache.k[0]))
        refused(ValueError, "contiguous", f, cache=cache._replace(
            k_scale=torch.zeros(2, 4).t()))
        odd = torch.zeros(4 * 2 * 16 * 64 + 1, dtype=torch.uint8)[1:].view(E4M3)
        refused(ValueError, "aligned", f, cache=cache._replace(k=odd.view(4, 2, 16, 64)))
    refused(ValueError, "blocks of 8", attend, cache=cache._replace(k=cache.k[:, :, :8]))
    refused(ValueError, "k has shape", append, k=k[:, :1])
    refused(ValueError, "k has shape", append, k=k[0])
    refused(ValueError, "k has shape", append, k=k[..., :32], v=k[..., :32])
    refused(ValueError, "v has shape", append, v=k[:, :, :4])
    refused(TypeError, "v is", append, v=k.float())
    refused(TypeError, "k is", append, k=k.double(), v=k.double())
    refused(TypeError, "start is", append, start=lens.long())
    refused(ValueError, "count has shape", append, count=lens[:2])
    refused(ValueError, "unit stride", append, k=torch.zeros(3, 2, 64, 5, dtype=BF16).mT)
    refused(ValueError, "heads", attend, q=q[:, :5])
    refused(ValueError, "heads", attend, q=q[:, :0])
    refused(ValueError, "heads", attend, q=torch.zeros(3, 6, 5, 128, dtype=BF16))
    refused(TypeError, "q is", attend, q=q.float())
    refused(ValueError, "q has shape", attend, q=q[0])
    refused(TypeError, "lens is", attend, lens=lens.long())
    refused(ValueError, "lens has shape", attend, lens=lens[:1])
    refused(ValueError, "window", attend, window=0)
    refused(TypeError, "window", attend, window=3.0)
    refused(ValueError, "sinks", attend, sinks=-1, window=2)
    refused(ValueError, "sinks", attend, sinks=1)
    refused(ValueError, "out has shape", attend, out=q[:, :, :1])
    refused(TypeError, "out is", attend, out=q.half())
    refused(ValueError, "no blocks", attend, cache=workloads.KVCache(
        *(c[:0] for c in cache)))


def test_window_refusals(calls):
    f = workloads.window_attention
    q, k = torch.zeros(2, 4, 3, 64, dtype=BF16), torch.zeros(2, 2, 9, 64, dtype=BF16)
    start = torch.zeros(2, dtype=torch.int32)
    refused(Launched, "window_attention", f, q, k, k, window=3, sinks=2, q_start=start)
    refused(TypeError, "q is", f, q.float(), k.float(), k.float())
    refused(TypeError, "k is", f, q, k.half(), k)
    refused(TypeError, "v is", f, q, k, k.half())
    refused(ValueError, "k has shape", f, q, k[:1], k)
    refused(ValueError, "k has shape", f, q, k[0], k)
    refused(ValueError, "v has shape", f, q, k, k[:, :, 1:])
    refused(ValueError, "query heads", f, q[:, :3], k, k)
    refused(ValueError, "query heads", f, q, k[:, :0], k[:, :0])
    refused(ValueError, "head_dim", f, q[..., :32], k[..., :32], k[..., :32])
    refused(ValueError, "window", f, q, k, k, window=-2)
    refused(ValueError, "sinks", f, q, k, k, sinks=2)
    refused(TypeError, "q_start is", f, q, k, k, q_start=start.long())
    refused(ValueError, "q_start has shape", f, q, k, k, q_start=start[:1])
    refused(ValueError, "unit stride", f, q, torch.zeros(2, 2, 64, 9, dtype=BF16).mT, k)
    refused(ValueError, "unit stride", f, torch.zeros(2, 4, 64, 3, dtype=BF16).mT, k, k)
    refused(ValueError, "out has shape", f, q, k, k, out=q[:, :2])


# ---------------------------------------------------------------------------
# the C ABI
# ---------------------------------------------------------------------------
def declared():
    text = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    return sorted(set(re.findall(r"\b(newt_[a-z0-9_]+)\s*\(", text)))


def test_library_exports_every_declared_symbol():
    L = serving.lib()
    assert len(declared()) >= 10
    assert not [s for s in declared() if not hasattr(L, s)]
    assert L.newt_ops_abi_version() == 1


def test_structs_are_what_is_packed(tmp_path):
    """Sizes, and the last field's place, as a C compiler lays them out."""
    src = tmp_path / "sizes.c"
    names = {"newt_rmsnorm_params": serving._RMSNORM, "newt_logprobs_params": serving._LOGPROBS,
             "newt_kv_append_params": serving._APPEND,
             "newt_cached_attention_params": serving._CACHED,
             "newt_window_attention_params": serving._WINDOW}
    lines = "".join(f'printf("%zu %zu\\n", sizeof({n}), offsetof({n}, reserved));' for n in names)
    src.write_text(f'#include <stdio.h>\n#include "newt_ops.h"\nint main(void) {{ {lines} }}\n')
    subprocess.run(["gcc", "-std=c11", "-Wall", "-Werror", "-I" + os.path.dirname(HEADER), str(src),
                    "-o", str(tmp_path / "sizes")], check=True)
    out = subprocess.run([str(tmp_path / "sizes")], capture_output=True, text=True, check=True)
    for line, s in zip(out.stdout.splitlines(), names.values()):
        size, last = map(int, line.split())
        assert size == s.size and last == size - 4


def test_c_entries_refuse():
    """Null structs, null tensors, sizes and types that no kernel takes: an
    error and its message, before the GPU is touched."""
    L = serving.lib()

    def call(entry, params, message):
        assert entry(params, None) == 10002
        assert message in L.newt_ops_last_error(), L.newt_ops_last_error()

    for name in ("rmsnorm", "token_logprobs", "kv_append", "cached_attention", "window_attention"):
        call(getattr(L, "newt_" + name), None, b"null params")
    norm = lambda *a: serving._RMSNORM.pack(*a)  # noqa: E731
    P = 4096  # an address that nothing reads
    call(L.newt_rmsnorm, norm(0, 0, P, P, 0, 0, 1, 8, 8, 8, 8, 8, 1e-6, 0, 0, 0, 0, 0), b"null tensor")
    call(L.newt_rmsnorm, norm(P, P, P, P, 0, 0, 1, 8, 8, 8, 8, 8, 1e-6, 0, 0, 0, 0, 0), b"null tensor")
    call(L.newt_rmsnorm, norm(P, 0, P, P, 0, 0, 1, 0, 8, 8, 8, 8, 1e-6, 0, 0, 0, 0, 0), b"columns")
    call(L.newt_rmsnorm, norm(P, 0, P, P, 0, 0, 1, 8, 8, 8, 8, 8, 1e-6, 0, 0, 1, 0, 0), b"type")
    call(L.newt_rmsnorm, norm(P, 0, P, P, 0, P, 1, 96, 8, 8, 8, 8, 1e-6, 0, 0, 3, 64, 0), b"groups")
    call(L.newt_rmsnorm, norm(P, 0, P, P, 0, 0, 1, 8, 8, 8, 8, 8, 1e-6, 7, 0, 7, 0, 0), b"dtype")
    call(L.newt_rmsnorm, norm(P, 0, P, P, 0, 0, 1, 8, 8, 8, 8, 8, 1e-6, 1, 2, 1, 0, 0), b"w is")
    logs = lambda *a: serving._LOGPROBS.pack(*a)  # noqa: E731
    call(L.newt_token_logprobs, logs(P, P, P, 0, 0, 0, 0, 1, 8, 8, 1.0, 0, 0, 0), b"null tensor")
    call(L.newt_token_logprobs, logs(P, P, P, P, P, P, 0, 1, 8, 8, 1.0, 0, 9, 0), b"alternatives")
    call(L.newt_token_logprobs, logs(P, P, P, P, P, P, 0, 1, 0, 8, 1.0, 0, 0, 0), b"logits")
    call(L.newt_token_logprobs, logs(P, P, P, P, 0, 0, 0, 1, 8, 8, 0.0, 0, 0, 0), b"temperature")
    call(L.newt_token_logprobs, logs(P, P, P, P, 0, 0, 0, 1, 8, 8, 1.0, 3, 0, 0), b"dtype")
    call(L.newt_token_logprobs, logs(P, P, P, P, 0, 0, 0, 1, 200000, 8, 1.0, 0, 0, 0), b"workspace")
    cache = [P, P, P, P, 4, 2, 16, 64, 0]
    tokens = [P, P, P, P, 0, 1, 1, 1, 1, *[64] * 6, 2, 0]
    attend = [P, P, P, P, 0, 1, 1, 1, 1, *[64] * 6, 0, 0, 1.0, 4, 2, 0]
    for entry, s, rest in ((L.newt_kv_append, serving._APPEND, tokens),
                           (L.newt_cached_attention, serving._CACHED, attend)):
        for i, value, message in ((0, 0, b"null cache"), (4, -1, b"number of blocks"),
                                  (5, 0, b"heads"), (6, 24, b"blocks hold"), (7, 80, b"head_dim")):
            bad = list(cache)
            bad[i] = value
            call(entry, s.pack(*bad, *rest), message)
        call(entry, s.pack(*cache, 0, *rest[1:]), b"null tensor")
        call(entry, s.pack(*cache, *rest[:5], -1, *rest[6:]), b"negative")
    call(L.newt_kv_append, serving._APPEND.pack(*cache, *tokens[:-2], 3, 0), b"dtype")
    call(L.newt_cached_attention, serving._CACHED.pack(*cache, *attend[:-3], 3, 2, 0), b"multiple")
    call(L.newt_cached_attention, serving._CACHED.pack(*cache, *attend[:-3], 4, 0, 0), b"fp16")
    window = [P, P, P, P, 0, 0, 1, 1, 1, *[64] * 12, 0, 0, 1.0, 4, 2, 64, 2, 0]
    call(L.newt_window_attention, serving._WINDOW.pack(0, *window[1:]), b"null tensor")
    call(L.newt_window_attention, serving._WINDOW.pack(*window[:-3], 80, 2, 0), b"head_dim")
    call(L.newt_window_attention, serving._WINDOW.pack(*window[:-4], 3, 64, 2, 0), b"multiple")
    call(L.newt_window_attention, serving._WINDOW.pack(*window[:-2], 0, 0), b"fp16")


def test_empty_calls_launch_nothing():
    """No rows, tokens or sequences: success, without a GPU to launch on."""
    L = serving.lib()
    P = 4096
    assert L.newt_rmsnorm(serving._RMSNORM.pack(P, 0, P, P, 0, 0, 0, 8, 8, 8, 8, 8, 1e-6, 0, 0, 0, 0,
                                                0), None) == 0
    assert L.newt_token_logprobs(serving._LOGPROBS.pack(P, P, P, P, 0, 0, 0, 0, 8, 8, 1.0, 0, 0, 0),
                                 None) == 0
    cache = [P, P, P, P, 4, 2, 16, 64, 0]
    for batch, tokens in ((0, 1), (1, 0)):
        assert L.newt_kv_append(serving._APPEND.pack(
            *cache, P, P, P, P, 0, batch, tokens, 1, 1, *[64] * 6, 2, 0), None) == 0
        assert L.newt_cached_attention(serving._CACHED.pack(
            *cache, P, P, P, P, 0, batch, tokens, 1, 1, *[64] * 6, 0, 0, 1.0, 4, 2, 0), None) == 0
        assert L.newt_window_attention(serving._WINDOW.pack(
            P, P, P, P, 0, 0, batch, tokens, 1, *[64] * 12, 0, 0, 1.0, 4, 2, 64, 2, 0), None) == 0


# ---------------------------------------------------------------------------
# the definitions
# ---------------------------------------------------------------------------
def test_round_e4m3_is_the_format():
    numbers = torch.arange(256, dtype=torch.uint8).view(E4M3).double()
    finite = numbers[numbers.isfinite()]
    assert torch.equal(orc.round_e4m3(finite), finite)
    up = finite[finite >= 0].unique()
    middle = (up[1:] + up[:-1]) / 2
    for x, want in ((middle - 1e-9, up[:-1]), (middle + 1e-9, up[1:])):
        assert torch.equal(orc.round_e4m3(x), want)
    # ties go to the even one: every other number from 0 on
    even = torch.where(torch.arange(len(middle)) % 2 == 0, up[:-1], up[1:])
    assert torch.equal(orc.round_e4m3(middle), even)
    assert torch.equal(orc.round_e4m3(-middle), -even)
    x = torch.randn(1000) * 100
    assert torch.equal(orc.round_e4m3(x.clamp(-448, 448)), x.clamp(-448, 448).to(E4M3).double())


def test_power_of_two():
    for top, want in ((448.0, 1.0), (448.0001, 2.0), (224.0, 0.5), (3.5, 2.0 ** -7),
                      (0.0, 2.0 ** -100), (1e-38, 2.0 ** -100), (3e38, 2.0 ** 120)):
        assert orc.power_of_two(top) == want


def test_attention_definition():
    """One head against a masked softmax written out."""
    g = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn(2, n, 8, generator=g).double() for n in (5, 9, 9))
    o, a = orc.attention(q, k, v, range(4, 9), window=3, sinks=1)
    i, j = torch.arange(4, 9)[:, None], torch.arange(9)[None]
    seen = (j <= i) & ((i - j < 3) | (j < 1))
    w = torch.softmax((q @ k.transpose(1, 2) / 8 ** 0.5).masked_fill(~seen, float("-inf")), -1)
    torch.testing.assert_close(o, w @ v)
    torch.testing.assert_close(a, w @ v.abs())
    o, _ = orc.attention(q, k, v, range(-3, 2))
    assert bool((o[:, :3] == 0).all()) and bool((o[:, 3:] != 0).any())


def test_attention_refuses_overlapping_rows_and_scales():
    """Rows of an output that share memory, which programs would write at once,
    and scales that are not finite: an error before the GPU is touched."""
    L = serving.lib()
    P = 4096
    cache = [P, P, P, P, 4, 2, 16, 64, 0]

    def cached(o=(512, 128, 64), batch=2, q_len=2, heads=4, scale=1.0):
        return L.newt_cached_attention(serving._CACHED.pack(
            *cache, P, P, P, P, 0, batch, q_len, 1, 1, 512, 128, 64, *o, 0, 0, scale, heads, 2, 0),
            None)

    def window(o=(512, 128, 64), batch=2, q_len=2, heads=4, scale=1.0):
        return L.newt_window_attention(serving._WINDOW.pack(
            P, P, P, P, 0, 0, batch, q_len, 1, *[64] * 9, *o, 0, 0, scale, heads, 2, 64, 2, 0), None)

    cache[0] = P + 8
    assert cached() == 10002 and b"aligned" in L.newt_ops_last_error()
    cache[0] = P
    for call in (cached, window):
        for o in ((0, 128, 64), (512, 0, 64), (512, 128, 0)):
            assert call(o) == 10002
            assert b"overlap" in L.newt_ops_last_error()
        for scale in (float("inf"), -float("inf"), float("nan"), 2.0 ** 100):
            assert call(scale=scale) == 10002
            assert b"scale" in L.newt_ops_last_error()


def test_attention_refuses_rows_that_overlap_in_part():
    """Rows of an output that share some of their memory, in any order of the
    dimensions; what slices and permutations of a tensor give is taken."""
    L = serving.lib()
    P = 4096
    cache = [P, P, P, P, 4, 2, 16, 64, 0]

    def cached(o, batch=2, q_len=2, heads=4):
        # without a table: the check of the strides comes before that of null tensors
        return L.newt_cached_attention(serving._CACHED.pack(
            *cache, 0, P, P, P, 0, batch, q_len, 1, 1, 512, 128, 64, *o, 0, 0, 1.0, heads, 2, 0),
            None)

    def window(o, batch=2, q_len=2, heads=4):
        return L.newt_window_attention(serving._WINDOW.pack(
            0, P, P, P, 0, 0, batch, q_len, 1, *[64] * 9, *o, 0, 0, 1.0, heads, 2, 64, 2, 0), None)

    for call in (cached, window):
        for o in ((512, 128, 63), (512, 127, 64), (511, 128, 64), (512, 128, 1), (64, 128, 64),
                  (512, 64, 255), (64, 96, 512)):
            assert call(o) == 10002
            assert b"overlap" in L.newt_ops_last_error(), o
        for o in ((512, 128, 64), (512, 64, 256), (64, 128, 512), (64, 256, 128), (128, 512, 64),
                  (1000, 200, 70)):
            assert call(o) == 10002
            assert b"null tensor" in L.newt_ops_last_error(), o
        # dimensions of one have no stride
        assert call((0, 0, 64), batch=1, heads=2, q_len=2) == 10002
        assert b"overlap" in L.newt_ops_last_error()
        assert call((0, 64, 0), batch=1, q_len=1) == 10002
        assert b"null tensor" in L.newt_ops_last_error()


def test_cache_without_heads(calls):
    """A ValueError, as for other heads that do not go together."""
    q, table = torch.zeros(2, 4, 3, 64, dtype=BF16), torch.zeros(2, 1, dtype=torch.int32)
    cache = workloads.KVCache(*(c[:, :0].contiguous() for c in workloads.kv_cache(
        3, 2, 64, device="cpu")))
    lens = torch.zeros(2, dtype=torch.int32)
    refused(ValueError, "heads", workloads.cached_attention, q, cache, table, lens)


def test_required_tensors(monkeypatch):
    """None and other things in the place of a tensor that a call needs."""
    monkeypatch.setattr(serving._Dev, "device", classmethod(lambda cls: 0))
    monkeypatch.setattr(serving._Dev, "stream", staticmethod(lambda device: 0))
    x, t = torch.zeros(2, 64), torch.zeros(2, dtype=torch.int64)
    q, lens = torch.zeros(2, 2, 3, 64, dtype=BF16), torch.zeros(2, dtype=torch.int32)
    cache, table = workloads.kv_cache(2, 2, 64, device="cpu"), lens.view(2, 1)
    calls = {workloads.rmsnorm: {"x": x, "w": x[0]},
             workloads.token_logprobs: {"logits": x, "tokens": t},
             workloads.kv_append: {"cache": cache, "k": q, "v": q, "block_table": table,
                                   "start": lens},
             workloads.cached_attention: {"q": q, "cache": cache, "block_table": table,
                                          "lens": lens},
             workloads.window_attention: {"q": q, "k": q, "v": q}}
    for f, args in calls.items():
        refused(TypeError, "current GPU", f, **args)
        for name in args:
            if name == "cache":
                for wrong in (None, 3):
                    refused(TypeError, None, f, **{**args, name: wrong})
                refused(ValueError, None, f, **{**args, name: cache[:3]})
                for field in cache._fields:
                    refused(TypeError, "must be a tensor", f,
                            **{**args, name: cache._replace(**{field: None})})
                continue
            for wrong in (None, 1.0, [1, 2]):
                refused(TypeError, "must be a tensor", f, **{**args, name: wrong})
    for f, names in ((workloads.rmsnorm, ("residual", "out", "hidden")),
                     (workloads.kv_append, ("count",)), (workloads.cached_attention, ("out",)),
                     (workloads.window_attention, ("q_start", "out"))):
        for name in names:
            refused(TypeError, "current GPU", f, **{**calls[f], name: None})
            refused(TypeError, "must be a tensor", f, **{**calls[f], name: 1.0})


LAUNCH = serving._call  # before a test takes its place


def test_numbers_beyond_fp32(calls, monkeypatch):
    """A scale that fp32 does not hold is refused as one that is not finite; an
    eps that it does not hold is infinite, as in the calls made in C++. What is
    no number is a TypeError or ValueError."""
    launched = []
    monkeypatch.setattr(serving, "_call", lambda entry, what, params, device:
                        launched.append(params) if what == "rmsnorm" else
                        LAUNCH(entry, what, params, device))
    monkeypatch.setattr(serving._Dev, "stream", staticmethod(lambda device: 0))
    q, lens = torch.zeros(2, 2, 3, 64, dtype=BF16), torch.zeros(2, dtype=torch.int32)
    cache, table = workloads.kv_cache(2, 2, 64, device="cpu"), lens.view(2, 1)
    for scale in (1e39, -1e300, float("inf"), float("nan"), 10 ** 40):
        refused(ValueError, "scale", workloads.cached_attention, q, cache, table, lens, scale=scale)
        refused(ValueError, "scale", workloads.window_attention, q, q, q, scale=scale)
    for wrong in ("a", [1.0]):
        for f, args in ((workloads.window_attention, (q, q, q)),
                        (workloads.cached_attention, (q, cache, table, lens))):
            with pytest.raises((TypeError, ValueError)):
                f(*args, scale=wrong)
        with pytest.raises((TypeError, ValueError)):
            workloads.rmsnorm(torch.zeros(2, 64), torch.zeros(64), eps=wrong)
    with pytest.raises(TypeError):
        workloads.rmsnorm(torch.zeros(2, 64), torch.zeros(64), eps=None)
    workloads.rmsnorm(torch.zeros(2, 64), torch.zeros(64), eps=1e39)
    assert serving._RMSNORM.unpack(launched[0])[12] == float("inf")
