"""The serving operators on an MI355X against their definitions in 64 bits:
types, odd sizes, strides, lengths from one token on, empty rows, what masks
hide, and the operators together as a step runs them."""

import pytest
import torch

from oracle import serving as orc

pytestmark = pytest.mark.gpu

HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
E4M3 = torch.float8_e4m3fn
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
HALVES = [torch.float16, torch.bfloat16]


def rnd(*shape, dtype=torch.float32, seed=0, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def ints(*values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device="cuda")


def W():
    from newt_amd import workloads
    return workloads


# ---------------------------------------------------------------------------
# rmsnorm. Errors in fp32: a lane adds at most 64 squares (in rows that stay in
# registers; 16 for every 16384 columns of longer ones), the reductions 10 more,
# and each of about 8 further operations rounds once; the sum's error halves
# under the root. (64 + 10) / 2 + 8 < 64 roundings of 2^-24.
# ---------------------------------------------------------------------------
FP32 = 64 * 2.0 ** -24


def check_rmsnorm(x, w, residual=None, out_dtype=None, group=None, eps=1e-6, **kw):
    want, hidden = orc.rmsnorm(x, w, eps, residual)
    got, scale, got_hidden = W().rmsnorm(x, w, eps=eps, residual=residual, out_dtype=out_dtype,
                                         group=group, **kw)
    if residual is None:
        assert got_hidden is None
    else:
        assert torch.equal(got_hidden, hidden)
    if out_dtype is None:
        assert scale is None and got.dtype == x.dtype
        # below fp16's normal numbers a half step is 2^-25
        off = (got.double() - want).abs()
        assert bool((off <= (HALF_STEP[x.dtype] + FP32) * want.abs() + 2.0 ** -25).all())
        return got
    scales = orc.scales(want, group)
    assert scale.dtype == torch.float32 and scale.shape == scales.shape
    assert bool(((scale.double() - scales).abs() <= 2 * FP32 * scales).all())
    by = scale.double().repeat_interleave(x.shape[1] // scale.shape[1], 1)
    off = (got.double() * by - want).abs()
    # half a step of e4m3: 2^-4 of a normal number, 2^-10 of the scale below
    assert bool((off <= (2.0 ** -4 + 2 * FP32) * want.abs() + 2.0 ** -10 * by).all())
    # and it is the nearest number of the exact quotient, but for ties that
    # fp32 decides the other way
    nearest = orc.round_e4m3((want / by).clamp(-448, 448))
    assert float((got.double() != nearest).double().mean()) <= 1e-3
    return got


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N", [1, 7, 8, 63, 64, 65, 128, 200, 513, 1000, 1024, 2048, 4097, 8192,
                               16384, 20001, 32768, 40000])
def test_rmsnorm(dtype, N):
    for M, residual in ((1, True), (5, False), (9, True)):
        x = rnd(M, N, dtype=dtype, seed=N, scale=2.0)
        r = rnd(M, N, dtype=dtype, seed=N + 1, scale=5.0) if residual else None
        w = (rnd(N, seed=N + 2) * 0.3 + 1).to(dtype)
        check_rmsnorm(x, w, r)
        check_rmsnorm(x, w, r, out_dtype=E4M3)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N,group", [(32, 32), (64, 64), (128, 128), (256, 256), (320, 32),
                                     (384, 128), (2560, 256), (8192, 128), (8192, 32),
                                     (65536, 128), (33024, 256)])
def test_rmsnorm_groups(dtype, N, group):
    x = rnd(7, N, dtype=dtype, seed=N + group)
    r = rnd(7, N, dtype=dtype, seed=N + 1)
    check_rmsnorm(x, rnd(N, seed=3), r, out_dtype=E4M3, group=group)


def test_rmsnorm_strides_and_given_outputs():
    """Rows inside wider tensors, at odd addresses; outputs given; the residual
    updated in place; what lies around the outputs stays."""
    for dtype in DTYPES:
        x = rnd(33, 1003, dtype=dtype, seed=1)[:, 1:1000]
        r = rnd(33, 2001, dtype=dtype, seed=2)[:, 3:1002]
        w = rnd(1001, dtype=dtype, seed=3)[2:]
        around = torch.full((34, 1007), 7.0, dtype=dtype, device="cuda")
        kept = r.clone()
        want = W().rmsnorm(x.contiguous(), w, residual=kept)
        out, _, hidden = W().rmsnorm(x, w, residual=r, out=around[1:, 5:1004], hidden=r)
        assert hidden.data_ptr() == r.data_ptr() and torch.equal(r, want[2])
        assert torch.equal(out, want[0]) and torch.equal(around[1:, 5:1004], want[0])
        around[1:, 5:1004] = 7.0
        assert bool((around == 7.0).all())
        # x's own rows take the sum
        y = x.contiguous()
        assert torch.equal(W().rmsnorm(y, w, residual=kept, hidden=y)[0], want[0])
        assert torch.equal(y, want[2])


def test_rmsnorm_special_rows():
    """Zeros, tiny and huge values, infinities and NaN; no rows; the weight in
    fp32 beside 16-bit rows."""
    x = rnd(6, 512, seed=1)
    x[0] = 0.0
    x[1] = 1e-30
    x[2] = 1e15
    x[3, 5] = float("nan")
    x[4, 6] = float("inf")
    w = rnd(512, seed=2)
    for eps in (1e-6, 1e-12):
        want, _ = orc.rmsnorm(x, w, eps)
        got = W().rmsnorm(x, w, eps=eps)[0].double()
        for i in (0, 1, 2, 5):
            assert bool(((got[i] - want[i]).abs() <= 2 * FP32 * want[i].abs() + 1e-40).all())
        assert bool(got[3].isnan().all())
        assert bool((got[4].isnan() == (torch.arange(512, device="cuda") == 6)).all())
        assert bool((got[4, :6] == 0).all())
    q, scale, _ = W().rmsnorm(x, w, out_dtype=E4M3)
    assert bool((q[0].double() == 0).all()) and float(scale[0]) == 2.0 ** -126
    assert bool(q[3].double().isnan().all())
    got, _, hidden = W().rmsnorm(x[:0], w, residual=x[:0])
    assert got.shape == hidden.shape == (0, 512)
    for dtype in HALVES:
        check_rmsnorm(rnd(3, 777, dtype=dtype, seed=3), rnd(777, seed=4), rnd(3, 777, dtype=dtype))


def test_rmsnorm_many_rows():
    x = rnd(70001, 72, dtype=torch.bfloat16, seed=5)
    check_rmsnorm(x, rnd(72, dtype=torch.bfloat16, seed=6))


# ---------------------------------------------------------------------------
# token_logprobs. A lane adds n = V / 64 terms at most; every term's exponent
# carries 3 roundings of a number |d| <= 64 here, so a term is off by 64 * 3 *
# 2^-24 of itself; the result's own roundings are relative to what it is made of.
# ---------------------------------------------------------------------------
def check_logprobs(logits, tokens, top, temperature=1.0):
    want = orc.logprobs(logits, tokens, top, temperature)
    got = W().token_logprobs(logits, tokens, top=top, temperature=temperature)
    V = logits.shape[1]
    finite = torch.where(logits.isfinite(), logits.double(), 0.0)
    spread = (finite.amax(-1) - finite.amin(-1)).abs() / temperature + 1
    tol = (V / 64 + 16 + 200) * 2.0 ** -24 + spread * 2.0 ** -22
    for i, name in ((0, "logp"), (1, "entropy")):
        assert torch.equal(got[i].isnan(), want[i].isnan()), name
        assert torch.equal(got[i].isinf(), want[i].isinf()), name
        off = (got[i].double() - want[i]).nan_to_num(0.0, posinf=0.0, neginf=0.0).abs()
        # the entropy weighs up to `spread` with each term's error
        assert bool((off <= tol * (1 if i == 0 else 1 + spread)).all()), name
    if not top:
        assert got[2] is None and got[3] is None
        return
    assert torch.equal(got[3], want[3])
    live = want[3] >= 0
    assert torch.equal((got[2].isnan() | ~live), (want[2].isnan() | ~live))
    off = (got[2].double() - want[2]).nan_to_num(0.0, posinf=0.0, neginf=0.0).abs()
    assert bool((off <= tol[:, None])[live].all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,V,top", [(1, 1, 1), (1, 1, 0), (2, 3, 3), (3, 17, 5), (5, 64, 64),
                                     (4, 100, 64), (2, 511, 20), (3, 512, 1), (2, 513, 0),
                                     (7, 2049, 20), (1, 8193, 20), (1, 50021, 64), (3, 130001, 5),
                                     (300, 3001, 8), (1100, 1000, 3)])
def test_logprobs(dtype, T, V, top):
    x = rnd(T, V, dtype=dtype, seed=V + top, scale=3.0)
    g = torch.Generator(device="cuda").manual_seed(V)
    tokens = torch.randint(V, (T,), generator=g, device="cuda")
    check_logprobs(x, tokens, top)
    check_logprobs(x, tokens, top, temperature=0.6)


@pytest.mark.parametrize("V", [40, 1000, 30001])
def test_logprobs_ties_and_order(V):
    """Few distinct logits, rising and falling rows, equal rows: ids go up
    among equals wherever they lie."""
    g = torch.Generator(device="cuda").manual_seed(V)
    x = torch.stack([torch.randint(4, (V,), generator=g, device="cuda").float(),
                     torch.arange(V, device="cuda") / 512.0,
                     -torch.arange(V, device="cuda") / 512.0,
                     torch.full((V,), 3.25, device="cuda"),
                     torch.randint(2, (V,), generator=g, device="cuda") * -0.0])
    check_logprobs(x, torch.arange(5, device="cuda"), 20)


def test_logprobs_masked_rows():
    """Logits of -inf and of the type's lowest value, rows with fewer allowed
    tokens than alternatives, with none, with NaN or +inf; tokens that are none."""
    for dtype in DTYPES:
        for V in (100, 20001):
            x = rnd(10, V, dtype=dtype, seed=V, scale=2.0)
            x[0, 5:] = float("-inf")
            x[1, :-3] = float("-inf")
            x[2] = float("-inf")
            x[3, 7] = float("nan")
            x[4, 9] = float("inf")
            x[5, 1:] = torch.finfo(dtype).min
            x[6, ::2] = float("-inf")
            x[7, : V - 2] = float("nan")
            tokens = ints(0, 5, 1, 3, 2, 0, 1, 0, -1, V, dtype=torch.int64)
            got = W().token_logprobs(x, tokens, top=10)
            want = orc.logprobs(x, tokens, 10)
            keep = [0, 1, 5, 6, 8, 9]
            for i in range(2):
                assert torch.equal(got[i].isnan(), want[i].isnan())
                assert torch.equal(got[i].isinf(), want[i].isinf())
                a, b = got[i][keep].double(), want[i][keep]
                ok = b.isfinite()
                assert bool(((a - b)[ok].abs() <= 1e-4 + 1e-6 * b[ok].abs()).all())
            assert torch.equal(got[3], want[3])
            assert float(got[0][8]) == 0.0
            # a row whose logits all have the lowest value is uniform
            low = torch.full((1, V), torch.finfo(dtype).min, dtype=dtype, device="cuda")
            logp, entropy, _, ids = W().token_logprobs(low, ints(3, dtype=torch.int64), top=2)
            log = torch.tensor(float(V)).log()
            assert abs(float(entropy[0]) - float(log)) < 1e-4
            assert abs(float(logp[0]) + float(log)) < 1e-4 and ids.tolist() == [[0, 1]]


def test_logprobs_strides():
    x = rnd(9, 5003, dtype=torch.bfloat16, seed=1)[:, 1:5000]
    check_logprobs(x, torch.arange(9, device="cuda"), 4)
    one = rnd(1, 300, seed=2).expand(5, 300)
    check_logprobs(one, torch.arange(5, device="cuda"), 4)
    got = W().token_logprobs(x[:0], torch.arange(0, device="cuda"), top=4)
    assert got[0].shape == (0,) and got[2].shape == (0, 4)


# ---------------------------------------------------------------------------
# the cache
# ---------------------------------------------------------------------------
def make_cache(blocks, heads, size, D, seed, low=-9, high=-4):
    """A cache full of any numbers, NaN bytes among them, as memory that was in
    use before."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    at = {"generator": g, "device": "cuda"}
    k, v = (torch.randint(256, (blocks, heads, *s), dtype=torch.uint8, **at).view(E4M3)
            for s in ((size, D), (D, size)))
    scales = [torch.exp2(torch.randint(low, high, (blocks, heads), **at).float()) for _ in range(2)]
    return W().KVCache(k, v, *scales)


def numbers(cache):
    return [c.double() for c in cache]


def same(a, b):
    return all(torch.equal(x.isnan(), y.isnan()) and torch.equal(x.nan_to_num(), y.nan_to_num())
               for x, y in zip(a, b))


def check_append(cache, k, v, table, start, count=None):
    want = orc.append(cache, k, v, table, start, count)
    before = [c.view(torch.uint8).clone() for c in cache[:2]]
    W().kv_append(cache, k, v, table, start, count=count)
    assert same(numbers(cache), want)
    return before


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("size,D", [(16, 64), (32, 128), (64, 128), (128, 64), (256, 256)])
def test_append(dtype, size, D):
    """Prompts and single tokens behind them, at every place in a block."""
    for S, starts, counts in ((1, (0, 1, size - 1, size), None),
                              (1, (5, 2 * size, 3 * size - 1, 0), (1, 0, 1, 1)),
                              (7, (0, size - 3, size - 7, 2), (7, 7, 7, 3)),
                              (2 * size + 3, (0, 1, size - 1, 3), (2 * size + 3, 1, size + 1, 2 * size)),
                              (3 * size, (0, size, 7, 2), None)):
        heads = 3
        cache = make_cache(22, heads, size, D, seed=S)
        table = torch.randperm(20, device="cuda").to(torch.int32).view(4, 5)
        k = rnd(4, heads, S, D, dtype=dtype, seed=S + 1, scale=2.0)
        v = rnd(4, heads, S, D, dtype=dtype, seed=S + 2, scale=0.01)
        check_append(cache, k, v, table, ints(*starts), None if counts is None else ints(*counts))


def test_append_bytes_around_stay():
    cache = make_cache(12, 2, 32, 64, seed=1)
    table = torch.arange(12, device="cuda", dtype=torch.int32).view(3, 4)
    k, v = rnd(3, 2, 40, 64, seed=2) * 1e-4, rnd(3, 2, 40, 64, seed=3) * 1e-4
    before = check_append(cache, k, v, table, ints(32, 0, 70), ints(40, 0, 5))
    kb, vb = (c.view(torch.uint8) for c in cache[:2])
    assert torch.equal(kb[0], before[0][0]) and torch.equal(kb[3:8], before[0][3:8])
    assert torch.equal(kb[2, :, 8:], before[0][2, :, 8:])
    assert torch.equal(vb[2, :, :, 8:], before[1][2, :, :, 8:])
    assert torch.equal(kb[10, :, 11:], before[0][10, :, 11:])
    assert torch.equal(vb[10, :, :, 11:], before[1][10, :, :, 11:])
    assert torch.equal(kb[11], before[0][11])


def test_append_scales():
    """Growing and shrinking tokens, zeros, the borders of a scale, tiny and
    huge values, infinities and NaN; token by token as together."""
    size, D = 16, 64
    values = [0.0, 1e-38, 2.0 ** -110, 1.0, 448.0, 449.0, 3.5, 3.515625, 448.0 * 2 ** 20, 1e-3,
              3e38, 0.5, float("inf"), float("nan"), -447.9, 2.0]
    cache, whole = make_cache(3, 2, size, D, seed=1), make_cache(3, 2, size, D, seed=1)
    table = ints(2, 0, 1).view(1, 3)
    k = rnd(1, 2, len(values), D, seed=2).clamp(-1, 1)
    k[..., 0] = 1.0
    k = k * torch.tensor(values, device="cuda")[:, None]
    v = -k.flip(1)
    for t in range(len(values)):
        check_append(cache, k[:, :, t:t + 1], v[:, :, t:t + 1], table, ints(t + 20))
    check_append(whole, k, v, table, ints(20))
    # and in whole numbers of a scale, what fits stays what it is
    cache = W().kv_cache(1, 1, 64, block_size=16)
    x = torch.tensor([1.0, -0.5, 448.0, 2.0 ** -9], device="cuda").repeat(16).view(1, 1, 1, 64)
    W().kv_append(cache, x, x * 2 ** -30, ints(0).view(1, 1), ints(0))
    assert float(cache.k_scale[0, 0]) == 1.0 and float(cache.v_scale[0, 0]) == 2.0 ** -30
    assert torch.equal(cache.k[0, 0, 0].float(), x[0, 0, 0])
    assert torch.equal(cache.v[0, 0, :, 0].float(), x[0, 0, 0])
    W().kv_append(cache, x * 4, x * 2 ** -32, ints(0).view(1, 1), ints(1))
    assert float(cache.k_scale[0, 0]) == 4.0 and float(cache.v_scale[0, 0]) == 2.0 ** -30
    assert torch.equal(cache.k[0, 0, 0, :3].float() * 4, x[0, 0, 0, :3])


def test_append_drops_what_has_no_place():
    """Positions behind the table, blocks outside of the cache, a negative
    start, more tokens than there are; strided tokens, a strided table."""
    cache = make_cache(8, 2, 16, 64, seed=5)
    wide = torch.full((5, 6), 99, dtype=torch.int32, device="cuda")
    table = wide[:, 1:4]
    table[0] = ints(0, 8, 1)
    table[1] = ints(2, -1, 3)
    table[2] = ints(4, 5, 6)
    table[3] = ints(7, 7, 7)
    table[4] = ints(-2 ** 31, 2 ** 31 - 1, 100)
    k = rnd(5, 50, 2, 70, seed=6).transpose(1, 2)[..., 3:67]
    v = rnd(2, 5, 50, 64, dtype=torch.float32, seed=7).transpose(0, 1)
    check_append(cache, k, v, table, ints(3, 9, 40, -1, 0), ints(50, 30, 99, 50, 50))


# ---------------------------------------------------------------------------
# attention. Roundings: of each weight to the type that the second product
# takes it in (2^-8 for bf16; for fp16 2^-11, of a weight below 2^-14 2^-25, and
# for the cache 2^-16 in two parts), relative to a = sum p |v|; of the output;
# and fp32's: a score of D products is off by D * 2^-24 of its terms' sum, which
# is below 64 here, and its weight by that much of itself.
# ---------------------------------------------------------------------------
def check_attention(got, want, a, dtype, cached, n, vmax):
    D = got.shape[-1]
    weight = 2.0 ** -16 if cached and dtype == torch.float16 else HALF_STEP[dtype]
    tol = (weight + (D + 64) * 64 * 2.0 ** -24) * a + HALF_STEP[dtype] * want.abs() + 2.0 ** -25
    if dtype == torch.float16 and not cached:
        tol = tol + n * 2.0 ** -25 * vmax
    assert torch.equal(got.isnan(), want.isnan())
    off = (got.double() - want).nan_to_num(0.0).abs()
    assert bool((off <= tol.nan_to_num(0.0)).all()), float((off / tol).nan_to_num(0.0).max())


def check_window(q, k, v, window=None, sinks=0, scale=None, start=None, **kw):
    got = W().window_attention(q, k, v, window=window, sinks=sinks, scale=scale, q_start=start, **kw)
    B, H, S, D = q.shape
    for b in range(B):
        first = k.shape[2] - S if start is None else int(start[b])
        want, a = orc.attention(q[b], k[b], v[b], range(first, first + S), window, sinks, scale)
        vmax = float(v[b].nan_to_num(0.0, 0.0, 0.0).abs().max()) if v.shape[2] else 0.0
        check_attention(got[b], want, a, q.dtype, False, k.shape[2], vmax)
    return got


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("B,H,KV,S,Sk,window,sinks", [
    (1, 1, 1, 1, 1, None, 0), (2, 4, 2, 1, 77, None, 0), (1, 8, 1, 3, 300, 64, 0),
    (1, 2, 2, 130, 130, None, 0), (2, 6, 2, 70, 200, 33, 5), (1, 3, 1, 200, 333, 100, 70),
    (1, 2, 1, 65, 65, 1, 0), (1, 2, 1, 129, 129, 1, 1), (1, 1, 1, 300, 300, 64, 64),
    (1, 16, 1, 1, 1000, 200, 130), (1, 5, 5, 40, 640, 1000, 3)])
def test_window(dtype, D, B, H, KV, S, Sk, window, sinks):
    q = rnd(B, H, S, D, dtype=dtype, seed=S)
    k, v = rnd(B, KV, Sk, D, dtype=dtype, seed=Sk), rnd(B, KV, Sk, D, dtype=dtype, seed=Sk + 1)
    check_window(q, k, v, window, sinks)


@pytest.mark.parametrize("dtype", HALVES)
def test_window_positions(dtype):
    """Sequences that begin elsewhere: queries before the first key see nothing
    and get zeros, ones behind the last see what is left of their window."""
    q = rnd(6, 4, 90, 64, dtype=dtype, seed=1)
    k, v = rnd(6, 2, 150, 64, dtype=dtype, seed=2), rnd(6, 2, 150, 64, dtype=dtype, seed=3)
    start = ints(0, 60, -1, -90, 100, 1000)
    for window, sinks in ((None, 0), (40, 0), (40, 7), (200, 80)):
        got = check_window(q, k, v, window, sinks, start=start)
        assert bool((got[3] == 0).all())
    # more queries than keys
    check_window(q, k[:, :, :20], v[:, :, :20], 7, 2)
    check_window(q, k[:, :, :0], v[:, :, :0], 7, 2)
    check_window(q[:, :, :0], k, v)
    check_window(q[:0], k[:0], v[:0])


@pytest.mark.parametrize("dtype", HALVES)
def test_window_hidden_values(dtype):
    """NaN and infinities in keys and values that a query does not see do not
    reach it: behind the last query, before every window, and in the middle,
    where they reach exactly the queries that see them."""
    q = rnd(1, 4, 100, 64, dtype=dtype, seed=1)
    k, v = rnd(1, 2, 400, 64, dtype=dtype, seed=2), rnd(1, 2, 400, 64, dtype=dtype, seed=3)
    for bad in (float("nan"), float("inf"), float("-inf")):
        k2, v2 = k.clone(), v.clone()
        k2[:, :, 260:], v2[:, :, 260:] = bad, bad
        k2[:, :, 3:80], v2[:, :, 3:80] = bad, bad
        got = check_window(q, k2, v2, 60, 3, start=ints(150))
        assert bool(got.isfinite().all())
        v2[:, 1, 200, 5] = bad
        k2[:, 0, 210] = float("nan")
        got = check_window(q, k2, v2, 30, 3, start=ints(150))
        rows = torch.arange(100, device="cuda") + 150
        assert torch.equal(got[0, 2, :, 5].isfinite(), (rows < 200) | (rows >= 230))
        assert torch.equal(got[0, 0, :, 0].isfinite(), (rows < 210) | (rows >= 240))
    v2 = v.clone()
    v2[:, :, 200, 0], v2[:, :, 210, 0] = float("inf"), float("-inf")
    got = W().window_attention(q, k, v2, window=30, q_start=ints(150))
    rows = torch.arange(100, device="cuda") + 150
    assert torch.equal(got[0, 0, :, 0].isnan(), (rows >= 210) & (rows < 230))
    assert torch.equal(got[0, 0, :, 0] == float("inf"), (rows >= 200) & (rows < 210))
    assert torch.equal(got[0, 0, :, 0] == float("-inf"), (rows >= 230) & (rows < 240))


@pytest.mark.parametrize("dtype", HALVES)
def test_window_strides_and_scores(dtype):
    """Heads behind tokens, odd strides, shared tensors, a given output; scores
    that rise along the keys, so that every tile has a new maximum, and scales
    of either sign."""
    q = rnd(2, 50, 4, 67, dtype=dtype, seed=1).transpose(1, 2)[..., 1:65]
    kv = rnd(2, 130, 2, 2, 64, dtype=dtype, seed=2)
    k, v = kv[:, :, :, 0].transpose(1, 2), kv[:, :, :, 1].transpose(1, 2)
    around = torch.full((2, 50, 4, 70), 5.0, dtype=dtype, device="cuda")
    out = around.transpose(1, 2)[..., 3:67]
    got = check_window(q, k, v, 60, 2, out=out)
    assert got.data_ptr() == out.data_ptr()
    out.fill_(5.0)
    assert bool((around == 5.0).all())
    one = rnd(1, 1, 130, 64, dtype=dtype, seed=3).expand(2, 2, 130, 64)
    check_window(q, one, one, 100, 0)
    rise = (torch.arange(130, device="cuda") / 130.0 * 6)[:, None].to(dtype) * torch.ones_like(k)
    for scale in (0.125, -0.125, 0.0, 0.02):
        check_window(torch.ones_like(q), rise, v, None, 0, scale=scale)
        check_window(torch.ones_like(q), rise, v, 90, 3, scale=scale)


# the cache's attention ------------------------------------------------------
def fill_cache(heads, size, D, lens, seed, extra=3, outlier=True):
    """A cache with ordinary numbers, blocks in any order, and NaN bytes and
    scales wherever no sequence's token lies."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    B, per = len(lens), max(1, max(-(-n // size) for n in lens))
    n = B * per + extra
    at = {"generator": g, "device": "cuda"}
    k, v = ((torch.randn(n, heads, *s, **at) * 90).clamp(-448, 448)
            for s in ((size, D), (D, size)))
    ks, vs = (torch.exp2(torch.randint(-9, -5, (n, heads), **at).float()) for _ in range(2))
    table = torch.randperm(n, **at)[: B * per].view(B, per).to(torch.int32)
    unused = torch.ones(n, dtype=torch.bool, device="cuda")
    for b, length in enumerate(lens):
        for slot in range(-(-length // size)):
            page = int(table[b, slot])
            unused[page] = False
            tail = length - slot * size
            if tail < size:
                k[page, :, tail:], v[page, :, :, tail:] = float("nan"), float("nan")
            if outlier and slot % 3 == 1:
                vs[page] *= 1.3 * 2.0 ** 12  # any scale will do
        table[b, -(-length // size):] = 2 ** 30
    ks[unused], vs[unused], k[unused], v[unused] = (float("nan"),) * 4
    return W().KVCache(k.to(E4M3), v.to(E4M3), ks, vs), table


def check_cached(q, cache, table, lens, window=None, sinks=0, scale=None, **kw):
    got = W().cached_attention(q, cache, table, ints(*lens), window=window, sinks=sinks,
                               scale=scale, **kw)
    S = q.shape[2]
    for b, n in enumerate(lens):
        keys, values, has = orc.cached(cache, table, b, max(n, 0))
        want, a = orc.attention(q[b], keys, values, range(n - S, n), window, sinks, scale, has)
        check_attention(got[b], want, a, q.dtype, True, n, 0.0)
    return got


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("size,D", [(16, 64), (16, 128), (32, 128), (64, 64), (64, 128), (64, 256),
                                    (128, 128), (256, 64)])
@pytest.mark.parametrize("H,KV,S", [(1, 1, 1), (8, 2, 1), (6, 2, 3), (16, 1, 1), (24, 1, 1),
                                    (8, 2, 9)])
def test_cached(dtype, size, D, H, KV, S):
    lens = (1, 64, 15, 0, 333, 127)
    cache, table = fill_cache(KV, size, D, lens, seed=size + D)
    q = rnd(len(lens), H, S, D, dtype=dtype, seed=H + S)
    check_cached(q, cache, table, lens)
    check_cached(q, cache, table, lens, window=50, sinks=0)
    check_cached(q, cache, table, lens, window=100, sinks=4)
    check_cached(q, cache, table, lens, window=17, sinks=70)
    check_cached(q, cache, table, lens, window=1, sinks=1)


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("B,H,KV,n,S", [(1, 8, 2, 9001, 1), (2, 4, 4, 3000, 2), (1, 32, 8, 16000, 1),
                                        (1, 1, 1, 20000, 1), (40, 8, 8, 700, 1)])
def test_cached_long(dtype, B, H, KV, n, S):
    lens = [max(1, n - 97 * b) for b in range(B)]
    cache, table = fill_cache(KV, 64, 128, lens, seed=n, outlier=False)
    q = rnd(B, H, S, 128, dtype=dtype, seed=n)
    check_cached(q, cache, table, lens)
    check_cached(q, cache, table, lens, window=1000, sinks=4)


@pytest.mark.parametrize("size", [16, 64])
def test_cached_hidden_blocks(size):
    """Blocks that left the window: their table entries may be anything, and
    so may their bytes. Entries outside of the cache among the visible ones
    hide their tokens. Sequences longer than the table end with it."""
    lens = (400, 390, 200, 64)
    cache, table = fill_cache(2, size, 64, lens, seed=size)
    q = rnd(4, 4, 2, 64, dtype=torch.bfloat16, seed=1)
    want = check_cached(q, cache, table, lens, window=60, sinks=4)
    free = table.clone()
    for b, n in enumerate(lens):
        for slot in range(free.shape[1]):
            if slot * size >= 4 and (slot + 1) * size <= n - 2 + 1 - 60:
                free[b, slot] = (-7, 2 ** 31 - 1, -2 ** 31, cache.k.shape[0])[slot % 4]
    assert torch.equal(W().cached_attention(q, cache, free, ints(*lens), window=60, sinks=4), want)
    table[0, 1], table[1, 0], table[3] = -1, cache.k.shape[0], -5
    check_cached(q, cache, table, lens)
    got = check_cached(q, cache, table, lens, window=70, sinks=20)
    assert bool((got[3] == 0).all())
    check_cached(q, cache, table, (4000, 390, 200, 500))
    check_cached(q, cache, table[:, :0], lens)
    check_cached(q, cache, table, (-5, 0, 1, 2))


def test_cached_nan_values():
    """A NaN value reaches the queries that see its token and no others."""
    lens = (130, 70)
    cache, table = fill_cache(1, 32, 64, lens, seed=9, outlier=False)
    cache.v.view(torch.uint8)[int(table[0, 3]), 0, 5, 126 - 96] = 0xff
    cache.v.view(torch.uint8)[int(table[1, 0]), 0, 6, 3] = 0x7f
    q = rnd(2, 4, 6, 64, dtype=torch.bfloat16, seed=2)
    for dtype in HALVES:
        got = check_cached(q.to(dtype), cache, table, lens)
        assert torch.equal(got[0, 0, :, 5].isnan(), torch.arange(6, device="cuda") >= 2)
        assert bool(got[1, :, :, 6].isnan().all()) and not bool(got[1, :, :, 7].isnan().any())
        got = check_cached(q.to(dtype), cache, table, lens, window=3, sinks=1)
        assert torch.equal(got[0, 0, :, 5].isnan(),
                           (torch.arange(6, device="cuda") >= 2) & (torch.arange(6, device="cuda") < 5))
        assert bool(got[1].isfinite().all())


def test_cached_strides():
    lens = (100, 200, 5)
    cache, table = fill_cache(2, 64, 128, lens, seed=4)
    wide = torch.cat([torch.full_like(table, -3), table, table], 1)
    q = rnd(3, 2, 6, 131, dtype=torch.bfloat16, seed=5).transpose(1, 2)[..., 1:129]
    around = torch.full((3, 2, 6, 136), 5.0, dtype=torch.bfloat16, device="cuda")
    out = around.transpose(1, 2)[..., 4:132]
    want = check_cached(q, cache, table, lens)
    got = check_cached(q, cache, wide[:, table.shape[1]:2 * table.shape[1]], lens, out=out)
    assert torch.equal(got, want)
    out.fill_(5.0)
    assert bool((around == 5.0).all())


# ---------------------------------------------------------------------------
# together
# ---------------------------------------------------------------------------
def test_prompt_and_steps():
    """A layer's path over a prompt and single tokens: norms, products, the
    cache and its attention, scores of the last product. The cache's attention
    sees what was appended; attention over the keys before they went into the
    cache is near, by e4m3's half step of 2^-4."""
    w = W()
    B, H, KV, D, V, S = 2, 4, 2, 64, 1000, 70
    E = H * D
    bf16 = torch.bfloat16
    norm = (rnd(E, seed=1) * 0.1 + 1).to(bf16)
    wq, wk, wv = (rnd(E, n * D, dtype=bf16, seed=i, scale=E ** -0.5)
                  for i, n in ((2, H), (3, KV), (4, KV)))
    head = rnd(E, V, dtype=bf16, seed=5, scale=E ** -0.5)
    cache = w.kv_cache(20, KV, D, block_size=32)
    table = torch.randperm(20, device="cuda")[:B * 4].view(B, 4).to(torch.int32)
    lens = ints(0, 0)
    hidden = torch.zeros(B * S, E, dtype=bf16, device="cuda")
    keys = []
    for step, n in enumerate((S, 1, 1, 1)):
        x = rnd(B * n, E, dtype=bf16, seed=20 + step)
        hidden = hidden[:B * n]
        y, _, hidden = w.rmsnorm(x, norm, residual=hidden, hidden=hidden)
        q, k, v = ((y @ m).view(B, n, -1, D).transpose(1, 2) for m in (wq, wk, wv))
        keys.append((k, v))
        w.kv_append(cache, k, v, table, lens)
        lens = lens + n
        o = w.cached_attention(q, cache, table, lens, window=48, sinks=4)
        near = w.window_attention(q, torch.cat([a for a, _ in keys], 2),
                                  torch.cat([b for _, b in keys], 2), window=48, sinks=4)
        for b in range(B):
            ks, vs, has = orc.cached(cache, table, b, int(lens[b]))
            want, a = orc.attention(q[b], ks, vs, range(int(lens[b]) - n, int(lens[b])), 48, 4)
            check_attention(o[b], want, a, bf16, True, 100, 0.0)
        assert float((o - near).float().norm() / near.float().norm()) < 0.1
        flat = o.transpose(1, 2).reshape(B * n, E)
        q8, scale, _ = w.rmsnorm(flat, norm, out_dtype=E4M3, group=128)
        y8 = (q8.float().view(B * n, -1, 128) * scale[..., None]).view(B * n, E).to(bf16)
        logits = y8 @ head
        logp, entropy, top_logp, top_ids = w.token_logprobs(
            logits, torch.arange(B * n, device="cuda"), top=3)
        want = orc.logprobs(logits, torch.arange(B * n, device="cuda"), 3)
        assert torch.equal(top_ids, want[3])
        assert bool(((logp.double() - want[0]).abs() < 1e-4).all())
        assert bool(((entropy.double() - want[1]).abs() < 1e-3).all())


def step_calls(w, s):
    y, _, h = w.rmsnorm(s["x"], s["w"], residual=s["r"])
    w.kv_append(s["cache"], s["k"], s["v"], s["table"], s["start"])
    o = w.cached_attention(s["q"], s["cache"], s["table"], s["lens"], window=500, sinks=4)
    p = w.window_attention(s["q"], s["keys"], s["keys"], window=300, sinks=2)
    return [y, h, o, p, *w.token_logprobs(s["logits"], s["tokens"], top=5)]


def step_state(seed):
    bf16 = torch.bfloat16
    lens = (700, 33, 2000)
    cache, table = fill_cache(2, 64, 128, [n + 1 for n in lens], seed=seed)
    return {"x": rnd(3, 1024, dtype=bf16, seed=seed), "r": rnd(3, 1024, dtype=bf16, seed=seed + 1),
            "w": rnd(1024, dtype=bf16, seed=2), "cache": cache, "table": table,
            "k": rnd(3, 2, 1, 128, dtype=bf16, seed=seed + 3),
            "v": rnd(3, 2, 1, 128, dtype=bf16, seed=seed + 4), "start": ints(*lens),
            "lens": ints(*lens) + 1, "q": rnd(3, 8, 1, 128, dtype=bf16, seed=seed + 5),
            "keys": rnd(3, 2, 900, 128, dtype=bf16, seed=seed + 6),
            "logits": rnd(3, 70001, dtype=bf16, seed=seed + 7),
            "tokens": ints(5, 6, 7, dtype=torch.int64)}


def same_values(a, b):
    return all(torch.equal(x.nan_to_num(), y.nan_to_num()) for x, y in zip(a, b))


def test_graphs_and_streams():
    """Two captured steps, replayed in turn with new inputs and eager calls
    between, and steps on two streams at once give the eager results bit for
    bit."""
    w = W()
    states = [step_state(100), step_state(200)]
    others = [step_state(300), step_state(400)]
    for s in states:
        step_calls(w, s)
    torch.cuda.synchronize()
    graphs = []
    for s in states:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step_calls(w, s)
        graphs.append((g, out))
    for turn in range(3):
        for s, o in zip(states, others):
            for name in ("x", "q", "k", "v", "logits", "keys"):
                s[name].copy_(o[name] * (turn + 1) * 0.5)
        for g, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        for s, (_, out) in zip(states, graphs):
            kept = [t.clone() for t in out]
            assert same_values(kept, step_calls(w, s))
            torch.cuda.synchronize()
    eager = [step_calls(w, s) for s in states]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in states]
    got = [None, None]
    for _ in range(3):
        for i, (s, stream) in enumerate(zip(states, streams)):
            with torch.cuda.stream(stream):
                got[i] = step_calls(w, s)
    torch.cuda.synchronize()
    for a, b in zip(got, eager):
        assert same_values(a, b)


@pytest.mark.parametrize("D", [64, 128])
def test_window_many_rows(D):
    """Launches of 256-row programs: sampled queries of every head, at the
    window's edges and elsewhere, and NaN behind what a query sees."""
    B, H, KV, S = 2, 64, 32, 1111
    q = rnd(B, H, S, D, dtype=torch.bfloat16, seed=1)
    k, v = rnd(B, KV, S, D, dtype=torch.bfloat16, seed=2), rnd(B, KV, S, D, dtype=torch.bfloat16, seed=3)
    v[1, 3, 700] = float("nan")
    got = W().window_attention(q, k, v, window=200, sinks=5)
    at = [0, 1, 199, 200, 204, 205, 500, 699, 700, 899, 900, 1110]
    for b in range(B):
        want, a = orc.attention(q[b][:, at], k[b], v[b], at, 200, 5)
        check_attention(got[b][:, at], want, a, torch.bfloat16, False, S, 0.0)
    rows = torch.arange(S, device="cuda")
    assert torch.equal(got[1, 6, :, 0].isnan(), (rows >= 700) & (rows < 900))
    assert int(got.isnan().sum()) == 2 * 200 * D


def test_logprobs_uneven_parts():
    """Rows whose parts differ by much, so that some waves hold none of the
    alternatives and larger numbers come late: stairs up and down, a few large
    logits in front, all of them at the end."""
    V = 30001
    g = torch.Generator(device="cuda").manual_seed(3)
    noise = torch.randn(6, V, generator=g, device="cuda")
    at = torch.arange(V, device="cuda")
    base = torch.stack([at // 512 * 3.0, -(at // 512) * 3.0, (at // 512 % 4) * 40.0,
                        torch.where(at < 9, 300.0, 0.0), torch.where(at > V - 9, 300.0, -300.0),
                        ((at // 512 % 4) == 3) * 25.0])
    check_logprobs(base + noise, torch.full((6,), 17, device="cuda"), 20)
    check_logprobs((base + noise)[:, 3:], torch.full((6,), 17, device="cuda"), 5)
    check_logprobs((base * 0.1 + noise).half(), torch.full((6,), 17, device="cuda"), 0)


def test_append_to_calibrated_scales():
    """Blocks whose scales are no powers of two: kept while they do, whatever
    the new tokens' own need is."""
    for S in (3, 40):
        cache = make_cache(12, 2, 32, 64, seed=S, low=-7, high=-3)
        for c in cache[2:]:
            c.mul_(1.37)
        for c in cache[:2]:
            c.copy_(torch.where(c.float().isnan(), 0.0, c.float()).to(E4M3))
        table = torch.randperm(12, device="cuda").to(torch.int32).view(3, 4)
        k, v = rnd(3, 2, S, 64, seed=S), rnd(3, 2, S, 64, seed=S + 1) * 30
        want = orc.append(cache, k, v, table, ints(5, 31, 70))
        W().kv_append(cache, k, v, table, ints(5, 31, 70))
        got = numbers(cache)
        assert torch.equal(got[2], want[2]) and torch.equal(got[3], want[3])
        for a, b in zip(got[:2], want[:2]):
            # a quotient in fp32 may round to the other side of a tie
            assert float((a != b).double().mean()) <= 1e-4
            assert bool(((a - b).abs() <= 2.0 ** -3 * b.abs() + 2.0 ** -9).all())


@pytest.mark.parametrize("B", [3, 70])
@pytest.mark.parametrize("slots", [4, 40])
def test_cached_lengths_of_any_size(B, slots):
    """Lengths up to 2^31 - 1, far behind the table's end: by units and by
    shares, with more sequences than a wave has lanes."""
    some = (2 ** 31 - 1, 2 ** 31 - 65, 2 ** 30, 2 ** 30 + 77, 100, -2 ** 31, 2 ** 31 - 1024)
    lens = [some[b % len(some)] for b in range(B)]
    cache, table = fill_cache(1, 64, 64, [64 * slots] * 3, seed=slots)
    table = table[torch.arange(B, device="cuda") % 3].contiguous()
    q = rnd(B, 2, 2, 64, dtype=torch.bfloat16, seed=B)
    held = 64 * slots
    for window, sinks in ((None, 0), (64, 4), (500, 130), (2 ** 30 - 1, 0)):
        got = W().cached_attention(q, cache, table, ints(*lens), window=window, sinks=sinks)
        for b, n in enumerate(lens):
            keys, values, has = orc.cached(cache, table, b, max(0, min(n, held)))
            want, a = orc.attention(q[b], keys, values, range(n - 2, n), window, sinks, None, has)
            check_attention(got[b], want, a, q.dtype, True, held, 0.0)


def test_window_positions_of_any_size():
    """Queries far behind the keys or in front of them all."""
    starts = ints(2 ** 31 - 1, 2 ** 30, 2 ** 30 + 90, -2 ** 31, -2 ** 30, 2 ** 31 - 200)
    q = rnd(6, 2, 3, 64, dtype=torch.bfloat16, seed=1)
    k, v = (rnd(6, 1, 150, 64, dtype=torch.bfloat16, seed=i) for i in (2, 3))
    for window, sinks in ((None, 0), (64, 0), (64, 70), (2 ** 30 - 1, 0), (2 ** 30 - 1, 3)):
        check_window(q, k, v, window=window, sinks=sinks, start=starts)


def test_attention_refuses_expanded_outputs():
    """As Python errors, whichever way the call takes."""
    q = rnd(2, 4, 3, 64, dtype=torch.bfloat16)
    k = rnd(2, 2, 70, 64, dtype=torch.bfloat16)
    cache, table = fill_cache(2, 64, 64, (64, 64), seed=1)
    one = torch.empty(1, 4, 3, 64, dtype=torch.bfloat16, device="cuda").expand(2, 4, 3, 64)
    with pytest.raises(ValueError, match="overlap"):
        W().window_attention(q, k, k, out=one)
    with pytest.raises(ValueError, match="overlap"):
        W().cached_attention(q, cache, table, ints(64, 64), out=one)
    with pytest.raises(ValueError, match="scale"):
        W().window_attention(q, k, k, scale=float("inf"))
    # read-only operands may be expanded
    check_window(q, k[:, :1].expand(2, 2, 70, 64), k[:1].expand(2, 2, 70, 64))
    check_window(q[:, :, :1].expand(2, 4, 3, 64), k[:, :, :1].expand(2, 2, 70, 64), k)


def test_cached_many_sequences_and_rows():
    """More sequences than a wave has lanes, of uneven lengths, in runs and in
    parts, and row tiles of many queries over a long cache."""
    for B, longest, KV, H, S, D in ((130, 900, 2, 4, 1, 64), (300, 130, 1, 1, 2, 64),
                                    (66, 6000, 1, 4, 1, 128), (2, 5000, 2, 8, 40, 64),
                                    (3, 2500, 1, 8, 5, 256)):
        lens = [1 + (b * 7919) % longest for b in range(B)]
        lens[B // 2] = 0
        cache, table = fill_cache(KV, 64, D, lens, seed=B, outlier=False)
        q = rnd(B, H, S, D, dtype=torch.bfloat16, seed=B)
        check_cached(q, cache, table, lens)
        if S > 1:
            check_cached(q, cache, table, lens, window=700, sinks=3)


def test_offsets_past_32_bits():
    """Rows, keys and blocks whose byte offsets, and element offsets of the
    8-bit cache, pass 2^32."""
    bf16 = torch.bfloat16
    blocks = 2 ** 19 + 5  # of 8192 bytes
    cache = W().kv_cache(blocks, 1, 128)
    table = torch.tensor([[blocks - 1, 3, blocks - 2]], dtype=torch.int32, device="cuda")
    k, v = rnd(1, 1, 150, 128, dtype=bf16, seed=1), rnd(1, 1, 150, 128, dtype=bf16, seed=2)
    W().kv_append(cache, k, v, table, ints(0))
    small = W().kv_cache(3, 1, 128)
    order = torch.tensor([[2, 0, 1]], dtype=torch.int32, device="cuda")
    W().kv_append(small, k, v, order, ints(0))
    for big, little in zip(cache, small):
        for at, to in ((blocks - 1, 2), (3, 0), (blocks - 2, 1)):
            assert torch.equal(big[at].view(torch.uint8), little[to].view(torch.uint8))
    q = rnd(1, 4, 2, 128, dtype=bf16, seed=3)
    assert torch.equal(W().cached_attention(q, cache, table, ints(150)),
                       W().cached_attention(q, small, order, ints(150)))
    del cache, big
    # 2^32 bytes and more from the first key to the last: a stride of 2^23 numbers
    keys = torch.zeros(300 * 2 ** 23, dtype=bf16, device="cuda").view(300, 2 ** 23)
    k, v = rnd(1, 1, 300, 64, dtype=bf16, seed=4), rnd(1, 1, 300, 64, dtype=bf16, seed=5)
    keys[:, :64], keys[:, 64:128] = k[0, 0], v[0, 0]
    q = rnd(1, 2, 70, 64, dtype=bf16, seed=6)
    far = [keys[:, i:i + 64].view(1, 1, 300, 64) for i in (0, 64)]
    assert torch.equal(W().window_attention(q, *far, window=90, sinks=3),
                       W().window_attention(q, k, v, window=90, sinks=3))
    # and rows of the norm and of the logits
    x = keys[:, :1000]
    w = torch.ones(1000, dtype=bf16, device="cuda")
    assert torch.equal(W().rmsnorm(x, w)[0], W().rmsnorm(x.contiguous(), w)[0])
    t = torch.arange(300, device="cuda")
    for a, b in zip(W().token_logprobs(x, t, top=4), W().token_logprobs(x.contiguous(), t, top=4)):
        assert torch.equal(a, b)


def test_calls_of_both_paths_agree(monkeypatch):
    """The calls made in C++ and those made in Python give the same bytes."""
    from newt_amd import serving
    bf16 = torch.bfloat16
    x, r, w = (rnd(7, 512, dtype=bf16, seed=i) for i in (1, 2, 3))
    q, k = rnd(2, 4, 5, 64, dtype=bf16, seed=4), rnd(2, 2, 900, 64, dtype=bf16, seed=5)
    logits, t = rnd(3, 30000, dtype=bf16, seed=6), torch.tensor([5, -1, 29999], device="cuda")
    table = torch.arange(30, device="cuda").to(torch.int32).view(2, 15)

    def calls():
        cache = W().kv_cache(30, 2, 64)
        W().kv_append(cache, k, k, table, ints(0, 3), ints(900, 800))
        return [*W().rmsnorm(x, w[0], residual=r, out_dtype=E4M3, group=128),
                *W().token_logprobs(logits, t, top=6, temperature=0.7),
                W().window_attention(q, k, k, window=300, sinks=4, q_start=ints(800, 20)),
                W().cached_attention(q, cache, table, ints(900, 803), window=500, sinks=2), *cache]

    fast = calls()
    monkeypatch.setattr(serving, "_fast", lambda *a: None)
    for a, b in zip(fast, calls()):
        assert a.dtype == b.dtype and a.stride() == b.stride()
        assert torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


@pytest.mark.parametrize("V", [4000, 70001])
@pytest.mark.parametrize("offset,temperature", [(1e3, 1.0), (-1e3, 1.0), (1e4, 1.0), (-1e4, 1.0),
                                                (1e5, 1.0), (-1e5, 1.0), (20.0, 0.02),
                                                (-20.0, 0.02)])
def test_logprobs_far_from_zero(V, offset, temperature):
    """fp32 rows around a common offset: what a row's results are relative to
    drops out, so the bound is that of rows around 0. Maxima differ between
    waves and splits, and in half of the rows grow towards the end."""
    x = rnd(8, V, seed=V, scale=3.0)
    x[4:] += torch.linspace(0, 6, V, device="cuda")
    check_logprobs(x * temperature + offset, torch.arange(8, device="cuda") * (V // 8), 5,
                   temperature=temperature)


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("scale", [1e4, 1e7, -1e8, 3e9, 1e15, 1e28])
def test_window_large_scores(dtype, scale):
    """Scores far above 2^24, whose products with log2(e) are rounded by more
    than the exponent of a weight can be off: whole numbers, so that a row's
    weights are equal among its largest scores and 0 elsewhere."""
    g = torch.Generator(device="cuda").manual_seed(7)
    q, k = (torch.randint(-3, 4, s, generator=g, device="cuda").to(dtype)
            for s in ((2, 4, 70, 64), (2, 2, 300, 64)))
    v = rnd(2, 2, 300, 64, dtype=dtype, seed=8)
    check_window(q, k, v, scale=scale)
    check_window(q, k, v, window=100, sinks=3, scale=scale)
    check_window(q[:, :, :1], k, v, scale=scale)


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("scale", [1e4, 1e7, -1e8, 3e9, 1e15, 1e25])
def test_cached_large_scores(dtype, scale):
    """As test_window_large_scores, over whole numbers times powers of two."""
    lens = (300, 1, 64, 2500)
    cache, table = fill_cache(2, 64, 64, lens, seed=3, outlier=False)
    g = torch.Generator(device="cuda").manual_seed(7)
    cache.k.copy_(torch.randint(-3, 4, cache.k.shape, generator=g, device="cuda").to(E4M3))
    for S in (1, 5):
        q = torch.randint(-3, 4, (4, 4, S, 64), generator=g, device="cuda").to(dtype)
        check_cached(q, cache, table, lens, scale=scale)
        check_cached(q, cache, table, lens, window=100, sinks=3, scale=scale)


def test_window_small_weights():
    """fp16: one key that outweighs each of the others by e^18 and comes before
    them, and 2^16 others whose values alone are not 0. A weight is off by
    2^-11 of itself, from 2^-21 of the largest on; below by 2^-32 of that."""
    n, D = 2 ** 16 + 1, 64
    q, k, v = (torch.zeros(1, 1, m, D, dtype=torch.float16, device="cuda") for m in (1, n, n))
    q[..., 0] = 1.0
    k[0, 0, 1:, 0] = -18.0
    v[0, 0, 1:] = rnd(n - 1, D, dtype=torch.float16, seed=1).abs()
    # so many sequences that a row's keys are all one program's
    got = W().window_attention(q.expand(4, 128, 1, D), k.expand(4, 128, n, D),
                               v.expand(4, 128, n, D), scale=1.0)
    want, a = orc.attention(q[0], k[0], v[0], [n - 1], scale=1.0)
    tol = ((2.0 ** -11 + (D + 64) * 64 * 2.0 ** -24) * a + 2.0 ** -11 * want.abs() + 2.0 ** -25
           + n * 2.0 ** -32 * float(v.max()))
    assert bool(((got.double() - want).abs() <= tol).all())
    assert torch.equal(got, got[:1, :1].expand_as(got))


def test_ordinary_calls_go_through_cpp(monkeypatch):
    """The C++ extension takes every operator's ordinary call, and leaves wrong
    shapes, types, strides and numbers to Python."""
    from newt_amd import serving
    fast, results = serving._fast, []

    def recorded(*args):
        results.append(fast(*args))
        return results[-1]

    monkeypatch.setattr(serving, "_fast", recorded)
    bf16 = torch.bfloat16
    x, w = rnd(7, 512, dtype=bf16, seed=1), rnd(512, dtype=bf16, seed=2)
    q, k = rnd(2, 4, 5, 64, dtype=bf16, seed=3), rnd(2, 2, 90, 64, dtype=bf16, seed=4)
    logits, tokens = rnd(3, 3000, dtype=bf16, seed=5), torch.arange(3, device="cuda")
    cache = W().kv_cache(6, 2, 64, block_size=32)
    table = torch.arange(6, device="cuda").to(torch.int32).view(2, 3)
    calls = {"rmsnorm": (x, w, 1e-6, x, -1, None, None, None),
             "token_logprobs": (logits, tokens, 5, 1.0),
             "kv_append": (cache, k, k, table, ints(0, 3), ints(90, 80)),
             "cached_attention": (q, cache, table, ints(90, 83), None, 0, None, None),
             "window_attention": (q, k, k, 40, 2, 0.125, ints(80, 20), None)}
    W().rmsnorm(x, w, residual=x)
    W().rmsnorm(x, w, out_dtype=E4M3, group=64, out=torch.empty_like(x, dtype=E4M3))
    W().token_logprobs(logits, tokens, top=5, temperature=0.7)
    W().kv_append(*calls["kv_append"])
    W().cached_attention(q, cache, table, ints(90, 83), window=30, sinks=2, out=q.clone())
    W().window_attention(q, k, k)
    assert len(results) == 6 and all(r is not None for r in results)
    wrong = {"rmsnorm": {0: (x[0], x.double(), x.t(), x[:, ::2], None), 1: (w[1:], w.half(), None),
                         2: ("a",), 3: (x[1:], x.float()), 4: (0, -2), 5: (64, 32.0),
                         6: (x[1:], x.float(), x[:1].expand(7, 512)), 7: (x[1:], x.float())},
             "token_logprobs": {0: (logits[0], logits.double(), logits[:, ::2], None),
                                1: (tokens[1:], tokens.int(), None), 2: (65, -1, 2.0),
                                3: (0.0, -1.0, float("nan"), None)},
             "kv_append": {0: (cache[:3], tuple(cache[:2]) + (cache[2][:3], cache[3]),
                               (cache[1], cache[0], *cache[2:]), None),
                           1: (k[0], k[:, :1], k.half(), None), 2: (k[:, :, 1:], k.half(), None),
                           3: (table[:1], table.long(), None), 4: (ints(0), tokens[:2], None),
                           5: (ints(0), tokens[:2])},
             "cached_attention": {0: (q[0], q[:, :3], q.float(), q.half()[..., ::2], None),
                                  1: (cache[:3], None), 2: (table[:1], table.long(), None),
                                  3: (ints(0), tokens[:2], None), 4: (0, 2.0), 5: (-1, 3),
                                  6: ("a", float("inf")),
                                  7: (q[:, :1], q.half(), q[:, :1].expand(2, 4, 5, 64))},
             "window_attention": {0: (q[0], q[:, :3], q.float(), None), 1: (k[:1], k.half(), None),
                                  2: (k[:, :, 1:], k.half(), None), 3: (0, 2.0), 4: (-1, None),
                                  5: ("a", float("nan")), 6: (ints(0), tokens[:2]),
                                  7: (q[:, :1], q.half(), q[:, :1].expand(2, 4, 5, 64))}}
    for name, args in calls.items():
        assert fast(name, *args) is not None
        for i, values in wrong[name].items():
            for value in values:
                assert fast(name, *args[:i], value, *args[i + 1:]) is None, (name, i)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [4000, 70001])
@pytest.mark.parametrize("temperature", [1e-6, 3e-9, 1e-20, 2.0 ** -99])
def test_logprobs_tiny_temperatures(dtype, V, temperature):
    """Logits over the temperature far above 2^24: a row's largest logits share
    all of its probability. They are whole numbers, so that fp32 tells them
    apart at any temperature."""
    g = torch.Generator(device="cuda").manual_seed(V)
    x = torch.randint(-40, 40, (6, V), generator=g, device="cuda").to(dtype)
    x[3:] -= 100
    tokens = x.float().argmax(-1)
    check_logprobs(x, tokens, 5, temperature=temperature)
    logp, entropy, top_logp, _ = W().token_logprobs(x, tokens, top=5, temperature=temperature)
    n = (x == x.amax(-1, keepdim=True)).sum(-1).double()
    # what is left of the sum's and the logarithm's own roundings
    assert bool(((logp.double() + n.log()).abs() <= (V / 64 + 16) * 2.0 ** -24 * 10).all())
    assert bool(((entropy.double() - n.log()).abs() <= (V / 64 + 16) * 2.0 ** -24 * 10).all())
    assert torch.equal(logp, top_logp[:, 0])


@pytest.mark.parametrize("V", [4000, 70001])
def test_logprobs_huge_logits(V):
    """fp32 logits around 1e10, whose steps are 1024, and ones whose maximum
    grows through all sizes from far below 2^20 to far above it."""
    g = torch.Generator(device="cuda").manual_seed(V)
    x = 1024.0 * torch.randint(4, (4, V), generator=g, device="cuda")
    tokens = torch.full((4,), V // 2, device="cuda")
    for offset in (1e10, -1e10, 3e13):
        check_logprobs(x * (offset / 1e10 if offset > 1e12 else 1.0) + offset, tokens, 5)
    noise = torch.randn(4, V, generator=g, device="cuda")
    for middle in (2 ** 20 / 1.4426950408889634, -2 ** 20 / 1.4426950408889634):
        for ramp in (torch.linspace(-20, 20, V, device="cuda"),
                     torch.linspace(20, -20, V, device="cuda")):
            check_logprobs(middle + ramp + noise, tokens, 5)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [50, 20001])
def test_logprobs_of_lowest_values(dtype, V):
    """Tokens masked with the type's lowest value have log probabilities of that
    size, not of -inf, as themselves and as alternatives."""
    x = rnd(4, V, dtype=dtype, seed=V)
    x[0, 3:] = torch.finfo(dtype).min
    x[1, ::2] = torch.finfo(dtype).min
    x[2, :-1] = torch.finfo(dtype).min
    x[3, 1:] = float("-inf")
    tokens = ints(V - 1, 0, 0, 1, dtype=torch.int64)
    check_logprobs(x, tokens, 8)
    check_logprobs(x, tokens, 8, temperature=2.0)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N", [72, 4097, 40000])
def test_rmsnorm_in_place(dtype, N):
    """y over x or over the residual, with and without the sum beside it."""
    x, r = rnd(5, N, dtype=dtype, seed=N), rnd(5, N, dtype=dtype, seed=N + 1)
    w = rnd(N, dtype=dtype, seed=N + 2)
    y, _, h = W().rmsnorm(x, w, residual=r)
    for i in (0, 1):
        both = [x.clone(), r.clone()]
        out, _, hidden = W().rmsnorm(both[0], w, residual=both[1], out=both[i])
        assert out is both[i] or out.data_ptr() == both[i].data_ptr()
        assert torch.equal(out, y) and torch.equal(hidden, h)
        both = [x.clone(), r.clone()]
        out, _, hidden = W().rmsnorm(both[0], w, residual=both[1], out=both[i], hidden=both[1 - i])
        assert torch.equal(both[i], y) and torch.equal(both[1 - i], h)
    y = W().rmsnorm(x, w)[0]
    assert torch.equal(W().rmsnorm(x, w, out=x)[0], y) and torch.equal(x, y)


@pytest.mark.parametrize("V", [50, 20001])
def test_logprobs_gaps_beyond_fp32(V):
    """fp32 logits further apart than the largest number, which a temperature
    brings together again; -inf beside the lowest of them stays -inf."""
    x = rnd(3, V, seed=V) * 1e38
    x[0, :5], x[0, 5:9] = 3e38, -3e38
    x[1] = -3.3e38
    x[1, 3:8] = float("-inf")
    x[2, 7] = torch.finfo(torch.float32).max
    tokens = ints(7, 4, 9, dtype=torch.int64)
    for temperature in (10.0, 1e20, 2.0 ** 99):
        check_logprobs(x, tokens, 8, temperature=temperature)
    got = W().token_logprobs(x, tokens, top=8, temperature=0.5)[0]
    assert float(got[1]) == float("-inf")
