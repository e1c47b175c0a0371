"""rotate, q4_matmul, q4_gated and sample on the GPU against their definitions in
64 bits (oracle/decoding.py). Tolerances count roundings: half a step of the
output's type, and of fp32 for each operation in front of it."""

import decimal
import math

import pytest
import torch

from oracle import decoding as orc
from oracle import serving as sorc

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
EPS = 2.0 ** -24  # half a step of fp32
INF, NAN = float("inf"), float("nan")


def W():
    from newt_amd import workloads
    return workloads


def rnd(*shape, dtype=F32, seed=0, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dtype).cuda()


def ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device="cuda")


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


# ---------------------------------------------------------------------------
# rotary positions
# ---------------------------------------------------------------------------
def check_rotated(got, x, freqs, positions, amplitude=1.0, **kw):
    """cos and sin are off by 2^-22 at most (their sums' roundings), the products
    and their sum by three more roundings of fp32."""
    x = x.cpu()
    want = orc.rotate(x, freqs, positions.cpu(), amplitude=amplitude, **kw)
    reach = orc.rotate(x.abs(), freqs * 0, positions.cpu(), amplitude=abs(amplitude), **kw)
    n = len(freqs)
    ia = torch.arange(n) * 2 if kw.get("interleaved") else torch.arange(n)
    ib = ia + 1 if kw.get("interleaved") else ia + n
    both = reach[..., ia] + reach[..., ib]  # amplitude (|a| + |b|)
    bound = torch.zeros_like(want)
    bound[..., ia] = bound[..., ib] = both * 8 * EPS + 2.0 ** -126
    tiny = 2.0 ** -25 if x.dtype == F16 else 0.0  # half of fp16's smallest step
    turned = bound > 0
    bound += (want.abs() * half_step(x.dtype) * (1 + 2.0 ** -10) + tiny) * turned
    assert got.dtype == x.dtype
    assert bool(((got.double().cpu() - want).abs() <= bound).all())


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("D,dim", [(128, 128), (64, 32), (80, 40), (256, 256), (96, 2), (7, 6),
                                   (66, 66)])
def test_rotate(dtype, interleaved, D, dim):
    w = W()
    rot = w.rotary(dim, interleaved=interleaved)
    q, k = rnd(2, 6, 5, D, dtype=dtype, seed=1), rnd(2, 2, 5, D, dtype=dtype, seed=2)
    start = ints([0, 1000])
    got = w.rotate(q, k, rot, start)
    at = start[:, None] + torch.arange(5, device="cuda")
    for o, x in zip(got, (q, k)):
        check_rotated(o, x, orc.frequencies(dim), at, interleaved=interleaved)


@pytest.mark.parametrize("factor,ramp,base", [(4.0, None, 10000.0), (32.0, (4096, 1.0, 4.0), 5e5),
                                              (0.5, (64, 0.0, 0.1), 3.0)])
def test_rotate_scaled_and_transposed(factor, ramp, base):
    w = W()
    rot = w.rotary(64, base=base, factor=factor, ramp=ramp, amplitude=1.25)
    freqs = orc.frequencies(64, base, factor, ramp)
    q = rnd(3, 2, 9, 128, seed=3)
    at = torch.randint(0, 1 << 17, (3, 9), generator=torch.Generator().manual_seed(1)).int().cuda()
    o, none = w.rotate(q, None, rot, at)
    assert none is None
    check_rotated(o, q, freqs, at, amplitude=1.25)
    # the gradient: <rotate(q), g> = <q, rotate transposed(g)>, and differences
    g = rnd(3, 2, 9, 128, seed=4)
    back, _ = w.rotate(g, None, rot, at, transposed=True)
    check_rotated(back, g, freqs, at, amplitude=1.25, transposed=True)
    d = rnd(3, 2, 9, 128, seed=5) * 2.0 ** -4
    ahead, behind = w.rotate(q + d, None, rot, at)[0], w.rotate(q - d, None, rot, at)[0]
    rise = ((ahead.double() - behind.double()) * g.double()).sum() / 2
    along = (d[..., :].double() * torch.cat((back[..., :64], g[..., 64:]), -1).double()).sum()
    # every number is off by 8 roundings of fp32 of numbers below 8
    assert abs(float(rise - along)) < 3 * 9 * 2 * 128 * 8 * 8 * EPS


def test_rotate_far_positions():
    """Against angles in decimal: 64 bits do not hold them."""
    w = W()
    dim, positions = 16, [2 ** 31 - 1, -2 ** 31, 123456789, -1, 0, 2 ** 24 + 1]
    x = torch.ones(1, 1, len(positions), dim, device="cuda")
    x[..., dim // 2:] = 0.0
    o, _ = w.rotate(x, None, w.rotary(dim, base=500000.0), ints([positions]))
    with decimal.localcontext(decimal.Context(prec=60)):
        pi2 = 2 * decimal.Decimal("3.14159265358979323846264338327950288419716939937510")
        for i in range(dim // 2):
            f = decimal.Decimal(500000) ** (decimal.Decimal(-2 * i) / dim)
            for t, p in enumerate(positions):
                angle = float(f * p % pi2)
                assert abs(float(o[0, 0, t, i]) - math.cos(angle)) < 8 * EPS
                assert abs(float(o[0, 0, t, i + dim // 2]) - math.sin(angle)) < 8 * EPS
    # starts whose tokens run past 2^31
    o, _ = w.rotate(x[:, :, :2], None, w.rotary(2, frequencies=[1.0]), ints([2 ** 31 - 1]))
    for t in range(2):
        angle = float(decimal.Decimal(2 ** 31 - 1 + t) % decimal.Decimal(
            "6.28318530717958647692528676655900576839433879875021"))
        assert abs(float(o[0, 0, t, 0]) - math.cos(angle) + math.sin(angle)) < 16 * EPS


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_rotate_strides_and_given_outputs(dtype):
    w = W()
    rot = w.rotary(64)
    freqs = orc.frequencies(64)
    x = rnd(2, 7, 13, 64, dtype=dtype, seed=6)  # [B, S, q, k and v heads, D] of one product
    packed = x.transpose(1, 2)
    q, k = packed[:, :8], packed[:, 8:10]
    at = ints([[5 * i + j for j in range(9, -5, -2)] for i in range(2)])
    assert at.shape == (2, 7)
    a, b = w.rotate(q, k, rot, at)
    check_rotated(a, q, freqs, at)
    check_rotated(b, k, freqs, at)
    # transposed positions, and outputs that are the inputs
    wide = at.repeat_interleave(3, 0).t().contiguous().t()[::3]
    rest = packed[:, 10:].clone()
    got = w.rotate(q, k, rot, wide, q_out=q, k_out=k)
    assert got[0].data_ptr() == q.data_ptr() and torch.equal(q, a) and torch.equal(k, b)
    assert torch.equal(packed[:, 10:], rest)
    # rows of an odd stride and address
    odd = torch.zeros(2 * 8 * 7 * 65 + 1, dtype=dtype, device="cuda")[1:].view(2, 8, 7, 65)[..., :64]
    back, _ = w.rotate(a, None, rot, at, transposed=True, q_out=odd)
    check_rotated(odd, a, freqs, at, transposed=True)
    assert bool((odd.as_strided((2, 8, 7), odd.stride()[:3], odd.storage_offset() + 64) == 0).all())


def test_rotate_many_heads_and_tokens():
    w = W()
    rot = w.rotary(128)
    q, k = rnd(1, 33, 1500, 128, dtype=BF16), rnd(1, 1, 1500, 128, dtype=BF16, seed=1)
    start = ints([77])
    at = start[:, None] + torch.arange(1500, device="cuda")
    for o, x in zip(w.rotate(q, k, rot, start), (q, k)):
        check_rotated(o, x, orc.frequencies(128), at)
    empty = w.rotate(q[:, :, :0], k[:, :, :0], rot, start)
    assert empty[0].shape == (1, 33, 0, 128)
    # NaN and infinities stay in their pair
    q[0, 3, 7, 5] = NAN
    q[0, 4, 8, 70] = INF
    o = w.rotate(q, None, rot, start)[0]
    bad = (~o.isfinite()).nonzero().tolist()
    assert bad == [[0, 3, 7, 5], [0, 3, 7, 69], [0, 4, 8, 6], [0, 4, 8, 70]]


# ---------------------------------------------------------------------------
# products with 4-bit weights
# ---------------------------------------------------------------------------
def weights(N, K, group, zeros=True, dtype=BF16, seed=0):
    g = torch.Generator().manual_seed(seed)
    q = torch.randint(0, 256, (N, K // 2), generator=g, dtype=torch.uint8)
    s = (torch.rand(N, K // group, generator=g) * 0.02 + 0.002).to(dtype)
    s[::7] *= -1
    z = torch.randint(0, 16, s.shape, generator=g, dtype=torch.uint8) if zeros else None
    return q, s, z


def on_gpu(q, s, z, gated=False):
    return W().q4_weights(q.cuda(), s.cuda(), None if z is None else z.cuda(), gated=gated)


def q4_bound(x, q, s, z):
    """(y, its bound in fp32). Sums in fp32 hold x (16 + q) s and x (16 + z) s: of a
    group at most 128 additions each, rounded, then a product and an addition a
    group and one for each of 16 waves."""
    y, _ = orc.q4(x, q, s, z)
    K = x.shape[1]
    group = K // s.shape[1]
    numbers = torch.stack((q & 15, q >> 4), -1).flatten(1).double()
    zero = 8.0 if z is None else z.double().repeat_interleave(group, 1)
    reach = x.double().abs() @ ((32 + numbers + zero)
                                * s.double().abs().repeat_interleave(group, 1)).T
    return y, reach * (128 + 4 + K // group + 16) * EPS


def check_q4(x, raw, out_dtype=None, bias=None, laid_out=None, **kw):
    laid_out = on_gpu(*raw) if laid_out is None else laid_out
    got = W().q4_matmul(x, laid_out, out_dtype=out_dtype, bias=bias, **kw)
    want, bound = q4_bound(x.cpu(), *raw)
    if bias is not None:
        want = want + bias.double().cpu()
    step = half_step(got.dtype)
    assert got.dtype == (out_dtype or x.dtype)
    err = (got.double().cpu() - want).abs()
    assert bool((err <= bound * (1 + step) + want.abs() * step + 2.0 ** -25 * (step == 2 ** -11)).all())
    # all in all: sums' roundings in no order (2^-18), the output's own
    assert float(err.norm()) <= float(want.norm()) * (2.0 ** -18 + step)
    return got


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("M,N,K", [(1, 64, 512), (2, 1, 128), (5, 48, 384), (16, 130, 640),
                                   (17, 33, 256), (40, 95, 1024), (70, 257, 128), (129, 64, 2176)])
def test_q4_matmul(dtype, group, M, N, K):
    raw = weights(N, K, group, zeros=(M + group) % 3 > 0, dtype=BF16 if M % 2 else F16, seed=M)
    x = rnd(M, K, dtype=dtype, seed=M + 1)
    check_q4(x, raw)


@pytest.mark.parametrize("M,N,K,group", [(1, 20, 32, 32), (3, 17, 96, 32), (33, 40, 192, 64),
                                         (200, 100, 160, 32), (1, 300, 16384, 128), (7, 16, 11008, 64),
                                         (300, 24, 4160, 64), (260, 2003, 256, 128)])
def test_q4_matmul_odd_sizes(M, N, K, group):
    raw = weights(N, K, group, seed=N)
    x = rnd(M, K, dtype=BF16, seed=1)
    bias = rnd(N, dtype=BF16, seed=2)
    check_q4(x, raw, out_dtype=F32)
    check_q4(x, raw, bias=bias)


def test_q4_matmul_rows_alone():
    """A row's result does not depend on the others of its launch's kind."""
    raw = weights(333, 1024, 128, seed=5)
    laid_out = on_gpu(*raw)
    x = rnd(16, 1024, dtype=BF16, seed=6)
    all_rows = W().q4_matmul(x, laid_out)
    for i in (0, 7, 15):
        assert torch.equal(W().q4_matmul(x[i:i + 1], laid_out)[0], all_rows[i])


def test_q4_matmul_strides():
    raw = weights(50, 256, 64, seed=7)
    base = rnd(11, 300, dtype=F16, seed=8)
    x = base[::2, 7:263]
    out = torch.full((6, 77), -5.0, dtype=F16, device="cuda")
    got = check_q4(x, raw, out=out[:, 3:53])
    assert got.data_ptr() == out[:, 3:].data_ptr()
    assert bool((out[:, :3] == -5).all()) and bool((out[:, 53:] == -5).all())
    assert W().q4_matmul(x[:0], on_gpu(*raw)).shape == (0, 50)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_q4_matmul_many_rows_of_any_stride(dtype, group):
    """Rows that are not aligned to 16 bytes, the same row again and again, and the
    numbers of rows on either side of the tiles'."""
    raw = weights(300, 896, group, seed=group, dtype=F16)
    base = rnd(131, 1001, dtype=dtype, seed=8)
    laid_out = on_gpu(*raw)
    check_q4(base[1::2, 5:901], raw, laid_out=laid_out)
    check_q4(base[7:8, :896].expand(70, 896), raw, laid_out=laid_out)
    check_q4(base[7:8, :896].expand(9, 896), raw, laid_out=laid_out)
    aligned = base[:, :896].contiguous()
    for M in (48, 49, 64, 65, 128):
        check_q4(aligned[:M], raw, laid_out=laid_out, bias=rnd(300, dtype=dtype, seed=M))


def test_q4_matmul_common_offset():
    """Rows far from zero: what the products have too much is taken off again."""
    raw = weights(64, 2048, 128, seed=9)
    x = (rnd(4, 2048, seed=10) + 30.0).to(BF16)
    check_q4(x, raw, out_dtype=F32)


def test_q4_matmul_not_finite():
    """A row with an infinity or NaN gives no numbers, the others theirs."""
    raw = weights(40, 256, 128, seed=11)
    x = rnd(6, 256, dtype=BF16, seed=12)
    want = W().q4_matmul(x, on_gpu(*raw))
    y = x.clone()
    y[1, 3], y[4, 200] = INF, NAN
    got = W().q4_matmul(y, on_gpu(*raw))
    for i in range(6):
        if i in (1, 4):
            assert not bool(got[i].isfinite().any())
        else:
            assert torch.equal(got[i], want[i])


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("M,F,K,group", [(1, 64, 512, 128), (3, 37, 96, 32), (16, 16, 128, 64),
                                         (31, 100, 256, 64), (140, 90, 1024, 128)])
def test_q4_gated(act, dtype, M, F, K, group):
    raw = weights(2 * F, K, group, zeros=M != 3, dtype=dtype, seed=M + F)
    x = rnd(M, K, dtype=dtype, seed=3)
    got = W().q4_gated(x, on_gpu(*raw, gated=True), act=act).double().cpu()
    y, bound = q4_bound(x.cpu(), *raw)
    gate, up = y[:, :F], y[:, F:]
    a = orc.activate(gate, act)
    want = a * up
    # both slopes are below 1.13; the activation itself takes 8 roundings of fp32
    fp32 = (1.13 * bound[:, :F] + 8 * EPS * gate.abs()) * (up.abs() + bound[:, F:]) \
        + a.abs() * bound[:, F:]
    tiny = 2.0 ** -25 if dtype == F16 else 0.0
    err = (got - want).abs()
    assert bool((err <= fp32 + (want.abs() + fp32) * half_step(dtype) + tiny).all())
    assert float(err.norm()) <= float(want.norm()) * (2.0 ** -17 + half_step(dtype))


def test_q4_gated_far_gates():
    """Gates of any size: activations that vanish or pass everything."""
    q = torch.full((32, 64), 0x99, dtype=torch.uint8)  # weights of 1 everywhere
    raw = (q, torch.ones(32, 1, dtype=F16), None)
    x = torch.zeros(5, 128, dtype=F16, device="cuda")
    x[:, 0] = torch.tensor([0.0, 50.0, -50.0, 2000.0, -2000.0])
    for act in ("silu", "gelu"):
        got = W().q4_gated(x, on_gpu(*raw, gated=True), act=act)[:, 0].tolist()
        assert got == [0.0, 2500.0, 0.0, INF, 0.0]


# ---------------------------------------------------------------------------
# the next token
# ---------------------------------------------------------------------------
def check_sample(logits, u, **settings):
    got = W().sample(logits, u, **settings).tolist()
    for r, g in enumerate(got):
        row = {k: (v[r].item() if isinstance(v, torch.Tensor) else
                   v if k == "top_k" else torch.tensor(v, dtype=F32).item())
               for k, v in settings.items()}
        assert g == orc.sample(logits[r], u[r].item(), **row), (r, row)
    return got


def uniform(T, seed=0):
    return torch.rand(T, generator=torch.Generator().manual_seed(seed)).cuda()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("V", [1, 2, 63, 1000, 8191, 32001, 151937])
def test_sample(dtype, V):
    T = 9
    x = rnd(T, V, dtype=dtype, seed=V, scale=3.0)
    u = uniform(T, V)
    for settings in ({}, {"temperature": 0.7, "top_k": 50}, {"top_p": 0.9}, {"min_p": 0.05},
                     {"temperature": 1.3, "top_k": 500, "top_p": 0.8, "min_p": 0.01},
                     {"temperature": 0.0}, {"top_k": 1, "top_p": 0.3}, {"top_p": 0.0}):
        check_sample(x, u, **settings)


def test_sample_settings_of_rows():
    T, V = 64, 5000
    x = rnd(T, V, seed=1, scale=4.0)
    pick = lambda values, seed, dtype=F32: torch.tensor(values)[torch.randint(  # noqa: E731
        len(values), (T,), generator=torch.Generator().manual_seed(seed))].to(dtype).cuda()
    check_sample(x, uniform(T, 2), temperature=pick([0.0, 0.5, 1.0, 2.0, 1e-3, 100.0], 1),
                 top_k=pick([0, 1, 7, 100, 4999, 5000, 9999, -3], 2, torch.int32),
                 top_p=pick([1.0, 0.1, 0.5, 0.99, 2.0, 0.0, -1.0], 3),
                 min_p=pick([0.0, 0.01, 0.5, 1.0, 3.0], 4))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("V", [4003, 70001])
def test_sample_ties(dtype, V):
    """Equal logits: the lowest ids stay, in counts that top_k and top_p cut."""
    x = torch.full((8, V), 1.5, dtype=dtype, device="cuda")  # ties beyond any list
    x[1, ::2] = -0.0
    x[1, 1::2] = 0.0
    x[2, 100:] = 0.5
    x[3] = torch.arange(V).remainder(5).to(dtype)
    x[4, 17] = 1.515625  # one step of bf16 above
    x[5, -1] = 3.0
    x[6, :] = 2.0 ** -100
    x[6, 9] = -(2.0 ** -100)
    x[7, :] = -30000.0
    for i, u in enumerate((0.0, 0.3, 0.999999)):
        u = torch.full((8,), u, device="cuda")
        for settings in ({}, {"top_k": 10}, {"top_k": 2500}, {"top_p": 0.5}, {"top_p": 0.25},
                         {"top_k": 1001, "top_p": 0.75}, {"min_p": 1.0}, {"temperature": 0.0}):
            check_sample(x, u, **settings)


@pytest.mark.parametrize("V", [3000, 90000])
def test_sample_masked_and_bad_rows(V):
    x = rnd(12, V, seed=3, scale=2.0)
    x[0] = -INF
    x[1, 5] = NAN
    x[2, V - 1] = INF
    x[3] = -INF
    x[3, 1234] = -7.0
    x[4, :V - 10] = -INF
    x[5, 1:] = torch.finfo(F32).min
    x[6] = torch.finfo(F32).min
    x[7] = torch.linspace(-3e38, 3e38, V)
    x[8] *= 1e-30
    x[9, 2000] = -NAN
    u = uniform(12, 4)
    for settings in ({}, {"top_k": 20}, {"top_p": 0.9}, {"min_p": 0.1}, {"temperature": 0.0},
                     {"temperature": 1e-30, "top_k": 3}, {"temperature": 1e30, "top_p": 0.5}):
        got = check_sample(x, u, **settings)
        assert got[0] == got[1] == got[2] == got[9] == -1 and got[3] == 1234 and got[4] >= V - 10
    bad = {"temperature": [NAN, -1.0, INF, 1.0], "top_p": [1.0, 1.0, 1.0, NAN]}
    settings = {k: torch.tensor(v, device="cuda") for k, v in bad.items()}
    assert W().sample(x[8:9].expand(4, V), u[:4], **settings).tolist() == [-1] * 4
    edge = torch.tensor([NAN, -0.5, 1.0, 7.0], device="cuda")
    got = W().sample(torch.zeros(4, V, device="cuda"), edge)
    assert got.tolist() == [-1, 0, V - 1, V - 1]


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("T,V", [(150, 20001), (2, 66001)])
def test_sample_narrow_and_wide_rows(dtype, T, V):
    """Logits that all lie in a few bins of the histogram, or far apart, in rows of
    one program and of several: each way in which the end is found."""
    x = rnd(T, V, dtype=dtype, seed=9)
    for scale, temperature in ((0.01, 1.0), (1.0, 40.0), (1.0, 1.0), (4.0, 0.2), (200.0, 1.0)):
        y = x * scale
        for settings in ({"top_k": 3000}, {"top_k": 6000}, {"top_k": 19999}, {"top_p": 0.3},
                         {"top_p": 0.999}, {"top_k": 6000, "top_p": 0.5}, {"min_p": 0.3},
                         {"top_k": 2000, "top_p": 0.9, "min_p": 0.2},
                         {"top_p": 0.9, "min_p": 0.001}, {"min_p": 1e-13}):
            got = W().sample(y, uniform(T, 3), temperature=temperature, **settings).tolist()
            for r in range(0, T, 75):
                row = {k: v if k == "top_k" else torch.tensor(v, dtype=F32).item()
                       for k, v in {"temperature": temperature, **settings}.items()}
                assert got[r] == orc.sample(y[r], uniform(T, 3)[r].item(), **row), (r, scale, row)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_sample_many_rows(dtype):
    x = rnd(3000, 70, dtype=dtype, seed=12, scale=3.0)
    check_sample(x, uniform(3000, 13), top_k=20, top_p=0.8)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_sample_longest_vocabularies(dtype):
    """Segments of several chunks, weights of fewer bits."""
    V = 1300003
    x = rnd(2, V, dtype=dtype, seed=11, scale=2.0)
    x[1] = 0.25
    for settings in ({}, {"top_p": 0.9}, {"top_k": 1000, "top_p": 0.5}, {"min_p": 0.01}):
        check_sample(x, uniform(2, 5), **settings)


def test_sample_strides():
    base = rnd(5, 2000, dtype=F16, seed=5, scale=3.0)
    x = base[1::2, 3:1500]
    check_sample(x, uniform(2, 6), top_k=30, top_p=0.9)
    one = base[2, 9:1009].expand(20, 1000)
    check_sample(one, uniform(20, 7), top_p=0.95)
    assert W().sample(base[:0], base[:0, 0].float()).shape == (0,)


def test_sample_follows_the_weights():
    """Ids as often as their weights say: u at all steps of a row's border count."""
    x = torch.log(torch.tensor([0.1, 0.4, 0.0, 0.3, 0.2], device="cuda"))
    n = 10000
    u = (torch.arange(n, device="cuda") + 0.5) / n
    ids = W().sample(x.expand(n, 5), u)
    assert torch.bincount(ids, minlength=5).tolist() == [1000, 4000, 0, 3000, 2000]
    ids = W().sample(x.expand(n, 5), u, top_p=0.65)  # 0.4 and 0.3 stay
    count = torch.bincount(ids, minlength=5).tolist()
    assert count[0] == count[2] == count[4] == 0 and abs(count[1] - n * 4 / 7) <= 1


# ---------------------------------------------------------------------------
# together
# ---------------------------------------------------------------------------
def layer(seed, D=64, H=4, KV=2, hidden=256, F=192, V=1000):
    """A decoder of one layer, its weights as they are and laid out."""
    sizes = {"qkv": ((H + 2 * KV) * D, hidden), "out": (hidden, H * D), "up": (2 * F, hidden),
             "down": (hidden, F), "vocab": (V, hidden)}
    raw = {n: weights(*size, 64, seed=seed + i) for i, (n, size) in enumerate(sizes.items())}
    return raw, {n: on_gpu(*r, gated=n == "up") for n, r in raw.items()}


def step(w, laid_out, s, D=64, H=4, KV=2):
    """One step of S tokens a sequence; what it computed on the way, and the ids."""
    B, S = s["x"].shape[:2]
    x, _, hidden = w.rmsnorm(s["x"].flatten(0, 1), s["norm"], residual=s["residual"].flatten(0, 1))
    qkv = w.q4_matmul(x, laid_out["qkv"]).view(B, S, -1, D).transpose(1, 2)
    q, k, v = qkv.split((H, KV, KV), 1)
    start = s["lens"] - S
    q, k = w.rotate(q, k, s["rotary"], start)
    w.kv_append(s["cache"], k, v, s["table"], start)
    o = w.cached_attention(q, s["cache"], s["table"], s["lens"])
    o = o.transpose(1, 2).reshape(B * S, H * D)
    y, _, hidden = w.rmsnorm(w.q4_matmul(o, laid_out["out"]), s["norm"], residual=hidden)
    up = w.q4_gated(y, laid_out["up"])
    z, _, _ = w.rmsnorm(w.q4_matmul(up, laid_out["down"]), s["norm"], residual=hidden)
    logits = w.q4_matmul(z.view(B, S, -1)[:, -1], laid_out["vocab"], out_dtype=F32)
    ids = w.sample(logits, s["u"], s["temperature"], top_k=40, top_p=0.95)
    return [x, qkv, q, k, o, y, up, z, logits, ids]


def step_state(w, seed, S):
    lens = [S, S + 70]
    cache = w.kv_cache(8, 2, 64)
    table = ints([[3, 1, 0, 5], [7, 2, 6, 4]])
    if lens[1] > S:  # earlier tokens of the second sequence
        k, v = (rnd(1, 2, 70, 64, dtype=BF16, seed=seed + i) for i in range(2))
        w.kv_append(cache, k, v, table[1:], ints([0]))
    return {"x": rnd(2, S, 256, dtype=BF16, seed=seed + 2), "lens": ints(lens), "table": table,
            "residual": rnd(2, S, 256, dtype=BF16, seed=seed + 3), "cache": cache,
            "norm": rnd(256, dtype=BF16, seed=seed + 4), "rotary": w.rotary(64),
            "u": uniform(2, seed), "temperature": torch.tensor([0.8, 0.0], device="cuda")}


@pytest.mark.parametrize("S", [1, 40])
def test_a_decoder_step(S):
    """Each operator of the step on what the one before it gave."""
    w = W()
    raw, laid_out = layer(20)
    s = step_state(w, 30, S)
    x, qkv, q, k, o, y, up, z, logits, ids = step(w, laid_out, s)
    check_q4(x, raw["qkv"], laid_out=laid_out["qkv"])
    at = (s["lens"] - S)[:, None] + torch.arange(S, device="cuda")
    check_rotated(q, qkv[:, :4], orc.frequencies(64), at)
    check_rotated(k, qkv[:, 4:6], orc.frequencies(64), at)
    for b, n in enumerate(s["lens"].tolist()):
        keys, values, has = sorc.cached(s["cache"], s["table"], b, n)
        want, _ = sorc.attention(q[b], keys, values, list(range(n - S, n)), has=has)
        got = o.view(2, S, 4, 64)[b].transpose(0, 1).double()
        assert float((got - want.to(got)).norm()) < 1e-2 * float(want.norm())
    check_q4(o, raw["out"], laid_out=laid_out["out"])
    check_q4(up, raw["down"], laid_out=laid_out["down"])
    last = z.view(2, S, -1)[:, -1]
    assert torch.equal(logits, check_q4(last, raw["vocab"], out_dtype=F32, laid_out=laid_out["vocab"]))
    assert ids.tolist() == check_sample(logits, s["u"], temperature=s["temperature"], top_k=40,
                                        top_p=0.95)


def test_graphs_and_streams():
    """Two captured steps, replayed in turn with new inputs and eager calls
    between, and steps on two streams at once give the eager results."""
    w = W()
    _, laid_out = layer(40)
    states = [step_state(w, 50, 1), step_state(w, 60, 7)]
    for s in states:
        step(w, laid_out, s)
    torch.cuda.synchronize()
    graphs = []
    for s in states:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step(w, laid_out, s)
        graphs.append((g, out))
    for turn in range(3):
        for i, s in enumerate(states):
            s["x"].copy_(rnd(*s["x"].shape, dtype=BF16, seed=100 * turn + i))
            s["u"].copy_(uniform(2, turn))
        for g, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        for s, (_, out) in zip(states, graphs):
            kept = [t.clone() for t in out]
            assert all(torch.equal(a, b) for a, b in zip(kept, step(w, laid_out, s)))
            torch.cuda.synchronize()
    eager = [step(w, laid_out, s) for s in states]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in states]
    got = [None, None]
    for _ in range(3):
        for i, (s, stream) in enumerate(zip(states, streams)):
            with torch.cuda.stream(stream):
                got[i] = step(w, laid_out, s)
    torch.cuda.synchronize()
    for a, b in zip(got, eager):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_ordinary_calls_go_through_cpp(monkeypatch):
    from newt_amd import serving
    w = W()
    raw, laid_out = layer(70)
    s = step_state(w, 80, 3)
    want = step(w, laid_out, s)
    monkeypatch.setattr(serving, "_call", None)  # the Python path would fail
    assert all(torch.equal(a, b) for a, b in zip(step(w, laid_out, s), want))
    monkeypatch.undo()
    monkeypatch.setattr(serving, "_fast", lambda *a: None)
    assert all(torch.equal(a, b) for a, b in zip(step(w, laid_out, s), want))


def test_offsets_past_32_bits():
    """Rows that lie more than 2^31 numbers behind the first."""
    w = W()
    wide = torch.empty(2, (1 << 31) + 64, dtype=BF16, device="cuda")
    x = wide[:, :4096]
    x.copy_(rnd(2, 4096, dtype=BF16, seed=1))
    raw = weights(32, 4096, 128, seed=2)
    check_q4(x, raw)
    check_sample(x, uniform(2), top_p=0.9)
    q = x.view(2, 1, 32, 128)
    far = wide[:, 8192:8192 + 4096].view(2, 1, 32, 128)
    rot = w.rotary(128)
    w.rotate(q, None, rot, ints([0, 9]), q_out=far)
    at = ints([0, 9])[:, None] + torch.arange(32, device="cuda")
    check_rotated(far, q, orc.frequencies(128), at)


# ---------------------------------------------------------------------------
# what lies at the borders of the products with 4-bit weights
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("M", [1, 20, 48, 49, 130])
@pytest.mark.parametrize("N,K,group", [(40, 96, 32), (40, 32, 32), (2100, 160, 32), (40, 192, 64),
                                       (8200, 320, 64)])
def test_q4_what_lies_behind_weighs_nothing(dtype, M, N, K, group):
    """Weights, zeros and scales behind the last column and row are any finite numbers."""
    raw = weights(N, K, group, seed=M + K)
    w = on_gpu(*raw)
    g = torch.Generator().manual_seed(K)
    words = w.q.clone()
    scales, zeros = w.scales.clone(), w.zeros.clone()
    for i in range(K % 128 // 32, 4):  # 32 columns each: a word of all lanes
        words[:, -1, :, i] = torch.randint(-2 ** 31, 2 ** 31, words.shape[:1] + (64,), generator=g).cuda()
    first = K // group
    scales[:, first:] = torch.randn(scales[:, first:].shape, generator=g).to(scales) * 100
    zeros[:, first:] = torch.randint(0, 256, zeros[:, first:].shape, generator=g).to(zeros)
    rows = N % 16  # of the last tile
    scales[-1, :, rows:], zeros[-1, :, rows:] = -1000.0, 200
    words[-1].view(-1, 4, 16, 4)[:, :, rows:] = 0x7abcdef0
    x = rnd(M, K, dtype=dtype, seed=M + 1)
    check_q4(x, raw, laid_out=w._replace(q=words, scales=scales, zeros=zeros))


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("M", [3, 33, 48, 49, 130])
def test_q4_matmul_zeros_of_any_byte(M, group):
    q, s, z = weights(100, 384, group, seed=M)
    z = torch.randint(0, 256, z.shape, generator=torch.Generator().manual_seed(M)).to(torch.uint8)
    z[:40] |= 0xf1  # odd ones from 241 on
    x = rnd(M, 384, dtype=BF16, seed=M)
    check_q4(x, (q, s, z), out_dtype=F32)
    check_q4(x.half(), (q, s, z))


def check_q4_bound(x, raw, laid_out=None, out_dtype=F32):
    """Each number within the roundings of its sums, whatever the sums' cancellation."""
    got = W().q4_matmul(x, on_gpu(*raw) if laid_out is None else laid_out, out_dtype=out_dtype)
    want, bound = q4_bound(x.cpu(), *raw)
    step = half_step(out_dtype)
    assert bool(((got.double().cpu() - want).abs() <= bound * (1 + step) + want.abs() * step).all())


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("M", [3, 33, 60, 200])
def test_q4_matmul_of_the_largest_numbers(M, group):
    """Rows of one sign near the largest bf16, with finite results: their sums are far
    beyond fp32, and so are those of x times a number."""
    q, s, z = weights(70, 512, group, seed=M)
    s = s * 2.0 ** -13
    z[::3] = 255
    g = torch.Generator().manual_seed(M)
    x = ((torch.rand(M, 512, generator=g) + 1.0) * 2.0 ** 126 * 1.98).to(BF16)
    x[::2] *= -1
    x[1::4] *= torch.randint(0, 2, x[1::4].shape, generator=g) * 2 - 1
    x = x.cuda()
    assert bool(x.isfinite().all())
    check_q4_bound(x, (q, s, z))
    check_q4_bound(x, (q, s, None))


@pytest.mark.parametrize("M", [3, 60])
def test_q4_matmul_of_the_smallest_numbers(M):
    """Sums are held 2^16 times smaller than the results: 160 roundings of at most
    2^-149 each, times the scale."""
    q, s, z = weights(70, 256, 64, seed=M)
    g = torch.Generator().manual_seed(M)
    x = (torch.randn(M, 256, generator=g) * 2.0 ** torch.randint(-126, -90, (M, 256), generator=g))
    x = x.to(BF16).cuda()
    s = (s * 64).contiguous()
    got = W().q4_matmul(x, on_gpu(q, s, z), out_dtype=F32)
    want, bound = q4_bound(x.cpu(), q, s, z)
    bound = bound + (160 * 4 * 2.0 ** -133 * s.double().abs().amax(1) + 2.0 ** -149)[None]
    assert bool(((got.double().cpu() - want).abs() <= bound * (1 + EPS)).all())


@pytest.mark.parametrize("M", [1, 20, 60])
def test_q4_gated_gelu_of_negative_gates(M):
    """v (1 + erf(v / sqrt 2)) / 2 cancels below 0 unless it is v erfc(-v / sqrt 2) / 2. The
    argument is off by 1.3 roundings of fp32, of which erfc's relative slope there, 2 v^2 / 2
    + 1, makes 190 at v = -12; erfc itself by 32 at most, three products by 3."""
    q = torch.full((32, 64), 0x99, dtype=torch.uint8)  # weights of 1 everywhere
    laid_out = on_gpu(q, torch.ones(32, 1, dtype=BF16), None, gated=True)
    for v in torch.linspace(-12.0, -0.25, 48).to(BF16).tolist():
        x = torch.zeros(M, 128, dtype=BF16, device="cuda")
        x[:, 0] = v
        got = W().q4_gated(x, laid_out, act="gelu").double().cpu()
        want = 0.5 * v * math.erfc(-v / math.sqrt(2.0)) * v
        assert bool(((got - want).abs() <= abs(want) * (2.0 ** -16 + half_step(BF16))).all()), v


def test_weights_are_what_q4_weights_gives():
    """A plain tuple of the same seven is not taken, in C++ or Python."""
    raw = weights(40, 256, 128)
    w, x = on_gpu(*raw), rnd(3, 256, dtype=BF16)
    for bad in (tuple(w), list(w)):
        with pytest.raises(TypeError, match="Q4Weights"):
            W().q4_matmul(x, bad)


@pytest.mark.parametrize("M", [5, 48, 100])
def test_q4_outputs_beside_their_inputs(M):
    """Columns of the same rows, rows between x's rows; over x or bias they are refused."""
    raw = weights(64, 256, 64, seed=13)
    laid_out, x = on_gpu(*raw), rnd(M, 256, dtype=BF16, seed=14)
    base = torch.zeros(2 * M + 1, 400, dtype=BF16, device="cuda")
    base[:M, 64:320], base[M:2 * M, 300:364] = x, 7.0
    a = base[:M, 64:320]
    for out in (base[:M, :64], base[:M, 320:384]):
        check_q4(a, raw, laid_out=laid_out, out=out)
    base[1:2 * M:2, :256] = x
    b = base[1:2 * M:2, :256]
    check_q4(b, raw, laid_out=laid_out, out=base[:2 * M:2, 100:164])
    check_q4(b, raw, laid_out=laid_out, out=base[2:2 * M + 1:2, :64])
    kept = base.clone()
    for out in (base[1:2 * M:2, :64], base[1:2 * M:2, 250:314], base[:M, 100:164]):
        with pytest.raises(ValueError, match="overlaps"):
            W().q4_matmul(b, laid_out, out=out)
    with pytest.raises(ValueError, match="overlaps"):
        W().q4_matmul(x, laid_out, bias=base[M + 1, 300:364], out=base[:M + 2, 300:364][2:])
    gated = on_gpu(*raw, gated=True)
    with pytest.raises(ValueError, match="overlaps"):
        W().q4_gated(b, gated, out=base[1:2 * M:2, 224:256])
    assert torch.equal(base, kept)


# ---------------------------------------------------------------------------
# the instances and loops that large sizes take
# ---------------------------------------------------------------------------
def tiles_of(outputs, gated=False):
    return -(-outputs // 16) * (2 if gated else 1)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("M,N", [(1, 2100), (16, 2100), (4, 33000), (5, 16500), (20, 8200), (40, 8200)])
def test_q4_matmul_of_many_outputs(dtype, group, M, N):
    """More than 128 tiles of weights (two a wave), 1024 and 2048 (four a wave, few
    waves), and for 17 rows and more 512 (four a wave); of nine blocks of columns the
    first waves have two."""
    assert tiles_of(N) in (132, 513, 1032, 2063)
    raw = weights(N, 1152, group, zeros=M % 2 > 0, dtype=dtype, seed=M)
    check_q4(rnd(M, 1152, dtype=dtype, seed=M + 1), raw)


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("M,F,act", [(1, 1100, "silu"), (1, 16400, "gelu"), (9, 8200, "silu"),
                                     (20, 4100, "gelu"), (48, 4100, "silu")])
def test_q4_gated_of_many_outputs(group, M, F, act):
    raw = weights(2 * F, 1152, group, dtype=BF16, seed=M + F)
    x = rnd(M, 1152, dtype=BF16, seed=3, scale=0.25)
    check_gated(x, raw, act)


def check_gated(x, raw, act):
    got = W().q4_gated(x, on_gpu(*raw, gated=True), act=act).double().cpu()
    y, bound = q4_bound(x.cpu(), *raw)
    F = y.shape[1] // 2
    gate, up = y[:, :F], y[:, F:]
    a = orc.activate(gate, act)
    want = a * up
    # slopes below 1.13, 8 roundings of fp32 in the activation, as in test_q4_gated
    fp32 = (1.13 * bound[:, :F] + 8 * EPS * gate.abs()) * (up.abs() + bound[:, F:]) \
        + a.abs() * bound[:, F:]
    tiny = 2.0 ** -25 if x.dtype == F16 else 0.0
    assert bool(((got - want).abs() <= fp32 + (want.abs() + fp32) * half_step(x.dtype) + tiny).all())


def parts(M, N, K, group, act=0):
    """How many parts q4_many splits the columns into, from what it asks for."""
    from newt_amd import serving
    need = serving.lib().newt_q4_matmul_workspace(serving._Q4.pack(
        *[4096] * 4, 0, 4096, 0, M, K, N, K, N, group, 2, 2, 2, act, 0))
    return need // (4 * M * tiles_of(N, act > 0) * 16) or 1


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("group,K", [(32, 2080), (64, 2112), (128, 2176)])
def test_q4_matmul_many_rows_long_programs(dtype, group, K):
    """17 blocks of columns in a program, the last one ragged: each stage of LDS and
    each set of sums is used again and again."""
    M, N = 500, 8190
    assert parts(M, N, K, group) == 1 and -(-K // 128) == 17
    raw = weights(N, K, group, zeros=dtype == F16, dtype=dtype, seed=K)
    check_q4(rnd(M, K, dtype=dtype, seed=1), raw)


@pytest.mark.parametrize("group,N,K", [(32, 4003, 9312), (64, 2003, 8000), (128, 2003, 16384)])
def test_q4_matmul_many_rows_long_parts(group, N, K):
    """Parts of seven blocks and more, the last one shorter."""
    M = 130
    n = parts(M, N, K, group)
    assert n > 1 and -(-K // 128) // n >= 7, n
    raw = weights(N, K, group, seed=K)
    check_q4(rnd(M, K, dtype=BF16, seed=1), raw)
    odd = rnd(M, K + 3, dtype=BF16, seed=2)[:, 3:]  # not aligned to 16 bytes
    check_q4(odd, raw)


@pytest.mark.parametrize("group,K", [(32, 1056), (64, 1728), (128, 1664)])
def test_q4_gated_many_rows_long_programs(group, K):
    M, F = 500, 4090
    assert parts(M, F, K, group, 1) == 1
    check_gated(rnd(M, K, dtype=BF16, seed=1, scale=0.25), weights(2 * F, K, group, seed=K), "silu")


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("D,dim,S", [(128, 128, 2100), (128, 64, 2100), (80, 40, 3500)])
def test_rotate_two_heads_a_thread(dtype, interleaved, D, dim, S):
    """As many tokens as give a thread two heads, an odd number of heads in all."""
    w = W()
    H, KV = 32, 1
    wide = 16 // dtype.itemsize
    V = wide if dim % (2 * wide) == 0 else 4
    units = dim // 2 // V + -(-(D - dim) // V)
    assert units * S * (H + KV) >= 2 * 256 * 1024
    rot = w.rotary(dim, interleaved=interleaved)
    q, k = rnd(1, H, S, D, dtype=dtype, seed=1), rnd(1, KV, S, D, dtype=dtype, seed=2)
    at = ints([5])[:, None] + torch.arange(S, device="cuda")
    for o, x in zip(w.rotate(q, k, rot, ints([5])), (q, k)):
        check_rotated(o, x, orc.frequencies(dim), at, interleaved=interleaved)
    # the same in place, and heads of more than one tensor in a thread
    want = w.rotate(q, k, rot, ints([5]))
    w.rotate(q, k, rot, ints([5]), q_out=q, k_out=k)
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])


# ---------------------------------------------------------------------------
# rows of logits with little to choose
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("T,V", [(3, 3000), (3, 90000), (150, 20001)])
def test_sample_of_few_tokens_with_weight(dtype, T, V):
    """Fewer tokens than top_k that are not masked, or that have any weight at a low
    temperature."""
    x = rnd(T, V, dtype=dtype, seed=V, scale=2.5)
    u = uniform(T, 3)
    few = torch.full_like(x, -INF)
    for r in range(T):
        n = 5 + 7 * r % 26
        at = torch.randperm(V, generator=torch.Generator().manual_seed(r))[:n].cuda()
        few[r, at] = x[r, at]
    rows = slice(None, None, 1 + T // 40)
    for settings in ({"top_k": 50, "top_p": 0.9}, {"top_k": 50}, {"top_k": 5, "top_p": 0.99},
                     {"top_k": 30, "top_p": 0.5, "min_p": 0.02}, {"top_p": 0.9}):
        check_rows(few, u, rows, settings)
    low = torch.finfo(dtype).min
    check_rows(few.clamp(min=low), u, rows, {"top_k": 50, "top_p": 0.9})
    for temperature in (0.02, 0.05, 0.1, 0.2):
        check_rows(x, u, rows, {"temperature": temperature, "top_k": 50, "top_p": 0.9})
        check_rows(x, u, rows, {"temperature": temperature, "top_k": 2000, "top_p": 0.999,
                                "min_p": 0.001})


def check_rows(logits, u, rows, settings):
    got = W().sample(logits, u, **settings)[rows].tolist()
    row = {k: v if k == "top_k" else torch.tensor(v, dtype=F32).item() for k, v in settings.items()}
    for g, x, v in zip(got, logits[rows], u[rows].tolist()):
        assert g == orc.sample(x, v, **row), settings


def test_sample_top_k_beyond_the_list():
    """A bin that fits a list, behind more tokens than fit one."""
    x = rnd(4, 40000, seed=21)
    for V in (40000, 20000):
        for top_k in (4095, 4097, 9000, 15000):
            for settings in ({}, {"top_p": 0.9}, {"top_p": 0.3, "min_p": 0.1}):
                check_rows(x[:, :V], uniform(4, 1), slice(None), {"top_k": top_k, **settings})


def test_sample_more_rows_than_a_launch_takes():
    """2^22 programs of 1024 threads are 2^32 work-items."""
    T = (1 << 22) + 70
    x = rnd(97, 5, seed=22, scale=2.0).repeat(T // 97 + 1, 1)[:T]
    u = uniform(97, 23).repeat(T // 97 + 1)[:T]
    t = torch.tensor([0.0, 0.7, 1.5], device="cuda").repeat(T // 3 + 1)[:T]
    k = torch.tensor([0, 2, 3, 5], dtype=torch.int32, device="cuda").repeat(T // 4 + 1)[:T]
    for settings in ({"top_p": 0.8}, {"temperature": t, "top_k": k}):
        ids = W().sample(x, u, **settings)
        n = 97 * 12  # rows until everything comes again
        few = {name: v[:n] if isinstance(v, torch.Tensor) else v for name, v in settings.items()}
        again = W().sample(x[:n], u[:n], **few)
        assert torch.equal(ids, again.repeat(T // n + 1)[:T])
    check_rows(x, u, slice(T - 40, T), {"top_p": 0.8})
