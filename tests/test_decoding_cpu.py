"""rotate, q4_matmul, q4_gated and sample without a GPU: what the Python entry
points and the C entries refuse, the C structs against the packed fields, the
weights' layout, frequencies, and the definitions that the GPU tests compare with."""

import decimal
import math
import os
import subprocess

import pytest
import torch

from newt_amd import serving, workloads
from oracle import decoding as orc

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
INT = torch.int32


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


def refused(kind, match, f, *args, **kw):
    with pytest.raises(kind, match=match):
        f(*args, **kw)


def launched(f, *args, **kw):
    refused(Launched, None, f, *args, **kw)


def test_tensors_have_to_be_on_the_gpu(monkeypatch):
    """Through the C++ calls too, which leave such tensors to Python."""
    monkeypatch.setattr(serving._Dev, "device", classmethod(lambda cls: 0))
    monkeypatch.setattr(serving._Dev, "stream", staticmethod(lambda device: 0))
    assert serving._Fast.load()
    rot = workloads.rotary(64, device="cpu")
    q, at = torch.zeros(1, 2, 3, 64), torch.zeros(1, dtype=INT)
    refused(TypeError, "current GPU", workloads.rotate, q, None, rot, at)
    refused(TypeError, "must be a tensor", workloads.rotate, None, None, rot, at)
    w = workloads.q4_weights(torch.zeros(4, 64, dtype=torch.uint8), torch.zeros(4, 1, dtype=F16))
    refused(TypeError, "current GPU", workloads.q4_matmul, torch.zeros(1, 128, dtype=F16), w)
    refused(TypeError, "must be a tensor", workloads.q4_matmul, [1.0], w)
    refused(TypeError, "current GPU", workloads.sample, torch.zeros(2, 9), torch.zeros(2))
    refused(TypeError, "must be a tensor", workloads.sample, torch.zeros(2, 9), 0.5)


# ---------------------------------------------------------------------------
# refusals
# ---------------------------------------------------------------------------
def test_rotary_refusals():
    f = workloads.rotary
    refused(ValueError, "odd", f, 7, device="cpu")
    refused(ValueError, "out of range", f, 0, device="cpu")
    refused(TypeError, "int", f, 64.0, device="cpu")
    for bad in (0.0, -1.0, math.inf, math.nan):
        refused(ValueError, "base", f, 64, base=bad, device="cpu")
        refused(ValueError, "factor", f, 64, factor=bad, device="cpu")
    for bad in (math.inf, math.nan, 1e300):
        refused(ValueError, "amplitude", f, 64, amplitude=bad, device="cpu")
    for bad in ((0, 1.0, 4.0), (4096, 4.0, 1.0), (4096, -1.0, 4.0), (4096, 1.0, math.inf)):
        refused(ValueError, "ramp", f, 64, ramp=bad, device="cpu")
    refused(TypeError, "bool", f, 64, interleaved=1, device="cpu")
    refused(ValueError, "32 finite frequencies", f, 64, frequencies=[1.0], device="cpu")
    refused(ValueError, "finite frequencies", f, 2, frequencies=[math.nan], device="cpu")


def test_rotate_refusals(calls):
    f = workloads.rotate
    rot = workloads.rotary(64, device="cpu")
    q, k = torch.zeros(2, 4, 5, 64, dtype=BF16), torch.zeros(2, 1, 5, 64, dtype=BF16)
    at, each = torch.zeros(2, dtype=INT), torch.zeros(2, 5, dtype=INT)
    launched(f, q, k, rot, at)
    launched(f, q, None, rot, each, transposed=True)
    launched(f, q, k, rot, at, q_out=q, k_out=k)
    refused(TypeError, "must be a Rotary", f, q, k, rot.turns, at)
    refused(TypeError, "must be a Rotary", f, q, k, (rot.turns.int(), 1.0, False), at)
    refused(ValueError, "q has shape", f, q[0], k, rot, at)
    refused(ValueError, "k has shape", f, q, k[0], rot, at)
    refused(ValueError, "k has shape", f, q, k[:, :, :4], rot, at)
    refused(TypeError, "k is", f, q, k.half(), rot, at)
    refused(TypeError, "q is", f, q.double(), None, rot, at)
    refused(ValueError, "rotary of 64 dimensions", f, q[..., :32], None, rot, at)
    refused(TypeError, "positions are", f, q, k, rot, at.long())
    refused(ValueError, "positions have shape", f, q, k, rot, each[:, :4])
    refused(ValueError, "positions have shape", f, q, k, rot, at[:1])
    refused(ValueError, "unit stride", f, q.transpose(2, 3).contiguous().transpose(2, 3), k, rot, at)
    refused(ValueError, "q_out has shape", f, q, k, rot, at, q_out=q[:, :3])
    refused(TypeError, "k_out is", f, q, k, rot, at, k_out=k.float())
    refused(ValueError, "output of k", f, q, None, rot, at, k_out=k)


def test_q4_refusals(calls):
    lay_out = workloads.q4_weights
    q, s = torch.zeros(6, 128, dtype=torch.uint8), torch.zeros(6, 4, dtype=BF16)
    z = torch.zeros(6, 4, dtype=torch.uint8)
    refused(TypeError, "must be a tensor", lay_out, [1], s)
    refused(TypeError, "not uint8", lay_out, q.int(), s)
    refused(TypeError, "scales are", lay_out, q, s.float())
    refused(ValueError, "scales of shape", lay_out, q, s[:5])
    refused(ValueError, "scales of shape", lay_out, q, torch.zeros(6, 16, dtype=BF16))
    refused(ValueError, "scales of shape", lay_out, q, torch.zeros(6, 0, dtype=BF16))
    refused(ValueError, "zeros has shape", lay_out, q, s, z[:, :3])
    refused(TypeError, "zeros is", lay_out, q, s, z.int())
    refused(ValueError, "two dimensions", lay_out, q[0], s)
    refused(ValueError, "not a gate's", lay_out, q[:5], s[:5], gated=True)
    refused(ValueError, "no rows", lay_out, q[:0], s[:0])
    refused(TypeError, "bool", lay_out, q, s, z, 1)
    w, g = lay_out(q, s, z), lay_out(q, s, z, gated=True)
    x = torch.zeros(3, 256, dtype=F16)
    f = workloads.q4_matmul
    launched(f, x, w)
    launched(f, x, w, bias=torch.zeros(6, dtype=F16), out_dtype=F32, out=torch.zeros(3, 6))
    refused(TypeError, "Q4Weights", f, x, (q, s, z))
    refused(ValueError, "laid out gated", f, x, g)
    refused(ValueError, "x has shape", f, x[0], w)
    refused(TypeError, "x is", f, x.float(), w)
    refused(ValueError, "columns", f, x[:, :128], w)
    refused(ValueError, "unit stride", f, torch.zeros(256, 3, dtype=F16).t(), w)
    refused(TypeError, "bias is", f, x, w, bias=torch.zeros(6))
    refused(ValueError, "bias has shape", f, x, w, bias=torch.zeros(5, dtype=F16))
    refused(ValueError, "bias needs", f, x, w, bias=torch.zeros(12, dtype=F16)[::2])
    refused(TypeError, "output", f, x, w, out_dtype=BF16)
    refused(TypeError, "out is", f, x, w, out=torch.zeros(3, 6))
    refused(ValueError, "out has shape", f, x, w, out=torch.zeros(3, 5, dtype=F16))
    refused(ValueError, "rows of out overlap", f, x, w, out=torch.zeros(6, dtype=F16).expand(3, 6))
    refused(ValueError, "rows of out need", f, x, w, out=torch.zeros(6, 3, dtype=F16).t())
    refused(ValueError, "contiguous", f, x, w._replace(q=w.q.transpose(2, 3).contiguous().transpose(2, 3)))
    refused(ValueError, "scales has shape", f, x, w._replace(scales=w.scales[:, :1]))
    refused(ValueError, "no groups", f, x, w._replace(group=16))
    f = workloads.q4_gated
    launched(f, x, g)
    launched(f, x, g, act="gelu", out=torch.zeros(3, 3, dtype=F16))
    refused(ValueError, "not laid out gated", f, x, w)
    refused(ValueError, "act=", f, x, g, act="relu")
    refused(TypeError, "out is", f, x, g, out=torch.zeros(3, 3))


def test_sample_refusals(calls):
    f = workloads.sample
    x, u = torch.zeros(3, 50, dtype=BF16), torch.zeros(3)
    launched(f, x, u)
    launched(f, x, u, 0, 5, 1, 0)
    launched(f, x, u, torch.zeros(3), torch.zeros(3, dtype=INT), torch.zeros(3), torch.zeros(3))
    refused(ValueError, "logits have shape", f, x[0], u)
    refused(ValueError, "logits have shape", f, x[:, :0], u)
    refused(TypeError, "logits are", f, x.double(), u)
    refused(ValueError, "u has shape", f, x, u[:2])
    refused(TypeError, "u is", f, x, u.double())
    refused(ValueError, "unit stride", f, x, torch.zeros(6)[::2])
    refused(ValueError, "rows of logits", f, torch.zeros(50, 3).t(), u)
    for name in ("temperature", "top_p", "min_p"):
        refused(ValueError, "out of range", f, x, u, **{name: -0.5})
        refused(ValueError, "out of range", f, x, u, **{name: math.nan})
        refused(TypeError, "number", f, x, u, **{name: None})
        refused(TypeError, "number", f, x, u, **{name: True})
        refused(ValueError, "has shape", f, x, u, **{name: torch.zeros(2)})
        refused(TypeError, f"{name} is", f, x, u, **{name: torch.zeros(3, dtype=INT)})
    refused(ValueError, "out of range", f, x, u, temperature=math.inf)
    refused(ValueError, "out of range", f, x, u, temperature=10 ** 400)
    refused(ValueError, "out of range", f, x, u, min_p=1.5)
    refused(ValueError, "top_k", f, x, u, top_k=-1)
    refused(TypeError, "top_k", f, x, u, top_k=2.0)
    refused(TypeError, "top_k is", f, x, u, top_k=torch.zeros(3, dtype=torch.int64))


# ---------------------------------------------------------------------------
# the C ABI
# ---------------------------------------------------------------------------
def test_structs_are_what_is_packed(tmp_path):
    src = tmp_path / "sizes.c"
    names = {"newt_rotate_params": serving._ROTATE, "newt_q4_params": serving._Q4,
             "newt_sample_params": serving._SAMPLE}
    lines = "".join(f'printf("%zu %zu\\n", sizeof({n}), offsetof({n}, reserved));' for n in names)
    src.write_text(f'#include <stdio.h>\n#include "newt_ops.h"\nint main(void) {{ {lines} }}\n')
    subprocess.run(["gcc", "-std=c11", "-Wall", "-Werror", "-I" + os.path.join(ROOT, "include"),
                    str(src), "-o", str(tmp_path / "sizes")], check=True)
    out = subprocess.run([str(tmp_path / "sizes")], capture_output=True, text=True, check=True)
    for line, s in zip(out.stdout.splitlines(), names.values()):
        size, last = map(int, line.split())
        assert size == s.size and last == size - 4


def test_c_entries_refuse():
    L = serving.lib()
    P = 4096  # an address that nothing reads

    def call(entry, params, message):
        assert entry(params, None) == 10002
        assert message in L.newt_ops_last_error(), L.newt_ops_last_error()

    for name in ("rotate", "q4_matmul", "sample"):
        call(getattr(L, "newt_" + name), None, b"null params")
    rotate = [P] * 6 + [2, 4, 1, 5, 64, 64] + [1280, 320, 64] * 4 + [1, 0, 1.0, 2, 0, 0, 0, 0]
    for i, value, message in ((0, 0, b"null tensor"), (3, 0, b"null tensor"), (4, 0, b"null tensor"),
                              (5, 0, b"null tensor"), (6, -1, b"negative"), (10, 0, b"head_dim"),
                              (11, 63, b"rot_dim"), (11, 66, b"rot_dim"), (6, 1 << 30, b"too many"),
                              (15, 100, b"overlap"), (21, 64, b"overlap"), (26, math.inf, b"finite"),
                              (27, 3, b"dtype")):
        bad = list(rotate)
        bad[i] = value
        call(L.newt_rotate, serving._ROTATE.pack(*bad), message)
    q4 = [P, P, P, P, 0, P, 0, 3, 256, 40, 256, 40, 64, 2, 1, 2, 0, 0]
    for i, value, message in ((0, 0, b"null tensor"), (5, 0, b"null tensor"), (1, P + 8, b"aligned"),
                              (2, P + 2, b"aligned"), (3, P + 4, b"aligned"), (7, -1, b"size"),
                              (8, 1 << 30, b"2^30"), (8, 200, b"whole groups"), (11, 39, b"overlap"),
                              (12, 16, b"groups are"), (13, 0, b"x is"), (14, 0, b"scales are"),
                              (15, 1, b"out is"), (16, 3, b"activation")):
        bad = list(q4)
        bad[i] = value
        call(L.newt_q4_matmul, serving._Q4.pack(*bad), message)
    gated = list(q4)
    gated[4], gated[16] = P, 1
    call(L.newt_q4_matmul, serving._Q4.pack(*gated), b"no bias")
    many = list(q4)
    many[7], many[8], many[10] = 100, 1 << 20, 1 << 20
    assert L.newt_q4_matmul_workspace(serving._Q4.pack(*many)) > 0
    call(L.newt_q4_matmul, serving._Q4.pack(*many), b"workspace")
    many[8] = 1 << 26
    call(L.newt_q4_matmul, serving._Q4.pack(*many), b"columns")
    sample = [P, P, P, 0, 0, 0, 0, 0, 2, 100, 100, 1.0, 1.0, 0.0, 0, 2, 0]
    for i, value, message in ((0, 0, b"null tensor"), (1, 0, b"null tensor"), (2, 0, b"null tensor"),
                              (8, -1, b"rows"), (9, 0, b"logits"), (9, 1 << 30, b"logits"),
                              (11, -1.0, b"temperature"), (11, math.nan, b"temperature"),
                              (12, -1.0, b"top_p"), (13, 2.0, b"min_p"), (15, 3, b"dtype"),
                              (9, 1 << 20, b"workspace")):
        bad = list(sample)
        bad[i] = value
        call(L.newt_sample, serving._SAMPLE.pack(*bad), message)


def test_q4_refuses_an_out_over_its_inputs():
    L = serving.lib()
    P = 1 << 40

    def refused(rows, out, bias=0, out_dtype=2, workspace=1 << 20):
        assert L.newt_q4_matmul(serving._Q4.pack(
            P, 1 << 20, 1 << 20, 0, bias, out, workspace, rows, 256, 40, 256, 40, 64, 2, 1, out_dtype,
            0, 0), None) == 10002
        assert b"out overlaps x or bias" in L.newt_ops_last_error()

    for rows in (1, 3, 48, 49, 500):
        for out in (P, P + 2, P - 78, P + 512 * rows - 2):
            refused(rows, out)
        refused(rows, P - 158, out_dtype=0)
        for bias in (1 << 30, (1 << 30) + 80 * rows - 2, (1 << 30) - 78):
            refused(rows, 1 << 30, bias)


def test_rows_that_meet(tmp_path):
    """The check of outputs over inputs against every pair of rows."""
    src = tmp_path / "meet.cpp"
    src.write_text('''
#include <cstdio>
#include <cstdlib>
#include "byte_rows.h"
using namespace newt_ops;
int main() {
  srand(1);
  int seen[2] = {0, 0};
  for (int n = 0; n < 400000; ++n) {
    int64_t v[8];
    for (int i = 0; i < 2; ++i) {
      v[4 * i] = 1000 + rand() % 200;
      v[4 * i + 1] = rand() % 6;
      v[4 * i + 2] = rand() % 81 - 20;
      v[4 * i + 3] = 1 + rand() % 30;
    }
    if (n % 2) v[6] = v[2];
    bool meet = false;
    for (int64_t i = 0; i < v[1]; ++i)
      for (int64_t j = 0; j < v[5]; ++j) {
        const int64_t a = v[0] + i * v[2], b = v[4] + j * v[6];
        meet |= a < b + v[7] && b < a + v[3];
      }
    const ByteRows a((void*)v[0], v[1], v[2], v[3]), b((void*)v[4], v[5], v[6], v[7]);
    if (rows_meet(a, b) != meet || rows_meet(b, a) != meet) {
      for (int64_t x : v) printf("%ld ", (long)x);
      return 1;
    }
    ++seen[meet];
  }
  return seen[0] < 100000 || seen[1] < 100000;
}
''')
    subprocess.run(["g++", "-std=c++17", "-I" + os.path.join(ROOT, "newt_amd/csrc/ops"), str(src), "-o",
                    str(tmp_path / "meet")], check=True)
    out = subprocess.run([str(tmp_path / "meet")], capture_output=True, text=True)
    assert out.returncode == 0, out.stdout


def test_q4_workspace_has_to_be_aligned():
    """Splits' sums are written 16 bytes at a time."""
    L = serving.lib()
    P = 4096
    many = [P, P, P, P, 0, P, 0, 100, 1 << 20, 40, 1 << 20, 40, 64, 2, 1, 2, 0, 0]
    assert L.newt_q4_matmul_workspace(serving._Q4.pack(*many)) > 0
    for workspace in (0, P + 4, P + 8):
        many[6] = workspace
        assert L.newt_q4_matmul(serving._Q4.pack(*many), None) == 10002
        assert b"workspace" in L.newt_ops_last_error()


def test_empty_calls_launch_nothing():
    L = serving.lib()
    P = 4096
    for batch, heads, tokens in ((0, 4, 5), (2, 0, 5), (2, 4, 0)):
        assert L.newt_rotate(serving._ROTATE.pack(*[P] * 6, batch, heads, 0, tokens, 64, 64,
                                                  *[1280, 320, 64] * 4, 1, 0, 1.0, 2, 0, 0, 0, 0),
                             None) == 0
    for rows, outputs in ((0, 40), (3, 0)):
        assert L.newt_q4_matmul(serving._Q4.pack(P, P, P, P, 0, P, 0, rows, 256, outputs, 256, 40, 64,
                                                 2, 1, 2, 0, 0), None) == 0
    assert L.newt_sample(serving._SAMPLE.pack(P, P, P, 0, 0, 0, 0, 0, 0, 100, 100, 1.0, 1.0, 0.0, 0,
                                              2, 0), None) == 0
    assert L.newt_sample_workspace(0, 100000, 2) == 0


def test_launches_of_too_many_programs_are_refused():
    """2^32 work-items and more, of which the runtime would leave some out: rows that
    no memory holds, but for a stride of 0. Nothing is launched."""
    L = serving.lib()
    P = 4096
    rows = (1 << 31) - 1
    sizes = serving._RMSNORM.pack(P, 0, P, P, 0, 0, rows, 64, 0, 0, 64, 0, 1e-6, 2, 2, 2, 0, 0)
    q4 = serving._Q4.pack(P, P, P, 0, 0, 1 << 40, 0, 40, 64, (1 << 30) - 1, 0, 1 << 30, 64, 2, 2, 2, 0,
                          0)
    for entry, params in ((L.newt_rmsnorm, sizes), (L.newt_q4_matmul, q4)):
        assert entry(params, None) == 10002
        assert b"more than a launch takes" in L.newt_ops_last_error(), L.newt_ops_last_error()


# ---------------------------------------------------------------------------
# layouts and definitions
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("N,K,group,gated", [(40, 96, 32, False), (34, 256, 64, True),
                                             (16, 128, 128, False), (2, 320, 64, True)])
def test_weights_lie_where_the_header_says(N, K, group, gated):
    g = torch.Generator().manual_seed(N)
    q = torch.randint(0, 256, (N, K // 2), generator=g, dtype=torch.uint8)
    s = torch.rand(N, K // group, generator=g).half()
    z = torch.randint(0, 16, s.shape, generator=g, dtype=torch.uint8)
    w = workloads.q4_weights(q, s, z, gated=gated)
    halves = 2 if gated else 1
    assert w.outputs == N // halves and w.q.shape[0] == halves * -(-w.outputs // 16)
    numbers = torch.stack((q & 15, q >> 4), -1).flatten(1).tolist()
    words = (w.q.long() & 0xffffffff).tolist()
    for n in range(N):
        half, row = divmod(n, w.outputs)
        tile, row = row // 16 * halves + half, row % 16
        for k in range(K):
            word = words[tile][k // 128][16 * (k % 32 // 8) + row][k % 128 // 32]
            word = (word >> 3 | word << 29) & 0xffffffff
            i = k % 8
            assert word >> (14 + 2 * i if i % 2 else 2 * i) & 15 == numbers[n][k]
        for i in range(K // group):
            assert w.scales[tile, i, row] == s[n, i] and w.zeros[tile, i, row] == z[n, i]
    assert bool((w.scales[:, K // group:] == 0).all())  # what lies behind weighs nothing


def test_rotary_turns():
    """Fractions of a turn to 2^-64, stretched where they turn slowly."""
    rot = workloads.rotary(64, base=500000.0, device="cpu")
    with decimal.localcontext(decimal.Context(prec=60)):
        for i, t in enumerate(rot.turns.tolist()):
            f = decimal.Decimal(500000) ** (decimal.Decimal(-2 * i) / 64)
            f /= 2 * decimal.Decimal("3.14159265358979323846264338327950288419716939937510")
            assert abs(f * 2 ** 64 - t % 2 ** 64) <= 1
    for factor, ramp in ((4.0, None), (32.0, (4096, 1.0, 4.0))):
        got = workloads.rotary(128, factor=factor, ramp=ramp, device="cpu").turns
        want = orc.frequencies(128, factor=factor, ramp=ramp) / (2 * math.pi)
        assert torch.allclose(got.double() / 2.0 ** 64, want, rtol=1e-12, atol=2.0 ** -60)
    # whole turns do not count; negative ones turn back
    turns = workloads.rotary(4, frequencies=[2 * math.pi * 5.25, -math.pi], device="cpu").turns
    assert abs(int(turns[0]) / 2 ** 64 - 0.25) < 1e-14
    assert abs(abs(int(turns[1])) / 2 ** 64 - 0.5) < 1e-14


def test_rotary_of_high_frequencies():
    """Whole turns in any number that 50 digits of pi leave a fraction of; more are refused."""
    with decimal.localcontext(decimal.Context(prec=80)):
        pi2 = 2 * decimal.Decimal("3.1415926535897932384626433832795028841971693993751058209749445923")
        for f in (1e6, 1e15, -1e20, 1e29, 6e30):
            t = int(workloads.rotary(2, frequencies=[f], device="cpu").turns[0])
            off = int((decimal.Decimal(f) / pi2 * 2 ** 64).to_integral_value()) - t
            assert min(off % 2 ** 64, -off % 2 ** 64) <= 1, f
    for kw in ({"frequencies": [1.0, -1e31]}, {"frequencies": [1e300, 0.0]}, {"factor": 1e-31},
               {"base": 1e-64}, {"frequencies": [1e20, 1.0], "factor": 1e-12},
               {"factor": 1e-31, "ramp": (4096, 1000.0, 2000.0)}):
        refused(ValueError, "1e30 turns", workloads.rotary, 4, device="cpu", **kw)


def test_rotate_definition():
    """Turning by p and q is turning by p + q, and back again by -(p + q)."""
    x = torch.randn(1, 2, 3, 8, generator=torch.Generator().manual_seed(0))
    f = orc.frequencies(6)
    at = torch.tensor([[1, 20, 300]])
    for kw in ({}, {"interleaved": True}):
        once = orc.rotate(x, f, at * 3, **kw)
        assert torch.allclose(orc.rotate(orc.rotate(x, f, at, **kw), f, 2 * at, **kw), once)
        assert torch.allclose(orc.rotate(once, f, at * 3, transposed=True, **kw), x.double())
        assert torch.equal(once[..., 6:], x.double()[..., 6:])


def test_sample_definition():
    """Against a loop over the sorted tokens."""
    g = torch.Generator().manual_seed(1)
    for _ in range(200):
        V = int(torch.randint(1, 12, (1,), generator=g))
        x = torch.randint(-3, 3, (V,), generator=g).double()
        t, u, p, m = (torch.rand(4, generator=g) + torch.tensor([0.1, 0.0, 0.05, 0.0])).tolist()
        k = int(torch.randint(0, 8, (1,), generator=g))
        w = [math.exp((v - float(x.max())) / t) for v in x.tolist()]
        ranked = sorted(range(V), key=lambda i: (-float(x[i]), i))[:k or V]
        mass, before, kept = sum(w[i] for i in ranked), 0.0, []
        for i in ranked:
            if not kept or ((p >= 1 or before < p * mass) and w[i] >= m):
                kept.append(i)
            before += w[i]
        total, run = sum(w[i] for i in kept), 0.0
        for i in sorted(kept):
            run += w[i]
            if run > u * total:
                break
        # borders that rounding decides are left out
        assert orc.sample(x, u, t, k, p, m) == i or abs(run - w[i] - u * total) < 1e-9
