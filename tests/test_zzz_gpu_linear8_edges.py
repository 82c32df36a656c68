"""8-bit linear layer on the GPU: the widest rows, and other calls at the edges of what the entry points take."""
import numpy as np
import pytest

from intel_gaudi3_software_amd import abi
from linear8_helpers import U, check_codes, code_tensor, gate64, real_tensor

pytestmark = pytest.mark.gpu


def _codes_of(t):
    import torch
    return t.cpu().view(torch.uint8).numpy()


@pytest.mark.parametrize("width", [(1 << 31) - 1, (1 << 31) - 8192 + 9])
def test_widest_rows(calc, width):
    """One row of nearly 2^31 elements: the place behind the last step of a lane is not a 32-bit signed number.  Everything but the two ends
    is zero, so the codes are the ends' own and no others."""
    import torch
    rng = np.random.default_rng(width % 1000)
    ends = torch.from_numpy(rng.standard_normal((2, 20000)).astype(np.float32)).cuda().bfloat16()
    x = torch.zeros(width, dtype=torch.bfloat16, device="cuda")
    x[:20000], x[-20000:] = ends[0], ends[1]
    codes, scales = torch.full((width,), 85, dtype=torch.uint8, device="cuda"), torch.zeros(2, device="cuda")
    X, O = real_tensor(x, [width, 1]), code_tensor(codes, [width, 1], "int8")
    short = code_tensor(torch.zeros(40000, dtype=torch.uint8, device="cuda"), [40000, 1], "int8")
    calc.quantizeRows(O, scales[:1], X)
    calc.quantizeRows(short, scales[1:], real_tensor(ends.reshape(-1).contiguous(), [40000, 1]))
    calc.synchronize()
    want = short.data().view(2, 20000)
    assert scales[0] == scales[1] and torch.equal(codes[:20000], want[0]) and torch.equal(codes[-20000:], want[1])
    assert int(torch.count_nonzero(codes)) == int(torch.count_nonzero(want))
    # the norm, in place of x: the codes are the same (no gamma), the sum is x twice
    calc.rmsNormQuantize(O, scales[:1], X, None, X, X, 0.0)
    calc.synchronize()
    assert torch.equal(codes[:20000], want[0]) and torch.equal(codes[-20000:], want[1])
    assert int(torch.count_nonzero(codes)) == int(torch.count_nonzero(want))
    assert torch.equal(x[:20000], 2 * ends[0]) and torch.equal(x[-20000:], 2 * ends[1]) and int(torch.count_nonzero(x)) == int(torch.count_nonzero(ends))
    v = 2 * ends.cpu().double().numpy()
    rms = np.sqrt(np.sum(v * v) / width)
    # (at most 40 of a lane's squares are not zero: the roundings of the sum are those of a short row)
    top = np.max(np.abs(v)) / rms / 127
    assert abs(float(scales[0]) - top) <= 40 * U * top


@pytest.mark.parametrize("gate,low,high,op", [("silu", -91.0, -87.01, abi.GATE_SILU), ("gelu", -10.15, -10.0, abi.GATE_GELU_TANH)])
@pytest.mark.parametrize("width", [40, 700, 9000, 20001])
def test_rows_in_the_gates_tail(calc, gate, low, high, op, width):
    """Rows whose gates all lie where 1 + e^-g leaves the range of fp32 and g / (1 + e^-g) does not yet, beside ordinary and very large
    values; one row has them among ordinary gates, with factors that make up for them."""
    import torch
    rng = np.random.default_rng(width)
    g = rng.uniform(low, high, (4, width)).astype(np.float32)
    x = (rng.standard_normal((4, width)) * np.array([1.0, 1e10, 1e37, 1.0])[:, None]).astype(np.float32)
    plain = rng.random(width) < 0.5
    g[3, plain] = rng.standard_normal(int(plain.sum()))
    x[3, ~plain] *= np.float32(3e36)
    codes, scales = torch.zeros(4, width, dtype=torch.uint8, device="cuda"), torch.zeros(4, device="cuda")
    calc.quantizeRows(code_tensor(codes, [width, 4], "e5m2"), scales, real_tensor(torch.from_numpy(x).cuda(), [width, 4]), real_tensor(torch.from_numpy(g).cuda(), [width, 4]), op)
    calc.synchronize()
    # fp32 roundings: those of the gate elsewhere (12; the gelu's argument has five, which its size, at most 91 here, magnifies), and the
    # factor's argument, its exponential and its product (4)
    roundings = 16 if gate == "silu" else 16 + 5 * 91
    v = gate64(g.astype(np.float64), gate) * x.astype(np.float64)
    check_codes(v, _codes_of(codes), scales.cpu().double().numpy(), "e5m2", roundings, roundings + 2)


def test_gates_where_fp32_ends(calc):
    """Gated values below 2^-126 have a denormal's bits, those below 2^-150 are zero, whatever multiplies them."""
    import torch
    g = np.array([-95.0, -100.0, -103.0, -110.0, -200.0, -1e30], np.float32)
    scales, codes = torch.zeros(6, device="cuda"), torch.zeros(6, 8, dtype=torch.uint8, device="cuda")
    gt, x = torch.from_numpy(np.repeat(g[:, None], 8, 1)).cuda(), torch.full((6, 8), 1e30, device="cuda")
    calc.quantizeRows(code_tensor(codes, [8, 6], "int8"), scales, real_tensor(x, [8, 6]), real_tensor(gt, [8, 6]), abi.GATE_SILU)
    calc.synchronize()
    with np.errstate(over="ignore"):
        want = np.abs(gate64(g.astype(np.float64), "silu"))
    got = scales.cpu().double().numpy() * 127 / np.float64(np.float32(1e30))
    assert np.all(np.abs(got - want) <= 16 * U * want + 2.0 ** -149), (got, want)
    assert np.all(got[3:] == 0) and np.all(got[:3] > 0)
    assert np.all(_codes_of(codes).view(np.int8)[:3] == -127) and not codes[3:].any()


@pytest.mark.parametrize("width", [40, 700, 5000, 9000, 20001])
@pytest.mark.parametrize("factor,gamma", [(1e37, 1e37), (1e37, 1e20), (1e-36, 1e-36), (1e-20, 1e-36), (1e-37, 1e37), (1e37, 1e-37)])
def test_norm_of_values_and_gammas_of_any_size(calc, width, factor, gamma):
    """Products of a value and its gamma may lie anywhere, as long as the normalised value is one of fp32's."""
    import torch
    rng = np.random.default_rng(width)
    x = (rng.standard_normal((3, width)) * factor).astype(np.float32)
    g = (rng.uniform(0.5, 2.0, width) * gamma).astype(np.float32)
    g[::7] *= np.float32(1e-3)
    codes, scales = torch.zeros(3, width, dtype=torch.uint8, device="cuda"), torch.zeros(3, device="cuda")
    X, G = real_tensor(torch.from_numpy(x).cuda(), [width, 3]), real_tensor(torch.from_numpy(g).cuda(), [width])
    for kind in ("int8", "e4m3"):
        calc.rmsNormQuantize(code_tensor(codes, [width, 3], kind), scales, X, G, eps=0.0)
        calc.synchronize()
        s = x.astype(np.float64)
        v = s * g.astype(np.float64)[None] / np.sqrt(np.mean(s * s, axis=1, keepdims=True))
        # (roundings: the product, its power of two exactly, the quotient in two parts, the last one; the sum's as in the other tests, halved by the root)
        check_codes(v, _codes_of(codes), scales.cpu().double().numpy(), kind, 4, 8 + ((16 if width <= 16384 else 24) + 16) / 2)


def test_rows_repeated_by_a_stride_of_zero(calc):
    """A tensor of one row in memory and many by its strides, as an operand of each call."""
    import torch
    x = torch.randn(64, device="cuda")
    codes, one = torch.zeros(9, 64, dtype=torch.uint8, device="cuda"), torch.zeros(1, 64, dtype=torch.uint8, device="cuda")
    scales, single = torch.zeros(9, device="cuda"), torch.zeros(1, device="cuda")
    many = real_tensor(x, [64, 9], strides=[1, 0])
    calc.quantizeRows(code_tensor(one, [64, 1], "int8"), single, real_tensor(x, [64, 1]))
    calc.quantizeRows(code_tensor(codes, [64, 9], "int8"), scales, many)
    calc.synchronize()
    assert torch.equal(codes, one.expand(9, 64)) and torch.equal(scales, single.expand(9))
    calc.rmsNormQuantize(code_tensor(codes, [64, 9], "int8"), scales, many)
    calc.synchronize()
    assert torch.equal(codes, one.expand(9, 64)) and torch.all(scales == scales[0])
    out = torch.zeros(9, 9, dtype=torch.int32, device="cuda")
    calc.scaledGemm(real_tensor(out, [9, 9]), code_tensor(one, [64, 9], "int8", strides=[1, 0]), None, code_tensor(codes, [64, 9], "int8"), None)
    calc.synchronize()
    v = one.view(torch.int8).long()
    assert torch.all(out == (v * v).sum())


def test_rows_behind_a_dimension_of_one_index(calc):
    """Rows whose dimensions do not make one pitch, with a dimension of one index between them whose stride looks as if they did."""
    import torch
    rng = np.random.default_rng(4)
    W, R, Q = 64, 3, 4
    buf = torch.from_numpy(rng.standard_normal(700 * Q).astype(np.float32)).cuda()
    X = real_tensor(buf, [700 * Q, 1]).window(0, [W, R, 1, Q], [1, 100, 700, 700, 2800])
    codes, scales = torch.full((900 * Q,), 85, dtype=torch.uint8, device="cuda"), torch.zeros(R * Q, device="cuda")
    O = code_tensor(codes, [900 * Q, 1], "int8").window(0, [W, R, 1, Q], [1, 80, 900, 900, 3600])
    calc.quantizeRows(O, scales, X)
    calc.synchronize()
    at = np.arange(Q)[:, None, None] * 700 + np.arange(R)[None, :, None] * 100 + np.arange(W)
    to = np.arange(Q)[:, None, None] * 900 + np.arange(R)[None, :, None] * 80 + np.arange(W)
    got = _codes_of(codes)
    check_codes(buf.cpu().double().numpy()[at].reshape(R * Q, W), got[to].reshape(R * Q, W), scales.cpu().double().numpy(), "int8", 2, 8)
    rest = np.ones(got.size, bool)
    rest[to.ravel()] = False
    assert np.all(got[rest] == 85)


@pytest.mark.parametrize("op", [abi.OP_FWD, abi.OP_DEDX, abi.OP_DEDW])
def test_convolution_weights_behind_a_dimension_of_one_index(calc, op):
    """The same for a 1 x 3 filter whose taps lie further apart than its channels: the results of the dense filter."""
    import torch
    from intel_gaudi3_software_amd import ConvolutionParams, MmeSimTensor
    C, K, W, H, B = 16, 24, 9, 8, 2
    g = torch.Generator(device="cuda")
    g.manual_seed(5)
    xs, ws, ys, pitch = [C, W, H, 1, B], [K, C, 1, 3, 1], [K, W, H - 2, 1, B], K * C + 40
    t = lambda sizes: torch.randn(int(np.prod(sizes)), generator=g, device="cuda").bfloat16()
    x, y, w = t(xs), t(ys), t(ws)
    apart = torch.zeros(3 * pitch, dtype=torch.bfloat16, device="cuda")
    apart.view(3, pitch)[:, :K * C] = w.view(3, K * C)
    strides = [1, K, pitch, pitch, 3 * pitch]
    cp = ConvolutionParams(2, [0, 0, 0, 0], [1, 1, 1, 1], [1, 1, 1, 1])
    T = lambda v, sizes, dt=abi.BF16, st=None: MmeSimTensor(sizes, 5, dt, v, strides=st)
    outs = []
    for dense in (True, False):
        if op == abi.OP_DEDW:
            n = 3 * (K * C if dense else pitch)
            out = torch.full((n,), 7.0, device="cuda")
            o = T(out, ws, abi.FP32, None if dense else strides)
            calc.doConvolution(o, T(x, xs), o, T(y, ys), cp, op)
            calc.synchronize()
            assert torch.all(out.view(3, -1)[:, K * C:] == 7.0)
            outs.append(out.view(3, -1)[:, :K * C].contiguous())
        else:
            sizes = ys if op == abi.OP_FWD else xs
            out = torch.zeros(int(np.prod(sizes)), device="cuda")
            o, f = T(out, sizes, abi.FP32), T(w, ws) if dense else T(apart, ws, abi.BF16, strides)
            calc.doConvolution(o, T(x, xs), f, o, cp, op) if op == abi.OP_FWD else calc.doConvolution(o, o, f, T(y, ys), cp, op)
            calc.synchronize()
            outs.append(out)
    assert torch.equal(outs[0], outs[1]) and torch.any(outs[0] != 0)


FIRST_CALLS = """
import torch
from intel_gaudi3_software_amd import HipCalculator, MmeSimTensor, abi
g = torch.Generator(device="cuda"); g.manual_seed(1)
T = lambda x, t, *fp8: MmeSimTensor(list(x.shape)[::-1], x.dim(), t, x, *fp8)
codes = lambda *s: torch.randint(0, 0x70, s, generator=g, device="cuda", dtype=torch.int32).to(torch.uint8)
real = lambda *s: torch.randn(*s, generator=g, device="cuda").bfloat16()
calls, outs = [], []
side = torch.cuda.Stream()
c = HipCalculator()
c.setStream(side.cuda_stream)
for t in ((abi.INT8,), (abi.FP8_143, 7, abi.MINIMAL_INF_NAN), (abi.FP8_152, 15)):
    for M, N, K in ((4, 512, 512), (4, 512, 520), (20, 16384, 512), (70, 4000, 512), (70, 4000, 333), (2001, 2001, 392), (2001, 2001, 385), (4000, 4001, 512)):
        o = torch.zeros(M, N, dtype=torch.bfloat16, device="cuda")
        outs.append(o)
        calls.append(lambda a=(T(o, abi.BF16), T(codes(M, K), *t), None, T(codes(N, K), *t), None): c.scaledGemm(*a))
for rows, width in ((40, 100), (300, 4096), (300, 14336), (20, 20000)):
    q, s = torch.zeros(rows, width, dtype=torch.uint8, device="cuda"), torch.zeros(rows, device="cuda")
    outs += [q, s]
    calls.append(lambda a=(T(q, abi.INT8), s, T(real(rows, width), abi.BF16), T(real(rows, width), abi.BF16)): c.quantizeRows(*a))
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph, stream=side):
    for f in calls:
        f()
torch.cuda.synchronize()
assert not any(bool(o.any()) for o in outs)
got = []
for k in range(3):
    for o in outs:
        o.zero_()
    torch.cuda.synchronize()
    graph.replay()
    torch.cuda.synchronize()
    got.append([o.clone() for o in outs])
for o in outs:
    o.zero_()
torch.cuda.synchronize()
for f in calls:
    f()
c.synchronize()
for k in range(3):
    assert all(bool(a.any()) and torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(got[k], outs)), k
print("the same")
"""


def test_first_calls_of_a_process_are_recorded():
    """Every form recorded into a graph by a process that has made no call before: nothing is asked of the runtime that a recording refuses."""
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-u", "-c", FIRST_CALLS], cwd=root, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, timeout=100)
    assert r.returncode == 0 and b"the same" in r.stdout, r.stdout.decode(errors="replace")[-2000:]
