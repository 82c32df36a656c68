"""8-bit linear layer on the GPU: every form of the kernels with every kind of operand and output it is made for, each call's form asserted."""
import numpy as np
import pytest

from intel_gaudi3_software_amd import abi
from linear8_helpers import HALF_STEP, U, check_codes, code_tensor, gate64, real_tensor, torch_real

pytestmark = pytest.mark.gpu

FP8_PAIRS = [("e4m3", "e4m3"), ("e4m3", "e5m2"), ("e5m2", "e4m3"), ("e5m2", "e5m2")]


def _random_codes(g, kind, *shape):
    """Any code of int8; any finite one of the 8-bit floats."""
    import torch
    if kind == "int8":
        return torch.randint(-128, 128, shape, generator=g, device="cuda", dtype=torch.int32).to(torch.int8).view(torch.uint8)
    c = torch.randint(0, 0x78 if kind == "e4m3" else 0x6C, shape, generator=g, device="cuda", dtype=torch.int32)
    return (c + 128 * torch.randint(0, 2, shape, generator=g, device="cuda", dtype=torch.int32)).to(torch.uint8)


def _values(codes, kind):
    import torch
    return codes.view({"int8": torch.int8, "e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}[kind]).double()


def _check(out, vx, vw, sx, sw, bias, int8, out_name):
    """One batch element, on the GPU in 64 bits, held to the bounds of linear8_helpers.sums_error and check_product."""
    import torch
    sums, scale = vx @ vw.T, sx.double()[:, None] * sw.double()[None, :]
    exact = sums * scale
    part = exact.abs()
    if bias is not None:
        exact = exact + bias.double()[None, :]
    error = 0.0
    if not int8:
        pad = -vx.shape[1] % 8
        tops = [torch.nn.functional.pad(v.abs(), (0, pad)).reshape(v.shape[0], -1, 8).amax(2) for v in (vx, vw)]
        error = (7 * 2.0 ** -13 * (tops[0] @ tops[1].T) + vx.shape[1] * 2.0 ** -23 * (vx.abs() @ vw.abs().T)) * scale * (1 + 4 * U)
    before = 2.01 * U * part + 1.01 * U * exact.abs() + error
    rel, least = HALF_STEP[out_name]
    bound = before + 2 * rel * (exact.abs() + before) + least
    assert torch.all(exact.abs() + bound < torch.finfo(torch_real(out_name)).max)  # (nothing here leaves the output's range)
    off = (out.double() - exact).abs() - bound
    assert float(off.max()) <= 0, (int(off.argmax()), float(off.max()))


def _product(calc, M, N, K, a, b, out_name, bias, batch, x_batch, w_batch, rows, waves, aligned=True, seed=0):
    import torch
    g = torch.Generator(device="cuda")
    g.manual_seed(M + 7 * N + 3 * K + seed)
    x, w = _random_codes(g, a, x_batch, M, K), _random_codes(g, b, w_batch, N, K)
    # scales that take the codes, whose root mean squares these are, and the sums to about one
    size = {"int8": 74.0, "e4m3": 130.0, "e5m2": 1000.0}
    sx, sw = (torch.exp(0.5 * torch.randn(*s, generator=g, device="cuda")) for s in ((x_batch, M), (w_batch, N)))
    sx *= 1.0 / size[a]
    sw *= 1.0 / (size[b] * K ** 0.5)
    bi = torch.randn(w_batch, N, generator=g, device="cuda") if bias else None
    first = 0 if aligned else 1
    pitch = -(-K // 16) * 16 + 16 if aligned else K + 2
    held = []
    for v, n in ((x, x_batch * M), (w, w_batch * N)):  # rows on a pitch, with other codes behind their ends
        t = torch.full((first + n * pitch,), 0x55, dtype=torch.uint8, device="cuda")
        t[first:].view(n, pitch)[:, :K] = v.reshape(n, K)
        held.append(t)
    X = code_tensor(held[0], [held[0].numel(), 1], a).window(first, [K, M, x_batch], [1, pitch, M * pitch, x_batch * M * pitch, x_batch * M * pitch])
    W = code_tensor(held[1], [held[1].numel(), 1], b).window(first, [K, N, w_batch], [1, pitch, N * pitch, w_batch * N * pitch, w_batch * N * pitch])
    guard = 512
    to = torch.full((batch * M * N + guard,), 77, dtype=torch_real(out_name), device="cuda")
    calc.scaledGemm(real_tensor(to, [N, M, batch]), X, sx, W, sw, bi)
    form = calc.lastContractionForm()
    calc.synchronize()
    assert (form["tile_rows"], form["wavefronts"]) == (rows, waves), form
    assert torch.all(to[batch * M * N:] == 77)
    out = to[:batch * M * N].view(batch, M, N)
    for c in range(batch):
        cx, cw = (c if x_batch > 1 else 0), (c if w_batch > 1 else 0)
        _check(out[c], _values(x[cx], a), _values(w[cw], b), sx[cx], sw[cw], bi[cw] if bias else None, a == "int8", out_name)
    return out


# M, N, K of the 128 x 128 and the 256 x 256 form: ragged on both sides, reductions that end inside a stage
TILES = [(2001, 2001, 392, 128, True), (2003, 2002, 645, 128, False), (4000, 4001, 592, 256, True), (2050, 8001, 336, 256, True)]


@pytest.mark.parametrize("M,N,K,rows,aligned", TILES)
@pytest.mark.parametrize("out,bias", [("bf16", True), ("fp16", True), ("fp32", True), ("bf16", False), ("fp32", False)])
def test_large_tiles_int8(calc, M, N, K, rows, aligned, out, bias):
    _product(calc, M, N, K, "int8", "int8", out, bias, 1, 1, 1, rows, 8, aligned)


@pytest.mark.parametrize("M,N,K,rows,aligned", TILES)
@pytest.mark.parametrize("a,b", FP8_PAIRS)
def test_large_tiles_fp8(calc, M, N, K, rows, aligned, a, b):
    _product(calc, M, N, K, a, b, "bf16", False, 1, 1, 1, rows, 8, aligned)
    _product(calc, M, N, K, a, b, "fp16", True, 1, 1, 1, rows, 8, aligned, seed=1)


@pytest.mark.parametrize("xb,wb", [(2, 2), (1, 2), (2, 1), (1, 1)])
@pytest.mark.parametrize("M,N,K,rows", [(1400, 1405, 1040, 128), (1100, 2500, 336, 256)])
@pytest.mark.parametrize("a,b,out", [("int8", "int8", "bf16"), ("int8", "int8", "fp32"), ("e4m3", "e5m2", "fp16")])
def test_large_tiles_batches(calc, M, N, K, rows, xb, wb, a, b, out):
    _product(calc, M, N, K, a, b, out, True, 2, xb, wb, rows, 8)


# (for up to 16 rows of x four wavefronts mean 64 rows of w per workgroup; for 32, where 32 rows of w have four too, N is so large that the
# planner's estimate for 64, in whole rounds over 256 compute units, is the least: 1 or 2 rounds against 2 or 3)
@pytest.mark.parametrize("M,N,K,rows", [(1, 16387, 1040, 8), (8, 16384, 1555, 8), (9, 14336, 4096, 16), (16, 14339, 2064, 16), (17, 16384, 4096, 32), (32, 16400, 529, 32)])
@pytest.mark.parametrize("a,b,out", [("int8", "int8", "bf16"), ("int8", "int8", "fp32"), ("e4m3", "e4m3", "bf16"), ("e4m3", "e5m2", "fp16"), ("e5m2", "e4m3", "bf16"), ("e5m2", "e5m2", "bf16")])
def test_few_rows_with_64_rows_of_w(calc, M, N, K, rows, a, b, out):
    _product(calc, M, N, K, a, b, out, out != "bf16", 1, 1, 1, rows, 4)


def test_int8_rows_have_the_same_bits_in_every_form(calc):
    """Whole sums and one order of scaling: a token's outputs are the same alone, in a chunk and in a prompt."""
    import torch
    g = torch.Generator(device="cuda")
    g.manual_seed(3)
    N, K = 4000, 528
    x, w = _random_codes(g, "int8", 4001, K), _random_codes(g, "int8", N, K)
    sx, sw, bias = (torch.randn(n, generator=g, device="cuda") for n in (4001, N, N))
    W = code_tensor(w, [K, N], "int8")
    for name in ("bf16", "fp32"):
        seen, first = set(), None
        for M in (4001, 1024, 300, 33, 16, 3):
            out = torch.zeros(M, N, dtype=torch_real(name), device="cuda")
            calc.scaledGemm(real_tensor(out, [N, M]), code_tensor(x[:M], [K, M], "int8"), sx, W, sw, bias)
            seen.add(calc.lastContractionForm()["tile_rows"])
            calc.synchronize()
            first = out if first is None else first
            assert torch.equal(out, first[:M]), M
        assert {8, 16, 64, 128, 256} <= seen


@pytest.mark.parametrize("M,N,K", [(5, 600, 1000), (100, 700, 1040), (2001, 2001, 392), (4000, 4001, 512)])
def test_fp8_rows_do_not_see_each_other(calc, M, N, K):
    """A row's outputs are the same bits whatever the other rows hold, NaN among it."""
    import torch
    g = torch.Generator(device="cuda")
    g.manual_seed(M)
    x, w, other = (_random_codes(g, "e4m3", n, K) for n in (M, N, M))
    keep = torch.arange(M, device="cuda") % 3 == 0
    other[keep] = x[keep]
    other[~keep, 0] = 0x7F  # NaN
    outs = []
    for v in (x, other):
        outs.append(torch.zeros(M, N, dtype=torch.bfloat16, device="cuda"))
        torch.cuda.synchronize()
        calc.scaledGemm(real_tensor(outs[-1], [N, M]), code_tensor(v, [K, M], "e4m3"), None, code_tensor(w, [K, N], "e4m3"), None)
        calc.synchronize()
    assert torch.equal(outs[0][keep], outs[1][keep]) and torch.all(torch.isnan(outs[1][~keep])) and not torch.any(torch.isnan(outs[0]))


@pytest.mark.parametrize("name", ["bf16", "fp16"])
@pytest.mark.parametrize("width", [8193, 11008, 14336, 16379, 16384])
@pytest.mark.parametrize("gate", ["", "silu", "gelu"])
def test_rows_of_32_elements_a_lane(calc, gate, width, name):
    """The form of long prompts' gated rows: as many rows as compute units, wider than 8192."""
    import torch
    rng = np.random.default_rng(width)
    rows, dt = 260, torch_real(name)
    both = torch.from_numpy(rng.standard_normal((rows, 2 * width)).astype(np.float32)).cuda().to(dt)
    both[3] = 0
    both[5, width + width // 2] = float("nan")
    t = real_tensor(both, [2 * width, rows])
    kind = {"": "int8", "silu": "e4m3", "gelu": "e5m2"}[gate]
    codes, scales = torch.full((rows * width + 64,), 85, dtype=torch.uint8, device="cuda"), torch.zeros(rows, device="cuda")
    O, X, G = code_tensor(codes, [width, rows], kind), t.window(width, [width, rows]), t.window(0, [width, rows]) if gate else None
    cus = torch.cuda.get_device_properties(0).multi_processor_count
    form = abi.plan_quantize_rows(O.desc, scales.data_ptr(), X.desc, G.desc if gate else None, num_cus=cus)
    assert form["elements"] == 32 and form["rows_per_group"] == 1, form
    calc.quantizeRows(O, scales, X, G, abi.GATE_GELU_TANH if gate == "gelu" else abi.GATE_SILU)
    calc.synchronize()
    assert torch.all(codes[rows * width:] == 85)
    b = both.cpu().double().numpy()
    v = b[:, width:] if not gate else gate64(b[:, :width], gate) * b[:, width:]
    # (the roundings that the narrower forms' tests count; |g| < 6 here, so that the gelu's argument stays below 28)
    n = {"": 2, "silu": 12, "gelu": 12 + 5 * 28}[gate]
    check_codes(v, codes[:rows * width].cpu().numpy().reshape(rows, width), scales.cpu().double().numpy(), kind, n, max(8, n + 2))


@pytest.mark.parametrize("M,N,K", [(4, 600, 512), (70, 4000, 512), (2001, 2001, 385), (4000, 4001, 512)])
@pytest.mark.parametrize("name,power", [("fp16", -34), ("fp16", -2), ("bf16", -146), ("bf16", 111), ("fp32", -146)])
def test_outputs_at_the_ends_of_their_type(calc, M, N, K, name, power):
    """Whole sums times powers of two are exact in fp32: what comes out is one rounding of them, to denormals and infinities too."""
    import torch
    g = torch.Generator(device="cuda")
    g.manual_seed(M)
    x, w = _random_codes(g, "int8", M, K), _random_codes(g, "int8", N, K)
    out = torch.zeros(M, N, dtype=torch_real(name), device="cuda")
    sx, sw = torch.full((M,), 2.0 ** (power // 2), device="cuda"), torch.full((N,), 2.0 ** (power - power // 2), device="cuda")
    torch.cuda.synchronize()
    calc.scaledGemm(real_tensor(out, [N, M]), code_tensor(x, [K, M], "int8"), sx, code_tensor(w, [K, N], "int8"), sw)
    calc.synchronize()
    sums = _values(x, "int8") @ _values(w, "int8").T
    want = (sums * 2.0 ** power).float()
    assert torch.equal(want.double(), sums * 2.0 ** power) or name == "bf16" and power > 0
    assert torch.equal(out, want.cpu().to(out.dtype).cuda())
    if name != "fp32":
        assert bool(torch.any(torch.isinf(out))) == (power in (-2, 111)) and (power > -30 or bool(torch.any((out != 0) & (out.abs() < torch.finfo(out.dtype).tiny))))


@pytest.mark.parametrize("M,N", [(100, 300), (3, 20)])
def test_no_reduction_leaves_the_bias(calc, M, N):
    import torch
    out, bias = torch.full((M, N), 9.0, device="cuda"), torch.randn(N, device="cuda")
    one = code_tensor(torch.zeros(max(M, N), 16, dtype=torch.uint8, device="cuda"), [16, max(M, N)], "int8")
    calc.scaledGemm(real_tensor(out, [N, M]), one.window(0, [0, M]), None, one.window(0, [0, N]), None, bias)
    calc.synchronize()
    assert torch.equal(out, bias.expand(M, N))


@pytest.mark.parametrize("name", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("width", [40, 3001, 20000])
def test_residual_sums_at_the_ends_of_their_type(calc, name, width):
    """The sum that is kept is one rounding of the sum in fp32, denormals, infinities and NaN among it."""
    import torch
    rng = np.random.default_rng(width)
    dt = torch_real(name)
    tiny, top = torch.finfo(dt).smallest_normal, torch.finfo(dt).max
    x, r = (torch.from_numpy(rng.standard_normal((4, width)).astype(np.float32)) for _ in range(2))
    for v in (x, r):
        v[0] *= tiny
        v[1] *= 0.4 * top
    x, r = x.clamp(-top, top).to(dt), r.clamp(-top, top).to(dt)
    x[2, 1], r[2, 1], x[2, 3], r[2, 5] = float("inf"), float("-inf"), float("inf"), float("nan")
    want = (x.float() + r.float()).to(dt)
    x, r, out = x.cuda(), r.cuda(), torch.zeros(4, width, dtype=dt, device="cuda")
    codes, scales = torch.zeros(4, width, dtype=torch.uint8, device="cuda"), torch.zeros(4, device="cuda")
    calc.rmsNormQuantize(code_tensor(codes, [width, 4], "int8"), scales, real_tensor(x, [width, 4]), None, real_tensor(r, [width, 4]), real_tensor(out, [width, 4]))
    calc.synchronize()
    got = out.cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(got.nan_to_num(7.0), want.nan_to_num(7.0))
    assert torch.isnan(scales[2]) and not codes[2].any() and torch.all(torch.isfinite(scales[[0, 3]]))
