"""8-bit linear layer on the GPU: quantizeRows, rmsNormQuantize, scaledGemm against 64-bit arithmetic.

(Collected behind the test of the allocation-free entry point, which compares the device's free memory before and after: the runtime gives a
hardware queue memory when the first kernel with private memory runs there, and which queue a new handle's stream gets depends on the
streams that earlier tests have used.)"""
import math

import numpy as np
import pytest

from intel_gaudi3_software_amd import MMEStackException, MmeSimTensor, abi
from linear8_helpers import (CODES, U, check_codes, check_product, code_tensor, code_values, gate64, real_tensor, sums_error,
                             torch_real)

pytestmark = pytest.mark.gpu


def _rows(rng, rows, width, spread=1.0):
    return rng.standard_normal((rows, width)) * np.exp(spread * rng.standard_normal((rows, 1)))


def _cuda(a, name):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.float32)).to(torch_real(name)).cuda()


def _f64(t):
    return t.cpu().double().numpy()


def _codes_of(t):
    import torch
    return t.cpu().view(torch.uint8).numpy()


def _scale_roundings(width, norm):
    # |v|'s own roundings (2), the final one, the squares' sum: at most 16 additions in a lane (a row gone over in memory: one more
    # for every 8192 elements), 12 between lanes, the square itself and s's rounding twice; the root halves them
    return 4.0 + ((16 if width <= 16384 else 8 * math.ceil(width / 8192)) + 12 + 4) / 2 if norm else 8.0


WIDTHS = [1, 7, 8, 9, 63, 64, 511, 512, 513, 1024, 1025, 2047, 2048, 2049, 4096, 4097, 8191, 8192, 8200, 16384, 16385, 40007]


@pytest.mark.parametrize("width", WIDTHS)
@pytest.mark.parametrize("name", ["bf16", "fp16", "fp32"])
def test_quantize_rows_widths(calc, width, name):
    import torch
    rng = np.random.default_rng(width)
    for rows, kind in ((1, "int8"), (5, "e4m3"), (4, "e5m2")):
        x = _cuda(_rows(rng, rows, width), name)
        codes, scales = torch.full((rows, width), 85, dtype=torch.uint8, device="cuda"), torch.full((rows,), -1.0, device="cuda")
        calc.quantizeRows(code_tensor(codes, [width, rows], kind), scales, real_tensor(x, [width, rows]))
        calc.synchronize()
        check_codes(_f64(x), _codes_of(codes), _f64(scales), kind, 2, _scale_roundings(width, False))


@pytest.mark.parametrize("kind", list(CODES))
def test_quantize_rows_types(calc, kind):
    import torch
    rng = np.random.default_rng(3)
    x = _cuda(_rows(rng, 37, 384), "bf16")
    codes, scales = torch.zeros(37, 384, dtype=torch.uint8, device="cuda"), torch.zeros(37, device="cuda")
    calc.quantizeRows(code_tensor(codes, [384, 37], kind), scales, real_tensor(x, [384, 37]))
    calc.synchronize()
    check_codes(_f64(x), _codes_of(codes), _f64(scales), kind, 2, 8)


@pytest.mark.parametrize("gate", ["silu", "gelu"])
@pytest.mark.parametrize("name,width", [("bf16", 96), ("fp16", 1000), ("fp32", 777), ("bf16", 5632), ("bf16", 14336), ("fp32", 20001)])
def test_gated_rows_side_by_side(calc, gate, name, width):
    """Gate and up halves as windows of one tensor: the second half starts wherever the first one ends."""
    import torch
    rng = np.random.default_rng(width)
    rows = 6
    both = _cuda(rng.standard_normal((rows, 2 * width)) * 3, name)
    t = real_tensor(both, [2 * width, rows])
    codes, scales = torch.zeros(rows, width, dtype=torch.uint8, device="cuda"), torch.zeros(rows, device="cuda")
    for kind in ("int8", "e4m3"):
        calc.quantizeRows(code_tensor(codes, [width, rows], kind), scales, t.window(width, [width, rows]), t.window(0, [width, rows]),
                          {"silu": abi.GATE_SILU, "gelu": abi.GATE_GELU_TANH}[gate])
        calc.synchronize()
        b = _f64(both)
        # fp32 roundings: the gate's argument (gelu: five, magnified by it: checked apart), e^x to two units, one addition, one quotient,
        # one product, the factor and the last product.  e^-a against 1 + e^-a: an error of a's rounding d moves the gate by at most
        # |a| d relative, and |a| <= 2 sqrt(2 / pi) (|g| + 0.044715 |g|^3) < 90 for gelu where the gate is not negligible (|g| < 8 here
        # gives 49); silu's argument is exact
        roundings = 12 if gate == "silu" else 12 + 5 * 60
        check_codes(gate64(b[:, :width], gate) * b[:, width:], _codes_of(codes), _f64(scales), kind, roundings, roundings + 2)


def test_gate_extremes(calc):
    import torch
    g = np.array([-1e30, -200.0, -100.0, -88.5, -87.5, -20.0, -1e-30, 0.0, 1e-30, 5.0, 50.0, 87.5, 90.0, 1000.0], np.float32)
    for gate, op in (("silu", abi.GATE_SILU), ("gelu", abi.GATE_GELU_TANH)):
        gt, x = torch.from_numpy(g).cuda(), torch.ones(len(g), device="cuda")
        codes, scales = torch.zeros(len(g), dtype=torch.uint8, device="cuda"), torch.zeros(1, device="cuda")
        calc.quantizeRows(code_tensor(codes, [len(g), 1], "e5m2"), scales, real_tensor(x, [len(g), 1]), real_tensor(gt, [len(g), 1]), op)
        calc.synchronize()
        want = gate64(g.astype(np.float64), gate)
        want[~np.isfinite(want)] = 0.0
        check_codes(want[None], _codes_of(codes)[None], _f64(scales), "e5m2", 400, 400)


@pytest.mark.parametrize("width", WIDTHS)
@pytest.mark.parametrize("name,gamma_name,residual", [("bf16", "bf16", True), ("fp16", "fp32", False), ("fp32", "fp32", True), ("bf16", None, False)])
def test_norm_widths(calc, width, name, gamma_name, residual):
    import torch
    rng = np.random.default_rng(width + 1)
    for rows, kind in ((1, "e4m3"), (5, "int8")):
        x = _cuda(_rows(rng, rows, width), name)
        res = _cuda(_rows(rng, rows, width), name) if residual else None
        gamma = _cuda(1 + 0.3 * rng.standard_normal(width), gamma_name) if gamma_name else None
        codes, scales = torch.zeros(rows, width, dtype=torch.uint8, device="cuda"), torch.zeros(rows, device="cuda")
        out = torch.zeros_like(x)
        calc.rmsNormQuantize(code_tensor(codes, [width, rows], kind), scales, real_tensor(x, [width, rows]), real_tensor(gamma, [width]) if gamma_name else None,
                             real_tensor(res, [width, rows]) if residual else None, real_tensor(out, [width, rows]) if residual else None, 1e-5)
        calc.synchronize()
        s = _f64(x)
        if residual:
            s = s + _f64(res)
            # (the sum is rounded to fp32, then to its type)
            want = (x.float() + res.float()).to(x.dtype)
            assert torch.equal(out, want)
        v = s / np.sqrt(np.mean(s * s, axis=1, keepdims=True) + np.float64(np.float32(1e-5)))
        if gamma_name:
            v = v * _f64(gamma)[None]
        # the sum's rounding may be large against a sum that cancels: it is part of the input here
        if residual:
            s32 = (x.float() + res.float()).cpu().double().numpy()
            v = s32 / np.sqrt(np.mean(s32 * s32, axis=1, keepdims=True) + np.float64(np.float32(1e-5)))
            if gamma_name:
                v = v * _f64(gamma)[None]
        check_codes(v, _codes_of(codes), _f64(scales), kind, 3, _scale_roundings(width, True))


def _norm64(s, gamma, eps):
    with np.errstate(all="ignore"):
        v = s * gamma
        return v / np.sqrt(np.mean(s * s, axis=1, keepdims=True) + eps)


@pytest.mark.parametrize("width", [40, 600, 3000, 9000, 20000])
def test_rows_at_the_ends_of_the_range(calc, width):
    """Rows of zeros, of denormals, of values whose squares or products overflow, rows that hold an inf or NaN; neighbours of such
    rows are ordinary."""
    import torch
    rng = np.random.default_rng(width)
    base = rng.standard_normal((11, width))
    factors = [1.0, 0.0, 1e-41, 1e-38, 1e-30, 1e-20, 1e15, 1e25, 5e36, 1.0, 1.0]
    x64 = base * np.array(factors)[:, None]
    x64[9, width // 2] = np.inf
    x64[10, width - 1] = np.nan
    x = torch.from_numpy(x64.astype(np.float32)).cuda()
    xs = _f64(x)
    codes, scales = torch.zeros(11, width, dtype=torch.uint8, device="cuda"), torch.zeros(11, device="cuda")
    X = real_tensor(x, [width, 11])
    for kind in ("int8", "e4m3"):
        O = code_tensor(codes, [width, 11], kind)
        calc.quantizeRows(O, scales, X)
        calc.synchronize()
        # (a scale below 2^-126 is a denormal: the bound's absolute part; row 2's are all of that kind)
        check_codes(xs, _codes_of(codes), _f64(scales), kind, 2, 8)
        for eps in (0.0, 1e-6):
            for gamma in (None, 1.0, 1e-25, 1e25):
                G = None if gamma is None else torch.full((width,), gamma, device="cuda")
                calc.rmsNormQuantize(O, scales, X, None if gamma is None else real_tensor(G, [width]), eps=eps)
                calc.synchronize()
                g = 1.0 if gamma is None else np.float64(np.float32(gamma))
                v = _norm64(xs, g, np.float64(np.float32(eps)))
                v[1] = 0.0
                # (s gamma below 2^-126 has fewer bits; those rows are checked for their scales' size only)
                fine = [r for r in range(11) if factors[r] == 0.0 or not np.isfinite(x64[r]).all() or abs(factors[r] * g) > 1e-34]
                check_codes(v[fine], _codes_of(codes)[fine], _f64(scales)[fine], kind, 4, _scale_roundings(width, True) + 4)


def test_zero_gamma_hides_no_nan(calc):
    import torch
    x = torch.ones(3, 200, device="cuda")
    x[1, 50] = float("inf")
    gamma = torch.ones(200, device="cuda")
    gamma[50] = 0.0
    codes, scales = torch.ones(3, 200, dtype=torch.uint8, device="cuda"), torch.zeros(3, device="cuda")
    calc.rmsNormQuantize(code_tensor(codes, [200, 3], "int8"), scales, real_tensor(x, [200, 3]), real_tensor(gamma, [200]))
    calc.synchronize()
    s = _f64(scales)
    assert np.isnan(s[1]) and np.all(np.isfinite(s[[0, 2]])) and not _codes_of(codes)[1].any()


def test_norm_in_place_strided_and_gaps(calc):
    """residual_out in place of the residual, rows with a pitch, dimensions whose strides do not collapse; what lies between the
    rows stays."""
    import torch
    rng = np.random.default_rng(8)
    W, P, R, Q = 72, 100, 5, 3  # rows of 72 on a pitch of 100, 5 rows per plane, planes 700 apart
    buf = [torch.from_numpy(rng.standard_normal(700 * Q).astype(np.float32)).bfloat16().cuda() for _ in range(2)]
    st = [1, P, 700, 700 * Q, 700 * Q]
    xt, rt = (real_tensor(b, [700 * Q, 1]).window(0, [W, R, Q], st) for b in buf)
    codes = torch.full((7, 2000), 85, dtype=torch.uint8, device="cuda")
    ct = code_tensor(codes, [14000, 1], "e4m3").window(3, [W, R, Q], [1, 80, 401, 1300, 1300])
    gamma = torch.from_numpy(rng.standard_normal(W).astype(np.float32)).bfloat16().cuda()
    scales = torch.zeros(R * Q + 2, device="cuda")
    before = [b.clone() for b in buf]
    calc.rmsNormQuantize(ct, scales, xt, real_tensor(gamma, [W]), rt, rt, 1e-6)
    calc.synchronize()
    at = (np.arange(Q)[:, None, None] * 700 + np.arange(R)[None, :, None] * P + np.arange(W)[None, None, :]).reshape(R * Q, W)
    x, r = _f64(before[0])[at], _f64(before[1])[at]
    s = (before[0].float() + before[1].float()).cpu()
    want = before[1].cpu().clone()
    want[torch.from_numpy(at.ravel())] = s.bfloat16()[torch.from_numpy(at.ravel())]
    assert torch.equal(buf[1].cpu(), want) and torch.equal(buf[0], before[0])
    at_c = (3 + np.arange(Q)[:, None, None] * 401 + np.arange(R)[None, :, None] * 80 + np.arange(W)[None, None, :]).reshape(R * Q, W)
    got = _codes_of(codes).ravel()
    check_codes(_norm64(s.double().numpy()[at], _f64(gamma)[None], np.float64(np.float32(1e-6))), got[at_c], _f64(scales), "e4m3", 3, 24)
    rest = np.ones(got.size, bool)
    rest[at_c.ravel()] = False
    assert np.all(got[rest] == 85) and not _f64(scales)[R * Q:].any()


@pytest.mark.parametrize("width", [100, 500, 4000, 5001, 14336, 20000, 70001])
@pytest.mark.parametrize("place", ["x", "residual"])
def test_norm_in_place_in_every_form(calc, width, place):
    """The same bits as with an output of its own, ordinary rows and ones that are gone over twice."""
    import torch
    rng = np.random.default_rng(width)
    x, r = (torch.from_numpy((rng.standard_normal((6, width)) * np.array([1, 1e30, 1e-30, 1, 0, 1])[:, None]).astype(np.float32)).cuda() for _ in range(2))
    got = []
    for own in (True, False):
        X, R = x.clone(), r.clone()
        out = torch.zeros_like(x) if own else X if place == "x" else R
        codes, scales = torch.zeros(6, width, dtype=torch.uint8, device="cuda"), torch.zeros(6, device="cuda")
        tx, tr = real_tensor(X, [width, 6]), real_tensor(R, [width, 6])
        calc.rmsNormQuantize(code_tensor(codes, [width, 6], "e4m3"), scales, tx, None, tr, real_tensor(out, [width, 6]) if own else tx if place == "x" else tr)
        calc.synchronize()
        assert torch.equal(out, x + r)
        got.append((codes, scales))
    assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1])


def test_broadcast_rows_and_no_rows(calc):
    import torch
    x = torch.randn(64, device="cuda")
    codes, scales = torch.zeros(9, 64, dtype=torch.uint8, device="cuda"), torch.zeros(9, device="cuda")
    one = real_tensor(x, [64, 1]).window(0, [64, 9], [1, 0, 0, 0, 0])
    calc.quantizeRows(code_tensor(codes, [64, 9], "int8"), scales, one)
    calc.synchronize()
    check_codes(np.repeat(_f64(x)[None], 9, 0), _codes_of(codes), _f64(scales), "int8", 2, 8)
    before = codes.clone()
    calc.quantizeRows(code_tensor(codes, [64, 9], "int8").window(0, [64, 0]), scales[:0], real_tensor(x, [64, 1]).window(0, [64, 0]))
    calc.synchronize()
    assert torch.equal(codes, before)


# ---- scaled product ----------------------------------------------------------------------------------------------------
def _random_codes(rng, kind, *shape):
    if kind == "int8":
        return rng.integers(-128, 128, shape).astype(np.int8).view(np.uint8)
    c = rng.integers(0, 0x78 if kind.startswith("e4m3") else 0x6C, shape).astype(np.uint8)
    return c | (rng.integers(0, 2, shape).astype(np.uint8) << 7)


def _product(calc, rng, M, N, K, a="int8", b="int8", out="bf16", batch=1, bias=False, scales=True, x_batch=None, w_batch=None):
    import torch
    xb, wb = x_batch or batch, w_batch or batch
    x, w = _random_codes(rng, a, xb, M, K), _random_codes(rng, b, wb, N, K)
    sx, sw = (np.exp(rng.standard_normal((xb, M))) * 1e-2).astype(np.float32), (np.exp(rng.standard_normal((wb, N))) * 1e-3).astype(np.float32)
    bi = rng.standard_normal((wb, N)).astype(np.float32)
    # (one element in front: nothing is aligned beyond its own element)
    tx, tw = (torch.from_numpy(np.concatenate([np.zeros(1, np.uint8), v.ravel()])).cuda() for v in (x, w))
    guard = 64
    to = torch.full((batch * M * N + guard,), 77, dtype=torch_real(out), device="cuda")
    return dict(x=x, w=w, sx=sx, sw=sw, bias=bi if bias else None, tx=tx, tw=tw, to=to, guard=guard, scales=scales, M=M, N=N, K=K, a=a, b=b, out=out,
                batch=batch, xb=xb, wb=wb, tsx=torch.from_numpy(sx).cuda(), tsw=torch.from_numpy(sw).cuda(), tbias=torch.from_numpy(bi).cuda())


def _run_product(calc, p, aligned=True):
    M, N, K, batch = p["M"], p["N"], p["K"], p["batch"]
    import torch
    if aligned:
        tx, tw = p["tx"][1:].clone(), p["tw"][1:].clone()
        X, W = code_tensor(tx, [K, M, p["xb"]], p["a"]), code_tensor(tw, [K, N, p["wb"]], p["b"])
    else:
        X = code_tensor(p["tx"], [p["tx"].numel(), 1], p["a"]).window(1, [K, M, p["xb"]], [1, K, M * K, M * K * p["xb"], M * K * p["xb"]])
        W = code_tensor(p["tw"], [p["tw"].numel(), 1], p["b"]).window(1, [K, N, p["wb"]], [1, K, N * K, N * K * p["wb"], N * K * p["wb"]])
    O = real_tensor(p["to"], [N, M, batch])
    s = p["scales"]
    calc.scaledGemm(O, X, p["tsx"] if s else None, W, p["tsw"] if s else None, p["tbias"] if p["bias"] is not None else None)
    calc.synchronize()
    assert torch.all(p["to"][batch * M * N:] == 77)
    return p["to"][:batch * M * N].cpu().numpy() if p["out"] in ("int32", "fp32") else p["to"][:batch * M * N].cpu().double().numpy()


def _check(p, out):
    M, N, K, batch = p["M"], p["N"], p["K"], p["batch"]
    out = out.reshape(batch, M, N)
    for c in range(batch):
        cx, cw = (c if p["xb"] > 1 else 0), (c if p["wb"] > 1 else 0)
        x, w = code_values(p["x"][cx], p["a"]).reshape(M, K), code_values(p["w"][cw], p["b"]).reshape(N, K)
        sums = x @ w.T
        if p["out"] == "int32":
            assert np.array_equal(out[c], sums.astype(np.int64))
            continue
        error = sums_error(x, w, p["a"])
        one_x, one_w = np.ones(M), np.ones(N)
        check_product(out[c].astype(np.float64), sums, error, p["sx"][cx].astype(np.float64) if p["scales"] else one_x,
                      p["sw"][cw].astype(np.float64) if p["scales"] else one_w, p["bias"][cw].astype(np.float64) if p["bias"] is not None else None, p["out"])


SIZES = [(1, 1, 1), (1, 64, 64), (1, 65, 16), (2, 1, 100), (3, 17, 31), (16, 128, 256), (17, 130, 129), (31, 33, 15), (32, 64, 1024), (33, 63, 48),
         (64, 256, 272), (65, 257, 500), (100, 512, 512), (128, 384, 640), (129, 385, 1000), (250, 520, 1040), (256, 256, 4096), (257, 300, 2064),
         (512, 1024, 512), (700, 515, 333), (1, 4096, 4096), (8, 1000, 14336), (48, 2048, 2048)]


@pytest.mark.parametrize("M,N,K", SIZES)
@pytest.mark.parametrize("a,b", [("int8", "int8"), ("e4m3", "e4m3"), ("e5m2", "e4m3")])
def test_product_sizes(calc, M, N, K, a, b):
    rng = np.random.default_rng(M * 7 + N * 3 + K)
    for out, bias in (("bf16", False), ("fp32", True), ("int32", False)) if a == "int8" else (("bf16", False), ("fp16", True)):
        p = _product(calc, rng, M, N, K, a, b, out, bias=bias, scales=out != "int32")
        _check(p, _run_product(calc, p))


@pytest.mark.parametrize("M,N,K", [(1, 70, 130), (20, 100, 256), (70, 260, 96), (300, 300, 1024)])
@pytest.mark.parametrize("a,b,out", [("int8", "int8", "int32"), ("int8", "int8", "fp16"), ("e4m3", "e5m2", "fp16"), ("e5m2", "e5m2", "bf16"), ("e4m3_b3", "e5m2_b20", "bf16")])
def test_product_unaligned_and_types(calc, M, N, K, a, b, out):
    rng = np.random.default_rng(5)
    p = _product(calc, rng, M, N, K, a, b, out, bias=out != "int32", scales=out != "int32")
    if out == "fp16" and a != "int8":
        p["tsx"] *= 0.01  # (sums of such codes reach 1e5)
        p["sx"] *= np.float32(0.01)
        p["sx"] = p["tsx"].cpu().numpy()
    _check(p, _run_product(calc, p, aligned=False))
    _check(p, _run_product(calc, p, aligned=True))


@pytest.mark.parametrize("batch,xb,wb", [(3, 3, 3), (3, 1, 3), (3, 3, 1), (5, 1, 1)])
@pytest.mark.parametrize("M,N,K", [(2, 100, 64), (40, 130, 200), (150, 300, 512)])
def test_product_batches(calc, batch, xb, wb, M, N, K):
    rng = np.random.default_rng(11)
    for a, out in (("int8", "int32"), ("int8", "bf16"), ("e4m3", "bf16")):
        p = _product(calc, rng, M, N, K, a, a, out, batch=batch, bias=out != "int32", scales=out != "int32", x_batch=xb, w_batch=wb)
        _check(p, _run_product(calc, p))


@pytest.mark.parametrize("M", [1, 5, 40, 200])
def test_product_strided(calc, M):
    """Rows on pitches, batch dimensions in another order than memory, an output with gaps that stay."""
    import torch
    rng = np.random.default_rng(M)
    N, K = 96, 160
    x, w = _random_codes(rng, "int8", M, 2, K), _random_codes(rng, "int8", N, 208)  # x: the batch lies between the rows
    tx, tw = torch.from_numpy(x).cuda(), torch.from_numpy(w).cuda()
    X = code_tensor(tx, [K * 2 * M, 1], "int8").window(0, [K, M, 2], [1, 2 * K, K, 2 * K * M, 2 * K * M])
    W = code_tensor(tw, [208, N], "int8").window(16, [K, N])
    to = torch.full((M * 2 * 128,), 77, dtype=torch.int32, device="cuda")
    O = real_tensor(to, [to.numel(), 1]).window(4, [N, M, 2], [1, 256, 128, 256 * M, 256 * M])
    calc.scaledGemm(O, X, None, W, None)
    calc.synchronize()
    got = to.cpu().numpy().reshape(M, 2, 128)
    want = np.einsum("mbk,nk->mbn", x.view(np.int8).astype(np.int64), w[:, 16:16 + K].view(np.int8).astype(np.int64))
    assert np.array_equal(got[:, :, 4:4 + N], want)
    assert np.all(got[:, :, :4] == 77) and np.all(got[:, :, 4 + N:] == 77)


@pytest.mark.parametrize("M,N,rows,aligned", [(70, 4000, 64, True), (70, 4000, 64, False), (2001, 2001, 128, True), (2001, 2001, 128, False), (4000, 4001, 256, True)])
def test_product_tiles_at_every_kind_of_end(calc, M, N, rows, aligned):
    """Reductions that end at every place of a stage, fewer stages than the ring holds and more, rows at even and at odd addresses."""
    import torch
    rng = np.random.default_rng(M)
    seen = set()
    for K in (1, 7, 15, 16, 17, 31, 100, 127, 128, 129, 255, 256, 272, 330, 384, 400, 511, 512, 513, 640, 645, 766, 1025):
        x, w = _random_codes(rng, "int8", M, K), _random_codes(rng, "int8", N, K)
        pitch, first = (-(-K // 16) * 16 + 16, 16) if aligned else (K + 3, 5)
        tx, tw = torch.full((first + M * pitch,), 99, dtype=torch.uint8, device="cuda"), torch.full((first + N * pitch,), 99, dtype=torch.uint8, device="cuda")
        tx[first:].view(M, pitch)[:, :K] = torch.from_numpy(x).cuda()
        tw[first:].view(N, pitch)[:, :K] = torch.from_numpy(w).cuda()
        out = torch.full((M, N), 77, dtype=torch.int32, device="cuda")
        X = code_tensor(tx, [tx.numel(), 1], "int8").window(first, [K, M], [1, pitch, M * pitch, M * pitch, M * pitch])
        W = code_tensor(tw, [tw.numel(), 1], "int8").window(first, [K, N], [1, pitch, N * pitch, N * pitch, N * pitch])
        calc.scaledGemm(real_tensor(out, [N, M]), X, None, W, None)
        seen.add(calc.lastContractionForm()["tile_rows"])
        calc.synchronize()
        value = lambda c: torch.from_numpy(c.view(np.int8)).cuda().double()
        assert torch.equal(out.double(), value(x) @ value(w).T), K  # (exact: sums below 2^53)
    assert rows in seen


def test_offsets_beyond_32_bits(calc):
    """Rows that lie further apart than 2^31 elements, of values, codes and outputs."""
    import torch
    rng = np.random.default_rng(8)
    pitch, K, N = (1 << 31) + 4096, 256, 80
    big = torch.empty(3 * pitch, dtype=torch.uint8, device="cuda")  # (6.4 GB)
    far = lambda t, width: MmeSimTensor([big.numel() // (2 if t == abi.BF16 else 1)], 1, t, big.view(torch.bfloat16) if t == abi.BF16 else big).window(
        0, [width, 3], [1, pitch // (2 if t == abi.BF16 else 1)] + [3 * pitch] * 3)
    x = torch.from_numpy(rng.standard_normal((3, K))).cuda().bfloat16()
    big.view(torch.bfloat16).view(3, pitch // 2)[:, :K] = x
    codes, scales = torch.zeros(3, K, dtype=torch.uint8, device="cuda"), torch.zeros(3, device="cuda")
    calc.quantizeRows(code_tensor(codes, [K, 3], "int8"), scales, far(abi.BF16, K))
    near, near_scales = torch.zeros_like(codes), torch.zeros_like(scales)
    calc.quantizeRows(code_tensor(near, [K, 3], "int8"), near_scales, real_tensor(x, [K, 3]))
    calc.synchronize()
    assert torch.equal(codes, near) and torch.equal(scales, near_scales)
    calc.quantizeRows(far(abi.INT8, K), scales, real_tensor(x, [K, 3]))
    w = torch.from_numpy(_random_codes(rng, "int8", N, K)).cuda()
    out = torch.zeros(3, N, dtype=torch.bfloat16, device="cuda")
    calc.scaledGemm(real_tensor(out, [N, 3]), far(abi.INT8, K), scales, code_tensor(w, [K, N], "int8"), None)
    near_out = torch.zeros_like(out)
    calc.scaledGemm(real_tensor(near_out, [N, 3]), code_tensor(near, [K, 3], "int8"), scales, code_tensor(w, [K, N], "int8"), None)
    calc.synchronize()
    assert torch.equal(out, near_out)
    # the rows of w, in tiles, and the output
    many = torch.from_numpy(_random_codes(rng, "int8", 200, K)).cuda()
    calc.scaledGemm(far(abi.BF16, 3).window(0, [3, 3]), code_tensor(near, [K, 3], "int8"), scales, code_tensor(near, [K, 3], "int8"), None)
    want = torch.zeros(3, 3, dtype=torch.bfloat16, device="cuda")
    calc.scaledGemm(real_tensor(want, [3, 3]), code_tensor(near, [K, 3], "int8"), scales, code_tensor(near, [K, 3], "int8"), None)
    calc.synchronize()
    assert torch.equal(big.view(torch.bfloat16).view(3, pitch // 2)[:, :3], want)
    big.view(3, pitch)[:, :K] = near
    torch.cuda.synchronize()
    tall, want = torch.zeros(200, 3, dtype=torch.bfloat16, device="cuda"), torch.zeros(200, 3, dtype=torch.bfloat16, device="cuda")
    calc.scaledGemm(real_tensor(tall, [3, 200]), code_tensor(many, [K, 200], "int8"), None, far(abi.INT8, K), scales)
    calc.scaledGemm(real_tensor(want, [3, 200]), code_tensor(many, [K, 200], "int8"), None, code_tensor(near, [K, 3], "int8"), scales)
    calc.synchronize()
    assert torch.equal(tall, want)


def test_product_without_reduction_and_without_rows(calc):
    import torch
    bias = torch.tensor([1.0, -2.0, 3.0], device="cuda")
    out = torch.full((4, 3), 9.0, device="cuda")
    w = torch.zeros(3, 16, dtype=torch.uint8, device="cuda")
    W = code_tensor(w, [16, 3], "int8")
    calc.scaledGemm(real_tensor(out, [3, 4]), W.window(0, [0, 4]), None, W.window(0, [0, 3]), None, bias)
    calc.synchronize()
    assert torch.equal(out, bias.expand(4, 3))
    calc.scaledGemm(real_tensor(out, [3, 4]).window(0, [3, 0]), W.window(0, [16, 0]), None, W, None)
    calc.synchronize()
    assert torch.equal(out, bias.expand(4, 3))


def test_product_at_the_ends_of_the_range(calc):
    """The longest reduction of the largest codes; scales of opposite extremes; NaN and inf scales touch their own row only."""
    import torch
    K = 131071
    x, w = torch.full((2, K), -128, dtype=torch.int8, device="cuda"), torch.full((70, K), -128, dtype=torch.int8, device="cuda")
    w[69] = 127
    out = torch.zeros(2, 70, dtype=torch.int32, device="cuda")
    calc.scaledGemm(real_tensor(out, [70, 2]), code_tensor(x, [K, 2], "int8"), None, code_tensor(w, [K, 70], "int8"), None)
    calc.synchronize()
    assert torch.all(out[:, :69] == 16384 * K) and torch.all(out[:, 69] == -128 * 127 * K)
    x, w = torch.full((5, 64), 2, dtype=torch.int8, device="cuda"), torch.full((6, 64), 3, dtype=torch.int8, device="cuda")
    sx = torch.tensor([1e-30, 1.0, float("nan"), float("inf"), 0.0], device="cuda")
    sw = torch.tensor([1e30, 1.0, 1e-3, 2.0, 1e38, 1.0], device="cuda")
    for name in ("fp32", "bf16", "fp16"):
        o = torch.zeros(5, 6, dtype=torch_real(name), device="cuda")
        calc.scaledGemm(real_tensor(o, [6, 5]), code_tensor(x, [64, 5], "int8"), sx, code_tensor(w, [64, 6], "int8"), sw)
        calc.synchronize()
        want = (384.0 * sx[:, None] * sw[None, :]).to(o.dtype)
        assert torch.equal(torch.isnan(o), torch.isnan(want)) and torch.allclose(o.float().nan_to_num(7), want.float().nan_to_num(7), rtol=2.0 ** -7, atol=1e-35)


def test_product_rows_do_not_depend_on_each_other(calc):
    """fp8 sums have an order: a row's outputs are the same bits again in a second call."""
    import torch
    rng = np.random.default_rng(2)
    for M, N, K in ((3, 500, 4096), (100, 700, 3000), (300, 600, 2048)):
        p = _product(calc, rng, M, N, K, "e4m3", "e4m3", "bf16")
        first = _run_product(calc, p).copy()
        p["to"].fill_(77)
        assert np.array_equal(first, _run_product(calc, p))


def test_full_mode_codes_need_the_promise(calc):
    import torch
    rng = np.random.default_rng(4)
    x = _cuda(rng.standard_normal((20, 256)), "bf16")
    w = _cuda(rng.standard_normal((30, 256)), "bf16")
    c = calc
    try:
        q, s = [], []
        for t in (x, w):
            q.append(torch.zeros(t.shape, dtype=torch.uint8, device="cuda"))
            s.append(torch.zeros(t.shape[0], device="cuda"))
            c.quantizeRows(code_tensor(q[-1], [256, t.shape[0]], "e4m3_full"), s[-1], real_tensor(t, [256, t.shape[0]]))
        c.synchronize()
        o = torch.zeros(20, 30, dtype=torch.float16, device="cuda")
        call = lambda: c.scaledGemm(real_tensor(o, [30, 20]), code_tensor(q[0], [256, 20], "e4m3_full"), s[0], code_tensor(q[1], [256, 30], "e4m3_full"), s[1])
        with pytest.raises(MMEStackException) as e:
            call()
        assert e.value.status == abi.EUNSUPPORTED
        c.setFp8SpecialsPolicy(abi.FP8_SPECIALS_ASSUME_NONE)
        call()
        c.synchronize()
        vx, vw = code_values(_codes_of(q[0]), "e4m3_full"), code_values(_codes_of(q[1]), "e4m3_full")
        check_product(_f64(o), vx @ vw.T, sums_error(vx, vw, "e4m3_full"), _f64(s[0]), _f64(s[1]), None, "fp16")
    finally:
        c.setFp8SpecialsPolicy(abi.FP8_SPECIALS_CHECK)


# ---- streams, graphs, devices, refusals -----------------------------------------------------------------------------------
def _block(c, t, out):
    """Norm, up and gate projection, gated rows, down projection: a feed-forward block in 8 bits."""
    M, H, F = t["M"], t["H"], t["F"]
    c.rmsNormQuantize(t["xq"], t["xs"], t["x"], t["gamma"], t["res"], t["sum"], 1e-6)
    c.scaledGemm(t["gu"], t["xq"], t["xs"], t["w1"], t["w1s"])
    c.quantizeRows(t["hq"], t["hs"], t["gu"].window(F, [F, M]), t["gu"].window(0, [F, M]))
    c.scaledGemm(out, t["hq"], t["hs"], t["w2"], t["w2s"])


def _block_tensors(c, M, H, F, kind, seed):
    import torch
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")
    t = {"M": M, "H": H, "F": F, "raw": {"x": rnd(M, H).bfloat16(), "res": (2 * rnd(M, H)).bfloat16(), "gamma": (1 + 0.2 * rnd(H)).bfloat16()}}
    t["raw"]["sum"] = torch.zeros_like(t["raw"]["x"])
    for n in ("x", "res", "sum"):
        t[n] = real_tensor(t["raw"][n], [H, M])
    t["gamma"] = real_tensor(t["raw"]["gamma"], [H])
    for n, rows, width in (("w1", 2 * F, H), ("w2", H, F)):
        w = (rnd(rows, width) / math.sqrt(width)).bfloat16()
        t["raw"][n] = torch.zeros(rows, width, dtype=torch.uint8, device="cuda")
        t[n], t[n + "s"] = code_tensor(t["raw"][n], [width, rows], kind), torch.zeros(rows, device="cuda")
        torch.cuda.synchronize()
        c.quantizeRows(t[n], t[n + "s"], real_tensor(w, [width, rows]))
        c.synchronize()
    for n, width in (("xq", H), ("hq", F)):
        t["raw"][n] = torch.zeros(M, width, dtype=torch.uint8, device="cuda")
        t[n], t[n[0] + "s"] = code_tensor(t["raw"][n], [width, M], kind), torch.zeros(M, device="cuda")
    t["raw"]["gu"] = torch.zeros(M, 2 * F, dtype=torch.bfloat16, device="cuda")
    t["gu"] = real_tensor(t["raw"]["gu"], [2 * F, M])
    return t


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("M", [1, 19, 300])
def test_feed_forward_block(calc, kind, M):
    """The operators in the order a model calls them, each stage against 64-bit arithmetic on the stage's own inputs."""
    import torch
    H, F = 512, 1360
    t = _block_tensors(calc, M, H, F, kind, M)
    out = torch.zeros(M, H, dtype=torch.bfloat16, device="cuda")
    torch.cuda.synchronize()
    _block(calc, t, real_tensor(out, [H, M]))
    calc.synchronize()
    raw = t["raw"]
    s = (raw["x"].float() + raw["res"].float()).cpu().double().numpy()
    assert torch.equal(raw["sum"], (raw["x"].float() + raw["res"].float()).bfloat16())
    check_codes(_norm64(s, _f64(raw["gamma"])[None], np.float64(np.float32(1e-6))), _codes_of(raw["xq"]), _f64(t["xs"]), kind, 3, _scale_roundings(H, True))
    for a, b, sa, sb, o in (("xq", "w1", "xs", "w1s", raw["gu"]), ("hq", "w2", "hs", "w2s", out)):
        va, vb = code_values(_codes_of(raw[a]), kind), code_values(_codes_of(raw[b]), kind)
        check_product(_f64(o), va @ vb.T, sums_error(va, vb, kind), _f64(t[sa]), _f64(t[sb]), None, "bf16")
    gu = _f64(raw["gu"])
    check_codes(gate64(gu[:, :F], "silu") * gu[:, F:], _codes_of(raw["hq"]), _f64(t["hs"]), kind, 12, 14)


@pytest.mark.parametrize("M", [2, 130])
def test_block_in_a_graph_and_on_another_stream(calc, M):
    """Recorded on a caller's stream after one call there, replayed with other inputs, eager calls of another size in between."""
    import torch
    c = calc
    try:
        side = torch.cuda.Stream()
        c.setStream(side.cuda_stream)
        H, F = 256, 400
        t = _block_tensors(c, M, H, F, "int8", 1)
        other = _block_tensors(c, 3 * M + 1, 2 * H, 2 * F, "int8", 2)
        out, out2 = torch.zeros(M, H, dtype=torch.bfloat16, device="cuda"), torch.zeros(3 * M + 1, 2 * H, dtype=torch.bfloat16, device="cuda")
        O, O2 = real_tensor(out, [H, M]), real_tensor(out2, [2 * H, 3 * M + 1])
        torch.cuda.synchronize()
        _block(c, t, O)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            _block(c, t, O)
        torch.cuda.synchronize()
        for k in range(4):
            t["raw"]["x"].copy_(torch.randn(M, H, device="cuda").bfloat16())
            torch.cuda.synchronize()
            out.zero_()
            t["raw"]["gu"].zero_()
            _block(c, other, O2)
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            got = out.clone()
            out.zero_()
            torch.cuda.synchronize()
            _block(c, t, O)
            c.synchronize()
            assert torch.equal(got, out), k
    finally:
        torch.cuda.synchronize()
        c.setStream(None)


FORMS = [(4, 512, 512), (70, 4000, 512), (2001, 2001, 385), (4000, 4001, 512)]  # few rows, tiles of 64, 128 and 256


def _products(seed):
    import torch
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    cases = []
    for M, N, K in FORMS:
        x, w = (torch.randint(-127, 128, (r, K), generator=g, device="cuda", dtype=torch.int8) for r in (M, N))
        out = torch.zeros(M, N, dtype=torch.int32, device="cuda")
        cases.append((x, w, out, real_tensor(out, [N, M]), code_tensor(x, [K, M], "int8"), None, code_tensor(w, [K, N], "int8"), None))
    torch.cuda.synchronize()
    return cases


def test_every_form_in_a_graph(calc):
    import torch
    cases = _products(1)
    try:
        side = torch.cuda.Stream()
        calc.setStream(side.cuda_stream)
        forms = set()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            for c in cases:
                calc.scaledGemm(*c[3:])
                forms.add(calc.lastContractionForm()["tile_rows"])
        assert forms == {8, 64, 128, 256}
        for k in range(3):
            for x, _, out, *_ in cases:
                x.add_(1)
                out.zero_()
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            for x, w, out, *_ in cases:
                assert torch.equal(out.double(), x.double() @ w.double().T), k
    finally:
        torch.cuda.synchronize()
        calc.setStream(None)


def test_two_calculators_at_once(calc):
    """Calls of two handles on two streams, enqueued in turn, share nothing."""
    import torch
    from intel_gaudi3_software_amd import HipCalculator
    second = HipCalculator()
    try:
        a, b = _products(2), _products(3)
        for _ in range(5):
            for p, q in zip(a, reversed(b)):
                calc.scaledGemm(*p[3:])
                second.scaledGemm(*q[3:])
        calc.synchronize()
        second.synchronize()
        for x, w, out, *_ in a + b:
            assert torch.equal(out.double(), x.double() @ w.double().T)
    finally:
        second.close()


def test_own_stream_waits_for_torch(calc):
    """On its own stream the calculator waits for what torch's stream has enqueued."""
    import torch
    x = torch.zeros(2000, 4096, dtype=torch.bfloat16, device="cuda")
    codes, scales = torch.zeros(2000, 4096, dtype=torch.uint8, device="cuda"), torch.zeros(2000, device="cuda")
    for k in range(3):
        x.fill_(float(k + 1))
        calc.quantizeRows(code_tensor(codes, [4096, 2000], "int8"), scales, real_tensor(x, [4096, 2000]))
        calc.synchronize()
        assert torch.all(codes == 127) and torch.all(scales == torch.tensor((k + 1) / 127, device="cuda"))


def test_refusals(calc):
    import torch
    f = lambda *s, dtype=torch.float32: torch.zeros(*s, dtype=dtype, device="cuda")
    u = lambda *s: torch.zeros(*s, dtype=torch.uint8, device="cuda")
    C8 = lambda rows=4, kind="int8", w=64: code_tensor(u(rows, w), [w, rows], kind)
    X = lambda rows=4, w=64, dt=torch.float32: real_tensor(f(rows, w, dtype=dt), [w, rows])

    def refused(call, status, word):
        with pytest.raises(MMEStackException) as e:
            call()
        assert e.value.status == status and word in str(e.value), str(e.value)

    sc = f(4)
    refused(lambda: calc.quantizeRows(C8(5), sc, X()), abi.EINVAL, "rowScales")
    refused(lambda: calc.quantizeRows(C8(4, w=32), sc, X()), abi.EINVAL, "sizes differ")
    refused(lambda: calc.quantizeRows(C8(), None, X()), abi.EINVAL, "row_scales")
    refused(lambda: calc.quantizeRows(X(), sc, X()), abi.EINVAL, "int8, fp8_143 or fp8_152")
    refused(lambda: calc.quantizeRows(C8(), sc, C8()), abi.EINVAL, "bf16, fp16 or fp32")
    refused(lambda: calc.quantizeRows(C8(), sc, X(), X(dt=torch.bfloat16)), abi.EINVAL, "type differs")
    refused(lambda: calc.quantizeRows(C8(), sc, X(), X(), 2), abi.EINVAL, "invalid gate")
    refused(lambda: calc.quantizeRows(C8().window(0, [0, 4]), sc, X().window(0, [0, 4])), abi.EINVAL, "zero elements")
    bad = MmeSimTensor([64, 4], 2, abi.FP8_143, u(4, 64), 7, abi.NO_INF_NAN)
    refused(lambda: calc.quantizeRows(bad, sc, X()), abi.EUNSUPPORTED, "full or minimal")
    bad = MmeSimTensor([64, 4], 2, abi.FP8_152, u(4, 64), 15, abi.MINIMAL_INF_NAN)
    refused(lambda: calc.quantizeRows(bad, sc, X()), abi.EUNSUPPORTED, "full inf/NaN")
    bad = MmeSimTensor([64, 4], 2, abi.FP8_143, u(4, 64), 5, abi.FULL_INF_NAN)
    refused(lambda: calc.quantizeRows(bad, sc, X()), abi.EINVAL, "exponent bias")
    bad = MmeSimTensor([64, 4], 2, abi.FP16, f(4, 64, dtype=torch.float16), 14)
    refused(lambda: calc.quantizeRows(C8(), sc, bad), abi.EUNSUPPORTED, "fp16")
    overlapping = code_tensor(u(4, 64), [256, 1], "int8").window(0, [64, 4], [1, 63, 256, 256, 256])
    refused(lambda: calc.quantizeRows(overlapping, sc, X()), abi.EINVAL, "rows overlap")
    buf = f(4, 64)
    inside = code_tensor(buf.view(torch.uint8).view(4, 256), [256, 4], "int8").window(0, [64, 4])
    refused(lambda: calc.quantizeRows(inside, sc, real_tensor(buf, [64, 4])), abi.EINVAL, "meets")
    refused(lambda: calc.rmsNormQuantize(C8(), sc, X(), eps=-1.0), abi.EINVAL, "eps")
    refused(lambda: calc.rmsNormQuantize(C8(), sc, X(), eps=float("nan")), abi.EINVAL, "eps")
    refused(lambda: calc.rmsNormQuantize(C8(), sc, X(), residualOut=X()), abi.EINVAL, "without a residual")
    refused(lambda: calc.rmsNormQuantize(C8(), sc, X(), real_tensor(f(63), [63])), abi.EINVAL, "gamma")
    refused(lambda: calc.rmsNormQuantize(C8(), sc, X(), real_tensor(f(64, dtype=torch.bfloat16), [64])), abi.EINVAL, "gamma")
    r = f(5, 64)
    whole = real_tensor(r, [64, 5])
    refused(lambda: calc.rmsNormQuantize(C8(), sc, X(), None, whole.window(0, [64, 4]), whole.window(64, [64, 4])), abi.EINVAL, "meets")

    O = lambda m=4, n=8, dt=torch.float32: real_tensor(f(m, n, dtype=dt), [n, m])
    refused(lambda: calc.scaledGemm(O(), C8(), None, C8(8, "e4m3"), None), abi.EINVAL, "int8 both")
    refused(lambda: calc.scaledGemm(O(), X(), None, X(8), None), abi.EINVAL, "int8 both")
    refused(lambda: calc.scaledGemm(O(), C8(), None, C8(8, w=32), None), abi.EINVAL, "Common dim")
    refused(lambda: calc.scaledGemm(O(n=9), C8(), None, C8(8), None), abi.EINVAL, "output width")
    refused(lambda: calc.scaledGemm(O(m=3), C8(), None, C8(8), None), abi.EINVAL, "output height")
    refused(lambda: calc.scaledGemm(C8(4, w=8), C8(), None, C8(8), None), abi.EINVAL, "output")
    refused(lambda: calc.scaledGemm(O(dt=torch.int32), C8(), sc, C8(8), None), abi.EINVAL, "sums themselves")
    refused(lambda: calc.scaledGemm(O(dt=torch.int32), C8(4, "e4m3"), None, C8(8, "e4m3"), None), abi.EINVAL, "output")
    refused(lambda: calc.scaledGemm(O(), C8(4, "e4m3"), None, C8(8, "e4m3"), None), abi.EUNSUPPORTED, "bf16 or fp16")
    refused(lambda: calc.scaledGemm(O(), C8(), f(3), C8(8), None), abi.EINVAL, "xScales")
    refused(lambda: calc.scaledGemm(O(), C8(), sc, C8(8), f(8), f(8).double()), abi.EINVAL, "bias")
    long = u(1, 131072)
    refused(lambda: calc.scaledGemm(O(1, 1), code_tensor(long, [131072, 1], "int8"), None, code_tensor(long, [131072, 1], "int8"), None), abi.EUNSUPPORTED, "131071")
    o = f(4, 64)
    refused(lambda: calc.scaledGemm(real_tensor(o, [64, 4]).window(0, [8, 4]), code_tensor(o.view(torch.uint8).view(4, 256), [256, 4], "int8").window(0, [64, 4]), None,
                                    C8(8), None), abi.EINVAL, "meets")
    host = MmeSimTensor([64, 4], 2, abi.FP32)
    refused(lambda: calc.quantizeRows(C8(), sc, host), abi.EINVAL, "device tensors")
    refused(lambda: calc.doActivation(X(), X().window(0, [64, 4])), abi.EUNSUPPORTED, "windows")
    with pytest.raises(ValueError):
        X().window(1, [64, 4])
    # a tensor of another device, sizes that a descriptor does not hold
    away, huge = X(), X()
    away._gpu, huge._fits = calc._gpu + 1, False
    refused(lambda: calc.quantizeRows(C8(), sc, away), abi.EINVAL, "calculator's device")
    refused(lambda: calc.quantizeRows(C8(), sc, huge), abi.EINVAL, "32-bit")
    refused(lambda: calc.quantizeRows(C8(), sc.cpu(), X()), abi.EINVAL, "calculator's device")
    # (and the other entry points do not take the new types)
    refused(lambda: calc.doBatchGemm(O(), C8(), C8(8), abi.OP_ABT), abi.EINVAL, "")
    calc.synchronize()
