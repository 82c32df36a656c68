"""8-bit linear layer without a GPU: which kernel form the planner picks, that it stays inside what the kernels assume, and every
refusal (the real calls go through the same checks)."""
import os
import subprocess

import numpy as np
import pytest

from intel_gaudi3_software_amd import MmeSimTensor, abi

MIB = 1 << 20


@pytest.fixture(autouse=True)
def _library():
    if not os.path.exists(abi.LIB_PATH):
        pytest.skip("libmme_hip.so has not been built (python -m intel_gaudi3_software_amd.build)")


def T(at, sizes, dtype, bias=0, mode=0, strides=None):
    """A descriptor at `at` MiB."""
    t = abi.make_tensor(at * MIB, sizes, dtype, bias, mode, None, dim=5)
    if strides is not None:
        for d in range(5):
            t.strides[d] = strides[d] if d < len(strides) else t.strides[d]
    return t


def product(M, N, K, out=abi.BF16, dtype=abi.INT8, batch=1, **kw):
    bias, mode = {abi.INT8: (0, 0), abi.FP8_143: (7, abi.MINIMAL_INF_NAN), abi.FP8_152: (15, 0)}[dtype]
    o, x, w = T(4096, [N, M, batch], out), T(1, [K, M, batch], dtype, bias, mode), T(2048, [K, N, batch], dtype, bias, mode)
    return abi.plan_scaled_gemm(o, x, w, **kw)


def test_forms_of_the_product():
    # one token, sixteen: the few-rows form with as many rows of x as needed
    assert product(1, 4096, 4096) == {"large_tile": 3, "tile_rows": 8, "split_k": 1, "wavefronts": 8}
    assert product(16, 14336, 4096, dtype=abi.FP8_143) == {"large_tile": 3, "tile_rows": 16, "split_k": 1, "wavefronts": 4}
    # few outputs in all keep it at any number of rows
    assert product(64, 1024, 16384)["large_tile"] == 3 and product(100, 512, 16384)["tile_rows"] == 32
    # more outputs: 64 x 64, 128 x 128, 256 x 256
    assert product(250, 4096, 14336) == {"large_tile": 1, "tile_rows": 64, "split_k": 1, "wavefronts": 8}
    assert product(1024, 4096, 4096)["tile_rows"] == 128
    assert product(4096, 4096, 4096)["tile_rows"] == 256 and product(2048, 14336, 4096, batch=4, dtype=abi.FP8_152)["tile_rows"] == 256
    # rows that do not start at multiples of 16 bytes, and short reductions, stay with the forms that take them
    assert product(4096, 4096, 4095)["tile_rows"] == 128 and product(4096, 4096, 128)["tile_rows"] < 256
    assert product(5, 0, 64)["large_tile"] == -1


def test_planned_products_respect_what_the_kernels_assume():
    """256 x 256 tiles: aligned rows and four whole stages of 64; 32 rows of x or fewer never leave the few-rows form; an unaligned
    operand never meets a direct copy (the few-rows form then has 16 rows of w, which the planner's wavefronts show)."""
    rng = np.random.default_rng(7)
    seen = set()
    for _ in range(3000):
        M, N, K = (int(np.exp(rng.uniform(0, np.log(16384)))) for _ in range(3))
        if rng.random() < 0.6:
            K = max(16, K // 16 * 16)
        f = product(M, N, K)
        seen.add((f["large_tile"], f["tile_rows"], f["wavefronts"]))
        assert f["split_k"] == 1
        if M <= 32:
            assert f["large_tile"] == 3 and f["tile_rows"] == (8 if M <= 8 else 16 if M <= 16 else 32)
        if f["tile_rows"] == 256:
            assert K >= 256 and K % 16 == 0
        if K % 16 and f["large_tile"] == 3 and N > 1 and M > 1:
            assert f["wavefronts"] == 8
    assert {s[1] for s in seen} == {8, 16, 32, 64, 128, 256}


def rows(width, n=5, out=abi.INT8, dtype=abi.BF16, **kw):
    mode = abi.MINIMAL_INF_NAN if out == abi.FP8_143 else 0
    return abi.plan_quantize_rows(T(2048, [width, n], out, {abi.FP8_143: 7, abi.FP8_152: 15}.get(out, 0), mode), 4096 * MIB, T(1, [width, n], dtype, 15 if dtype == abi.FP16 else 0), **kw)


def test_forms_of_the_row_quantisers():
    assert rows(64) == {"lanes": 16, "elements": 8, "rows_per_group": 16, "one_pitch": 1}
    assert rows(4096) == {"lanes": 512, "elements": 8, "rows_per_group": 1, "one_pitch": 1}
    assert rows(14336, 8192) == {"lanes": 448, "elements": 32, "rows_per_group": 1, "one_pitch": 1}
    assert rows(14336, 16)["elements"] == 16 and rows(14336, 8192, dtype=abi.FP32)["elements"] == 16
    n = abi.plan_rms_norm_quantize(T(2048, [14336, 8192], abi.INT8), 4096 * MIB, T(1, [14336, 8192], abi.BF16))
    assert n["elements"] == 16 and n["lanes"] == 896
    for width in list(range(1, 1200)) + [4095, 4096, 4097, 8191, 8192, 8193, 16383, 16384, 16385, 200000]:
        for many in (1, 1000):
            f = rows(width, many)
            # every element has a lane, no workgroup is over 1024 lanes, a lane's share is whole
            assert f["elements"] == 0 or f["lanes"] * f["elements"] >= width
            assert f["lanes"] * f["rows_per_group"] <= 1024 and (f["rows_per_group"] > 1 or f["lanes"] % 64 == 0)
            assert f["elements"] in (0, 8, 16, 32) and (f["elements"] != 8 or f["lanes"] <= 512) and (f["elements"] != 32 or f["lanes"] <= 512)


def test_pitches():
    """One pitch for all rows only where the dimensions' strides allow it for every tensor."""
    sizes = [64, 3, 4]
    o = lambda st=None: T(2048, sizes, abi.INT8, strides=st)
    x = lambda st=None: T(1, sizes, abi.BF16, strides=st)
    plan = lambda a, b: abi.plan_quantize_rows(a, 4096 * MIB, b)["one_pitch"]
    assert plan(o(), x()) == 1 and plan(o(), x([1, 100, 300, 1200, 1200])) == 1
    assert plan(o(), x([1, 100, 301, 1204, 1204])) == 0 and plan(o([1, 64, 200, 800, 800]), x()) == 0
    assert plan(o(), x([1, 0, 64, 256, 256])) == 0


def refused(word, call, *args, **kw):
    with pytest.raises(ValueError) as e:
        call(*args, **kw)
    assert word in str(e.value), str(e.value)


def test_refusals_of_the_quantisers():
    S = 4096 * MIB
    x, o = T(1, [64, 4], abi.FP32), T(64, [64, 4], abi.INT8)
    q, n = abi.plan_quantize_rows, abi.plan_rms_norm_quantize
    q(o, S, x), n(o, S, x)
    refused("got null pointer", q, None, S, x)
    refused("got null pointer", q, o, S, None)
    refused("got null pointer", q, o, None, x)
    refused("got null pointer", q, T(0, [64, 4], abi.INT8), S, x)
    refused("not aligned", q, o, S + 2, x)
    odd = T(1, [64, 4], abi.FP32)
    odd.data = MIB + 2
    refused("not aligned", q, o, S, odd)
    refused("type not supported", q, o, S, T(1, [64, 4], abi.TF32))
    refused("type not supported", q, T(64, [64, 4], 99), S, x)
    refused("int8, fp8_143 or fp8_152", q, T(64, [64, 4], abi.BF16), S, x)
    refused("bf16, fp16 or fp32", q, o, S, T(1, [64, 4], abi.INT32))
    refused("sizes differ", q, T(64, [64, 5], abi.INT8), S, x)
    refused("zero elements", q, T(64, [0, 4], abi.INT8), S, T(1, [0, 4], abi.FP32))
    assert q(T(64, [64, 0], abi.INT8), S, T(1, [64, 0], abi.FP32))["lanes"] == -1
    refused("2^31", q, T(64, [1 << 16, 1 << 15], abi.INT8), S, T(8192, [1 << 16, 1 << 15], abi.FP32))
    refused("2^31", q, T(64, [1 << 31, 1 << 31, 1 << 31, 1 << 31, 1 << 31], abi.INT8), S, x)
    refused("one launch", q, T(8192, [1, (1 << 28) + 1], abi.INT8), 16384 * MIB, T(1, [1, (1 << 28) + 1], abi.FP32))
    assert q(T(8192, [1, (1 << 28) - 16], abi.INT8), 16384 * MIB, T(1, [1, (1 << 28) - 16], abi.FP32))["lanes"] == 16
    refused("contiguous", q, o, S, T(1, [64, 4], abi.FP32, strides=[2, 128]))
    refused("rows overlap", q, T(64, [64, 4], abi.INT8, strides=[1, 63]), S, x)
    refused("rows overlap", q, T(64, [64, 4, 2], abi.INT8, strides=[1, 128, 63]), S, T(1, [64, 4, 2], abi.FP32))
    # (rows of two dimensions may lie between each other)
    assert q(T(64, [64, 4, 2], abi.INT8, strides=[1, 128, 64]), S, T(1, [64, 4, 2], abi.FP32))["lanes"] == 16
    refused("exponent bias", q, T(64, [64, 4], abi.FP8_143, 6), S, x)
    refused("exponent bias", q, T(64, [64, 4], abi.FP8_152, 31), S, x)
    refused("infNanMode", q, T(64, [64, 4], abi.FP8_143, 7, 3), S, x)
    refused("full or minimal", q, T(64, [64, 4], abi.FP8_143, 7, abi.NO_INF_NAN), S, x)
    refused("full inf/NaN", q, T(64, [64, 4], abi.FP8_152, 15, abi.MINIMAL_INF_NAN), S, x)
    refused("fp16", q, o, S, T(1, [64, 4], abi.FP16, 14))
    refused("fp16", q, o, S, T(1, [64, 4], abi.FP16, 15, abi.NO_INF_NAN))
    refused("invalid gate", q, o, S, x, T(32, [64, 4], abi.FP32), 2)
    refused("type differs", q, o, S, x, T(32, [64, 4], abi.BF16))
    refused("sizes differ", q, o, S, x, T(32, [64, 3], abi.FP32))
    # outputs that meet inputs: the codes on x, the scales on x's last bytes, the codes on the gate
    refused("meets", q, T(1, [64, 4], abi.INT8), S, x)
    refused("meets", q, o, MIB + 64 * 4 * 4 - 4, x)
    assert q(o, MIB + 64 * 4 * 4, x)["lanes"] == 16
    refused("meets", q, o, S, x, T(64, [64, 4], abi.FP32))
    refused("meets", q, o, 64 * MIB + 252, x)
    # the norm's own
    refused("eps", n, o, S, x, eps=-1e-9)
    refused("eps", n, o, S, x, eps=float("inf"))
    refused("eps", n, o, S, x, eps=float("nan"))
    refused("without a residual", n, o, S, x, residual_out=T(32, [64, 4], abi.FP32))
    refused("gamma", n, o, S, x, T(32, [63], abi.FP32))
    refused("gamma", n, o, S, x, T(32, [64, 4], abi.FP32))
    refused("gamma", n, o, S, x, T(32, [64], abi.BF16))
    r = T(32, [64, 4], abi.FP32)
    for same in (x, r):  # in place is allowed for the very same tensor only
        assert n(o, S, x, residual=r, residual_out=same)["lanes"] == 16
    shifted = T(32, [64, 4], abi.FP32)
    shifted.data = 32 * MIB + 4
    refused("meets", n, o, S, x, residual=r, residual_out=shifted)
    refused("rows overlap", n, o, S, x, residual=r, residual_out=T(40, [64, 4], abi.FP32, strides=[1, 0]))
    refused("meets", n, o, S, x, residual=r, residual_out=T(64, [64, 4], abi.FP32))
    refused("meets", n, o, S, x, T(48, [64], abi.FP32), residual=r, residual_out=T(48, [64, 4], abi.FP32))


def test_refusals_of_the_product():
    g = abi.plan_scaled_gemm
    o, x, w = T(4096, [8, 4], abi.BF16), T(1, [64, 4], abi.INT8), T(2048, [64, 8], abi.INT8)
    e4 = lambda at, s, mode=abi.MINIMAL_INF_NAN, bias=7: T(at, s, abi.FP8_143, bias, mode)
    e5 = lambda at, s, mode=0, bias=15: T(at, s, abi.FP8_152, bias, mode)
    assert g(o, x, w)["large_tile"] == 3 and g(o, e4(1, [64, 4]), e5(2048, [64, 8]))["large_tile"] == 3
    assert g(T(4096, [8, 4], abi.INT32), x, w)["large_tile"] == 3
    refused("int8 both", g, o, x, e4(2048, [64, 8]))
    refused("int8 both", g, o, T(1, [64, 4], abi.BF16), T(2048, [64, 8], abi.BF16))
    refused("output", g, T(4096, [8, 4], abi.INT8), x, w)
    refused("output", g, T(4096, [8, 4], abi.INT32), e4(1, [64, 4]), e4(2048, [64, 8]))
    refused("bf16 or fp16", g, T(4096, [8, 4], abi.FP32), e4(1, [64, 4]), e4(2048, [64, 8]))
    refused("fp16", g, T(4096, [8, 4], abi.FP16, 14), x, w)
    refused("Common dim", g, o, x, T(2048, [65, 8], abi.INT8))
    refused("output width", g, T(4096, [9, 4], abi.BF16), x, w)
    refused("output height", g, T(4096, [8, 5], abi.BF16), x, w)
    refused("batch dims", g, T(4096, [8, 4, 2], abi.BF16), T(1, [64, 4, 3], abi.INT8), w)
    assert g(T(4096, [8, 4, 2], abi.BF16), T(1, [64, 4, 2], abi.INT8), w)["large_tile"] == 3
    refused("65535", g, T(4096, [1, 1, 65536], abi.BF16), T(1, [16, 1, 65536], abi.INT8), T(2048, [16, 1], abi.INT8))
    refused("131071", g, T(4096, [1, 1], abi.BF16), T(1, [131072, 1], abi.INT8), T(2048, [131072, 1], abi.INT8))
    assert g(T(4096, [1, 1], abi.BF16), T(1, [131071, 1], abi.INT8), T(2048, [131071, 1], abi.INT8))["large_tile"] == 3
    long = (1 << 30) + 1
    refused("2^30", g, T(4096, [1, 1], abi.BF16), e4(1, [long, 1]), e4(2048, [long, 1]))
    assert g(T(4096, [1, 1], abi.BF16), e4(1, [long - 1, 1]), e4(2048, [long - 1, 1]))["large_tile"] == 3
    wide = (1 << 27) + 1
    refused("one launch", g, T(4096, [wide, 1], abi.BF16), T(1, [1, 1], abi.INT8), T(2048, [1, wide], abi.INT8))
    assert g(T(4096, [wide - 17, 1], abi.BF16), T(1, [1, 1], abi.INT8), T(2048, [1, wide - 17], abi.INT8))["large_tile"] == 3
    refused("rows overlap", g, T(4096, [8, 4], abi.BF16, strides=[1, 7]), x, w)
    refused("exponent bias", g, o, e4(1, [64, 4], bias=8), e4(2048, [64, 8]))
    for a, b in ((e4(1, [64, 4], 0), e4(2048, [64, 8])), (e4(1, [64, 4]), e5(2048, [64, 8], 1)), (e4(1, [64, 4], 1), e4(2048, [64, 8]))):
        refused("ASSUME_NONE", g, o, a, b)
        assert g(o, a, b, fp8_specials_policy=abi.FP8_SPECIALS_ASSUME_NONE)["large_tile"] == 3
    # nothing to do is no error
    assert g(T(4096, [8, 0], abi.BF16), T(1, [64, 0], abi.INT8), w)["large_tile"] == -1
    assert g(o, T(1, [0, 4], abi.INT8), T(2048, [0, 8], abi.INT8))["large_tile"] == 3
    # the other entry points do not take the new types
    with pytest.raises(ValueError):
        abi.plan_batch_gemm(T(4096, [8, 4], abi.FP32), x, w, abi.OP_ABT)


def test_windows():
    t = MmeSimTensor([20, 3], 2, abi.FP32)
    w = t.window(10, [10, 3])
    assert w.desc.data == t.desc.data + 40 and list(w.desc.strides)[:2] == [1, 20] and w.getSizes()[:2] == [10, 3]
    assert w.window(3, [7, 3]).desc.data == t.desc.data + 52
    assert list(t.window(0, [20, 9], [1, 0, 0, 0, 0]).desc.strides) == [1, 0, 0, 0, 0]
    for bad in ((11, [10, 3]), (0, [20, 4]), (-1, [10, 3])):
        with pytest.raises(ValueError):
            t.window(*bad)
    with pytest.raises(ValueError):
        w.window(3, [8, 3])


def test_cpp_surface():
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    exe = os.path.join(root, "tests", "cpp", "linear8_calculator")
    if not os.path.exists(exe):  # (host code only: g++ over the header, two seconds)
        from intel_gaudi3_software_amd import build
        build.build_cpp_tests()
    r = subprocess.run([exe], stdout=subprocess.PIPE, stderr=subprocess.STDOUT, timeout=60)
    text = r.stdout.decode(errors="replace")
    assert r.returncode == 0 and "all ok" in text, text


def test_windows():
    """Part of a buffer, inside it, with strides that a descriptor holds (on host memory: a window is a descriptor)."""
    t = MmeSimTensor([16, 8], 2, abi.FP32)
    w = t.window(20, [4, 3])
    assert list(w.desc.sizes) == [4, 3, 1, 1, 1] and w.desc.strides[1] == 16 and w.desc.data == t.desc.data + 80
    assert t.window(0, [16, 5], [1, 0]).desc.strides[1] == 0 and t.window(64, [16, 4]).window(16, [16, 3]).desc.data == t.desc.data + 320
    assert t.window(0, [16, 1], [1, 1 << 40]).sizes[1] == 1  # (the stride of a single row is never used)
    for offset, sizes, strides in ((0, [16, 9], None), (-1, [4, 3], None), (1, [16, 8], None), (64, [4, 3], [1, -16]), (0, [4, 2], [1, 1 << 32]), (0, [-1, 2], None),
                                   (0, [1 << 32, 0], None)):
        with pytest.raises(ValueError):
            t.window(offset, sizes, strides)
    long = MmeSimTensor([16, 8], 2, abi.FP32, np.zeros(128, np.float32), strides=[1, -16])
    assert not long._fits and t._fits
