"""The measured cases of the 8-bit linear layer: rms_norm_quantize, quantize_rows and scaled_gemm.

A language model's linear layer in 8 bits goes: normalise a token's activations (with the residual's addition) and write them as
8-bit codes with one scale per token; multiply codes by codes; scale the sums back per token and output channel.  The input of the
second half of a feed-forward block is a gated product that is quantised the same way, and the weights are quantised once, a scale
per output channel.  No backward pass: these are the operators of serving.

``run`` computes an operator in elementary torch operations, or, where ``own`` is set, through ``HipCalculator``.  8-bit codes are
returned as the values they stand for (fp8 codes viewed as such, int8 codes as bf16, which holds every one of them), the
scales beside them."""
import math

import torch

own = False

# int8: 127; fp8_143 in minimal inf/NaN mode (bias 7) and fp8_152 (bias 15): their largest finite values
QMAX = {"int8": 127.0, "fp8_143": 448.0, "fp8_152": 57344.0}
CODE = {"int8": torch.int8, "fp8_143": torch.float8_e4m3fn, "fp8_152": torch.float8_e5m2}
FLOAT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"int8": 1, "fp8_143": 1, "fp8_152": 1, "bf16": 2, "fp16": 2, "fp32": 4, "int32": 4}
EPS = 1e-6


def listed():
    return [
        # norm: the tokens of sixteen sequences that each produce one token; a long prompt; ragged rows of an odd width
        {"name": "norm of 16 tokens", "op": "norm", "rows": 16, "width": 4096, "type": "bf16", "out": "int8", "residual": True},
        {"name": "norm of a long prompt", "op": "norm", "rows": 8192, "width": 4096, "type": "bf16", "out": "fp8_143", "residual": True},
        {"name": "norm of an odd width", "op": "norm", "rows": 1111, "width": 5001, "type": "fp16", "out": "fp8_152", "residual": False},
        # rows: gate and up halves of one projection's output on their way to the down projection (few tokens, a long prompt); weights,
        # quantised once per output channel
        {"name": "gated rows of 16 tokens", "op": "rows", "rows": 16, "width": 14336, "type": "bf16", "out": "fp8_143", "gate": "silu"},
        {"name": "gated rows of a long prompt", "op": "rows", "rows": 8192, "width": 14336, "type": "bf16", "out": "fp8_143", "gate": "silu"},
        {"name": "rows of a weight matrix", "op": "rows", "rows": 14336, "width": 4096, "type": "fp32", "out": "int8", "gate": ""},
        # product: one token; sixteen tokens; a ragged chunk of a prompt with a bias; an odd slice of a vocabulary for a few tokens; a
        # prompt; four groups of tokens with weights of their own (8-bit floats of both flavours)
        {"name": "product for one token", "op": "product", "batch": 1, "m": 1, "n": 4096, "k": 4096, "a": "int8", "b": "int8", "out": "bf16", "bias": False},
        {"name": "product for 16 tokens", "op": "product", "batch": 1, "m": 16, "n": 14336, "k": 4096, "a": "fp8_143", "b": "fp8_143", "out": "bf16", "bias": False},
        {"name": "product for a chunk", "op": "product", "batch": 1, "m": 250, "n": 4096, "k": 14336, "a": "int8", "b": "int8", "out": "fp16", "bias": True},
        {"name": "product of odd sizes", "op": "product", "batch": 1, "m": 33, "n": 10007, "k": 1555, "a": "int8", "b": "int8", "out": "fp32", "bias": False},
        {"name": "product for a prompt", "op": "product", "batch": 1, "m": 4096, "n": 4096, "k": 4096, "a": "int8", "b": "int8", "out": "bf16", "bias": True},
        {"name": "product for four groups", "op": "product", "batch": 4, "m": 2048, "n": 14336, "k": 4096, "a": "fp8_143", "b": "fp8_152", "out": "bf16", "bias": False},
    ]


MOST_MACS = 4 * 2048 * 14336 * 4096  # of the largest listed product
MOST_CELLS = 8192 * 14336            # of the largest listed matrix of rows


def _size(rng, low, high, step=1):
    return max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high))) / step)) * step)


def draw(rng):
    op = rng.choice(["norm", "rows", "product", "product"])
    if op == "product":
        batch = rng.choice([1, 1, 1, 2, 3])
        n, k = (_size(rng, 64, 16384, s) for s in (rng.choice([1, 16, 64]), rng.choice([1, 16, 16, 64])))
        m = _size(rng, 1, max(1, min(8192, MOST_MACS // (batch * n * k))))
        a = rng.choice(["int8", "int8", "fp8_143", "fp8_152"])
        b = "int8" if a == "int8" else rng.choice(["fp8_143", "fp8_152"])
        out = rng.choice(["bf16", "bf16", "fp16"] + (["fp32", "int32"] if a == "int8" else []))
        return {"op": op, "batch": batch, "m": m, "n": n, "k": k, "a": a, "b": b, "out": out, "bias": out != "int32" and rng.random() < 0.5}
    width = _size(rng, 64, 16384, rng.choice([1, 8, 64]))
    case = {"op": op, "rows": _size(rng, 1, min(16384, MOST_CELLS // width)), "width": width, "type": rng.choice(["bf16", "bf16", "fp16", "fp32"]),
            "out": rng.choice(["int8", "fp8_143", "fp8_143", "fp8_152"])}
    if op == "norm":
        case["residual"] = rng.random() < 0.7
    else:
        case["gate"] = rng.choice(["", "silu", "silu", "gelu"])
    return case


def work(case):
    """Each input read once, each output written once."""
    if case["op"] == "product":
        c, m, n, k = case["batch"], case["m"], case["n"], case["k"]
        scales = 0 if case["out"] == "int32" else 4 * c * (m + n + (n if case["bias"] else 0))
        return {"bytes": c * (m * k + n * k + m * n * SIZE[case["out"]]) + scales, "flops": 2 * c * m * n * k}
    r, w, s = case["rows"], case["width"], SIZE[case["type"]]
    if case["op"] == "norm":
        return {"bytes": r * w * (s * (3 if case["residual"] else 1) + 1) + w * s + 4 * r, "flops": r * w * 6}
    return {"bytes": r * w * (s * (2 if case["gate"] else 1) + 1) + 4 * r, "flops": r * w * (12 if case["gate"] else 3)}


def _values(case, seed):
    """The inputs, on the GPU, from the seed alone."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def normal(*shape, std=1.0):
        return torch.randn(*shape, generator=g, device="cuda") * std

    if case["op"] == "product":
        c, m, n, k = case["batch"], case["m"], case["n"], case["k"]

        def codes(kind, *shape):  # what a quantiser makes of normal values: the largest of a row is the type's largest
            if kind == "int8":
                return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float16).mul_(32.0).round_().clamp_(-127, 127).to(torch.int8)
            return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float16).mul_(QMAX[kind] / 4).clamp_(-QMAX[kind], QMAX[kind]).to(CODE[kind])

        v = {"x": codes(case["a"], c, m, k), "w": codes(case["b"], c, n, k), "sx": None, "sw": None, "bias": None}
        if case["out"] != "int32":
            # scales of rows whose largest magnitudes lie within a factor of four
            v["sx"] = torch.exp(normal(c, m, std=0.3)) * (4.0 / QMAX[case["a"]])
            v["sw"] = torch.exp(normal(c, n, std=0.3)) * (4.0 / QMAX[case["b"]] / math.sqrt(k))
        if case["bias"]:
            v["bias"] = normal(c, n)
        return v
    t, r, w = FLOAT[case["type"]], case["rows"], case["width"]
    spread = torch.exp(normal(w, std=0.5))  # a few channels are larger than the rest
    if case["op"] == "norm":
        return {"x": (normal(r, w) * spread).to(t), "residual": normal(r, w, std=2.0).to(t) if case["residual"] else None,
                "gamma": (1.0 + normal(w, std=0.2)).to(t)}
    if case["gate"]:  # the gate half and the up half of one projection's output, side by side in its rows
        both = normal(r, 2 * w).to(t)
        return {"both": both, "gate": both[:, :w], "x": both[:, w:]}
    return {"both": None, "gate": None, "x": (normal(r, w) * spread).to(t)}


_kept = {}


def _calculator():
    """The program's calculator, on a stream of its own."""
    if not _kept:
        from intel_gaudi3_software_amd import HipCalculator
        _kept["stream"] = torch.cuda.Stream()
        _kept["calc"] = HipCalculator()
        _kept["calc"].setStream(_kept["stream"].cuda_stream)
    return _kept["calc"]


def prepare(case, seed):
    s = {"case": dict(case), **_values(case, seed)}
    if own:
        _describe(s)
        torch.cuda.synchronize()  # the calculator's stream does not wait for torch's
    return s


def _describe(s):
    """Output buffers and the calculator's descriptors of all tensors: what a program that runs a layer again and again keeps."""
    from intel_gaudi3_software_amd import MmeSimTensor, abi
    case, device = s["case"], "cuda"
    _calculator()
    code = {"int8": (abi.INT8, 0, abi.FULL_INF_NAN), "fp8_143": (abi.FP8_143, 7, abi.MINIMAL_INF_NAN), "fp8_152": (abi.FP8_152, 15, abi.FULL_INF_NAN)}
    real = {"bf16": (abi.BF16, 0), "fp16": (abi.FP16, 15), "fp32": (abi.FP32, 0), "int32": (abi.INT32, 0)}
    if case["op"] == "product":
        c, m, n, k = case["batch"], case["m"], case["n"], case["k"]
        s["out"] = torch.empty(c, m, n, dtype=torch.int32 if case["out"] == "int32" else FLOAT[case["out"]], device=device)
        t, bias = real[case["out"]]
        s["out_t"] = MmeSimTensor([n, m, c], 3, t, s["out"], bias)
        for name, kind, rows in (("x", case["a"], m), ("w", case["b"], n)):
            t, bias, mode = code[kind]
            s[name + "_t"] = MmeSimTensor([k, rows, c], 3, t, s[name], bias, mode)
        return
    r, w = case["rows"], case["width"]
    s["codes"] = torch.empty(r, w, dtype=CODE[case["out"]], device=device)
    s["scales"] = torch.empty(r, dtype=torch.float32, device=device)
    t, bias, mode = code[case["out"]]
    s["codes_t"] = MmeSimTensor([w, r], 2, t, s["codes"], bias, mode)
    t, bias = real[case["type"]]
    if case["op"] == "norm":
        s["x_t"] = MmeSimTensor([w, r], 2, t, s["x"], bias)
        s["gamma_t"] = MmeSimTensor([w], 1, t, s["gamma"], bias)
        s["residual_t"] = s["sum_t"] = s["sum"] = None
        if case["residual"]:
            s["sum"] = torch.empty_like(s["x"])
            s["residual_t"] = MmeSimTensor([w, r], 2, t, s["residual"], bias)
            s["sum_t"] = MmeSimTensor([w, r], 2, t, s["sum"], bias)
    elif case["gate"]:
        both = MmeSimTensor([2 * w, r], 2, t, s["both"], bias)
        s["gate_t"], s["x_t"] = both.window(0, [w, r]), both.window(w, [w, r])
        s["gate_op"] = {"silu": abi.GATE_SILU, "gelu": abi.GATE_GELU_TANH}[case["gate"]]
    else:
        s["gate_t"], s["x_t"], s["gate_op"] = None, MmeSimTensor([w, r], 2, t, s["x"], bias), abi.GATE_SILU


def _own(s):
    calc, case = _calculator(), s["case"]
    if case["op"] == "product":
        calc.scaledGemm(s["out_t"], s["x_t"], s["sx"], s["w_t"], s["sw"], s["bias"])
        return {"out": s["out"]}
    if case["op"] == "norm":
        calc.rmsNormQuantize(s["codes_t"], s["scales"], s["x_t"], s["gamma_t"], s["residual_t"], s["sum_t"], EPS)
    else:
        calc.quantizeRows(s["codes_t"], s["scales"], s["x_t"], s["gate_t"], s["gate_op"])
    codes = s["codes"]
    if case["out"] == "int8":
        with torch.cuda.stream(_kept["stream"]):
            codes = codes.to(torch.bfloat16)
    out = {"codes": codes, "scales": s["scales"]}
    if case.get("residual"):
        out["sum"] = s["sum"]
    return out


def _gate(g, kind, dtype):
    g = g.to(dtype)
    if kind == "silu":
        return g / (1.0 + torch.exp(-g))
    return 0.5 * g * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (g + 0.044715 * g * g * g)))


def _quantised(v, kind):
    """Codes of rows of values, and their scales: the largest magnitude of a row gets the type's largest code."""
    top = v.abs().amax(-1, keepdim=True)
    scale = top / QMAX[kind]
    q = v / torch.where(top > 0, scale, torch.ones_like(scale))
    if kind == "int8":
        return torch.round(q).clamp_(-127, 127).to(torch.bfloat16), scale[:, 0]
    return q.clamp_(-QMAX[kind], QMAX[kind]).to(torch.float32).to(CODE[kind]), scale[:, 0]


def run(s):
    if own:
        return _own(s)
    case = s["case"]
    if case["op"] == "product":
        if case["out"] == "int32":  # whole sums: 64 bits hold them
            return {"out": torch.matmul(s["x"].double(), s["w"].double().transpose(1, 2)).to(torch.int32)}
        out = torch.matmul(s["x"].float(), s["w"].float().transpose(1, 2))
        out = out * s["sx"][:, :, None] * s["sw"][:, None, :]
        if case["bias"]:
            out = out + s["bias"][:, None, :]
        return {"out": out.to(FLOAT[case["out"]])}
    x, out = s["x"].float(), {}
    if case["op"] == "norm":
        if case["residual"]:
            x = x + s["residual"].float()
            out["sum"] = x.to(FLOAT[case["type"]])
        v = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * s["gamma"].float()
    else:
        v = _gate(s["gate"], case["gate"], torch.float32) * x if case["gate"] else x
    out["codes"], out["scales"] = _quantised(v, case["out"])
    return out


def _nearest_code(q, kind):
    """The value of the code nearest to q (ties to the code with an even last bit), in 64 bits."""
    if kind == "int8":
        return torch.round(q)
    mantissa, lowest = {"fp8_143": (3, -6), "fp8_152": (2, -14)}[kind]
    step = torch.exp2(torch.clamp(torch.frexp(q)[1] - 1, min=lowest).double() - mantissa)
    return torch.round(q / step) * step


def exact(case, seed):
    """The same from the definitions, in 64 bits: products of the codes' values; codes as the nearest value of their type."""
    v = _values(case, seed)
    if case["op"] == "product":
        sums = torch.stack([v["x"][c].double() @ v["w"][c].double().t() for c in range(case["batch"])])
        if case["out"] == "int32":
            return {"out": sums.round().to(torch.int64)}
        sums *= v["sx"].double()[:, :, None]
        sums *= v["sw"].double()[:, None, :]
        if case["bias"]:
            sums += v["bias"].double()[:, None, :]
        return {"out": sums}
    y, out = v["x"].double(), {}
    if case["op"] == "norm":
        if case["residual"]:
            y = y + v["residual"].double()
            out["sum"] = y
        y = y * v["gamma"].double() / torch.sqrt(torch.sum(y * y, -1, keepdim=True) / case["width"] + EPS)
    elif case["gate"]:
        y = y * _gate(v["gate"], case["gate"], torch.float64)
    largest = torch.max(torch.abs(y), -1).values
    out["scales"] = largest / QMAX[case["out"]]
    out["codes"] = _nearest_code(y * (QMAX[case["out"]] / largest)[:, None], case["out"])
    return out
