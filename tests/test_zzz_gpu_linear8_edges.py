"""8-bit linear layer on the GPU: the widest rows, and other calls at the edges of what the entry points take."""
import numpy as np
import pytest

from intel_gaudi3_software_amd import abi
from linear8_helpers import CODES, U, check_codes, code_tensor, code_values, real_tensor

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
