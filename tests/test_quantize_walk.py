"""Which block a thread of the row quantisation reaches (csrc/quantize.cu): the
walk is followed here step by step, and the rule that gives it 32-bit indices
has to leave room for all of it; the last row counts under 2^31 on a GPU."""
import os
import re

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
GROUPS = 32  # of a CTA, 8 lanes each


def walked(total, grid, u):
    """The furthest block that any group of lanes steps to: u blocks are fetched
    ahead, a warp's four groups go on until all of them are past the end."""
    groups, furthest = grid * GROUPS, 0
    for first in range(0, groups, 4):
        at = held = first  # of the warp's first group; the others are 1 to 3 further on
        at += u * groups
        while held < total:
            held, at = at, at + u * groups
        furthest = max(furthest, at + 3)
    return furthest


def source():
    return open(os.path.join(ROOT, "onnx_b200", "csrc", "quantize.cu")).read()


def test_walk_constants():
    src = source()
    assert "static constexpr int GROUPS = 256 / LANES;" in src and "LANES = 8, NV = QB / LANES / VN;" in src
    assert "static constexpr int U = 4 / NV;" in src  # 1 for floats, 2 for 16-bit types


def test_32_bit_indices_hold_the_whole_walk():
    rule = re.search(r"const int64_t furthest = (.*);\s*if \(furthest < \(1ll << 31\)", source())
    assert rule, "the rule for 32-bit indices"
    rule = rule.group(1).replace("(int64_t)", "").replace("W::U", "u").replace("W::GROUPS", str(GROUPS))
    for u in (1, 2):
        for grid in (1, 2, 3, 7):
            for total in (1, 3, 4, 31, 32, 33, 64, 65, 1000, 4097):
                assert walked(total, grid, u) <= eval(rule, dict(total=total, grid=grid, u=u))
    # one block a row and 444 CTAs: these row counts reach past 2^31
    assert eval(rule, dict(total=2147455231, grid=444, u=2)) >= 2 ** 31


@pytest.fixture
def device_memory():
    """Given back to the device afterwards, for tests in other processes."""
    import torch
    yield
    torch.cuda.empty_cache()


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [2147426000, 2147455231, 2147483647])
def test_rows_up_to_the_last_32_bit_index(device_memory, rows):
    """One block a row in 16 bits; all but a few rows hold whatever the memory held."""
    import torch

    from onnx_b200 import _native as N
    from onnx_b200.tensor import Context
    if torch.cuda.mem_get_info()[0] < 100 << 30:
        pytest.skip("needs 60 GB of device memory")
    ctx = Context(0, stream=torch.cuda.current_stream().cuda_stream)
    cols, ld = 5, 8
    x = torch.empty(rows, ld, dtype=torch.float16, device="cuda")
    q = torch.empty(rows, ld, dtype=torch.uint8, device="cuda")
    scale = torch.empty(rows, device="cuda")
    at = [0, 1, rows // 2, rows - 14209, rows - 2, rows - 1]
    part = torch.randn(len(at), ld, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda").half()
    for i, r in enumerate(at):
        x[r] = part[i]
        q[r] = 7
    N.check(N.lib.lonnx_quantize_fp8(ctx.handle, x.data_ptr(), 10, rows, cols, ld, 1, q.data_ptr(), ld,
                                     scale.data_ptr(), 1))
    ctx.sync()
    amax = part[:, :cols].double().abs().amax(1)
    quotient = 448 * part[:, :cols].double() / amax[:, None]
    step = torch.exp2(torch.floor(torch.log2(quotient.abs().clamp_min(2.0 ** -6))) - 3)
    want = torch.round(quotient / step) * step
    for i, r in enumerate(at):
        got = q[r]
        assert torch.equal(got[:cols].view(torch.float8_e4m3fn).double(), want[i])
        assert (got[cols:] == 7).all()
        assert float(scale[r]) == float(np.float32(amax[i].item()) / np.float32(448))
