"""CPU checks of what ``matmul_fp8`` refuses besides wrong shapes: sizes past the
library's, which are 32-bit arguments there, and an element type that is not
that of the tensor to write."""
import numpy as np
import pytest

from onnx_b200 import _native as N
from onnx_b200 import scoring
from onnx_b200.tensor import BFLOAT16
from test_scoring import fp8, t

F16 = np.float16


@pytest.mark.parametrize("m, n, k", [(2 ** 32 + 4, 8, 16), (4, 2 ** 32 + 8, 16), (4, 8, 2 ** 32 + 16),
                                     (2 ** 30 + 1, 8, 16), (4, 2 ** 31, 16)])
def test_product_sizes_past_the_library(m, n, k):
    with pytest.raises(ValueError, match="2\\^30"):
        scoring.matmul_fp8(fp8(m, k, 1), fp8(n, k, 128), out=t((m, n)))


@pytest.mark.parametrize("dtype, held", [(np.float32, F16), (F16, np.float32), (BFLOAT16, F16), ("float32", BFLOAT16)])
def test_product_type_other_than_outs(dtype, held):
    with pytest.raises(ValueError, match="dtype"):
        scoring.matmul_fp8(fp8(4, 256, 1), fp8(8, 256, 128), dtype=dtype, out=t((4, 8), held))


@pytest.mark.parametrize("dtype, held", [(None, F16), (F16, F16), (BFLOAT16, BFLOAT16), ("float32", np.float32)])
def test_product_type_of_out(dtype, held):
    """Past the checks, to the library's own, which has no context here."""
    with pytest.raises(N.LonnxError, match="null context"):
        scoring.matmul_fp8(fp8(4, 256, 1), fp8(8, 256, 128), dtype=dtype, out=t((4, 8), held))
