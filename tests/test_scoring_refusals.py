"""CPU checks of what ``matmul_fp8`` refuses besides wrong shapes: sizes past the
library's, which are 32-bit arguments there."""
import pytest

from onnx_b200 import scoring
from test_scoring import fp8, t


@pytest.mark.parametrize("m, n, k", [(2 ** 32 + 4, 8, 16), (4, 2 ** 32 + 8, 16), (4, 8, 2 ** 32 + 16),
                                     (2 ** 30 + 1, 8, 16), (4, 2 ** 31, 16)])
def test_product_sizes_past_the_library(m, n, k):
    with pytest.raises(ValueError, match="2\\^30"):
        scoring.matmul_fp8(fp8(m, k, 1), fp8(n, k, 128), out=t((m, n)))
