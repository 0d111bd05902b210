"""CPU checks of the scoring operators' argument handling: the Python calls
refuse wrong types, shapes and options before the library sees them, and the
C entry points refuse bad arguments before they look at their context."""
import numpy as np
import pytest

from onnx_b200 import _native as N
from onnx_b200 import scoring
from onnx_b200.tensor import BFLOAT16, FLOAT8E4M3, ONNX_DTYPE, DeviceTensor

F32, I64 = np.float32, np.int64
BADARG, SHAPE, UNSUPPORTED = -1, -2, -7


class FakeContext:
    device, stream, handle = 0, 7, None


CTX = FakeContext()


def t(shape, dtype=F32, ctx=CTX, ptr=4096):
    return DeviceTensor(ctx, shape, dtype, ptr=ptr)


def fp8(rows, cols, block_rows, ld=None, scale=None):
    return scoring.Fp8Matrix(t((rows, ld or -(-cols // 16) * 16), FLOAT8E4M3),
                             t(scale or (-(-rows // block_rows), -(-cols // 128))), cols, block_rows)


def test_type_tags_are_distinct():
    assert BFLOAT16 != np.uint16 and FLOAT8E4M3 != np.uint8
    assert (BFLOAT16.itemsize, FLOAT8E4M3.itemsize) == (2, 1)
    assert (ONNX_DTYPE[BFLOAT16], ONNX_DTYPE[FLOAT8E4M3], ONNX_DTYPE[np.dtype(np.uint8)]) == (16, 17, 2)


@pytest.mark.parametrize("call", [
    lambda: scoring.quantize_fp8(t((4, 4), I64)),
    lambda: scoring.quantize_fp8(t((4,))),
    lambda: scoring.quantize_fp8(t((4, 4)), block_rows=64),
    lambda: scoring.quantize_fp8(t((4, 200)), out=(t((4, 200), FLOAT8E4M3), t((4, 1)))),
    lambda: scoring.quantize_fp8(t((4, 200)), out=(t((4, 199), FLOAT8E4M3), t((4, 2)))),
    lambda: scoring.quantize_fp8(t((4, 200)), out=(t((4, 200), np.uint8), t((4, 2)))),
    lambda: scoring.matmul_fp8(fp8(4, 256, 128), fp8(8, 256, 128), out=t((4, 8))),
    lambda: scoring.matmul_fp8(fp8(4, 256, 1), fp8(8, 256, 1), out=t((4, 8))),
    lambda: scoring.matmul_fp8(fp8(4, 256, 1), fp8(8, 255, 128), out=t((4, 8))),
    lambda: scoring.matmul_fp8(fp8(4, 250, 1, ld=250), fp8(8, 250, 128), out=t((4, 8))),
    lambda: scoring.matmul_fp8(fp8(4, 250, 1, scale=(4, 1)), fp8(8, 250, 128), out=t((4, 8))),
    lambda: scoring.matmul_fp8(fp8(4, 256, 1), fp8(8, 256, 128), out=t((8, 4))),
    lambda: scoring.matmul_fp8(fp8(4, 256, 1), fp8(8, 256, 128), out=t((4, 8), I64)),
    lambda: scoring.matmul_fp8(fp8(4, 256, 1), fp8(8, 256, 128), activation="tanh", out=t((4, 8))),
    lambda: scoring.matmul_fp8(fp8(4, 256, 1), fp8(8, 256, 128), bias=t((4,)), out=t((4, 8))),
    lambda: scoring.token_logprobs(t((4, 8), np.float64)),
    lambda: scoring.token_logprobs(t((4, 8)), targets=t((5,), I64)),
    lambda: scoring.token_logprobs(t((4, 8)), targets=t((4,), np.int32)),
    lambda: scoring.token_logprobs(t((4, 8)), k=9),
    lambda: scoring.token_logprobs(t((4, 100)), k=33),
    lambda: scoring.token_logprobs(t((4, 100)), k=-1),
    lambda: scoring.token_logprobs(t((4, 100)), vocab=101),
    lambda: scoring.token_logprobs(t((4, 0)), vocab=0),
    lambda: scoring.token_logprobs(t((4, 100)), out={"logprob": t((4,))}),
    lambda: scoring.token_logprobs(t((4, 100)), k=2, out={"top_id": t((4, 2), I64)}),
    lambda: scoring.token_logprobs(t((4, 100)), k=2, out={"top_id": t((4, 2), I64), "top_logprob": t((4, 3))}),
])
def test_python_calls_refuse(call):
    with pytest.raises(ValueError):
        call()


@pytest.mark.parametrize("call", [
    lambda: scoring.quantize_fp8(np.zeros((4, 4), F32)),
    lambda: scoring.token_logprobs(np.zeros((4, 4), F32)),
    lambda: scoring.token_logprobs(t((4, 4)), targets=np.zeros(4, I64)),
])
def test_python_calls_want_device_tensors(call):
    with pytest.raises(TypeError):
        call()


def test_python_calls_refuse_another_stream():
    class Other(FakeContext):
        stream = 8
    with pytest.raises(ValueError, match="another context"):
        scoring.token_logprobs(t((4, 8)), targets=t((4,), I64, ctx=Other()))


def quantize(x=4096, dtype=1, rows=4, cols=200, ldx=200, block_rows=1, q=4096, ldq=208, scale=4096, lds=2):
    return N.lib.lonnx_quantize_fp8(None, x, dtype, rows, cols, ldx, block_rows, q, ldq, scale, lds)


def gemm(A=4096, lda=208, sA=4096, ldsA=2, B=4096, ldb=208, sB=4096, ldsB=2, bias=None, C=4096, dtype=1, ldc=8, M=4,
         Nn=8, K=200, epi=0):
    return N.lib.lonnx_gemm_fp8(None, A, lda, sA, ldsA, B, ldb, sB, ldsB, bias, C, dtype, ldc, M, Nn, K, epi)


def logprobs(x=4096, dtype=1, rows=4, vocab=100, ld=100, targets=4096, temperature=1.0, lp=4096, ent=4096, k=2, tl=4096,
             ti=4096):
    return N.lib.lonnx_token_logprobs(None, x, dtype, rows, vocab, ld, targets, temperature, lp, ent, k, tl, ti)


@pytest.mark.parametrize("call, args, code, words", [
    (quantize, dict(dtype=7), UNSUPPORTED, "input type"),
    (quantize, dict(block_rows=2), BADARG, "blocks of 2 rows"),
    (quantize, dict(rows=-1), BADARG, "negative"),
    (quantize, dict(ldx=199), SHAPE, "leading dimension"),
    (quantize, dict(ldq=199), SHAPE, "leading dimension"),
    (quantize, dict(lds=1), SHAPE, "leading dimension"),
    (quantize, dict(x=4098), BADARG, "aligned"),
    (quantize, dict(scale=4097), BADARG, "aligned"),
    (quantize, dict(), BADARG, "null context"),
    (gemm, dict(dtype=17), UNSUPPORTED, "output type"),
    (gemm, dict(K=-1), BADARG, "negative"),
    (gemm, dict(M=(1 << 30) + 1), UNSUPPORTED, "2^30"),
    (gemm, dict(epi=3), BADARG, "epilogue"),
    (gemm, dict(lda=192), SHAPE, "leading dimension"),
    (gemm, dict(ldc=7), SHAPE, "leading dimension"),
    (gemm, dict(ldsB=1), SHAPE, "leading dimension"),
    (gemm, dict(lda=200), BADARG, "16 bytes"),
    (gemm, dict(B=4104), BADARG, "16 bytes"),
    (gemm, dict(C=4098), BADARG, "aligned"),
    (gemm, dict(bias=4097), BADARG, "aligned"),
    (gemm, dict(), BADARG, "null context"),
    (logprobs, dict(dtype=11), UNSUPPORTED, "type 11"),
    (logprobs, dict(vocab=0), BADARG, "0 tokens"),
    (logprobs, dict(vocab=(1 << 30) + 1, ld=1 << 31), BADARG, "tokens"),
    (logprobs, dict(rows=-1), BADARG, "rows"),
    (logprobs, dict(ld=99), SHAPE, "apart"),
    (logprobs, dict(temperature=0.0), BADARG, "temperature"),
    (logprobs, dict(temperature=float("nan")), BADARG, "temperature"),
    (logprobs, dict(temperature=float("inf")), BADARG, "temperature"),
    (logprobs, dict(k=33), BADARG, "alternatives"),
    (logprobs, dict(k=3, vocab=2), BADARG, "alternatives"),
    (logprobs, dict(x=4097), BADARG, "aligned"),
    (logprobs, dict(targets=4100), BADARG, "aligned"),
    (logprobs, dict(x=None), BADARG, "null pointer"),
    (logprobs, dict(ti=None), BADARG, "null pointer"),
    (logprobs, dict(targets=None), BADARG, "null pointer"),
    (logprobs, dict(), BADARG, "null context"),
])
def test_entry_points_refuse(call, args, code, words):
    assert call(**args) == code
    assert words in N.lib.lonnx_last_error().decode()
