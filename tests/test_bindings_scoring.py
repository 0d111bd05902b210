"""CPU checks of the C# source of the scoring operators (bindings/csharp)."""
import os
import re

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSHARP = os.path.join(ROOT, "bindings", "csharp")


def source(name):
    return open(os.path.join(CSHARP, name)).read()


def test_quantised_sizes_are_64_bit():
    """Row and column counts are int: sums and products of them are taken in long,
    or a count near 2^31 makes a buffer smaller than what the library writes."""
    body = re.search(r"public static Fp8Matrix Quantize\(.*?\n    }", source("Scoring.cs"), re.S).group(0)
    code = re.sub(r"(?m)^\s*///.*", "", body)
    for name in ("rows", "cols"):
        for at in re.finditer(rf"\b{name}\b(?=\s*[+*])", code):
            assert code[:at.start()].rstrip().endswith("(long)"), code[max(at.start() - 30, 0):at.end() + 20]


def test_every_scoring_entry_point_is_reached():
    """What Native.cs declares for scoring, some class calls, with the arguments that
    the C functions have: a caller's stream, and rows wider than they are long."""
    rest = "".join(source(f) for f in os.listdir(CSHARP) if f != "Native.cs")
    for name in ("lonnx_ctx_create_on_stream", "lonnx_quantize_fp8", "lonnx_gemm_fp8", "lonnx_token_logprobs"):
        assert f"Native.{name}(" in rest, name
    scoring = source("Scoring.cs")
    assert re.search(r"void MatMul\([^)]*long ldc = 0\)", scoring) and "ldc == 0 ? w.Rows : ldc" in scoring
    assert re.search(r"void TokenLogprobs\([^)]*long ld = 0\)", scoring) and "ld == 0 ? vocab : ld" in scoring
    assert re.search(r"public CudaContext\(int device, IntPtr stream\)", source("DeviceTensor.cs"))
