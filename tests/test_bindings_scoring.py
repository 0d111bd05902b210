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
