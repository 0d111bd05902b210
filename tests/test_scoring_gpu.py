"""The scoring operators (8-bit block quantisation, the block-scaled product,
token log-probabilities) against their formulas in 64 bits."""
import numpy as np
import pytest
import torch

from onnx_b200 import _native as N
from onnx_b200 import scoring
from onnx_b200.tensor import BFLOAT16, FLOAT8E4M3, Context, DeviceTensor

pytestmark = pytest.mark.gpu

TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
OWN = {torch.float32: np.dtype(np.float32), torch.float16: np.dtype(np.float16), torch.bfloat16: BFLOAT16,
       torch.float8_e4m3fn: FLOAT8E4M3, torch.int64: np.dtype(np.int64)}
HALF = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}  # half a step of each type
U = 2.0 ** -24


@pytest.fixture(scope="module")
def tctx():
    """A context on torch's stream, so that torch tensors are operands in order."""
    return Context(0, stream=torch.cuda.current_stream().cuda_stream)


def dev(ctx, t, shape=None):
    """A torch tensor's memory as an operand (shape: [rows, leading dimension] of a wider one)."""
    return DeviceTensor(ctx, shape or t.shape, OWN[t.dtype], ptr=t.data_ptr(), owner=t)


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(*shape, seed=0):
    return torch.randn(*shape, generator=gen(seed), device="cuda")


# ---- quantisation -------------------------------------------------------------

def to_e4m3(t):
    """float64 -> the nearest e4m3 value, ties to even, saturating."""
    step = torch.exp2(torch.floor(torch.log2(t.abs().clamp_min(2.0 ** -6))) - 3)
    return (torch.round(t / step) * step).clamp(-448, 448)


def quantize_reference(x, block_rows):
    """(values, scales) by the definition: the quotient 448 x / amax, exact or far
    from a halfway point in 64 bits, to 8 bits; amax / 448 rounded to fp32."""
    r, c = x.shape
    br, bc = -(-r // block_rows), -(-c // 128)
    tall = torch.zeros(br * block_rows, bc * 128, device="cuda")
    tall[:r, :c] = x.float().abs()
    amax = tall.view(br, block_rows, bc, 128).amax((1, 3)).clamp_min(2.0 ** -96)
    wide = amax.repeat_interleave(block_rows, 0)[:r].repeat_interleave(128, 1)[:, :c].double()
    return to_e4m3(x.double() * 448.0 / wide), amax / torch.full_like(amax, 448.0)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("rows, cols", [(1, 1), (1, 128), (3, 127), (5, 129), (128, 128), (129, 384), (130, 1001),
                                        (257, 640), (1000, 72)])
def test_quantize(tctx, rows, cols, block_rows, dtype):
    x = (randn(rows, cols, seed=rows + cols) * torch.exp2(4 * randn(cols, seed=3))).to(TORCH[dtype])
    m = scoring.quantize_fp8(dev(tctx, x), block_rows)
    q = torch.full((rows, m.q.shape[1]), 7, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    scale = torch.zeros(m.scale.shape, device="cuda")
    scoring.quantize_fp8(dev(tctx, x), block_rows, out=(dev(tctx, q), dev(tctx, scale)))
    want, want_scale = quantize_reference(x, block_rows)
    assert torch.equal(scale, want_scale)
    assert torch.equal(q[:, :cols].double(), want)
    assert (q.view(torch.uint8)[:, cols:] == 7).all()  # past a row's end: left as it was
    assert np.array_equal(m.scale.to_host(), scale.cpu().numpy())
    assert np.array_equal(m.q.to_host().view(np.uint8)[:, :cols], q.view(torch.uint8)[:, :cols].cpu().numpy())


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("ldx, ldq, offset", [(205, 333, 0), (208, 208, 1), (224, 204, 2)])
@pytest.mark.parametrize("block_rows", [1, 128])
def test_quantize_strides_and_alignment(tctx, block_rows, ldx, ldq, offset, dtype):
    rows, cols = 133, 203
    x = randn(rows * ldx + offset, seed=1).to(TORCH[dtype])
    q = torch.full((rows * ldq + offset,), 7, dtype=torch.uint8, device="cuda")
    lds = 5
    scale = torch.full((rows, lds), -1.0, device="cuda")
    N.check(N.lib.lonnx_quantize_fp8(tctx.handle, x[offset:].data_ptr(), {"f32": 1, "bf16": 16}[dtype], rows, cols, ldx,
                                     block_rows, q[offset:].data_ptr(), ldq, scale.data_ptr(), lds))
    want, want_scale = quantize_reference(x[offset:].view(rows, ldx)[:, :cols], block_rows)
    got = q[offset:].view(rows, ldq)
    assert torch.equal(got[:, :cols].contiguous().view(torch.float8_e4m3fn).double(), want)
    assert torch.equal(scale[:want_scale.shape[0], :2], want_scale)
    assert (got[:, cols:] == 7).all() and (q[:offset] == 7).all()
    assert (scale[:, 2:] == -1).all() and (scale[want_scale.shape[0]:] == -1).all()


@pytest.mark.parametrize("block_rows", [1, 128])
def test_quantize_special_values(tctx, block_rows):
    x = randn(256, 512, seed=5)
    x[:, :128] = 0                       # a block of zeros
    x[0, 130] = float("nan")             # NaN beside numbers
    x[0, 300] = float("inf")             # an infinite block
    x[0, 400] = 3e38                     # near the type's largest
    x[128:, 384:] *= 2.0 ** -140         # subnormal: below the smallest block magnitude
    m = scoring.quantize_fp8(dev(tctx, x), block_rows)
    v = torch.from_numpy(m.q.to_host().view(np.uint8).copy()).cuda().view(torch.float8_e4m3fn).float()
    s = torch.from_numpy(m.scale.to_host()).cuda()
    assert (v[:, :128] == 0).all() and (s[:, 0] == np.float32(2.0 ** -96) / np.float32(448)).all()
    assert v[0, 130].isnan() and not v[0, 131:256].isnan().any() and s[0, 1].isfinite()
    assert s[0, 2] == float("inf") and (v[0, 256:384] * s[0, 2]).isnan().all()
    assert v[0, 400] == 448 and (s[128 // block_rows:, 3] == np.float32(2.0 ** -96) / np.float32(448)).all()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_quantize_halfway_points(tctx, dtype):
    """Values on and next to the points halfway between two e4m3 values, in blocks of many magnitudes."""
    grid = torch.arange(0, 128, dtype=torch.uint8, device="cuda")[:127].view(torch.float8_e4m3fn).float()
    mid = (grid[1:] + grid[:-1]) / 2  # 126 halfway points, exact in fp32
    amax = torch.cat([torch.tensor([448.0, 7.0, 1.0, 3.0, 5.0, 0.1], device="cuda"), randn(250, seed=8).abs() + 0.01])
    amax = amax.to(TORCH[dtype]).float()
    x = torch.zeros(256, 128, device="cuda")
    x[:, :126] = mid * amax[:, None] / 448
    x[:, 126] = amax
    x = x.to(TORCH[dtype])
    x[64:128] = torch.nextafter(x[64:128], torch.zeros_like(x[64:128]))
    want, want_scale = quantize_reference(x, 1)
    m = scoring.quantize_fp8(dev(tctx, x))
    got = torch.from_numpy(m.q.to_host().view(np.uint8).copy()).cuda().view(torch.float8_e4m3fn)
    assert torch.equal(got.double(), want)


def test_quantize_nothing(tctx):
    q = torch.full((4, 16), 7, dtype=torch.uint8, device="cuda")
    s = torch.zeros(4, 1, device="cuda")
    for rows, cols in ((0, 16), (4, 0)):
        N.check(N.lib.lonnx_quantize_fp8(tctx.handle, None, 1, rows, cols, 16, 1, q.data_ptr(), 16, s.data_ptr(), 1))
    tctx.sync()
    assert (q == 7).all()


# ---- the product ---------------------------------------------------------------

def fp8_operands(m, n, k, seed=0, lda=None, ldb=None):
    """Quantised operands in padded rows whose padding is NaN: (a, sa, b, sb), scales spread over decades."""
    lda, ldb = lda or -(-k // 16) * 16, ldb or -(-k // 16) * 16
    out = []
    for rows, ld, br, sd in ((m, lda, 1, seed), (n, ldb, 128, seed + 1)):
        kb = -(-k // 128)
        q = torch.full((rows, ld), 0x7F, dtype=torch.uint8, device="cuda")
        q[:, :k] = (randn(rows, k, seed=sd) * 100).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
        s = torch.exp2(3 * randn(-(-rows // br), kb, seed=sd + 10)) / 448
        out += [q, s]
    return out


def product_reference(a, sa, b, sb, k, bias=None):
    """(A . B^T + bias, the same of absolute values) in 64 bits."""
    y = mag = 0.0
    for i in range(-(-k // 128)):
        at = slice(128 * i, min(k, 128 * i + 128))
        x, w = a.view(torch.float8_e4m3fn)[:, at].double(), b.view(torch.float8_e4m3fn)[:, at].double()
        s = sa[:, i].double()[:, None] * sb[:, i].double().repeat_interleave(128)[:b.shape[0]]
        y, mag = y + s * (x @ w.t()), mag + s * (x.abs() @ w.abs().t())
    if bias is not None:
        y, mag = y + bias.double(), mag + bias.double().abs()
    return y, mag


def product_bound(mag, k, dtype, y):
    """A block's 128 products are summed in fp32 with at most a step (2^-23) lost
    per addition; each block's scale is a rounded product, its FMA and the bias
    addition round to nearest; then one rounding to the output type, whose
    smallest steps (f16: 2^-24, half of it lost) are absolute."""
    return (128 * 2 * U + (-(-k // 128) + 3) * U) * mag + HALF[dtype] * y.abs() * (1 + 1e-3) + (2.0 ** -25 if dtype == "f16" else 0)


def run_product(ctx, a, sa, b, sb, k, dtype="f32", act=None, bias=None, ldc=None):
    m, n = a.shape[0], b.shape[0]
    ldc = ldc or n
    c = torch.full((m, ldc), 5.0, dtype=TORCH[dtype], device="cuda")
    N.check(N.lib.lonnx_gemm_fp8(ctx.handle, a.data_ptr(), a.shape[1], sa.data_ptr(), sa.shape[1], b.data_ptr(),
                                 b.shape[1], sb.data_ptr(), sb.shape[1], bias.data_ptr() if bias is not None else None,
                                 c.data_ptr(), {"f32": 1, "f16": 10, "bf16": 16}[dtype], ldc, m, n, k,
                                 scoring.ACTIVATIONS[act]))
    ctx.sync()
    assert (c[:, n:] == 5).all()
    return c[:, :n]


SHAPES = [(1, 1, 1), (1, 128, 128), (1, 1000, 257), (2, 129, 4096), (7, 384, 384), (8, 4096, 512), (16, 250, 1111),
          (17, 513, 640), (31, 65, 33), (32, 2000, 384), (33, 640, 1152), (64, 300, 2048), (65, 1536, 384),
          (127, 127, 127), (128, 256, 128), (129, 257, 129), (200, 1000, 1001), (256, 256, 8192), (300, 4100, 384),
          (777, 1000, 1111), (1024, 192, 96), (1500, 2100, 300), (2048, 2300, 2100), (1700, 1900, 1100),
          (2600, 4000, 130), (4000, 5000, 520), (19000, 380, 640), (20000, 640, 300)]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("m, n, k", SHAPES)
def test_product(tctx, m, n, k, dtype):
    a, sa, b, sb = fp8_operands(m, n, k, seed=m + n + k)
    got = run_product(tctx, a, sa, b, sb, k, dtype).double()
    want, mag = product_reference(a, sa, b, sb, k)
    limit = 65504.0 if dtype == "f16" else float("inf")
    fine = want.abs() < limit
    err = (got - want).abs()[fine]
    assert (err <= product_bound(mag, k, dtype, want)[fine]).all(), float((err / mag[fine]).max())


@pytest.mark.parametrize("m, n, k", [(1, 1000, 384), (5, 130, 640), (40, 500, 129), (300, 700, 384), (513, 1024, 1152)])
@pytest.mark.parametrize("act", [None, "relu", "gelu"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_product_bias_and_activation(tctx, m, n, k, act, dtype):
    a, sa, b, sb = fp8_operands(m, n, k, seed=m + n)
    sa, sb = sa / 20, sb / 20
    bias = randn(n, seed=9)
    got = run_product(tctx, a, sa, b, sb, k, dtype, act, bias).double()
    want, mag = product_reference(a, sa, b, sb, k, bias)
    # an activation's slope is at most 1.13; the GELU's erf is within 1.5e-7 (A&S 7.1.26) and its
    # evaluation within a few steps of its argument
    bound = 1.13 * product_bound(mag, k, "f32", want * 0)
    if act == "relu":
        want = want.clamp_min(0)
    elif act == "gelu":
        bound = bound + want.abs() * (1.5e-7 + 16 * U)
        want = 0.5 * want * torch.special.erfc(-want / 2 ** 0.5)
    assert ((got - want).abs() <= bound + HALF[dtype] * (want.abs() + bound)).all()


@pytest.mark.parametrize("m, n, k, lda, ldb, ldc", [(3, 129, 200, 256, 208, 131), (150, 300, 200, 208, 512, 304),
                                                     (260, 515, 390, 400, 416, 517), (40, 515, 390, 400, 416, 600),
                                                     (500, 495, 390, 400, 400, 496), (700, 1463, 24, 32, 32, 1464)])
@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_product_strides(tctx, m, n, k, lda, ldb, ldc, dtype):
    a, sa, b, sb = fp8_operands(m, n, k, seed=4, lda=lda, ldb=ldb)
    wide_a, wide_b = torch.full((m, 7), 9.0, device="cuda"), torch.full((len(sb), 6), 9.0, device="cuda")
    wide_a[:, :sa.shape[1]], wide_b[:, :sb.shape[1]] = sa / 30, sb / 30
    got = run_product(tctx, a, wide_a, b, wide_b, k, dtype, ldc=ldc).double()
    want, mag = product_reference(a, sa / 30, b, sb / 30, k)
    assert ((got - want).abs() <= product_bound(mag, k, dtype, want)).all()


@pytest.mark.parametrize("m, n", [(1, 300), (20, 300), (200, 300)])
def test_product_special_values(tctx, m, n):
    k = 300
    a, sa, b, sb = fp8_operands(m, n, k)
    a[0, 5] = 0x7F                       # NaN in a row of A
    b[7, 299] = 0x7F                     # and in a row of B
    got = run_product(tctx, a, sa, b, sb, k)
    assert got[0].isnan().all() and got[:, 7].isnan().all()
    rest = got[1:, [j for j in range(n) if j != 7]]
    assert not rest.isnan().any()
    a[0, 5] = 0
    sa[m - 1] = 0                        # a row whose scales are zero
    got = run_product(tctx, a, sa, b, sb, k)
    assert (got[m - 1, :7] == 0).all()


def test_product_without_columns(tctx):
    """K = 0: the bias through the activation; M = 0 or N = 0: nothing."""
    bias = randn(300, seed=2)
    c = torch.zeros(3, 300, device="cuda")
    N.check(N.lib.lonnx_gemm_fp8(tctx.handle, None, 0, None, 0, None, 0, None, 0, bias.data_ptr(), c.data_ptr(), 1, 300,
                                 3, 300, 0, scoring.ACTIVATIONS["relu"]))
    tctx.sync()
    assert torch.equal(c, bias.clamp_min(0).expand(3, 300))
    for m, n in ((0, 300), (3, 0)):
        N.check(N.lib.lonnx_gemm_fp8(tctx.handle, None, 16, None, 1, None, 16, None, 1, None, c.data_ptr(), 1, 300, m, n,
                                     16, 0))
    tctx.sync()
    assert torch.equal(c, bias.clamp_min(0).expand(3, 300))


@pytest.mark.parametrize("m, n, k", [(1, 4096, 4096), (50, 1111, 3000), (700, 900, 1000)])
def test_product_is_repeatable(tctx, m, n, k):
    a, sa, b, sb = fp8_operands(m, n, k)
    first = run_product(tctx, a, sa, b, sb, k)
    assert all(torch.equal(first, run_product(tctx, a, sa, b, sb, k)) for _ in range(3))


# ---- log-probabilities ---------------------------------------------------------

def scores_reference(x, target, k, temperature):
    """The definition in 64 bits, z = (x - max x) / T (logits of the lowest value
    would absorb the sum's logarithm without the difference): log-softmax,
    entropy, stable order."""
    z = (x.double() - x.double().amax(1, keepdim=True)) / float(np.float32(temperature))
    lse = torch.logsumexp(z, 1, keepdim=True)
    lp = z - lse
    p = torch.exp(lp)
    order = torch.sort(x.float() + 0.0, dim=1, descending=True, stable=True).indices[:, :k]
    return dict(logprob=lp.gather(1, target.clamp_min(0)[:, None])[:, 0], entropy=-torch.special.xlogy(p, p).sum(1),
                top_logprob=lp.gather(1, order), top_id=order), z


def check_scores(got, want, z, vocab, temperature):
    """fp32 bounds: (x - m) / T to three roundings; S to its terms' error (the
    exponential's 2 steps and its argument's rounding, at most 0.54 steps of the
    sum's weight each) and the additions: a thread sums at most vocab / 256 + 64
    terms, then about 24 join."""
    d = z.abs()
    s = (vocab / 256 + 64 + 24 + 8) * U * 2
    for name, of in (("logprob", got["logprob"]), ("top_logprob", got["top_logprob"])):
        w = want[name]
        bound = 4 * U * (w.abs() + 40) + s
        err = (of.double() - w).abs()
        assert ((err <= bound) | (of == w)).all(), (name, float(err.nan_to_num(0).max()))
    p = torch.exp(z - torch.logsumexp(z, 1, keepdim=True))
    mean = (p * torch.where(p > 0, d, 0.0)).sum(1)
    err = (got["entropy"].double() - want["entropy"]).abs()
    assert (err <= 2 * s * (1 + mean) + 4 * U * (40 + mean)).all(), float(err.max())
    assert torch.equal(got["top_id"], want["top_id"])


def run_scores(ctx, x, target, k, temperature=1.0, vocab=None):
    rows = x.shape[0]
    hold = {"logprob": torch.full((rows + 1,), 9.0, device="cuda"), "entropy": torch.full((rows + 1,), 9.0, device="cuda"),
            "top_logprob": torch.full((rows + 1, k), 9.0, device="cuda"),
            "top_id": torch.full((rows + 1, k), 9, dtype=torch.int64, device="cuda")}
    names = ["entropy"] + (["logprob"] if target is not None else []) + (["top_logprob", "top_id"] if k else [])
    scoring.token_logprobs(dev(ctx, x), dev(ctx, target) if target is not None else None, k=k, temperature=temperature,
                           vocab=vocab, out={n: dev(ctx, hold[n][:rows]) for n in names})
    torch.cuda.synchronize()
    assert all((t[rows] == 9).all() for t in hold.values())
    return {n: t[:rows] for n, t in hold.items()}


VOCABS = [1, 2, 3, 31, 32, 33, 100, 1001, 2048, 2049, 4096, 4099, 8191, 20011, 32768, 65537, 250037]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("vocab", VOCABS)
@pytest.mark.parametrize("rows", [1, 5, 700])
def test_logprobs(tctx, rows, vocab, dtype):
    if rows == 700 and vocab > 40000:
        rows = 310  # past the sizes at which a row is shared by several blocks
    for k in sorted({0, 1, min(5, vocab), min(32, vocab)}):
        x = (3 * randn(rows, vocab, seed=vocab + k)).to(TORCH[dtype])
        target = torch.randint(0, vocab, (rows,), generator=gen(k), device="cuda")
        got = run_scores(tctx, x, target, k)
        want, z = scores_reference(x, target, k, 1.0)
        check_scores(got, want, z, vocab, 1.0)


@pytest.mark.parametrize("vocab, ld, offset", [(1000, 1003, 1), (1003, 1003, 3), (9001, 9007, 5), (40000, 40001, 7),
                                               (33, 47, 1), (5, 8, 2)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("temperature", [0.25, 1.7])
def test_logprobs_strides_alignment_temperature(tctx, vocab, ld, offset, dtype, temperature):
    rows, k = 9, min(7, vocab)
    flat = (2 * randn(rows * ld + offset, seed=ld)).to(TORCH[dtype])
    x = flat[offset:].view(rows, ld)
    x[:, vocab:] = float("nan")  # columns past the vocabulary are not read
    target = torch.randint(0, vocab, (rows,), generator=gen(1), device="cuda")
    got = run_scores(tctx, x, target, k, temperature, vocab=vocab)
    want, z = scores_reference(x[:, :vocab], target, k, temperature)
    check_scores(got, want, z, vocab, temperature)


@pytest.mark.parametrize("vocab", [40, 1500, 9000, 100003])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_logprobs_masks_and_ties(tctx, vocab, dtype):
    x = randn(8, vocab, seed=vocab).to(TORCH[dtype])
    low = torch.finfo(TORCH[dtype]).min
    x[0] = 0.5                                            # every logit equal
    x[1, torch.rand(vocab, generator=gen(2), device="cuda") < 0.97] = float("-inf")
    x[1, vocab // 2] = 1.0
    x[2] = low                                            # the type's lowest value, everywhere
    x[3, : vocab - 1] = low                               # and everywhere but in one place
    x[4] = torch.round(2 * x[4].float()).to(x.dtype)      # a few values, many ties
    x[5] = torch.arange(vocab, device="cuda").float().clamp_max(60000).to(x.dtype)            # rising
    x[6] = -torch.arange(vocab, device="cuda").float().clamp_max(60000).to(x.dtype)           # falling
    x[7, ::2], x[7, 1::2] = 0.0, -0.0                     # both zeros are one value
    target = torch.tensor([vocab - 1, 0, 5, vocab - 1, 1, vocab - 1, 0, 3], device="cuda")
    for k in (0, 1, 32):
        got = run_scores(tctx, x, target, k)
        want, z = scores_reference(x, target, k, 1.0)
        check_scores(got, want, z, vocab, 1.0)


@pytest.mark.parametrize("vocab", [40, 1500, 9000, 100003])
def test_logprobs_rows_without_tokens_and_nan(tctx, vocab):
    x = randn(5, vocab, seed=1)
    x[0] = float("-inf")
    x[1, vocab - 1] = float("nan")
    x[2, vocab // 2] = float("inf")
    x[3] = float("nan")
    target = torch.zeros(5, dtype=torch.int64, device="cuda")
    got = run_scores(tctx, x, target, 4)
    assert got["logprob"][0] == float("-inf") and got["entropy"][0] == 0
    assert (got["top_logprob"][0] == float("-inf")).all() and got["top_id"][0].tolist() == [0, 1, 2, 3]
    assert got["logprob"][1:4].isnan().all() and got["entropy"][1:4].isnan().all()
    assert torch.equal(got["top_id"][1], torch.topk(x[1].nan_to_num(-9e9), 4).indices)  # NaN comes last
    assert got["top_id"][2, 0] == vocab // 2 and got["top_id"][3].tolist() == [0, 1, 2, 3]
    want, z = scores_reference(x[4:], target[4:], 4, 1.0)
    check_scores({n: t[4:] for n, t in got.items()}, want, z, vocab, 1.0)


@pytest.mark.parametrize("vocab", [700, 12345])
def test_logprobs_padding_rows(tctx, vocab):
    x = randn(6, vocab, seed=3)
    target = torch.tensor([3, -1, 4, -100, 5, -1], device="cuda")
    x[target < 0] = float("nan")  # not read
    got = run_scores(tctx, x, target, 3)
    pad = target < 0
    assert (got["logprob"][pad] == 0).all() and (got["entropy"][pad] == 0).all()
    assert (got["top_id"][pad] == -1).all() and (got["top_logprob"][pad] == float("-inf")).all()
    want, z = scores_reference(x[~pad], target[~pad], 3, 1.0)
    check_scores({n: t[~pad] for n, t in got.items()}, want, z, vocab, 1.0)
    # without targets every row is scored; these rows start on other addresses, and the order of a
    # row's sums goes by its first 16-byte boundary, so the two agree within the bounds, not in bits
    bare = run_scores(tctx, x[~pad], None, 3)
    check_scores({**bare, "logprob": got["logprob"][~pad]}, want, z, vocab, 1.0)


@pytest.mark.parametrize("vocab", [700, 12345])
def test_logprobs_target_past_the_vocabulary(tctx, vocab):
    x = randn(3, vocab, seed=3)
    target = torch.tensor([1, vocab, 2], device="cuda")
    got = run_scores(tctx, x, target, 0)
    with pytest.raises(N.LonnxError) as e:
        tctx.sync()
    assert e.value.code == -6 and "target" in e.value.message
    assert got["logprob"][1].isnan() and got["logprob"][[0, 2]].isfinite().all() and got["entropy"].isfinite().all()
    tctx.sync()  # reported once


def test_logprobs_nothing(tctx):
    N.check(N.lib.lonnx_token_logprobs(tctx.handle, None, 1, 0, 10, 10, None, 1.0, None, None, 0, None, None))
    x = randn(2, 10)
    N.check(N.lib.lonnx_token_logprobs(tctx.handle, x.data_ptr(), 1, 2, 10, 10, None, 1.0, None, None, 0, None, None))
    tctx.sync()


def test_logprobs_offsets_past_32_bits(tctx):
    """Rows that start more than 2^31 elements into the logits."""
    vocab, rows = 1 << 16, 33000
    x = torch.empty(rows, vocab, dtype=torch.float16, device="cuda")
    x[-3:] = randn(3, vocab, seed=1).half()
    target = torch.full((rows,), -1, dtype=torch.int64, device="cuda")
    target[-3:] = torch.tensor([1, 2, 65535], device="cuda")
    got = run_scores(tctx, x, target, 5)
    want, z = scores_reference(x[-3:], target[-3:], 5, 1.0)
    check_scores({n: t[-3:] for n, t in got.items()}, want, z, vocab, 1.0)


@pytest.mark.parametrize("m, n, k", [(9000, 250048, 40), (9000, 250037, 40)])  # rows on 16 bytes, and not
def test_product_offsets_past_32_bits(tctx, m, n, k):
    """Rows that start more than 2^31 elements into C."""
    a, sa, b, sb = fp8_operands(m, n, k, seed=n)
    got = run_product(tctx, a, sa, b, sb, k, "bf16")
    at = torch.tensor([0, 1, m // 2, m - 2, m - 1], device="cuda")
    want, mag = product_reference(a[at], sa[at], b, sb, k)
    assert ((got[at].double() - want).abs() <= product_bound(mag, k, "bf16", want)).all()


def test_product_of_few_rows_offsets_past_32_bits(tctx):
    m, n, k, ldc = 20, 1000, 384, (1 << 27) + 8
    a, sa, b, sb = fp8_operands(m, n, k, seed=4)
    got = run_product(tctx, a, sa, b, sb, k, "bf16", ldc=ldc).double()
    want, mag = product_reference(a, sa, b, sb, k)
    assert ((got - want).abs() <= product_bound(mag, k, "bf16", want)).all()


@pytest.mark.parametrize("offset", [0, 1])
@pytest.mark.parametrize("block_rows", [1, 128])
def test_quantize_offsets_past_32_bits(tctx, block_rows, offset):
    """Rows that start more than 2^31 elements into x and q."""
    rows, cols, ld = 20, 300, (1 << 27) + 16
    x = torch.empty(rows * ld + offset, dtype=torch.float16, device="cuda")
    q = torch.empty(rows * ld + offset, dtype=torch.uint8, device="cuda")
    part = torch.as_strided(x, (rows, cols), (ld, 1), offset)
    part.copy_(randn(rows, cols, seed=5))
    scale = torch.empty(-(-rows // block_rows), 3, device="cuda")
    N.check(N.lib.lonnx_quantize_fp8(tctx.handle, x.data_ptr() + 2 * offset, 10, rows, cols, ld, block_rows,
                                     q.data_ptr() + offset, ld, scale.data_ptr(), 3))
    want, want_scale = quantize_reference(part, block_rows)
    got = torch.as_strided(q, (rows, cols), (ld, 1), offset).contiguous().view(torch.float8_e4m3fn)
    assert torch.equal(scale, want_scale) and torch.equal(got.double(), want)


# ---- together -------------------------------------------------------------------

def score(ctx, hidden, head, target, k, out=None):
    """Hidden states to scores, as a scorer runs it."""
    logits = scoring.matmul_fp8(scoring.quantize_fp8(dev(ctx, hidden)), head)
    return scoring.token_logprobs(logits, dev(ctx, target), k=k, out=out), logits


@pytest.mark.parametrize("tokens, hidden, vocab", [(1, 384, 5003), (7, 384, 5003), (150, 200, 1234)])
def test_scoring_run(tctx, tokens, hidden, vocab):
    h, w = randn(tokens, hidden, seed=1), randn(vocab, hidden, seed=2) * hidden ** -0.5
    target = torch.randint(0, vocab, (tokens,), generator=gen(3), device="cuda")
    head = scoring.quantize_fp8(dev(tctx, w), block_rows=128)
    got, logits = score(tctx, h, head, target, 5)
    got = {n: torch.from_numpy(t.to_host()).cuda() for n, t in got.items()}
    # the product of the quantised operands, by their definition
    (qa, sa), (qb, sb) = quantize_reference(h, 1), quantize_reference(w, 128)
    as_bytes = [q.float().to(torch.float8_e4m3fn).view(torch.uint8) for q in (qa, qb)]
    y, mag = product_reference(as_bytes[0], sa, as_bytes[1], sb, hidden)
    logits = torch.from_numpy(logits.to_host()).cuda()
    assert ((logits.double() - y).abs() <= product_bound(mag, hidden, "f32", y)).all()
    want, z = scores_reference(logits, target, 5, 1.0)
    check_scores(got, want, z, vocab, 1.0)
    # and the 8-bit head is near the fp32 one: two operands within 2^-4 of a value each, errors of random sign
    exact = torch.log_softmax(h.double() @ w.double().t(), 1).gather(1, target[:, None])[:, 0]
    assert (got["logprob"].double() - exact).abs().max() < 0.5


def test_scoring_captured_and_replayed():
    """The whole run recorded in a CUDA graph on the context's stream, replayed on new hidden states."""
    stream = torch.cuda.Stream()
    ctx = Context(0, stream=stream.cuda_stream)
    tokens, hidden, vocab = 6, 384, 4001
    h, w = randn(tokens, hidden, seed=1), randn(vocab, hidden, seed=2) * 0.05
    target = torch.randint(0, vocab, (tokens,), generator=gen(3), device="cuda")
    torch.cuda.synchronize()
    head = scoring.quantize_fp8(dev(ctx, w), block_rows=128)
    score(ctx, h, head, target, 3)  # first call outside the capture: buffers come from the context's cache after it
    ctx.sync()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        got, logits = score(ctx, h, head, target, 3)
    for seed in (5, 6):
        h.copy_(randn(tokens, hidden, seed=seed))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        replayed = {n: t.to_host() for n, t in got.items()}
        fresh, _ = score(ctx, h, head, target, 3)
        assert all(np.array_equal(replayed[n], fresh[n].to_host()) for n in replayed)


def test_scoring_capture_keeps_its_buffers():
    """What a captured run let go of (its quantised hidden states) is not given
    to tensors made later: a replay leaves them as they are."""
    stream = torch.cuda.Stream()
    ctx = Context(0, stream=stream.cuda_stream)
    tokens, hidden, vocab = 6, 384, 4001
    h, w = randn(tokens, hidden, seed=1), randn(vocab, hidden, seed=2) * 0.05
    target = torch.randint(0, vocab, (tokens,), generator=gen(3), device="cuda")
    torch.cuda.synchronize()
    head = scoring.quantize_fp8(dev(ctx, w), block_rows=128)
    score(ctx, h, head, target, 3)
    ctx.sync()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        got, logits = score(ctx, h, head, target, 3)
    others = [randn(tokens, hidden, seed=s) for s in (7, 8, 9)]
    torch.cuda.synchronize()
    later = [scoring.quantize_fp8(dev(ctx, x)) for x in others]
    before = [m.q.to_host() for m in later]
    h.copy_(randn(tokens, hidden, seed=5))
    torch.cuda.synchronize()
    graph.replay()
    torch.cuda.synchronize()
    assert all(np.array_equal(b, m.q.to_host()) for b, m in zip(before, later))


@pytest.mark.parametrize("tokens, other", [(40, 40), (1, 1500), (1500, 200)])
def test_scoring_on_two_streams(tctx, tokens, other):
    """Two contexts on one GPU, working at the same time on their own streams,
    also with kernels that share an SM's tensor memory."""
    a, b = Context(0), Context(0)
    h, w = randn(max(tokens, other), 640, seed=1), randn(3001, 640, seed=2) * 0.05
    target = torch.randint(0, 3001, (max(tokens, other),), generator=gen(3), device="cuda")
    torch.cuda.synchronize()
    heads = [scoring.quantize_fp8(dev(c, w), block_rows=128) for c in (a, b)]
    sizes = (tokens, other)
    alone = []
    for c, head, m in zip((a, b), heads, sizes):
        alone.append({n: t.to_host() for n, t in score(c, h[:m], head, target[:m], 4)[0].items()})
        c.sync()
    runs = [[score(c, h[:m], head, target[:m], 4)[0] for c, head, m in zip((a, b), heads, sizes)] for _ in range(20)]
    for pair in runs:
        for got, want in zip(pair, alone):
            assert all(np.array_equal(want[n], t.to_host()) for n, t in got.items())


def test_context_on_a_stream():
    s = torch.cuda.Stream()
    c = Context(0, stream=s.cuda_stream)
    assert c.stream == s.cuda_stream
    c.close()
    with torch.cuda.stream(s):
        assert float(torch.ones(4, device="cuda").sum()) == 4.0  # the stream outlives the context
