"""Token log-probabilities where rows are many (a warp to a row, from 24 rows an
SM on) and long, against 64 bits.  Most rows are padding, which is not read."""
import pytest
import torch

from onnx_b200 import _native as N
from onnx_b200.tensor import Context
from test_scoring_gpu import TORCH, U, check_scores, gen, randn, run_scores, scores_reference

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def tctx():
    return Context(0, stream=torch.cuda.current_stream().cuda_stream)


def spread(x, rows, ld=None, offset=0):
    """The rows of x among `rows` ones, of which the others are padding and hold
    anything: (wide, their places)."""
    n, vocab = x.shape
    ld = ld or vocab
    at = (torch.arange(n, device="cuda") * (rows - 1)) // max(n - 1, 1)
    wide = torch.empty(rows * ld + offset, dtype=x.dtype, device="cuda")[offset:].view(rows, ld)
    wide[at] = float("nan")
    wide[at, :vocab] = x
    return wide, at


def score_spread(ctx, x, target, rows, k, ld=None, offset=0):
    wide, at = spread(x, rows, ld, offset)
    all_targets = torch.full((rows,), -1, dtype=torch.int64, device="cuda")
    all_targets[at] = target
    got = run_scores(ctx, wide, all_targets, k, vocab=x.shape[1])
    pad = all_targets < 0
    assert (got["logprob"][pad] == 0).all() and (got["entropy"][pad] == 0).all()
    if k:
        assert (got["top_id"][pad] == -1).all() and (got["top_logprob"][pad] == float("-inf")).all()
    return {n: t[at] for n, t in got.items()}


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows", [1, 310, 700, 3600])
@pytest.mark.parametrize("k", [0, 5])
def test_one_peak_over_equal_logits(tctx, rows, k, dtype):
    """A first logit far above 110002 equal ones, whose terms are near or under half
    a step of the peak's: a sum that adds them one by one to it loses them.

    S: a term is wrong by 2 steps (4 U), and by 3 U |z| for its argument's three
    roundings; a sum of 64 terms by 64 U, the halves, their exact joining's
    remainder, the 5 and 4 rounds of the warp and the CTA by 12 U, two changes of
    the maximum by 4 U."""
    vocab = 110003
    below = [15.5, 16.0, 16.5, 16.75, 17.0, 17.5]
    below = below[3:4] if rows == 1 else below
    x = torch.zeros(len(below), vocab, dtype=TORCH[dtype], device="cuda")
    x[:, 1:] = -torch.tensor(below, device="cuda")[:, None].to(x.dtype)
    target = torch.zeros(len(below), dtype=torch.int64, device="cuda")
    target[-1] = 1 if rows > 1 else 0
    got = score_spread(tctx, x, target, rows, k)
    want, z = scores_reference(x, target, k, 1.0)
    p = torch.exp(z - torch.logsumexp(z, 1, keepdim=True))
    mean = (p * z.abs()).sum(1)
    s = (4 + 64 + 12 + 4 + 3 * mean) * U
    if k:
        assert torch.equal(got["top_id"], want["top_id"])
    for name in ("logprob", "top_logprob") if k else ("logprob",):
        w = want[name]
        bound = (s + 4 * U * 18).reshape(-1, *[1] * (w.ndim - 1))  # and roundings of terms up to 18
        assert ((got[name].double() - w).abs() <= bound).all(), (name, float((got[name].double() - w).abs().max()))
    # ln S - W / S: W is a sum like S of terms |z| as large
    bound = s + (2 * s + 8 * U) * mean + 4 * U
    err = (got["entropy"].double() - want["entropy"]).abs()
    assert (err <= bound).all(), float((err / bound).max())


@pytest.mark.parametrize("vocab, ld, offset", [(4500, 4500, 0), (9001, 9007, 3), (33000, 33000, 0)])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("k", [0, 1, 5, 32])
def test_many_rows(tctx, vocab, ld, offset, dtype, k):
    x = (3 * randn(40, vocab, seed=vocab + k)).to(TORCH[dtype])
    target = torch.randint(0, vocab, (40,), generator=gen(k), device="cuda")
    got = score_spread(tctx, x, target, 3600, k, ld, offset)
    want, z = scores_reference(x, target, k, 1.0)
    check_scores(got, want, z, vocab, 1.0)


@pytest.mark.parametrize("vocab, ld, offset", [(9000, 9000, 0), (9001, 9007, 3), (20011, 20013, 1)])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("k", [0, 5, 32])
def test_many_rows_masks_and_ties(tctx, vocab, ld, offset, dtype, k):
    x = randn(9, vocab, seed=vocab).to(TORCH[dtype])
    low = torch.finfo(TORCH[dtype]).min
    x[0] = 0.5                                            # every logit equal
    x[1, torch.rand(vocab, generator=gen(2), device="cuda") < 0.97] = float("-inf")
    x[1, vocab // 2] = 1.0
    x[2] = low                                            # the type's lowest value, everywhere
    x[3, : vocab - 1] = low                               # and everywhere but in one place
    x[4] = torch.round(2 * x[4].float()).to(x.dtype)      # a few values, many ties
    x[5] = torch.arange(vocab, device="cuda").float().to(x.dtype)   # rising
    x[6] = -torch.arange(vocab, device="cuda").float().to(x.dtype)  # falling
    x[7, ::2], x[7, 1::2] = 0.0, -0.0                     # both zeros are one value
    target = torch.tensor([vocab - 1, 0, 5, vocab - 1, 1, vocab - 1, 0, 3, 7], device="cuda")
    got = score_spread(tctx, x, target, 3600, k, ld, offset)
    want, z = scores_reference(x, target, k, 1.0)
    check_scores(got, want, z, vocab, 1.0)


@pytest.mark.parametrize("vocab", [4500, 9001])
def test_many_rows_without_tokens_and_nan(tctx, vocab):
    x = randn(5, vocab, seed=1)
    x[0] = float("-inf")
    x[1, vocab - 1] = float("nan")
    x[2, vocab // 2] = float("inf")
    x[3] = float("nan")
    target = torch.zeros(5, dtype=torch.int64, device="cuda")
    got = score_spread(tctx, x, target, 3600, 4)
    assert got["logprob"][0] == float("-inf") and got["entropy"][0] == 0
    assert (got["top_logprob"][0] == float("-inf")).all() and got["top_id"][0].tolist() == [0, 1, 2, 3]
    assert got["logprob"][1:4].isnan().all() and got["entropy"][1:4].isnan().all()
    assert torch.equal(got["top_id"][1], torch.topk(x[1].nan_to_num(-9e9), 4).indices)  # NaN comes last
    assert got["top_id"][2, 0] == vocab // 2 and got["top_id"][3].tolist() == [0, 1, 2, 3]
    want, z = scores_reference(x[4:], target[4:], 4, 1.0)
    check_scores({n: t[4:] for n, t in got.items()}, want, z, vocab, 1.0)

# ---- targets past the vocabulary ------------------------------------------------

def entropies(ctx, x, target):
    entropy = torch.empty(len(x), device="cuda")
    N.check(N.lib.lonnx_token_logprobs(ctx.handle, x.data_ptr(), 1, len(x), x.shape[1], x.shape[1], target.data_ptr(),
                                       1.0, None, entropy.data_ptr(), 0, None, None))
    return entropy


@pytest.mark.parametrize("rows, vocab", [(3, 700), (3, 12345), (3600, 2500)])
def test_target_past_the_vocabulary_without_its_logprob(tctx, rows, vocab):
    """Targets may be given for the padding alone; one past the vocabulary is reported all the same."""
    x = randn(rows, vocab, seed=3)
    target = torch.ones(rows, dtype=torch.int64, device="cuda")
    target[1] = vocab
    entropy = entropies(tctx, x, target)
    with pytest.raises(N.LonnxError) as e:
        tctx.sync()
    assert e.value.code == -6 and "target" in e.value.message
    assert entropy.isfinite().all()
    target[1] = vocab - 1
    entropies(tctx, x, target)
    tctx.sync()


def test_sync_reports_every_flag(tctx):
    """A Gather index and a target out of range before one sync: both are named."""
    x = randn(3, 100)
    entropies(tctx, x, torch.tensor([1, 100, 2], device="cuda"))
    data, y = randn(4, 8), torch.empty(1, 8, device="cuda")
    N.check(N.lib.lonnx_gather(tctx.handle, data.data_ptr(), 4, 1, 4, 8, torch.tensor([9], device="cuda").data_ptr(), 1,
                               y.data_ptr()))
    with pytest.raises(N.LonnxError) as e:
        tctx.sync()
    assert e.value.code == -6 and "Gather" in e.value.message and "target" in e.value.message
    tctx.sync()


def test_sync_reports_an_expired_wait_with_the_rest(tctx):
    x = randn(3, 100)
    entropies(tctx, x, torch.tensor([1, 100, 2], device="cuda"))
    N.check(N.lib.lonnx_debug_expire_wait(tctx.handle, 100000))
    with pytest.raises(N.LonnxError) as e:
        tctx.sync()
    assert e.value.code == -5 and "wait expired" in e.value.message and "target" in e.value.message
    tctx.sync()
