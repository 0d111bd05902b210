"""Workloads of the output-head operators: block quantisation to 8-bit float,
the block-scaled 8-bit product, and the log-probabilities of tokens.

A pass takes device data that a program already holds and returns the whole
result.  With ``own`` false an operator is its plain form (elementary torch
operations in 32 bits); with ``own`` true it is the call of
``onnx_b200.scoring`` on the same memory.
"""
import math

import torch

own = False

VOCAB = 250037   # rows of the multilingual encoder's embedding table
BLOCK = 128
E4M3_MAX = 448.0
TINY = 2.0 ** -96  # smallest block magnitude that sets a scale
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
DEV = "cuda"


def listed():
    return [
        # one decoding step's hidden states for 8 requests
        dict(name="quantize 8x4096 bf16", op="quantize", rows=8, cols=4096, dtype="bf16", block_rows=1),
        # the encoder's FFN activations at batch 256 x 128 tokens
        dict(name="quantize 32768x1536 f32", op="quantize", rows=32768, cols=1536, dtype="f32", block_rows=1),
        # an output head's weights (the embedding table), once at load
        dict(name="quantize head 250037x384 f32", op="quantize", rows=VOCAB, cols=384, dtype="f32", block_rows=128),
        # one token through a square projection: latency and the weights' bytes
        dict(name="product 1x4096x4096 bf16", op="product", m=1, n=4096, k=4096, out="bf16", act="none", bias=False),
        # the logits of 32 requests over the repository's vocabulary (odd width)
        dict(name="product 32x250037x384 f32", op="product", m=32, n=VOCAB, k=384, out="f32", act="none", bias=False),
        # ragged in every direction
        dict(name="product 777x1000x1111 f16", op="product", m=777, n=1000, k=1111, out="f16", act="relu", bias=True),
        # the encoder's first FFN product with its bias and GELU at batch 256
        dict(name="product 32768x1536x384 f32", op="product", m=32768, n=1536, k=384, out="f32", act="gelu", bias=True),
        # a long prompt through a large square projection
        dict(name="product 8192x8192x8192 bf16", op="product", m=8192, n=8192, k=8192, out="bf16", act="none",
             bias=False),
        # one decoding step: a single row over the whole vocabulary
        dict(name="logprobs 1x250037 f32 k20", op="logprobs", rows=1, vocab=VOCAB, dtype="f32", k=20, pad=0,
             masked=0.0, temperature=1.0),
        # a batch of decoding steps with most tokens masked by a grammar
        dict(name="logprobs 64x32768 bf16 k5", op="logprobs", rows=64, vocab=32768, dtype="bf16", k=5, pad=0,
             masked=0.9, temperature=0.7),
        # many rows over a small odd vocabulary, no alternatives, padded batch
        dict(name="logprobs 16384x1001 f16 k0", op="logprobs", rows=16384, vocab=1001, dtype="f16", k=0, pad=2000,
             masked=0.0, temperature=1.0),
        # scoring a prompt of 2048 tokens over the whole vocabulary
        dict(name="logprobs 2048x250037 f32 k20", op="logprobs", rows=2048, vocab=VOCAB, dtype="f32", k=20, pad=48,
             masked=0.0, temperature=1.0),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["quantize", "product", "logprobs"])
    if op == "quantize":
        block_rows = rng.choice([1, 128])
        cols = _log_uniform(rng, 64, 16384)
        rows = _log_uniform(rng, 1, min(65536, 96_000_000 // cols))
        return dict(op=op, rows=rows, cols=cols, dtype=rng.choice(["f32", "f16", "bf16"]), block_rows=block_rows)
    if op == "product":
        n = _log_uniform(rng, 100, 40000)
        k = _log_uniform(rng, 64, 12000)
        m = _log_uniform(rng, 1, max(2, min(32768, int(5e11 / (n * k)))))
        return dict(op=op, m=m, n=n, k=k, out=rng.choice(["f32", "f16", "bf16"]),
                    act=rng.choice(["none", "relu", "gelu"]), bias=rng.random() < 0.5)
    vocab = _log_uniform(rng, 100, 262144)
    rows = _log_uniform(rng, 1, min(32768, 400_000_000 // vocab))
    return dict(op=op, rows=rows, vocab=vocab, dtype=rng.choice(["f32", "f16", "bf16"]), k=rng.choice([0, 1, 5, 20, 32]),
                pad=rng.choice([0, rows // 8]), masked=rng.choice([0.0, 0.0, 0.5, 0.95]),
                temperature=rng.choice([0.6, 1.0, 1.3]))


def _amax(x, block_rows):
    """The largest magnitude of each block_rows x 128 block of x, in 32 bits."""
    r, c = x.shape
    x = torch.nn.functional.pad(x.float().abs(), (0, -c % BLOCK, 0, -r % block_rows))
    x = x.view(x.shape[0] // block_rows, block_rows, x.shape[1] // BLOCK, BLOCK)
    return x.amax(dim=(1, 3)).clamp_min(TINY)


def _spread(s, block_rows, rows, cols):
    """A value of each block, at each element of the block."""
    return s.repeat_interleave(block_rows, 0)[:rows].repeat_interleave(BLOCK, 1)[:, :cols]


def _quantize(x, block_rows):
    r, c = x.shape
    a = _amax(x, block_rows)
    q = (x.float() * _spread(E4M3_MAX / a, block_rows, r, c)).to(torch.float8_e4m3fn)
    return q, a / E4M3_MAX


def _values(g, rows, cols):
    """Normal values whose size differs from column to column, as hidden states' does."""
    x = torch.randn(rows, cols, generator=g, device=DEV)
    return x.mul_(torch.exp(0.5 * torch.randn(cols, generator=g, device=DEV)))


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    s = dict(case)
    if case["op"] == "quantize":
        s["x"] = _values(g, case["rows"], case["cols"]).to(TYPES[case["dtype"]])
    elif case["op"] == "product":
        m, n, k = case["m"], case["n"], case["k"]
        for name, rows, br in (("a", m, 1), ("w", n, BLOCK)):
            q, sc = _quantize(_values(g, rows, k) if name == "a" else 0.02 * torch.randn(rows, k, generator=g, device=DEV), br)
            # rows 16-byte aligned, as the library lays out its own 8-bit matrices
            held = torch.zeros(rows, -(-k // 16) * 16, dtype=torch.uint8, device=DEV)
            held[:, :k] = q.view(torch.uint8)
            s[name], s["s" + name] = held.view(torch.float8_e4m3fn), sc
        s["bias_v"] = torch.randn(n, generator=g, device=DEV) if case["bias"] else None
    else:
        rows, vocab = case["rows"], case["vocab"]
        x = torch.randn(rows, vocab, generator=g, device=DEV, dtype=torch.float32).mul_(2.5)
        target = torch.randint(0, vocab, (rows,), generator=g, device=DEV)
        x[torch.arange(rows, device=DEV), target] += 6.0  # given tokens are mostly likely ones
        x = x.to(TYPES[case["dtype"]])
        if case["masked"]:
            out = torch.rand(vocab, generator=g, device=DEV) < case["masked"]
            out[target[0]] = False  # a grammar always allows some token
            x.masked_fill_(out, -math.inf)
        if case["pad"]:
            target[rows - case["pad"]:] = -1
        s["x"], s["target"] = x, target
    return s


def _order(x):
    """64-bit keys in the order of (value, then lowest index first)."""
    bits = (x + 0.0).view(torch.int32).long()
    bits = torch.where(bits >= 0, bits, -2147483648 - bits)
    return bits * 4294967296 + (4294967295 - torch.arange(x.shape[1], device=x.device))


def _plain_logprobs(x, target, k, temperature):
    x = x.float()
    m = x.amax(1, keepdim=True)
    d = (x - m) / temperature
    e = torch.exp(d)
    total = e.sum(1, keepdim=True)
    log_total = torch.log(total)
    entropy = (log_total - (e * torch.where(e > 0, d, 0.0)).sum(1, keepdim=True) / total)[:, 0]
    pad = target < 0
    logprob = (d.gather(1, target.clamp_min(0)[:, None]) - log_total)[:, 0]
    out = dict(logprob=logprob.masked_fill(pad, 0.0), entropy=entropy.masked_fill(pad, 0.0))
    if k:
        top = 4294967295 - torch.topk(_order(x), k, dim=1).values % 4294967296
        out["top_logprob"] = (d.gather(1, top) - log_total).masked_fill(pad[:, None], -math.inf)
        out["top_id"] = top.masked_fill(pad[:, None], -1)
    return out


def _gelu(x):
    return 0.5 * x * (1.0 + torch.erf(x / math.sqrt(2.0)))


def _act(x, act):
    return torch.relu(x) if act == "relu" else _gelu(x) if act == "gelu" else x


def _plain(s):
    if s["op"] == "quantize":
        return _quantize(s["x"], s["block_rows"])
    if s["op"] == "product":
        m, n, k = s["m"], s["n"], s["k"]
        a = s["a"][:, :k].float() * _spread(s["sa"], 1, m, k)
        w = s["w"][:, :k].float() * _spread(s["sw"], BLOCK, n, k)
        y = a @ w.t()
        if s["bias_v"] is not None:
            y = y + s["bias_v"]
        return _act(y, s["act"]).to(TYPES[s["out"]])
    return _plain_logprobs(s["x"], s["target"], s["k"], s["temperature"])


_contexts = {}


def _context():
    """The library's context on torch's current stream: made once per stream."""
    from onnx_b200.tensor import Context
    device, stream = torch.cuda.current_device(), torch.cuda.current_stream().cuda_stream
    if (device, stream) not in _contexts:
        _contexts[device, stream] = Context(device, stream=stream)
    return _contexts[device, stream]


def _own(s):
    from onnx_b200 import scoring
    from onnx_b200.tensor import BFLOAT16, FLOAT8E4M3, DeviceTensor
    import numpy as np
    ctx = _context()
    types = {torch.float32: np.float32, torch.float16: np.float16, torch.bfloat16: BFLOAT16,
             torch.float8_e4m3fn: FLOAT8E4M3, torch.int64: np.int64}

    def dev(t):
        return None if t is None else DeviceTensor(ctx, t.shape, types[t.dtype], ptr=t.data_ptr(), owner=t)

    if s["op"] == "quantize":
        r, c, br = s["rows"], s["cols"], s["block_rows"]
        q = torch.empty(r, c, dtype=torch.float8_e4m3fn, device=DEV)
        scale = torch.empty(-(-r // br), -(-c // BLOCK), device=DEV)
        scoring.quantize_fp8(dev(s["x"]), block_rows=br, out=(dev(q), dev(scale)))
        return q, scale
    if s["op"] == "product":
        a = scoring.Fp8Matrix(dev(s["a"]), dev(s["sa"]), s["k"], 1)
        w = scoring.Fp8Matrix(dev(s["w"]), dev(s["sw"]), s["k"], BLOCK)
        y = torch.empty(s["m"], s["n"], dtype=TYPES[s["out"]], device=DEV)
        scoring.matmul_fp8(a, w, bias=dev(s["bias_v"]), activation=s["act"], out=dev(y))
        return y
    rows, k = s["rows"], s["k"]
    out = dict(logprob=torch.empty(rows, device=DEV), entropy=torch.empty(rows, device=DEV))
    if k:
        out["top_logprob"] = torch.empty(rows, k, device=DEV)
        out["top_id"] = torch.empty(rows, k, dtype=torch.int64, device=DEV)
    scoring.token_logprobs(dev(s["x"]), dev(s["target"]), k=k, temperature=s["temperature"],
                           out={name: dev(t) for name, t in out.items()})
    return out


def run(state):
    return _own(state) if own else _plain(state)


def work(case):
    size = {"f32": 4, "f16": 2, "bf16": 2}
    if case["op"] == "quantize":
        r, c, br = case["rows"], case["cols"], case["block_rows"]
        return {"bytes": r * c * (size[case["dtype"]] + 1) + 4 * -(-r // br) * -(-c // BLOCK), "flops": 2 * r * c}
    if case["op"] == "product":
        m, n, k = case["m"], case["n"], case["k"]
        kb = -(-k // BLOCK)
        return {"bytes": (m + n) * k + 4 * kb * (m + -(-n // BLOCK)) + m * n * size[case["out"]] + (4 * n if case["bias"] else 0),
                "flops": 2 * m * n * k}
    rows, v, k = case["rows"], case["vocab"], case["k"]
    held = rows - case["pad"]
    return {"bytes": held * v * size[case["dtype"]] + rows * (16 + 12 * k), "flops": 5 * held * v}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "quantize":
        # scales in 64 bits; an 8-bit value has the nearest representable one as its definition
        x, br = s["x"].double(), case["block_rows"]
        rows, cols = x.shape
        nr, nc = -(-rows // br), -(-cols // BLOCK)
        tall = torch.zeros(nr * br, nc * BLOCK, dtype=torch.float64, device=DEV)
        tall[:rows, :cols] = x.abs()
        amax = tall.reshape(nr, br, nc, BLOCK).permute(0, 2, 1, 3).flatten(2).max(2).values.clamp(min=TINY)
        del tall
        i = torch.arange(rows, device=DEV) // br
        j = torch.arange(cols, device=DEV) // BLOCK
        t = x * (E4M3_MAX / amax)[i][:, j]
        # steps of e4m3: 2^(exponent - 3), 2^-9 below the normal range
        step = torch.exp2(torch.frexp(t)[1].double().sub(1).clamp(min=-6) - 3)
        return torch.round(t / step) * step, amax / E4M3_MAX
    if case["op"] == "product":
        m, n, k = case["m"], case["n"], case["k"]
        y = torch.zeros(m, n, dtype=torch.float64, device=DEV)
        row = torch.arange(n, device=DEV) // BLOCK
        for b in range(-(-k // BLOCK)):
            at = slice(b * BLOCK, min(k, (b + 1) * BLOCK))
            part = (s["a"][:, at].double() * s["sa"][:, b].double()[:, None]) @ s["w"][:, at].double().t()
            y += part * s["sw"][row, b].double()
            del part
        if s["bias_v"] is not None:
            y += s["bias_v"].double()
        if case["act"] == "relu":
            y = y.clamp(min=0)
        elif case["act"] == "gelu":
            y = y * 0.5 * torch.special.erfc(-y * 0.5 ** 0.5)
        return y
    parts = []
    for x, target in zip(s["x"].split(256), s["target"].split(256)):
        z = x.double() / case["temperature"]
        lse = torch.logsumexp(z, 1)
        p = torch.exp(z - lse[:, None])
        entropy = -torch.special.xlogy(p, p).sum(1)
        pad = target < 0
        got = [torch.where(pad, 0.0, z[torch.arange(len(x), device=DEV), target.clamp(min=0)] - lse),
               torch.where(pad, 0.0, entropy)]
        if case["k"]:
            top = z.topk(case["k"], dim=1).values - lse[:, None]
            got.append(torch.where(pad[:, None], -math.inf, top))
        parts.append(got)
    cat = [torch.cat(t) for t in zip(*parts)]
    out = dict(logprob=cat[0], entropy=cat[1])
    if case["k"]:
        out["top_logprob"], out["top_id"] = cat[2], None
    return out
