"""The output end of a language model: hidden states to the scores of tokens.

``quantize_fp8`` turns weights (once, ``block_rows=128``) and activations
(each step, ``block_rows=1``) into 8-bit floats with one scale per block,
``matmul_fp8`` multiplies the two on the tensor cores, and ``token_logprobs``
reads the logits once for the log-probabilities of given tokens, the entropy
and the likeliest alternatives:

    head = quantize_fp8(embedding, block_rows=128)           # [vocab, hidden]
    logits = matmul_fp8(quantize_fp8(hidden), head)          # [tokens, vocab]
    scores = token_logprobs(logits, targets, k=5)

All take and give ``DeviceTensor``s and only enqueue work on the context's
stream (``lonnx_quantize_fp8``, ``lonnx_gemm_fp8``, ``lonnx_token_logprobs``
of include/lonnx.h, which has the formulas).
"""
from __future__ import annotations

from dataclasses import dataclass

import numpy as np

from . import _native as N
from .tensor import BFLOAT16, FLOAT8E4M3, ONNX_DTYPE, Context, DeviceTensor

BLOCK = 128          # columns of a quantisation block, and rows of a weight's
MAX_ALTERNATIVES = 32
FLOAT_TYPES = (np.dtype(np.float32), np.dtype(np.float16), BFLOAT16)
ACTIVATIONS = {None: 0, "none": 0, "relu": 1, "gelu": 2}


def _ceil(a: int, b: int) -> int:
    return -(-a // b)


def _need(t, what: str, ctx: Context, dtypes, shape=None) -> DeviceTensor:
    """``t`` if it is a tensor of this context's device, of these types and shape."""
    if not isinstance(t, DeviceTensor):
        raise TypeError(f"{what}: expected a DeviceTensor, got {type(t).__name__}")
    if t.ctx is not ctx and (t.ctx.device != ctx.device or t.ctx.stream != ctx.stream):
        raise ValueError(f"{what}: on another context's stream or device")
    if t.dtype not in dtypes:
        raise ValueError(f"{what}: type {t.dtype} is not supported")
    if shape is None and len(t.shape) != 2:
        raise ValueError(f"{what}: expected a matrix, got shape {t.shape}")
    if shape is not None and t.shape != shape:
        raise ValueError(f"{what}: expected shape {shape}, got {t.shape}")
    return t


@dataclass
class Fp8Matrix:
    """A block-quantised matrix [rows, cols]: ``q`` [rows, >= cols] holds e4m3
    values (columns past ``cols`` are alignment padding), ``scale`` one float
    per block of ``block_rows`` x 128."""
    q: DeviceTensor
    scale: DeviceTensor
    cols: int
    block_rows: int

    @property
    def rows(self) -> int:
        return self.q.shape[0]


def quantize_fp8(x: DeviceTensor, block_rows: int = 1, out=None) -> Fp8Matrix:
    """``x`` [rows, cols] (float32, float16, bfloat16) in 8 bits, with a scale
    per 1 x 128 (``block_rows=1``) or 128 x 128 block.  ``out``: (q, scale) to
    write; otherwise they are made, with rows of ``q`` 16-byte aligned as
    ``matmul_fp8`` needs them."""
    if not isinstance(x, DeviceTensor):
        raise TypeError(f"x: expected a DeviceTensor, got {type(x).__name__}")
    ctx = x.ctx
    _need(x, "x", ctx, FLOAT_TYPES)
    if block_rows not in (1, BLOCK):
        raise ValueError(f"block_rows: 1 or {BLOCK}, got {block_rows}")
    rows, cols = x.shape
    scales = (_ceil(rows, block_rows), _ceil(cols, BLOCK))
    if out is None:
        out = (DeviceTensor(ctx, (rows, _ceil(cols, 16) * 16), FLOAT8E4M3), DeviceTensor(ctx, scales, np.float32))
    q, scale = out
    _need(q, "out q", ctx, (FLOAT8E4M3,))
    _need(scale, "out scale", ctx, (np.dtype(np.float32),), scales)
    if q.shape[0] != rows or q.shape[1] < cols:
        raise ValueError(f"out q: expected [{rows}, >= {cols}], got {q.shape}")
    N.check(N.lib.lonnx_quantize_fp8(ctx.handle, x.ptr, ONNX_DTYPE[x.dtype], rows, cols, cols, block_rows, q.ptr,
                                     q.shape[1], scale.ptr, scales[1]))
    return Fp8Matrix(q, scale, cols, block_rows)


def matmul_fp8(a: Fp8Matrix, w: Fp8Matrix, bias: DeviceTensor | None = None, activation: str | None = None,
               dtype=np.float32, out: DeviceTensor | None = None) -> DeviceTensor:
    """act(a . w^T + bias) [a.rows, w.rows] from activations ``a``
    (``block_rows=1``) and weights ``w`` (``block_rows=128``) over the same
    columns; ``activation``: None, "relu" or "gelu"."""
    ctx = a.q.ctx
    if a.block_rows != 1 or w.block_rows != BLOCK:
        raise ValueError(f"blocks of {a.block_rows} and {w.block_rows} rows: a needs 1, w {BLOCK}")
    if a.cols != w.cols:
        raise ValueError(f"a has {a.cols} columns, w {w.cols}")
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation: None, 'relu' or 'gelu', got {activation!r}")
    m, n, k = a.rows, w.rows, a.cols
    kb = _ceil(k, BLOCK)
    f32 = np.dtype(np.float32)
    for x, what, rows in ((a, "a", m), (w, "w", _ceil(n, BLOCK))):
        _need(x.q, what, ctx, (FLOAT8E4M3,))
        _need(x.scale, f"{what} scale", ctx, (f32,), (rows, kb))
        if x.q.shape[1] < k or x.q.shape[1] % 16:
            raise ValueError(f"{what}: rows of {x.q.shape[1]} bytes (at least {k}, a multiple of 16)")
    if bias is not None:
        _need(bias, "bias", ctx, (f32,), (n,))
    if out is None:
        out = DeviceTensor(ctx, (m, n), dtype)
    _need(out, "out", ctx, FLOAT_TYPES, (m, n))
    N.check(N.lib.lonnx_gemm_fp8(ctx.handle, a.q.ptr, a.q.shape[1], a.scale.ptr, kb, w.q.ptr, w.q.shape[1],
                                 w.scale.ptr, kb, bias.ptr if bias is not None else None, out.ptr,
                                 ONNX_DTYPE[out.dtype], n, m, n, k, ACTIVATIONS[activation]))
    return out


def token_logprobs(logits: DeviceTensor, targets: DeviceTensor | None = None, k: int = 0, temperature: float = 1.0,
                   vocab: int | None = None, out: dict | None = None) -> dict:
    """Scores of ``logits`` [rows, vocab]: a dict of ``entropy`` [rows], with
    ``targets`` (int64 [rows], negative for a padding row) ``logprob`` [rows],
    and with ``k`` (at most 32) the likeliest tokens, ``top_logprob`` [rows, k]
    and ``top_id`` (int64).  ``vocab``: the columns to read, where the rows are
    wider than the vocabulary.  ``out``: tensors to write, by the same names;
    one that is left out is not computed (the alternatives come in pairs)."""
    if not isinstance(logits, DeviceTensor):
        raise TypeError(f"logits: expected a DeviceTensor, got {type(logits).__name__}")
    ctx = logits.ctx
    _need(logits, "logits", ctx, FLOAT_TYPES)
    rows, ld = logits.shape
    vocab = ld if vocab is None else int(vocab)
    if not 1 <= vocab <= ld:
        raise ValueError(f"vocab: 1 to {ld}, got {vocab}")
    if not 0 <= k <= min(MAX_ALTERNATIVES, vocab):
        raise ValueError(f"k: 0 to {min(MAX_ALTERNATIVES, vocab)}, got {k}")
    f32, i64 = np.dtype(np.float32), np.dtype(np.int64)
    if targets is not None:
        _need(targets, "targets", ctx, (i64,), (rows,))
    kinds = {"entropy": ((rows,), f32)}
    if targets is not None:
        kinds["logprob"] = ((rows,), f32)
    if k:
        kinds["top_logprob"], kinds["top_id"] = ((rows, k), f32), ((rows, k), i64)
    if out is None:
        out = {name: DeviceTensor(ctx, shape, dt) for name, (shape, dt) in kinds.items()}
    for name, t in out.items():
        if name not in kinds:
            raise ValueError(f"out: {name!r} is not an output of this call ({', '.join(sorted(kinds))})")
        _need(t, f"out {name}", ctx, (kinds[name][1],), kinds[name][0])
    if k and not ("top_logprob" in out and "top_id" in out):
        raise ValueError("out: top_logprob and top_id are both needed with k > 0")

    def ptr(name):
        return out[name].ptr if name in out else None

    N.check(N.lib.lonnx_token_logprobs(ctx.handle, logits.ptr, ONNX_DTYPE[logits.dtype], rows, vocab, ld,
                                       targets.ptr if targets is not None else None, float(temperature),
                                       ptr("logprob"), ptr("entropy"), k, ptr("top_logprob"), ptr("top_id")))
    return out
