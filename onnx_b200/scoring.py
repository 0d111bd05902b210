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
of include/lonnx.h, which has the formulas).  A tensor to write (``out``)
overlaps no other tensor of its call.
"""
from __future__ import annotations

from dataclasses import dataclass

import numpy as np

from . import _native as N
from .tensor import BFLOAT16, FLOAT8E4M3, ONNX_DTYPE, Context, DeviceTensor

BLOCK = 128          # columns of a quantisation block, and rows of a weight's
MAX_ALTERNATIVES = 32
MAX_SIZE = 1 << 30  # of a product, each way (32-bit arguments of the library)
F32, I64 = (np.dtype(np.float32),), (np.dtype(np.int64),)
FP8 = (FLOAT8E4M3,)
FLOAT_TYPES = F32 + (np.dtype(np.float16), BFLOAT16)
ACTIVATIONS = {None: 0, "none": 0, "relu": 1, "gelu": 2}

_quantize, _gemm, _logprobs = N.lib.lonnx_quantize_fp8, N.lib.lonnx_gemm_fp8, N.lib.lonnx_token_logprobs


def _need(t, what: str, ctx: Context, dtypes, shape=None) -> None:
    """Refuses a ``t`` that is not a tensor on this context's stream, of these
    types and of this shape (None: any matrix)."""
    if isinstance(t, DeviceTensor) and t.ctx is ctx and t.dtype in dtypes and \
            (t.shape == shape if shape is not None else len(t.shape) == 2):
        return
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
    ctx = getattr(x, "ctx", None)
    _need(x, "x", ctx, FLOAT_TYPES)
    if block_rows != 1 and block_rows != BLOCK:
        raise ValueError(f"block_rows: 1 or {BLOCK}, got {block_rows}")
    rows, cols = x.shape
    scales = (-(-rows // block_rows), -(-cols // BLOCK))
    if out is None:
        out = (DeviceTensor(ctx, (rows, -(-cols // 16) * 16), FLOAT8E4M3), DeviceTensor(ctx, scales, F32[0]))
    q, scale = out
    _need(q, "out q", ctx, FP8)
    _need(scale, "out scale", ctx, F32, scales)
    ldq = q.shape[1]
    if q.shape[0] != rows or ldq < cols:
        raise ValueError(f"out q: expected [{rows}, >= {cols}], got {q.shape}")
    rc = _quantize(ctx.handle, x.ptr, ONNX_DTYPE[x.dtype], rows, cols, cols, block_rows, q.ptr, ldq, scale.ptr, scales[1])
    if rc:
        N.check(rc)
    return Fp8Matrix(q, scale, cols, block_rows)


def matmul_fp8(a: Fp8Matrix, w: Fp8Matrix, bias: DeviceTensor | None = None, activation: str | None = None,
               dtype=None, out: DeviceTensor | None = None) -> DeviceTensor:
    """act(a . w^T + bias) [a.rows, w.rows] from activations ``a``
    (``block_rows=1``) and weights ``w`` (``block_rows=128``) over the same
    columns; ``activation``: None, "relu" or "gelu"; ``dtype``: the result's,
    float32 where neither it nor ``out`` says another."""
    ctx = a.q.ctx
    if a.block_rows != 1 or w.block_rows != BLOCK:
        raise ValueError(f"blocks of {a.block_rows} and {w.block_rows} rows: a needs 1, w {BLOCK}")
    k = a.cols
    if k != w.cols:
        raise ValueError(f"a has {k} columns, w {w.cols}")
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation: None, 'relu' or 'gelu', got {activation!r}")
    _need(a.q, "a", ctx, FP8)
    _need(w.q, "w", ctx, FP8)
    (m, lda), (n, ldw) = a.q.shape, w.q.shape
    if max(m, n, k) > MAX_SIZE:
        raise ValueError(f"{m} x {n} x {k}: at most 2^30 each")
    kb = -(-k // BLOCK)
    _need(a.scale, "a scale", ctx, F32, (m, kb))
    _need(w.scale, "w scale", ctx, F32, (-(-n // BLOCK), kb))
    if lda < k or ldw < k or lda % 16 or ldw % 16:
        raise ValueError(f"a and w: rows of {lda} and {ldw} bytes (at least {k}, multiples of 16)")
    if bias is not None:
        _need(bias, "bias", ctx, F32, (n,))
    if out is None:
        out = DeviceTensor(ctx, (m, n), F32[0] if dtype is None else dtype)
    _need(out, "out", ctx, FLOAT_TYPES, (m, n))
    if dtype is not None and np.dtype(dtype) != out.dtype:
        raise ValueError(f"dtype: {np.dtype(dtype)} asked for, out has {out.dtype}")
    rc = _gemm(ctx.handle, a.q.ptr, lda, a.scale.ptr, kb, w.q.ptr, ldw, w.scale.ptr, kb,
               None if bias is None else bias.ptr, out.ptr, ONNX_DTYPE[out.dtype], n, m, n, k, ACTIVATIONS[activation])
    if rc:
        N.check(rc)
    return out


def token_logprobs(logits: DeviceTensor, targets: DeviceTensor | None = None, k: int = 0, temperature: float = 1.0,
                   vocab: int | None = None, out: dict | None = None) -> dict:
    """Scores of ``logits`` [rows, vocab]: a dict of ``entropy`` [rows], with
    ``targets`` (int64 [rows], negative for a padding row) ``logprob`` [rows],
    and with ``k`` (at most 32) the likeliest tokens, ``top_logprob`` [rows, k]
    and ``top_id`` (int64).  ``vocab``: the columns to read, where the rows are
    wider than the vocabulary.  ``out``: tensors to write, by the same names;
    one that is left out is not computed (the alternatives come in pairs)."""
    ctx = getattr(logits, "ctx", None)
    _need(logits, "logits", ctx, FLOAT_TYPES)
    rows, ld = logits.shape
    vocab = ld if vocab is None else int(vocab)
    if not 1 <= vocab <= ld:
        raise ValueError(f"vocab: 1 to {ld}, got {vocab}")
    if not 0 <= k <= min(MAX_ALTERNATIVES, vocab):
        raise ValueError(f"k: 0 to {min(MAX_ALTERNATIVES, vocab)}, got {k}")
    each, top = (rows,), (rows, k)
    if targets is not None:
        _need(targets, "targets", ctx, I64, each)
    if out is None:
        out = {"entropy": DeviceTensor(ctx, each, F32[0])}
        if targets is not None:
            out["logprob"] = DeviceTensor(ctx, each, F32[0])
        if k:
            out["top_logprob"], out["top_id"] = DeviceTensor(ctx, top, F32[0]), DeviceTensor(ctx, top, I64[0])
    ptr = dict.fromkeys(("logprob", "entropy", "top_logprob", "top_id"))
    for name, t in out.items():
        if name not in ptr or (name == "logprob" and targets is None) or (name[0] == "t" and not k):
            raise ValueError(f"out: {name!r} is not an output of this call")
        _need(t, name, ctx, I64 if name == "top_id" else F32, top if name[0] == "t" else each)
        ptr[name] = t.ptr
    if k and (ptr["top_logprob"] is None or ptr["top_id"] is None):
        raise ValueError("out: top_logprob and top_id are both needed with k > 0")
    rc = _logprobs(ctx.handle, logits.ptr, ONNX_DTYPE[logits.dtype], rows, vocab, ld,
                   None if targets is None else targets.ptr, float(temperature), ptr["logprob"], ptr["entropy"], k,
                   ptr["top_logprob"], ptr["top_id"])
    if rc:
        N.check(rc)
    return out
