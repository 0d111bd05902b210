// The output end of a language model on the GPU: block quantisation to 8-bit
// float, the block-scaled product and the scores of tokens
// (lonnx_quantize_fp8, lonnx_gemm_fp8, lonnx_token_logprobs).  The managed
// counterpart of onnx_b200/scoring.py: operands are DeviceBuffers, calls only
// enqueue work on the context's stream.
namespace Lokad.Onnx.Cuda;

using System;

/// <summary>A block-quantised matrix: e4m3 values in rows of Ld bytes, one float per block of BlockRows x 128.</summary>
public sealed class Fp8Matrix
{
    public DeviceBuffer Q { get; init; } = null!;
    public DeviceBuffer Scale { get; init; } = null!;
    public int Rows { get; init; }
    public int Cols { get; init; }
    public long Ld { get; init; }
    public int BlockRows { get; init; }
    public long ScaleLd => ((long)Cols + 127) / 128;
}

public static class Scoring
{
    public const int Block = 128, MaxAlternatives = 32;

    /// <summary>x [rows, cols] of element type dtype (Native.DT_*) in 8 bits; blockRows: 1 (activations) or 128 (weights).</summary>
    public static Fp8Matrix Quantize(CudaContext ctx, IntPtr x, int dtype, int rows, int cols, int blockRows = 1)
    {
        if (blockRows != 1 && blockRows != Block) throw new ArgumentException($"blockRows: 1 or {Block}, got {blockRows}");
        long ld = ((long)cols + 15) / 16 * 16, scales = ((long)cols + Block - 1) / Block;
        var m = new Fp8Matrix
        {
            Q = new DeviceBuffer(ctx, (long)rows * ld),
            Scale = new DeviceBuffer(ctx, ((long)rows + blockRows - 1) / blockRows * scales * sizeof(float)),
            Rows = rows, Cols = cols, Ld = ld, BlockRows = blockRows
        };
        Native.Check(Native.lonnx_quantize_fp8(ctx.Handle, x, dtype, rows, cols, cols, blockRows, m.Q.Ptr, ld,
            m.Scale.Ptr, scales));
        return m;
    }

    /// <summary>
    /// act(a . w^T + bias) [a.Rows, w.Rows] into c (element type dtype, rows ldc elements apart, 0: w.Rows); bias:
    /// floats or IntPtr.Zero.
    /// </summary>
    public static void MatMul(CudaContext ctx, Fp8Matrix a, Fp8Matrix w, IntPtr bias, IntPtr c, int dtype,
        int epilogue = 0, long ldc = 0)
    {
        if (a.BlockRows != 1 || w.BlockRows != Block || a.Cols != w.Cols)
            throw new ArgumentException("a has blocks of 1 row, w of 128, over the same columns");
        Native.Check(Native.lonnx_gemm_fp8(ctx.Handle, a.Q.Ptr, a.Ld, a.Scale.Ptr, a.ScaleLd, w.Q.Ptr, w.Ld, w.Scale.Ptr,
            w.ScaleLd, bias, c, dtype, ldc == 0 ? w.Rows : ldc, a.Rows, w.Rows, a.Cols, epilogue));
    }

    /// <summary>
    /// Log-probabilities of `targets` (int64 per row, negative: a padding row; IntPtr.Zero: none), entropies and
    /// the k likeliest tokens of logits [rows, vocab], rows ld elements apart (0: vocab); an output that is
    /// IntPtr.Zero is not computed.
    /// </summary>
    public static void TokenLogprobs(CudaContext ctx, IntPtr logits, int dtype, int rows, int vocab, IntPtr targets,
        IntPtr logprob, IntPtr entropy, int k = 0, IntPtr topLogprob = default, IntPtr topId = default,
        float temperature = 1.0f, long ld = 0)
    {
        Native.Check(Native.lonnx_token_logprobs(ctx.Handle, logits, dtype, rows, vocab, ld == 0 ? vocab : ld, targets, temperature,
            logprob, entropy, k, topLogprob, topId));
    }
}
