"""Memory of a context's allocator that is used while the caller records the
stream into a CUDA graph: no later tensor gets it while the graph can still be
replayed, and it comes back when the graph is gone."""
import gc
import time

import numpy as np
import pytest
import torch

from onnx_b200 import _native as N
from onnx_b200 import scoring
from onnx_b200.tensor import Context, DeviceTensor
from test_scoring_gpu import dev, gen, randn, score

pytestmark = pytest.mark.gpu
SIZE = (1000, 77)


@pytest.fixture
def stream():
    return torch.cuda.Stream()


@pytest.fixture
def sctx(stream):
    return Context(0, stream=stream.cuda_stream)


def warm(ctx, n=4, shape=SIZE):
    """Blocks of that size in the context's cache, so that a recording finds them."""
    held = [DeviceTensor(ctx, shape, np.float32) for _ in range(n)]
    return {t.ptr for t in held}


def fill(ctx, t, byte):
    N.check(N.lib.lonnx_memset(ctx.handle, t.ptr, byte, t.nbytes))


def tensors(ctx, n, shape=SIZE):
    """n tensors, each with its number in every byte."""
    held = [DeviceTensor(ctx, shape, np.float32) for _ in range(n)]
    for i, t in enumerate(held):
        fill(ctx, t, i + 1)
    return held


def untouched(held):
    return all((t.to_host().view(np.uint8) == i + 1).all() for i, t in enumerate(held))


def until_reused(ctx, ptr, shape=SIZE, seconds=20):
    """Whether a new tensor gets that address within some seconds (a graph's end
    is told from a thread of the driver's)."""
    end = time.time() + seconds
    while time.time() < end:
        held = [DeviceTensor(ctx, shape, np.float32) for _ in range(8)]
        if ptr in {t.ptr for t in held}:
            return True
        del held
        time.sleep(0.05)
    return False


def test_results_let_go_of_after_the_recording(sctx, stream):
    """The whole scoring run recorded; its logits and scores are dropped before new tensors are made."""
    tokens, hidden, vocab = 6, 384, 4001
    h, w = randn(tokens, hidden, seed=1), randn(vocab, hidden, seed=2) * 0.05
    target = torch.randint(0, vocab, (tokens,), generator=gen(3), device="cuda")
    torch.cuda.synchronize()
    head = scoring.quantize_fp8(dev(sctx, w), block_rows=128)
    score(sctx, h, head, target, 3)
    sctx.sync()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        got, logits = score(sctx, h, head, target, 3)
    del got, logits
    later = tensors(sctx, 3, (tokens, vocab)) + tensors(sctx, 6, (tokens,))
    for i, t in enumerate(later):
        fill(sctx, t, i + 1)
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    assert untouched(later)


def test_block_of_one_recording_let_go_of_in_another(sctx, stream):
    """What a first recording made is not used by a second that drops it: the two graphs share nothing."""
    warm(sctx)
    one, two = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(one, stream=stream):
        a = DeviceTensor(sctx, SIZE, np.float32)
        fill(sctx, a, 9)
    ptr = a.ptr
    with torch.cuda.graph(two, stream=stream):
        del a
        b = DeviceTensor(sctx, SIZE, np.float32)
        fill(sctx, b, 5)
    assert b.ptr != ptr
    two.replay()
    one.replay()
    torch.cuda.synchronize()
    assert (b.to_host().view(np.uint8) == 5).all()


def test_a_recording_uses_its_own_blocks_again(sctx, stream):
    ptrs = warm(sctx, 1)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        for i in range(5):
            t = DeviceTensor(sctx, SIZE, np.float32)
            assert t.ptr in ptrs
            fill(sctx, t, i)
            del t
    later = tensors(sctx, 4)
    graph.replay()
    torch.cuda.synchronize()
    assert untouched(later) and not ptrs & {t.ptr for t in later}


@pytest.mark.parametrize("drop", ["during", "after", "once the graph is gone"])
def test_blocks_come_back_when_the_graph_is_gone(sctx, stream, drop):
    warm(sctx, 1)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        t = DeviceTensor(sctx, SIZE, np.float32)
        fill(sctx, t, 3)
        ptr = t.ptr
        if drop == "during":
            del t
    if drop == "after":
        del t
    graph.replay()
    torch.cuda.synchronize()
    if drop != "once the graph is gone":
        assert not until_reused(sctx, ptr, seconds=0.5)
    graph.reset()
    del graph
    gc.collect()
    if drop == "once the graph is gone":
        assert not until_reused(sctx, ptr, seconds=0.5)  # its owner still has it
        assert (t.to_host().view(np.uint8) == 3).all()
        del t
    assert until_reused(sctx, ptr)


def test_two_graphs_of_one_block(sctx, stream):
    """A block that two recordings had comes back when both are gone."""
    warm(sctx, 2)
    one, two = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(one, stream=stream):
        a = DeviceTensor(sctx, SIZE, np.float32)
        fill(sctx, a, 1)
    with torch.cuda.graph(two, stream=stream):
        fill(sctx, a, 2)
        ptr = a.ptr
        del a
    one.reset()
    assert not until_reused(sctx, ptr, seconds=1)
    two.reset()
    assert until_reused(sctx, ptr)


def test_many_recordings_do_not_grow_the_context(sctx, stream):
    """One graph after another, each of which lets its logits go: the memory is the same."""
    shape = (64, 250037)
    warm(sctx, 1, shape)
    sctx.sync()

    def record():
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            t = DeviceTensor(sctx, shape, np.float32)
            fill(sctx, t, 1)
            ptr = t.ptr
            del t
        graph.replay()
        torch.cuda.synchronize()
        graph.reset()
        return ptr

    assert until_reused(sctx, record(), shape)  # (leaves 8 blocks in the cache)
    free = torch.cuda.mem_get_info()[0]
    for _ in range(12):
        assert until_reused(sctx, record(), shape)
    assert torch.cuda.mem_get_info()[0] > free - (64 << 20)


def test_scratch_of_a_recorded_call(sctx, stream):
    """A recorded product's scratch is grown by a later one: the old one is not
    given to a tensor while the graph lives."""
    m, n, k = 256, 512, 256
    a, b = randn(m, k, seed=1), randn(k, n, seed=2)
    c, wide = torch.empty(m, n, device="cuda"), randn(k, 8 * n, seed=3)
    wide_c = torch.empty(m, 8 * n, device="cuda")
    torch.cuda.synchronize()

    def product(w, out):
        N.check(N.lib.lonnx_gemm_f32(sctx.handle, a.data_ptr(), w.data_ptr(), None, out.data_ptr(), 1, m, w.shape[1], k, 0,
                                     0, 0, 0, 1.0, 0.0, 0))
    product(b, c)
    sctx.sync()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        product(b, c)
    product(wide, wide_c)
    later = tensors(sctx, 4, (2 * k, n))
    graph.replay()
    torch.cuda.synchronize()
    assert untouched(later)
    assert torch.allclose(c, a @ b, atol=1e-3)


def test_eager_blocks_are_reused_as_before(sctx):
    ptrs = warm(sctx, 3)
    t = [DeviceTensor(sctx, SIZE, np.float32) for _ in range(3)]
    assert {x.ptr for x in t} == ptrs


def test_context_closed_before_its_graph(stream):
    """The context goes while a graph that it was recorded into lives: the graph
    is then only destroyed, which touches nothing of the context."""
    ctx = Context(0, stream=stream.cuda_stream)
    warm(ctx, 1)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        t = DeviceTensor(ctx, SIZE, np.float32)
        fill(ctx, t, 1)
        del t
    torch.cuda.synchronize()
    ctx.close()
    graph.reset()
    del graph
    gc.collect()
    time.sleep(0.3)
    other = Context(0, stream=stream.cuda_stream)
    assert untouched(tensors(other, 2))
