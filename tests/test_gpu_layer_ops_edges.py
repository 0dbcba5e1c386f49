"""The operators of a training step around the matrix products, on the GPU, at
the sizes, layouts and values where they can go wrong: kernels that walk many
rows or chunks, capped scores that fp32 resolves, results in another type than
the scores, overlapping operands, calls from several threads.

Tolerances as in test_gpu_layer_ops: bounds in fp32 carried along, u = 2^-24 a
rounding, and half a step of the stored type.
"""

import math

import numpy as np
import pytest
import torch

import torch_fl
from torch_fl import kernels as K

from .test_gpu_layer_ops import (DEV, TYPES, U, Num, check_rotary, close, gen, np64, random_spans,
                                 span_back_want)

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------- span softmax
def capped_want(x, spans, scale, cap):
    """softmax of cap * tanh(scale x / cap) over each span, and what fp32 may
    be off: scale / cap and its product with x are rounded (the tanh passes on
    u (1 - tanh^2) of that), tanhf is good to 2 units in the last place, its
    product with the cap is rounded."""
    n = x.shape[-1]
    key = np.arange(n)
    lo, hi = (np.clip(spans[..., i], 0, n)[:, None, :, None] for i in (0, 1))
    seen = np.broadcast_to((key >= lo) & (key < hi), x.shape)
    u = np.where(seen, x, 0.0) * scale / cap
    t = np.tanh(u)
    z, e = cap * t, cap * (np.abs(u) * (1 - t * t) * 2 * U + 5 * U * np.abs(t))
    top = np.where(seen, z, -np.inf).max(-1, keepdims=True)
    top = np.where(np.isfinite(top), top, 0)
    p = np.where(seen, np.exp(z - top), 0.0)
    # the scores' own error and the maximum's; the rounding of the difference
    # times log2 e, its conversion and ex2 (4 u)
    off = e + np.where(seen, e, 0).max(-1, keepdims=True) + 4 * U * (np.abs(z) + np.abs(top))
    ep = p * np.expm1(off) + 4 * U * p + seen * 2.0 ** -126
    s = p.sum(-1, keepdims=True)
    rel = (ep.sum(-1, keepdims=True) + (n / 512 + 60) * U * s) / np.where(s > 0, s, 1)
    y = p / np.where(s > 0, s, 1)
    return Num(y, np.where(seen, ep / np.where(s > 0, s, 1) + y * rel / (1 - rel) + 3 * U * y, 0)), seen


@pytest.mark.parametrize("n", [70, 700, 5000, 40000])
@pytest.mark.parametrize("dtype,out,cap", [
    (torch.float32, None, 50.0), (torch.float32, None, 1e5), (torch.bfloat16, torch.float32, 50.0),
    (torch.float16, None, 2000.0), (torch.bfloat16, None, 1e5)])
def test_capped_scores_keep_their_digits(dtype, out, cap, n):
    """Scores far below the cap, where tanh is nearly the identity: an absolute
    error of the tanh would be the cap times as large in the score."""
    g = gen(n)
    x = (3 * torch.randn(2, 2, 6, n, generator=g)).to(dtype).to(DEV)
    wide = torch.zeros(2, 2, 6, n + 9, dtype=dtype, device=DEV)
    shifted = wide[..., 1:n + 1].copy_(x)                       # rows in another step than their results
    spans = random_spans(2, 6, n, g)
    for xs in (x, shifted):
        y = torch_fl.ops.span_softmax(xs, spans, 0.5, cap, dtype=out)
        want, seen = capped_want(np64(x), spans.cpu().numpy(), 0.5, float(np.float32(cap)))
        close(y, want, y.dtype, "y")
        assert not np64(y)[~seen].any()
        dy = torch.randn(x.shape, generator=g).to(y.dtype).to(DEV)
        dx = torch.ops.flagos.span_softmax_backward(dy, y, xs, spans, 0.5, cap)
        close(dx, span_back_want(np64(dy), np64(y), np64(x), seen, 0.5, float(np.float32(cap))), dtype, "dx")


@pytest.mark.parametrize("K_", [12, 60, 700, 1004, 5004, 40004])
@pytest.mark.parametrize("cap", [None, 20.0])
def test_gradient_of_fp32_weights_at_the_edges_of_their_memory(K_, cap):
    """fp32 y and dy beside 16-bit x: a pack of x is two 16-byte words of them,
    of which the first or the last may hold nothing of the row.  Views in a
    buffer of NaN, results that begin inside a pack."""
    g = gen(K_)
    x = (2 * torch.randn(1, 1, 3, K_, generator=g)).bfloat16().to(DEV)
    spans = torch.tensor([[0, K_], [K_ - 3, K_], [1, 2]]).int().to(DEV)
    y = torch_fl.ops.span_softmax(x, spans, 0.5, cap, dtype=torch.float32)
    dy = torch.randn(1, 1, 3, K_, generator=g).to(DEV)
    want = torch.ops.flagos.span_softmax_backward(dy, y, x, spans, 0.5, cap)
    for at in (0, 4, 8):
        bufs = [torch.full((3 * K_ + 16,), math.nan, device=DEV) for _ in range(2)]
        views = [b[at:at + 3 * K_].view(1, 1, 3, K_).copy_(t) for b, t in zip(bufs, (y, dy))]
        got = torch.ops.flagos.span_softmax_backward(views[1], views[0], x, spans, 0.5, cap)
        assert torch.equal(got, want)
        # dx (and x) 4 elements into a pack, y and dy at the start of one
        xs, dx = (torch.full((3 * K_ + 16,), math.nan, device=DEV).bfloat16() for _ in range(2))
        xs[4:4 + 3 * K_] = x.flatten()
        K._abi.call("fl_b200_span_softmax_bwd", views[1].data_ptr(), K_, views[0].data_ptr(), K_, xs[4:].data_ptr(), K_,
                    spans.data_ptr(), 0, 2, dx[4:].data_ptr(), K_, 3, K_, 1, 3, 0.5, cap or 0.0, K._abi.F32,
                    K._abi.BF16, K._stream(x))
        # (another share of the sum for each thread: fp32 sums of some terms around 1)
        a, b = dx[4:4 + 3 * K_].double(), want.flatten().double()
        assert bool(((a - b).abs() <= 2.0 ** -7 * b.abs() + 60 * U * float(dy.abs().max())).all())
        assert bool(torch.isnan(dx[:4]).all()) and bool(torch.isnan(dx[4 + 3 * K_:]).all())


def test_calls_of_different_lengths_from_two_threads():
    """Rows of 1531 and of 2048 keys want different amounts of shared memory of
    one kernel: neither thread's calls may take it from the other's.  (The C
    entries themselves, so that both threads are in them at once.)"""
    import threading

    lib, made = K._abi.lib(), {}
    for n in (1531, 2048):
        x = (2 * torch.randn(1, 1, 4, n, generator=gen(n))).bfloat16().to(DEV)
        spans = torch.tensor([[0, n]] * 4).int().to(DEV)
        y = K.span_softmax(x, spans, 0.5, 20.0, out_dtype=torch.float32)
        dx = K.span_softmax_backward(y, y, x, spans, 0.5, 20.0)
        y2, dx2 = torch.zeros_like(y), torch.zeros_like(dx)
        stream = torch.cuda.Stream()
        fwd = (x.data_ptr(), n, spans.data_ptr(), 0, 2, None, 0, 0, None, y2.data_ptr(), n, 4, n, 1, 4, 0.5, 20.0,
               K._abi.BF16, K._abi.F32, stream.cuda_stream)
        bwd = (y.data_ptr(), n, y.data_ptr(), n, x.data_ptr(), n, spans.data_ptr(), 0, 2, dx2.data_ptr(), n, 4, n, 1, 4,
               0.5, 20.0, K._abi.F32, K._abi.BF16, stream.cuda_stream)
        made[n] = (x, spans, y, dx, y2, dx2, stream, fwd, bwd)
    torch.cuda.synchronize()
    ready, status = threading.Barrier(2), {n: set() for n in made}

    def work(n):
        fwd, bwd = made[n][-2:]
        ready.wait(60)
        for _ in range(5000):
            status[n].add(lib.fl_b200_span_softmax(*fwd))
            status[n].add(lib.fl_b200_span_softmax_bwd(*bwd))

    threads = [threading.Thread(target=work, args=(n,)) for n in made]
    [t.start() for t in threads]
    [t.join() for t in threads]
    torch.cuda.synchronize()
    assert status == {n: {0} for n in made}
    for x, spans, y, dx, y2, dx2, *_ in made.values():
        assert torch.equal(y, y2) and torch.equal(dx, dx2)


def test_rows_of_different_lengths_in_one_graph():
    g = gen(62)
    xs = [(2 * torch.randn(1, 1, 4, n, generator=g)).bfloat16().to(DEV) for n in (2048, 1531, 2056, 40)]
    spans = [torch.tensor([[0, x.shape[-1]]] * 4).int().to(DEV) for x in xs]
    run = lambda: [K.span_softmax(x, s, 0.5, 20.0) for x, s in zip(xs, spans)]
    want = run()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run()
    K.span_softmax(xs[3], spans[3])                         # the last length before the replay is the shortest
    K.span_softmax(xs[1], spans[1])
    [t.zero_() for t in got]
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


# --------------------------------------------------------------------- rotary
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [1, 2])
def test_rotary_of_overlapping_views(dtype, dim):
    """Windows of one row: tokens one element apart, of which a result laid
    out alike would have its heads' elements apart."""
    g = gen(71)
    row = torch.randn(64, generator=g).to(dtype).to(DEV)
    q = row.unfold(0, 16, 1)[:8][None, :, None]                            # [1, 8, 1, 16], strides (8, 1, 16, 1)
    k = row.unfold(0, 16, 3)[:8][None, :, None].expand(1, 8, 2, 16)
    assert torch.empty_like(q).stride(-1) != 1
    freq, pos = torch.rand(8, generator=g).to(DEV), torch.arange(8, device=DEV)
    if dim == 1:
        q, k = q.transpose(1, 2), k.transpose(1, 2)
    check_rotary(q, k, pos, freq, layout="bshd" if dim == 2 else "bhsd")
    layout = "bshd" if dim == 2 else "bhsd"
    got = K.rotary(q, k, pos, freq, layout=layout)
    want = K.rotary(q.contiguous(), k.contiguous(), pos, freq, layout=layout)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


# ------------------------------------------------------------------- clipping
def test_clip_refuses_expanded_outputs_before_it_writes_any():
    a, b = torch.full((1000,), 2.0, device=DEV), torch.ones(3, 1, device=DEV).expand(3, 4)
    c = torch.ones(8, 9, device=DEV)[:, :5]
    with pytest.raises(RuntimeError, match="share memory"):
        torch_fl.ops.clip_grads([a, c, b], 0.1, out=[a, c, b])
    assert bool((a == 2).all()) and bool((b == 1).all()) and bool((c == 1).all())
