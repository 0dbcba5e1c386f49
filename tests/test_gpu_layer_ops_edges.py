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

from .test_gpu_layer_ops import (DEV, TYPES, U, Num, check_clip, check_rotary, close, gen, np64, random_spans,
                                 sandwich_inputs, sandwich_want, span_back_want, span_want)
from .test_gpu_layer_ops import test_sandwich as check_sandwich

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


# ------------------------------------------------- kernels that walk many rows
def sms():
    return torch.cuda.get_device_properties(0).multi_processor_count


def mixed_spans(B, Q, n, g):
    """Of every kind in turn: empty, one key, a short run, up to 64 packs, all."""
    lo = torch.randint(0, n, (B, Q), generator=g, device=DEV)
    length = torch.stack([torch.zeros_like(lo), torch.ones_like(lo), torch.randint(2, 40, (B, Q), generator=g, device=DEV),
                          torch.randint(1, 500, (B, Q), generator=g, device=DEV), torch.full_like(lo, n)], -1)
    kind = torch.randint(0, 5, (B, Q, 1), generator=g, device=DEV)
    length = length.gather(-1, kind)[..., 0]
    lo = torch.where(length == n, 0, lo)
    return torch.stack([lo, (lo + length).clamp(max=n)], -1).int()


@pytest.mark.parametrize("dtype,out", [(torch.bfloat16, None), (torch.float16, torch.float32), (torch.float32, None)])
@pytest.mark.parametrize("cap,bias", [(None, False), (20.0, True)])
@pytest.mark.parametrize("n,many", [(43, True), (251, True), (252, False), (700, False), (1301, False)])
def test_span_softmax_walks_rows(dtype, out, cap, bias, n, many):
    """Rows enough that every resident warp takes a second one (5000), and runs
    of eight (from 32 rows a warp on): rows are what they are in launches where
    no warp has two, bit for bit, and picked ones are right in 64 bits."""
    H = 3
    rows = 32 * 28 * sms() + 2000 if many else 40 * sms()         # (28: the gradient's warps an SM)
    B, Q = (7, rows // 21 + 1) if many else (5, rows // 15 + 1)
    g = torch.Generator(device=DEV).manual_seed(n)
    wide = (3 * torch.randn(B, H, Q, n + 5, generator=g, device=DEV)).to(dtype)
    slopes = torch.tensor([0.5, 0.01, 0.0], device=DEV) if bias else None
    spans = mixed_spans(B, Q, n, g)
    pos = torch.randint(0, n, (B, Q), generator=g, device=DEV).int()
    for x in (wide[..., :n].contiguous(), wide[..., 4:n + 4]):
        y = torch_fl.ops.span_softmax(x, spans, 0.5, cap, slopes, pos, out)
        dy = torch.randn(x.shape, generator=g, device=DEV).to(y.dtype)
        dx = torch.ops.flagos.span_softmax_backward(dy, y, x, spans, 0.5, cap)
        step = 900                                                # 2700 rows: fewer than either kernel's warps
        assert H * step < 20 * sms()
        alike = 0
        for b in range(0, B, 2 if many else 1):
            for q0 in range(0, Q if x.is_contiguous() else 0, step):
                part, at = (slice(b, b + 1), slice(q0, q0 + step)), (slice(b, b + 1), slice(None), slice(q0, q0 + step))
                few = x[at].contiguous()
                y1 = torch_fl.ops.span_softmax(few, spans[part], 0.5, cap, slopes, pos[part], out)
                dx1 = torch.ops.flagos.span_softmax_backward(dy[at].contiguous(), y[at].contiguous(), few, spans[part], 0.5, cap)
                for h in range(H):
                    # a row that begins elsewhere in a 16-byte pack has its elements with other lanes, and so
                    # its sums in another order: the same bits are owed where it begins alike
                    moved = (b * H + h) * Q + q0 - h * few.shape[2]
                    if moved * n * few.element_size() % 16 == 0:
                        alike += 1
                        assert torch.equal(y1[:, h], y[at][:, h]) and torch.equal(dx1[:, h], dx[at][:, h])
        assert alike > 0 or not x.is_contiguous()
        pick = torch.randint(0, B * Q, (160,), generator=g, device=DEV).cpu()
        for h in range(H):
            take = lambda t: t[pick // Q, h, pick % Q][:, None, None]
            sp, ps = (t.reshape(B * Q, *t.shape[2:])[pick.to(DEV)][:, None] for t in (spans, pos))
            want, seen = span_want(np64(take(x)), sp.cpu().numpy(), 0.5, cap, None if slopes is None else np64(slopes[h:h + 1]),
                                   ps.cpu().numpy().astype(np.float64))
            close(take(y), want, y.dtype, f"y of head {h}")
            assert not np64(take(y))[~seen].any()
            close(take(dx), span_back_want(np64(take(dy)), np64(take(y)), np64(take(x)), seen, 0.5, cap), dtype, f"dx of head {h}")
            assert not np64(take(dx))[~seen].any()


@pytest.mark.parametrize("gate", ["none", "channel", "sequence", "token"])
@pytest.mark.parametrize("dtype,H", [(torch.bfloat16, 1032), (torch.float16, 1288), (torch.bfloat16, 2040)])
def test_sandwich_staged_rows_of_129_to_255_packs(dtype, H, gate):
    """Six resident CTAs an SM that walk at least eight rows each."""
    B, S = 5, 8 * 6 * sms() // 5 + 20
    x, res, post, pre, gt, *_ = sandwich_inputs((B, S, H), gate, dtype, H, 1.0)
    y, h = torch_fl.ops.sandwich_norm(x, res, post, pre, 1e-6, gt, 0.5, 1.0)
    pick = torch.cat([torch.tensor([0, 1, S - 1, S, B * S - 2, B * S - 1]),
                      torch.randint(0, B * S, (400,), generator=gen(H))]).to(DEV)
    flat = lambda t: np64(t.reshape(B * S, H)[pick])
    wide = None if gt is None else flat(gt.expand(B, S, H))
    wy, wh = sandwich_want(flat(x), flat(res), np64(post), np64(pre), wide, np.float32(1e-6), 0.5, 1.0)
    close(h.view(B * S, H)[pick], wh, dtype, "h")
    close(y.view(B * S, H)[pick], wy, dtype, "y")


@pytest.mark.parametrize("dtype,gate", [(torch.bfloat16, "none"), (torch.bfloat16, "channel"), (torch.bfloat16, "sequence"),
                                        (torch.float16, "token"), (torch.float32, "sequence")])
@pytest.mark.parametrize("team,packs", [(32, 33), (64, 125), (128, 255), (256, 512), (512, 1000)])
def test_sandwich_gradient_walks_chunks(dtype, gate, team, packs):
    """Five rows and more a team's chunk, of gate rows that end inside it."""
    H = packs * 16 // torch.finfo(dtype).bits * 8
    teams = sms() * (1 if team == 512 else 2) * max(1, 256 // team)
    S = 37
    B = 5 * teams // S + 2
    check_sandwich(dtype, gate, (B, S, H))


@pytest.mark.parametrize("kind", [2.0, math.inf])
@pytest.mark.parametrize("dtype", TYPES)
def test_clip_walks_chunks(dtype, kind):
    """More chunks of 32 KB than there are resident CTAs."""
    g = gen(81)
    sizes = [3000001, 5, 40000, 7000003, 64, 1, 2500000]
    ts = [(torch.randn(n, generator=g) * 0.01 * (1 + i % 3)).to(dtype).to(DEV) for i, n in enumerate(sizes)]
    assert sum(t.numel() * t.element_size() for t in ts) > 4 * sms() * 32768
    check_clip(ts, 0.003, kind)
    bucket = torch.zeros(sum(sizes) + 1, dtype=dtype, device=DEV)
    check_clip(ts, 0.003, kind, list(bucket[1:].split(sizes)))    # packed without gaps: by elements
    assert float(bucket[0]) == 0
    check_clip(ts, 0.003, kind, ts)


def test_clip_of_one_tensor_and_its_output():
    """A tensor stands for a list of one, as an output too."""
    a = torch.full((3, 1000), 2.0, device=DEV)
    for out in (torch.zeros_like(a), a):
        got, n = torch_fl.ops.clip_grads(a, 1.0, out=out)
        assert got[0] is out and abs(float(out.double().norm()) - 1) < 1e-5 and abs(float(n) - 12000 ** 0.5) < 1e-4


def test_dispatch_modes_see_the_norm_and_the_clipping():
    from torch.utils._python_dispatch import TorchDispatchMode

    seen = []

    class Watch(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            seen.append(func.name())
            return func(*args, **(kwargs or {}))

    ts = [torch.randn(n, generator=gen(n)).to(DEV) for n in (7, 5000)]
    out = [torch.empty_like(t) for t in ts]
    want, n = torch_fl.ops.clip_grads(ts, 0.5, out=[torch.empty_like(t) for t in ts])
    with Watch():
        got, n1 = torch_fl.ops.clip_grads(ts, 0.5, out=out)
        n2 = torch_fl.ops.grad_norm(ts)
    assert {"flagos::clip_grads_out", "flagos::grad_norm"} <= {s.split(".")[0] for s in seen}
    assert float(n) == float(n1) == float(n2) and all(a is o and torch.equal(a, b) for a, o, b in zip(got, out, want))
