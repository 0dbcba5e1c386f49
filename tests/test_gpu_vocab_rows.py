"""The vocabulary-row operators on the GPU against 64 bits: top-k, the
distillation loss on a teacher's top logits with its gradients, and the
verification of drafted tokens.

Tolerances, with u = 2^-24 (a rounding is off by at most half a step):

* top-k and verification are exact.
* Statistics.  An exponential 2^((z - m) c) carries 2 u |(z - m) c| ln 2 from
  its argument and 4 u from ex2.approx; the terms of S are positive, so S is
  off by at most (chain + 8) u relative, chain being the longest run of
  additions into one accumulator: a thread's share of the row plus the tree,
  V / 512 + 40 (weighted by its term, the argument's part stays below 2 u).
* loss = tau^2 (sum p d + log S - log S_t) with |d| <= D: each d carries
  6 u D, p as S does over k / 32 + 40 terms, logf one step of its value.
* A gradient w tau (q - p) adds the relative errors of q and p to those
  terms, and half a step of its type.
* Below 2^-126 fp32 has no relative precision: ex2.approx flushes such a q to
  0, and a p there is a multiple of 2^-149, so a relative bound on them means
  nothing.  Each of p and q is therefore granted 2^-126 absolutely, times what
  it is multiplied with: w tau, and for the teacher's gradient the gap too.
"""

import numpy as np
import pytest
import torch

import torch_fl
from oracle import ops
from tests import parity
from torch_fl import _abi
from torch_fl import kernels as K

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def gen(seed):
    return torch.Generator().manual_seed(seed)


def np64(t):
    return t.detach().cpu().double().numpy()


def half_step(dtype, ref):
    """Half a step of dtype at |ref|; half its smallest subnormal at least."""
    f = torch.finfo(dtype)
    tiny = f.tiny * f.eps
    return np.maximum(np.abs(ref) * f.eps / 2 * 1.0001, tiny * 0.5001)


# ---------------------------------------------------------------------- top-k
def check_topk(x, k, what="", fn=K.topk_lastdim):
    v, i = fn(x, k)
    assert v.dtype == x.dtype and i.dtype == torch.int64 and v.shape == i.shape
    x2 = x.reshape(-1, x.shape[-1])
    _, gi = ops.topk_golden(np64(x2), k)
    np.testing.assert_array_equal(i.cpu().numpy().reshape(-1, k), gi, err_msg=what)
    bits = torch.int32 if x.dtype == torch.float32 else torch.int16
    # gathered as integers: a gather of bfloat16 on the CPU may give a NaN other bits
    want = torch.gather(x2.cpu().view(bits), -1, torch.from_numpy(gi)).reshape(v.shape)
    assert torch.equal(v.cpu().view(bits), want), what  # the elements' own bits


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols,k", [
    (1, 1, 1), (2, 7, 7), (3, 33, 4), (5, 1000, 1), (1, 4096, 1024), (2, 1023, 1000), (3, 8193, 17),
    (4, 32000, 8), (7, 40003, 50), (2, 128256, 64), (1, 131073, 256), (300, 5000, 33), (700, 2048, 128),
])
def test_topk(dtype, rows, cols, k):
    x = (2.5 * torch.randn(rows, cols, generator=gen(rows + cols))).to(dtype).to(DEV)
    check_topk(x, k)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols,k", [(1300, 1001, 1), (1250, 4096, 130), (2500, 2053, 17), (1200, 513, 30),
                                         (1184, 8100, 256), (1500, 3003, 100), (593, 8001, 33), (900, 15999, 20)])
def test_topk_many_short_rows(dtype, rows, cols, k):
    x = (2.5 * torch.randn(rows, cols, generator=gen(rows + k))).to(dtype)
    x[3] = 1.0                                       # nothing but ties
    x[4] = torch.arange(cols)
    x[5] = -torch.arange(cols).float()
    x[6, 7:] = -float("inf")
    x[7, ::3] = float("nan")
    x[8] = torch.where(torch.arange(cols) % 2 == 0, -0.0, 0.0)
    x[9] = torch.finfo(dtype).min
    check_topk(x.to(DEV), k)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("copies", [1, 120])
def test_topk_special_rows(dtype, copies):
    V = 20011 if copies == 1 else 5003
    g = gen(3)
    base = torch.randn(V, generator=g)
    rows = [torch.zeros(V), torch.full((V,), -float("inf")), torch.arange(V, 0, -1).float(),
            torch.arange(V).float(), torch.full((V,), torch.finfo(dtype).min),
            torch.where(torch.arange(V) % 2 == 0, -0.0, 0.0), torch.sign(base), base]
    nan = base.clone()
    nan[[5, 700, V - 1]] = float("nan")
    inf = base.clone()
    inf[[9, V - 2]] = float("inf")
    few = torch.full((V,), -float("inf"))
    few[[V - 1, 3]] = torch.tensor([1.0, 2.0])
    last = torch.full((V,), -1.0)
    last[-300:] = 1.0
    x = torch.stack(rows + [nan, inf, few, last, torch.full((V,), float("nan"))]).to(dtype)
    x = x.repeat(copies, 1).to(DEV)
    for k in (1, 40, 300, 1024) if copies == 1 else (1, 40, 255):
        check_topk(x, k, f"k={k}")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("R,V,k", [(700, 4001, 64), (1300, 1024, 8), (640, 8150, 100), (2000, 2051, 17),
                                   (600, 15990, 20), (5, 20011, 50), (300, 40003, 64), (64, 128256, 200),
                                   (700, 9001, 400), (2, 300000, 1000), (4, 32000, 8)])
def test_topk_masked_rows(dtype, R, V, k):
    """Fewer live tokens than k, as many, a few more; ties below, between and
    above them, in the single elements at either end too; rows that rise."""
    g = gen(R + V)
    x = torch.randn(R, V + 7, generator=g)[:, 3:V + 3]
    mask = torch.full((R, V), -float("inf"))
    mask[1::4] = torch.finfo(dtype).min
    mask[2::4] = -0.5                                   # ties with live tokens on both sides
    live = torch.zeros(R, V, dtype=torch.bool)
    for r in range(R):
        n = (0, 1, k - 1, k, k + 1, k // 2, 3 * k)[r % 7]
        live[r, torch.randperm(V, generator=g)[:min(n, V)]] = True
    x = torch.where(live, x, mask)
    x[R // 2, V // 2] = float("nan")
    x[R // 3, -1] = float("inf")
    x[R - 1] = torch.arange(V) // 3                     # a rise, in threes
    if R > 8:
        x[4] = torch.where(torch.arange(V) % 2 == 0, 0.0, -0.0)
        x[5, V - 5:] = -float("inf")                    # the tail among the ties
        x[6, :V // 2] = 1.5                             # more ties than k, nothing above
        x[7] = -torch.arange(V).float()
    wide = torch.zeros(R, V + 7, dtype=dtype, device=DEV)
    wide[:, 3:V + 3] = x.to(dtype).to(DEV)
    check_topk(wide[:, 3:V + 3], k)
    check_topk(wide[:, 3:V + 3].contiguous(), k)


def replay_us(call, n=5):
    """Device time of a call, from replays of a graph of n of them."""
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for _ in range(n):
            call()
    best = float("inf")
    for _ in range(5):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        graph.replay()
        a.record()
        graph.replay()
        b.record()
        torch.cuda.synchronize()
        best = min(best, a.elapsed_time(b) * 1e3 / n)
    return best


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("R,V,k", [(8192, 4096, 64), (1500, 7000, 20), (1000, 128256, 64), (32, 128256, 64)])
def test_topk_masked_rows_take_no_multiple_of_ten(dtype, R, V, k):
    """Masked rows are walked a fixed number of times more, not once for each
    bit of a key: within 6 times the time of rows without ties (2.0 to 4.6
    measured; 7 to 34 when each bit of a key, or each tied element, had its turn)."""
    x = torch.randn(R, V, device=DEV).to(dtype)
    masked = x.masked_fill(torch.rand(R, V, device=DEV) * V > k // 3, -float("inf"))
    plain, tied = (replay_us(lambda: K.topk_lastdim(v, k)) for v in (x, masked))
    assert tied < 6 * plain, (plain, tied)


def test_topk_rows_that_rise_late():
    """Rows in ascending blocks: whatever a scan has kept is beaten later."""
    V = 65536
    x = torch.randn(6, V, generator=gen(1)) + torch.arange(V) // 512
    x[1] = torch.arange(V)
    x[2, : V // 2] = -5.0
    x[3] = x[3].flip(0)
    x[4, -2000:] = 1e4
    for dt in TYPES:
        check_topk(x.clamp(max=6e4).to(dt).to(DEV), 128, str(dt))


def test_topk_strides_and_shapes():
    x = torch.randn(6, 5, 3001, generator=gen(2)).to(torch.bfloat16).to(DEV)
    check_topk(x, 9)
    check_topk(x[:, 1], 9)                    # rows a stride apart
    check_topk(x[:, :, 3:2900], 9)            # rows that begin anywhere
    check_topk(x.transpose(0, 1), 9)          # copied first
    check_topk(x.transpose(0, 2), 3)
    check_topk(x[0, 0], 5)
    check_topk(x[:1].expand(4, 5, 3001), 5)
    check_topk(x[0, :1].expand(4, 3001), 5)
    check_topk(x[0, :1].expand(4, 3001), 5, fn=torch_fl.ops.topk)
    v, i = K.topk_lastdim(x[:0], 4)
    assert v.shape == (0, 5, 4)
    v, i = K.topk_lastdim(x, 0)
    assert v.shape == (6, 5, 0)
    check_topk(x, 9, fn=torch_fl.ops.topk)


def test_topk_gradient():
    x = torch.randn(4, 3, 513, generator=gen(4))
    xf = x.to("flagos").requires_grad_()
    v, i = torch_fl.ops.topk(xf, 6)
    assert not i.requires_grad
    w = torch.randn(4, 3, 6, generator=gen(5))
    (v * w.to("flagos")).sum().backward()
    xc = x.clone().requires_grad_()
    vc = torch.gather(xc, -1, i.cpu())
    (vc * w).sum().backward()
    assert torch.equal(xf.grad.cpu(), xc.grad)
    for dt in TYPES:
        d = torch.randn(5, 8, generator=gen(6)).to(dt).to(DEV)
        idx = torch.stack([torch.randperm(1001, generator=gen(r))[:8] for r in range(5)]).to(DEV)
        got = K.topk_backward(d, idx, 1001)
        assert torch.equal(got, torch.zeros(5, 1001, dtype=dt, device=DEV).scatter_(1, idx, d))


def test_topk_second_derivative():
    """A penalty on the gradient through topk: f = sum v^3 has the gradient 3 v^2
    at the indices, and sum of its squares 36 v^3.  Products of one sign
    throughout, each through at most 16 roundings."""
    x = torch.randn(4, 3, 257, generator=gen(8))
    xf = x.to("flagos").requires_grad_()
    v, i = torch_fl.ops.topk(xf, 5)
    g, = torch.autograd.grad((v * v * v).sum(), xf, create_graph=True)
    assert g.requires_grad
    (xf.sum() + (g * g).sum()).backward()
    vd = np64(torch.gather(x, -1, i.cpu()))
    ref = np.ones(x.shape)
    np.put_along_axis(ref, i.cpu().numpy(), 1 + 36 * vd ** 3, -1)
    size = np.ones(x.shape)
    np.put_along_axis(size, i.cpu().numpy(), 1 + 36 * np.abs(vd) ** 3, -1)
    within(xf.grad, ref, 16 * U * size, "second derivative")
    # by its own op, where an index may lie outside the row; and a third time
    d = torch.randn(2, 3, generator=gen(9)).to("flagos").requires_grad_()
    idx = torch.tensor([[5, -1, 0], [9, 3, 4]]).to("flagos")
    dx = torch.ops.flagos.topk_backward(d, idx, 9)
    c = torch.randn(2, 9, generator=gen(10))
    (dx * c.to("flagos")).sum().backward()
    want = torch.where((idx.cpu() >= 0) & (idx.cpu() < 9), torch.gather(c, -1, idx.cpu().clamp(0, 8)), 0.0)
    assert torch.equal(d.grad.cpu(), want)


# --------------------------------------------------------------- distillation
def make(R, V, k, dtype, seed, t_dtype=None, ids_dtype=torch.int64, holes=True):
    g = gen(seed)
    z = (2 * torch.randn(R, V, generator=g)).to(dtype)
    t = (6 - torch.cumsum(torch.rand(R, k, generator=g), -1)).to(t_dtype or dtype)
    ids = torch.stack([torch.randperm(V, generator=g)[:k] if k <= V else torch.randint(0, V, (k,), generator=g)
                       for _ in range(R)])
    if holes and R > 2:
        ids[R // 2] = -1                                # a row without a teacher
        if k > 2:
            ids[0, k // 2:] = -1                        # a list cut short
            ids[1, 1] = ids[1, 0]                       # the same token twice
            ids[R - 1, 0] = V + 5                       # outside the vocabulary
            ids[R - 1, 2] = V - 1
    w = torch.rand(R, generator=g) + 0.1
    return z.to(DEV), t.to(DEV), ids.to(ids_dtype).to(DEV), w.to(DEV)


def bounds(z, t, ids, tau, w):
    """Tolerances of (loss, dlogits, dteacher) before the output's rounding."""
    z, t, ids, w = np64(z) / tau, np64(t) / tau, np64(ids).astype(np.int64), np64(w)
    R, V = z.shape
    ok = (ids >= 0) & (ids < V)
    t = np.where(ok, t, -np.inf)
    taught = np.any(t > -np.inf, -1)
    z = np.where(taught[:, None], z, 0.0)       # rows without a teacher are exact zeros
    chain, tree = V / 512 + 48, t.shape[1] / 32 + 48
    flush = 2.0 ** -126

    def soft(v):
        """(softmax, |v - max| where it has weight, |log of the sum|) of the rows."""
        d = v - v.max(-1, keepdims=True)
        e = np.exp(d)
        s = e.sum(-1, keepdims=True)
        return e / s, np.where(e > 0, np.abs(d), 0.0), np.abs(np.log(s))

    q, qd, logs = soft(z)
    p, pd, logt = soft(np.where(taught[:, None], t, 0.0))
    p = np.where(ok & taught[:, None], p, 0.0)
    at = np.where(ok, ids, 0)
    d = np.where(p > 0, pd + np.take_along_axis(qd, at, -1), 0.0)
    row = U * (chain + tree + 4 * (logs + logt)[:, 0] + (p * (6 + tree) * d).sum(-1) + 8)
    tol_loss = tau * tau * row * taught
    gt = np.abs(w)[:, None] * tau * taught[:, None]
    tol_dz = gt * (U * q * (chain + 16 + 4 * qd) + flush)
    tol_p = gt * (U * p * (tree + 16 + 4 * pd) + flush)
    for r in range(R):
        np.add.at(tol_dz[r], ids[r][ok[r]], tol_p[r][ok[r]])
    gap = d + logs + logt
    tol_dt = gt * (p * (row[:, None] + U * (6 * d + 4 * (logs + logt) + (tree + 16) * (gap + 1)))
                   + flush * (gap + row[:, None] / U + 1))
    return tol_loss, tol_dz, tol_dt


def within(got, ref, tol, what):
    got = np64(got) if isinstance(got, torch.Tensor) else got
    err = np.abs(got - ref)
    bad = ~(err <= tol)
    assert not bad.any(), (what, int(bad.sum()), float((err / np.maximum(tol, 1e-300)).max()),
                           np.argwhere(bad)[0].tolist())


def check_distill(z, t, ids, w, tau, what=""):
    ref = ops.distill_topk_golden(np64(z), np64(t), np64(ids).astype(np.int64), tau, np64(w))
    tol = bounds(z, t, ids, tau, w)
    loss, stats = K.distill_topk(z, t, ids, tau)
    assert loss.dtype == torch.float32 and loss.shape == z.shape[:-1]
    within(loss, ref[0], tol[0] + half_step(torch.float32, ref[0]), what + " loss")
    dz, dt = K.distill_topk_backward(w, z, stats, t, ids, tau, need_teacher=True)
    assert dz.dtype == z.dtype and dt.dtype == t.dtype
    within(dz, ref[1], tol[1] + half_step(z.dtype, ref[1]), what + " dlogits")
    within(dt, ref[2], tol[2] + half_step(t.dtype, ref[2]), what + " dteacher")
    l2, dz2 = K.distill_topk_grad(z, t, ids, tau, w)
    within(l2, ref[0], tol[0] + half_step(torch.float32, ref[0]), what + " grad's loss")
    within(dz2, ref[1], tol[1] + half_step(z.dtype, ref[1]), what + " grad's dlogits")


SIZES = [(1, 1, 1), (3, 7, 3), (4, 100, 100), (5, 513, 17), (3, 4096, 1024), (33, 5001, 8),
         (2, 32000, 64), (9, 40003, 33), (300, 1111, 5), (4, 65536, 200), (3, 128256, 64),
         (2, 131077, 1000), (2, 300001, 16)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("R,V,k", SIZES)
def test_distill(dtype, R, V, k):
    check_distill(*make(R, V, k, dtype, R * 7 + V), tau=1.0 + (V % 3), what=f"{R}x{V}x{k}")


@pytest.mark.parametrize("tau", [0.05, 0.5, 20.0])
def test_distill_temperatures(tau):
    check_distill(*make(6, 2000, 12, torch.float32, 9), tau=tau)


def test_distill_mixed_types_and_strides():
    z, t, ids, w = make(6, 2048, 10, torch.bfloat16, 11, t_dtype=torch.float32, ids_dtype=torch.int32)
    check_distill(z, t, ids, w, 2.0, "f32 teacher, int32 ids")
    big = torch.zeros(6, 3000, dtype=torch.bfloat16, device=DEV)
    big[:, 5:2053] = z
    check_distill(big[:, 5:2053], t, ids, w, 2.0, "rows off every boundary, a stride apart")
    tt = torch.zeros(6, 32, device=DEV)
    tt[:, 3:13] = t
    ii = torch.full((6, 20), 7, dtype=torch.int64, device=DEV)
    ii[:, 10:] = ids
    check_distill(z, tt[:, 3:13], ii[:, 10:], w, 2.0, "strided lists")
    one = t[:1].expand(6, 10)
    check_distill(z, one, ids, w, 2.0, "one teacher list for every row")
    check_distill(z, t, ids, w[:1].expand(6), 2.0, "one weight for every row")
    # leading dims, out rows off the logits' phase
    l3, dz3 = K.distill_topk_grad(z.view(2, 3, 2048), t.view(2, 3, 10), ids.view(2, 3, 10), 2.0)
    l2, dz2 = K.distill_topk_grad(z, t, ids, 2.0)
    assert torch.equal(l3.view(6), l2) and torch.equal(dz3.view(6, 2048), dz2)
    out = torch.zeros(6, 2051, dtype=torch.bfloat16, device=DEV)
    lo, _ = K.distill_topk_grad(z, t, ids, 2.0, out=out[:, 1:2049])
    assert torch.equal(out[:, 1:2049], dz2) and not out[:, 0].any() and not out[:, 2049:].any()


def test_distill_gradient_between_the_logits_rows():
    """Logits and gradient as the two halves of one matrix's rows share no
    memory and are computed; an `out` that meets the logits is refused."""
    z, t, ids, w = make(6, 2048, 10, torch.bfloat16, 13)
    want = K.distill_topk_grad(z, t, ids, 2.0, w)
    both = torch.zeros(6, 4096, dtype=torch.bfloat16, device=DEV)
    both[:, :2048] = z
    loss, dz = K.distill_topk_grad(both[:, :2048], t, ids, 2.0, w, out=both[:, 2048:])
    assert torch.equal(loss, want[0]) and torch.equal(dz, want[1]) and torch.equal(both[:, :2048], z)
    wide = torch.zeros(7, 2048, dtype=torch.bfloat16, device=DEV)
    for out in (z, both[:, 1000:3048], both[:, 2047:4095]):
        logits = z if out is z else both[:, :2048]
        with pytest.raises(_abi.FlB200Error, match="invalid argument"):
            K.distill_topk_grad(logits, t, ids, 2.0, w, out=out)
    with pytest.raises(_abi.FlB200Error, match="invalid argument"):
        K.distill_topk_grad(wide[:6], t, ids, 2.0, w, out=wide[1:])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [999, 4096, 128256])
def test_distill_special_rows(dtype, V):
    R, k = 8, 6
    z, t, ids, w = make(R, V, k, dtype, 21, holes=False)
    low = torch.finfo(dtype).min
    z[0, V // 3:] = -float("inf")           # a masked vocabulary; teacher ids among what is left
    ids[0] = torch.arange(k, device=DEV) + 2
    z[1, V // 3:] = low                     # masked with the lowest value instead
    ids[1] = torch.arange(k, device=DEV) + 2
    z[2] = low                              # a row of nothing else is uniform
    t[3] = -float("inf")                    # a list without mass counts as empty
    z[3, 5] = float("nan")
    ids[4] = -1                             # nothing taught: NaN and inf do not matter
    z[4] = float("nan")
    z[4, 0] = float("inf")
    t[5, 1:] = -float("inf")                # a teacher that is sure
    t[6] = low
    z[7] = 0
    check_distill(z, t, ids, w, 2.0)
    loss, stats = K.distill_topk(z, t, ids, 2.0)
    dz, dt = K.distill_topk_backward(w, z, stats, t, ids, 2.0, need_teacher=True)
    for r in (3, 4):
        assert loss[r] == 0 and not dz[r].any() and not dt[r].any()
    # a taught row with a NaN, or of -inf alone, has no softmax; its neighbours do
    z[0, 1] = float("nan")
    z[1] = -float("inf")
    loss, dz = K.distill_topk_grad(z, t, ids, 2.0, w)
    assert torch.isnan(loss[:2]).all() and torch.isfinite(loss[2:]).all()
    assert torch.isnan(dz[:2]).all() and torch.isfinite(dz[2:]).all()
    # a token the student rules out: the loss is +inf as the formula has it
    z, t, ids, w = make(3, V, k, dtype, 22, holes=False)
    z[1, ids[1, 0]] = -float("inf")
    assert K.distill_topk(z, t, ids, 1.0)[0][1] == float("inf")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("R,V,k", [(593, 1000, 20), (2400, 2001, 64), (2500, 4090, 33), (600, 8000, 7),
                                   (1200, 511, 60), (5000, 37, 3), (2401, 1023, 1), (2402, 1024, 32),
                                   (1300, 2600, 40)])
def test_distill_many_short_rows(dtype, R, V, k):
    """Enough rows that each is a warp's; as elsewhere the rows between hold the edges."""
    z, t, ids, w = make(R, V, k, dtype, R + V)
    low = torch.finfo(dtype).min
    z[10, 9:] = -float("inf")
    ids[10] = torch.arange(k, device=DEV) % 7
    z[11, V // 2:] = low
    ids[11] = 3                             # one token throughout
    z[12] = low
    t[13] = -float("inf")
    z[13, 5] = float("nan")
    ids[14] = -1
    z[14] = float("nan")
    t[15, 1:] = -float("inf")
    t[16] = low
    z[17] = 0
    w[18] = 0
    check_distill(z, t, ids, w, 2.0)
    loss, stats = K.distill_topk(z, t, ids, 2.0)
    dz, dt = K.distill_topk_backward(w, z, stats, t, ids, 2.0, need_teacher=True)
    alone, none = K.distill_topk_backward(w, z, stats, t, ids, 2.0)
    assert none is None and torch.equal(alone, dz)
    for r in (13, 14):
        assert loss[r] == 0 and not dz[r].any() and not dt[r].any()
    # rows of a wider matrix, beside which nothing is written
    big = torch.zeros(R, V + 9, dtype=dtype, device=DEV)
    big[:, 3:V + 3] = z
    out = torch.full_like(big, 7.0)
    l2, _ = K.distill_topk_grad(big[:, 3:V + 3], t, ids, 2.0, w, out=out[:, 3:V + 3])
    l1, d1 = K.distill_topk_grad(z, t, ids, 2.0, w)
    tol = bounds(z, t, ids, 2.0, w)
    ref = ops.distill_topk_golden(np64(z), np64(t), np64(ids).astype(np.int64), 2.0, np64(w))
    within(l2, ref[0], tol[0] + half_step(torch.float32, ref[0]), "loss, in a wider matrix")
    within(out[:, 3:V + 3], ref[1], tol[1] + half_step(dtype, ref[1]), "gradient, in a wider matrix")
    assert (out[:, :3] == 7).all() and (out[:, V + 3:] == 7).all()
    # a row without a softmax is NaN, its neighbours are as they were
    z[20, 1] = float("nan")
    z[21] = -float("inf")
    ids[20:22, 0] = 1
    l3, d3 = K.distill_topk_grad(z, t, ids, 2.0, w)
    assert torch.isnan(l3[20:22]).all() and torch.isnan(d3[20:22]).all()
    rest = torch.tensor([r for r in range(R) if r not in (20, 21)], device=DEV)
    assert torch.equal(l3[rest], l1[rest]) and torch.equal(d3[rest], d1[rest])


@pytest.mark.parametrize("k", [2, 33, 64, 65, 128, 129, 300, 1024])
def test_distill_repeated_tokens(k):
    """Lists drawn from few tokens, one of a single token, one whose ids share
    their low bits; of every length that a kernel holds in another way."""
    R, V = 6, 70001
    z, t, ids, w = make(R, V, k, torch.float32, k, holes=False)
    g = gen(k + 1)
    ids = torch.randint(0, 7, (R, k), generator=g) * 9973
    ids[1] = 12345
    ids[2] = torch.arange(k) % 4 * 16384 + 5            # equal modulo 16384
    ids[3] = torch.arange(k) % 2 * 65536 + 3            # and modulo 65536
    ids[4] = torch.randint(0, V, (k,), generator=g)
    ids[5, ::2] = -1
    check_distill(z, t, ids.to(DEV), w, 1.5, f"k={k}")
    a = K.distill_topk_grad(z, t, ids.to(DEV), 1.5, w)
    for _ in range(3):                                  # whatever the marks' order
        b = K.distill_topk_grad(z, t, ids.to(DEV), 1.5, w)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_distill_without_lists_or_rows():
    z = torch.randn(3, 50, device=DEV)
    t, ids = torch.zeros(3, 0, device=DEV), torch.zeros(3, 0, dtype=torch.int64, device=DEV)
    loss, dz = K.distill_topk_grad(z, t, ids)
    assert not loss.any() and not dz.any()
    e = K.distill_topk_grad(z[:0], torch.zeros(0, 4, device=DEV),
                            torch.zeros(0, 4, dtype=torch.int64, device=DEV))
    assert e[0].shape == (0,) and e[1].shape == (0, 50)


def check_distill_ops(z, t, ids, w, tau, what=""):
    """The public ops on flagos tensors: the loss, both gradients through
    autograd for given row weights, and loss and gradient at once."""
    zf, tf, idf, wf = (v if v.device.type == "flagos" else v.cpu().to("flagos") for v in (z, t, ids, w))
    zf.requires_grad_(), tf.requires_grad_()
    ref = ops.distill_topk_golden(np64(z), np64(t), np64(ids).astype(np.int64), tau, np64(w))
    tol = bounds(z, t, ids, tau, w)
    loss = torch_fl.ops.distill_topk(zf, tf, idf, tau)
    within(loss, ref[0], tol[0] + half_step(torch.float32, ref[0]), what + " loss")
    loss.backward(wf)
    assert zf.grad.dtype == z.dtype and tf.grad.dtype == t.dtype
    within(zf.grad, ref[1], tol[1] + half_step(z.dtype, ref[1]), what + " dlogits")
    within(tf.grad, ref[2], tol[2] + half_step(t.dtype, ref[2]), what + " dteacher")
    l2, dz = torch_fl.ops.distill_topk_grad(zf.detach(), tf.detach(), idf, tau, wf)
    within(l2, ref[0], tol[0] + half_step(torch.float32, ref[0]), what + " grad's loss")
    within(dz, ref[1], tol[1] + half_step(z.dtype, ref[1]), what + " grad's dlogits")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("R,V,k", [(3, 7, 3), (5, 513, 17), (9, 40003, 33), (4, 65536, 200), (2, 131077, 1000),
                                   (700, 2001, 40), (3, 151936, 64)])
def test_public_distill(dtype, R, V, k):
    check_distill_ops(*make(R, V, k, dtype, R + 5 * V), tau=2.0, what=f"{R}x{V}x{k}")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("k", [6, 90, 300])
def test_public_distill_special_rows(dtype, k):
    """Masked vocabularies, sure and empty teachers, repeated and foreign tokens,
    other list types and strides, through the public ops."""
    V = 5003
    z, t, ids, w = make(10, V, k, dtype, 23, t_dtype=torch.float32, ids_dtype=torch.int32)
    low = torch.finfo(dtype).min
    z[0, V // 3:], ids[0] = -float("inf"), torch.arange(k, device=DEV) + 2
    z[1, V // 3:], ids[1] = low, torch.arange(k, device=DEV) + 2
    z[2] = low
    t[3], z[3, 5] = -float("inf"), float("nan")
    ids[4], z[4] = -1, float("nan")
    t[5, 1:] = -float("inf")
    ids[6] = 17                             # one token throughout
    ids[7] = torch.arange(k, device=DEV) % 3 * 1601 - 1
    w[8] = 0
    check_distill_ops(z, t, ids, w, 1.5, f"k={k}")
    wide = torch.zeros(10, V + 40, dtype=dtype)
    wide[:, 5:V + 5] = z.cpu()
    lists = torch.full((10, 2 * k + 3), 9.0)
    lists[:, 3:k + 3] = t.cpu()
    wide, lists, one = wide.to("flagos"), lists.to("flagos"), w[:1].cpu().to("flagos")
    check_distill_ops(wide[:, 5:V + 5], lists[:, 3:k + 3], ids, one.expand(10), 1.5, "strided")


@pytest.mark.parametrize("dtype", TYPES)
def test_public_topk_and_verify(dtype):
    """Special rows of every launch form, and both kinds of drafts, on flagos tensors."""
    for copies, V, ks in ((1, 20011, (1, 40, 300, 1024)), (150, 3001, (1, 40, 128))):
        x = torch.randn(5, V, generator=gen(12))
        x[0], x[1, 9:] = 2.0, -float("inf")
        x[2, ::3], x[3] = float("nan"), torch.arange(V) / 8
        x = x.to(dtype).repeat(copies, 1).to("flagos")
        for k in ks:
            check_topk(x, k, f"k={k}", fn=torch_fl.ops.topk)
    for with_q in (True, False):
        ids, p, q, u, lens = (None if v is None else v.cpu().to("flagos")
                              for v in drafts(7, 5, 9001, dtype, 14, with_q))
        check_verify(ids, p, q, u, lens, fn=torch_fl.ops.verify_draft)
        check_verify(ids, p, q, u, None, fn=torch_fl.ops.verify_draft)


def test_distill_autograd_on_flagos():
    """The op's autograd against the fp64 formula, through a mean over rows
    (a broadcast gradient), for both operands and with leading dims."""
    z, t, ids, _ = make(6, 1500, 8, torch.float32, 31)
    zf, tf = z.cpu().to("flagos").view(2, 3, 1500).requires_grad_(), t.cpu().to("flagos").view(2, 3, 8).requires_grad_()
    loss = torch_fl.ops.distill_topk(zf, tf, ids.cpu().to("flagos").view(2, 3, 8), 2.0)
    assert loss.shape == (2, 3) and loss.requires_grad
    loss.mean().backward()
    w = torch.full((6,), 1 / 6, device=DEV)
    ref = ops.distill_topk_golden(np64(z), np64(t), np64(ids).astype(np.int64), 2.0, np64(w))
    tol = bounds(z, t, ids, 2.0, w)
    within(zf.grad.view(6, -1), ref[1], tol[1] + half_step(torch.float32, ref[1]), "dlogits")
    within(tf.grad.view(6, -1), ref[2], tol[2] + half_step(torch.float32, ref[2]), "dteacher")
    # only the student's gradient, then none at all
    zf.grad = None
    torch_fl.ops.distill_topk(zf, tf.detach(), ids.cpu().to("flagos").view(2, 3, 8), 2.0).sum().backward()
    assert zf.grad is not None
    with torch.no_grad():
        assert not torch_fl.ops.distill_topk(zf, tf, ids.cpu().to("flagos").view(2, 3, 8), 2.0).requires_grad
    _, stats = torch.ops.flagos.distill_topk(zf, tf, ids.cpu().to("flagos").view(2, 3, 8), 2.0)
    assert not stats.requires_grad              # the row statistics have no gradient


def blocks_of(call):
    """Blocks of each kernel that the call launches, from a captured graph."""
    import ctypes

    class Params(ctypes.Structure):     # CUDA_KERNEL_NODE_PARAMS
        _fields_ = [("func", ctypes.c_void_p), ("grid", ctypes.c_uint * 3), ("block", ctypes.c_uint * 3),
                    ("smem", ctypes.c_uint), ("params", ctypes.c_void_p), ("extra", ctypes.c_void_p),
                    ("kern", ctypes.c_void_p), ("ctx", ctypes.c_void_p)]

    cuda = ctypes.CDLL("libcuda.so.1")
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph):
        call()
    raw, n = ctypes.c_void_p(graph.raw_cuda_graph()), ctypes.c_size_t()
    assert cuda.cuGraphGetNodes(raw, None, ctypes.byref(n)) == 0
    nodes = (ctypes.c_void_p * n.value)()
    assert cuda.cuGraphGetNodes(raw, nodes, ctypes.byref(n)) == 0
    blocks = []
    for node in nodes:
        kind = ctypes.c_int()
        assert cuda.cuGraphNodeGetType(ctypes.c_void_p(node), ctypes.byref(kind)) == 0
        if kind.value == 0:             # a kernel
            p = Params()
            assert cuda.cuGraphKernelNodeGetParams_v2(ctypes.c_void_p(node), ctypes.byref(p)) == 0
            blocks.append(p.grid[0] * p.grid[1] * p.grid[2])
    return blocks


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("R,V,k", [(1, 1000, 5), (4, 40003, 20), (9, 5001, 200), (300, 2000, 64), (700, 1000, 30)])
def test_distill_teacher_gradient_alone(dtype, R, V, k):
    """Without the student's gradient the teacher's is the same, and a block a
    row does all there is to do."""
    z, t, ids, w = make(R, V, k, dtype, 3 * R + k)
    _, stats = K.distill_topk(z, t, ids, 2.0)
    _, both = K.distill_topk_backward(w, z, stats, t, ids, 2.0, need_teacher=True)

    def alone():
        return K.distill_topk_backward(w, z, stats, t, ids, 2.0, need_logits=False, need_teacher=True)

    none, dt = alone()
    assert none is None
    ref = ops.distill_topk_golden(np64(z), np64(t), np64(ids).astype(np.int64), 2.0, np64(w))
    tol = bounds(z, t, ids, 2.0, w)
    for got in (dt, both):
        within(got, ref[2], tol[2] + half_step(dtype, ref[2]), "dteacher")
    assert blocks_of(alone) == [R]


def test_distill_second_derivative_is_refused():
    """The gradient itself is there under create_graph; to differentiate it
    again is an error, not a term that is missing."""
    z, t, ids, _ = make(5, 700, 6, torch.float32, 32)
    zf, tf = z.cpu().to("flagos").requires_grad_(), t.cpu().to("flagos").requires_grad_()
    idf = ids.cpu().to("flagos")
    plain = torch.autograd.grad(torch_fl.ops.distill_topk(zf, tf, idf, 2.0).sum(), (zf, tf))
    loss = torch_fl.ops.distill_topk(zf, tf, idf, 2.0)
    gz, gt = torch.autograd.grad(loss.sum(), (zf, tf), create_graph=True)
    assert torch.equal(gz, plain[0]) and torch.equal(gt, plain[1])
    for term in ((gz * gz).sum() + zf.sum(), (gt * gt).sum()):
        with pytest.raises(RuntimeError, match="second derivative"):
            term.backward(retain_graph=True)
    # one operand alone, and by the backward's own op
    loss = torch_fl.ops.distill_topk(zf, tf.detach(), idf, 2.0)
    gz, = torch.autograd.grad(loss.sum(), zf, create_graph=True)
    with pytest.raises(RuntimeError, match="second derivative"):
        (gz * gz).sum().backward()
    loss, stats = torch.ops.flagos.distill_topk(zf.detach(), tf.detach(), idf, 2.0)
    dx, _ = torch.ops.flagos.distill_topk_backward(torch.ones_like(loss), zf, stats, tf.detach(), idf, 2.0)
    with pytest.raises(RuntimeError, match="second derivative"):
        dx.sum().backward()


def test_forward_mode_is_refused():
    """There is no forward-mode formula; a tangent is not dropped unseen."""
    import torch.autograd.forward_ad as fwd

    z, t, ids, _ = make(5, 700, 6, torch.float32, 32)
    zf, tf, idf = (v.cpu().to("flagos") for v in (z, t, ids))
    with fwd.dual_level():
        zd, td = fwd.make_dual(zf, torch.ones_like(zf)), fwd.make_dual(tf, torch.ones_like(tf))
        for call in (lambda: torch_fl.ops.topk(zd, 3), lambda: torch_fl.ops.distill_topk(zd, tf, idf),
                     lambda: torch_fl.ops.distill_topk(zf, td, idf)):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()
        torch_fl.ops.topk(zf, 3)
        torch_fl.ops.distill_topk(zf, tf, idf)


def test_distill_shapes_of_every_rank():
    z, t, ids, w = make(12, 333, 5, torch.float32, 33)
    want = K.distill_topk_grad(z, t, ids, 2.0, w)
    one = torch_fl.ops.distill_topk_grad(z[7], t[7], ids[7], 2.0, w[7])
    # (a row off the boundary that its gradient's row begins on takes two
    # kernels: the formula's bounds hold, bit equality with one kernel does not)
    ref = ops.distill_topk_golden(np64(z), np64(t), np64(ids).astype(np.int64), 2.0, np64(w))
    tol = bounds(z, t, ids, 2.0, w)
    assert one[0].shape == () and one[1].shape == (333,)
    within(one[0].view(1), ref[0][7:8], tol[0][7:8] + half_step(torch.float32, ref[0][7:8]), "one row's loss")
    within(one[1], ref[1][7], tol[1][7] + half_step(torch.float32, ref[1][7]), "one row's gradient")
    four = torch_fl.ops.distill_topk_grad(z.view(2, 3, 2, 333), t.view(2, 3, 2, 5), ids.view(2, 3, 2, 5), 2.0,
                                          w.view(2, 3, 2))
    assert torch.equal(four[0].view(12), want[0]) and torch.equal(four[1].view(12, 333), want[1])
    # weights that broadcast, logits whose rows are one row, operands transposed
    a = torch_fl.ops.distill_topk_grad(z.view(3, 4, 333), t.view(3, 4, 5), ids.view(3, 4, 5), 2.0, w[:3, None])
    b = K.distill_topk_grad(z, t, ids, 2.0, w[:3].repeat_interleave(4))
    assert torch.equal(a[1].view(12, 333), b[1])
    same = z[:1].expand(12, 333)
    a, b = (torch_fl.ops.distill_topk_grad(v, t, ids, 2.0, w) for v in (same, same.contiguous()))
    c = K.distill_topk_grad(same, t, ids, 2.0, w)
    assert torch.equal(a[1], b[1]) and torch.equal(a[0], b[0]) and torch.equal(a[1], c[1])
    a = torch_fl.ops.distill_topk_grad(z.t().contiguous().t(), t.t().contiguous().t(),
                                       ids.t().contiguous().t(), 2.0, w)
    assert torch.equal(a[0], want[0]) and torch.equal(a[1], want[1])


def test_distill_results_repeat():
    z, t, ids, w = make(40, 32000, 64, torch.bfloat16, 41)
    a = K.distill_topk_grad(z, t, ids, 2.0, w)
    for _ in range(3):
        b = K.distill_topk_grad(z, t, ids, 2.0, w)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


# --------------------------------------------------------------- verification
def drafts(B, n, V, dtype, seed, with_q=True, near=0.3):
    g = gen(seed)
    logits = 2.5 * torch.randn(B, n + 1, V, generator=g)
    p = torch.softmax(logits, -1)
    q = torch.softmax(logits[:, :n] + near * torch.randn(B, n, V, generator=g), -1)
    ids = torch.multinomial(q.reshape(B * n, V), 1, generator=g).view(B, n) if n else torch.zeros(B, 0, dtype=torch.int64)
    u = torch.rand(B, n + 1, generator=g)
    lens = torch.randint(0, n + 1, (B,), generator=g)
    lens[::2] = n
    return (ids.to(DEV), p.to(dtype).to(DEV), q.to(dtype).to(DEV) if with_q else None, u.to(DEV), lens.to(DEV))


def check_verify(ids, p, q, u, lens=None, what="", fn=K.verify_draft):
    tok, acc = fn(ids, p, q, u, lens)
    gt, ga = ops.verify_draft_golden(ids.cpu().numpy(), np64(p), None if q is None else np64(q),
                                     u.cpu().numpy(), None if lens is None else lens.cpu().numpy())
    np.testing.assert_array_equal(acc.cpu().numpy(), ga, err_msg=what)
    np.testing.assert_array_equal(tok.cpu().numpy(), gt, err_msg=what)
    return tok, acc


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("with_q", [True, False])
@pytest.mark.parametrize("B,n,V", [(1, 1, 1), (2, 3, 5), (3, 0, 100), (1, 4, 32000), (5, 7, 40003),
                                   (40, 2, 1001), (2, 70, 333), (3, 5, 128256), (200, 1, 2048), (1, 2, 300007)])
def test_verify(dtype, with_q, B, n, V):
    check_verify(*drafts(B, n, V, dtype, B + n + V, with_q), what=f"{B}x{n}x{V}")


def test_verify_without_lens_and_through_ops():
    ids, p, q, u, lens = drafts(6, 4, 999, torch.float32, 5)
    check_verify(ids, p, q, u, None)
    check_verify(ids, p, q, u, lens, fn=torch_fl.ops.verify_draft)
    check_verify(ids, p, None, u, lens, fn=torch_fl.ops.verify_draft)
    check_verify(ids, p, q, u, lens + 3)                       # clamped to the drafts
    check_verify(ids, p, q, u, lens - 9)


def test_verify_strides():
    ids, p, q, u, lens = drafts(4, 3, 1003, torch.bfloat16, 6)
    wide = torch.zeros(4, 9, 1100, dtype=torch.bfloat16, device=DEV)
    wide[:, 2:6, 7:1010] = p
    wq = torch.zeros(3, 4, 1009, dtype=torch.bfloat16, device=DEV)
    wq[:, :, 1:1004] = q.transpose(0, 1)
    check_verify(ids, wide[:, 2:6, 7:1010], wq[:, :, 1:1004].transpose(0, 1), u, lens)
    check_verify(ids.t().contiguous().t(), p.transpose(1, 2).contiguous().transpose(1, 2), q,
                 u.t().contiguous().t(), lens)
    check_verify(ids, p[:1].expand(4, 4, 1003), q, u, lens)    # one target row set for all


def test_verify_edges():
    V = 4000
    B, n = 10, 2
    p = torch.full((B, n + 1, V), 1.0 / V)
    q = p[:, :n].clone()
    ids = torch.full((B, n), 17)
    u = torch.full((B, n + 1), 0.5)
    p[0], q[0] = 0, 0                       # no mass at all: -1
    q[1, 0, 17] = 0                         # a token its own draft rules out, kept
    p[2, 0, 17] = 0                         # the target rules it out
    p[3, 0], q[3, 0] = q[3, 0] * 0.25, q[3, 0]   # turned down, and nothing left of the residual
    ids[4, 0], ids[5, 1] = -1, V            # ids outside the vocabulary are turned down
    p[6] = 0
    p[6, :, V - 1] = 1                      # certain of the last token
    u[6, n] = 0.0
    p[7, 0, 5] = float("nan")               # NaN and infinities have no weight, or full
    p[7, 0, 17] = 0
    p[8, 0, 6], p[8, 0, 17] = float("inf"), 0
    u[9] = 1.0                              # past the range: as its end
    u[9, 0] = 0.0
    for dt in (torch.float32, torch.bfloat16):
        for qq in (q.to(dt).to(DEV), None):
            tok, acc = check_verify(ids.to(DEV), p.to(dt).to(DEV), qq, u.to(DEV))
            assert tok[0].tolist() == [-1, -1, -1] and acc[0] == 0
    # the draw at the ends of the range
    for val in (0.0, 1e-9, 1 - 2.0 ** -24, 0.5):
        u[:, n] = val
        check_verify(ids.to(DEV), p.to(DEV), q.to(DEV), u.to(DEV), what=str(val))


def test_verify_draws_each_token_by_its_share():
    """A row of whole multiples: every interval of the uniform number gives
    the token that owns it."""
    V, B = 64, 256
    p = torch.zeros(B, 1, V)
    p[:, 0, ::4] = 1.0 / 16
    u = (torch.arange(B).float() / B).view(B, 1)
    tok, acc = check_verify(torch.zeros(B, 0, dtype=torch.int64, device=DEV), p.to(DEV), None, u.to(DEV))
    assert torch.equal(tok[:, 0].cpu(), torch.arange(B) // 16 * 4)


# ------------------------------------------------------------- used together
def test_refusals_of_the_ops():
    x = torch.randn(4, 100, device=DEV)
    ids = torch.zeros(4, 3, dtype=torch.int64, device=DEV)
    t = torch.zeros(4, 3, device=DEV)
    F = torch.ops.flagos
    for bad in (lambda: F.topk(x, 101), lambda: F.topk(x, -1), lambda: F.topk(x.double(), 2),
                lambda: F.topk(torch.randn(2, 2000, device=DEV), 1025),
                lambda: F.topk(torch.tensor(1.0, device=DEV), 1),
                lambda: F.distill_topk(x, t[:3], ids[:3]), lambda: F.distill_topk(x, t, ids[:, :2]),
                lambda: F.distill_topk(x, t, ids.float()), lambda: F.distill_topk(x, t, ids, 0.0),
                lambda: F.distill_topk(x, t, ids, float("nan")), lambda: F.distill_topk(x, t, ids, -1.0),
                lambda: F.distill_topk(x.double(), t, ids), lambda: F.distill_topk(x, t.double(), ids),
                lambda: F.distill_topk(x, t, ids, 1e-60),
                lambda: F.distill_topk(x, torch.zeros(4, 1025, device=DEV), torch.zeros(4, 1025, dtype=torch.int64, device=DEV)),
                lambda: F.distill_topk(x[:, :0], t, ids),
                lambda: F.distill_topk_grad(x, t, ids, 1.0, torch.ones(3, device=DEV)),
                lambda: F.distill_topk_grad(x, t, ids, 1.0, torch.ones(4, device=DEV).double()),
                lambda: F.distill_topk_backward(t[:, 0], x, torch.zeros(4, 3, device=DEV), t, ids),
                lambda: F.distill_topk(x, t.cpu(), ids),
                lambda: F.verify_draft(ids, x.view(4, 1, 100).expand(4, 4, 100), None, torch.rand(4, 3, device=DEV)),
                lambda: F.verify_draft(ids, x.view(4, 1, 100), None, torch.rand(4, 4, device=DEV)),
                lambda: F.verify_draft(ids.int(), x.view(4, 1, 100).expand(4, 4, 100), None, torch.rand(4, 4, device=DEV)),
                lambda: F.verify_draft(ids, x.view(4, 1, 100).expand(4, 4, 100), x.view(4, 1, 100).expand(4, 3, 100).half(), torch.rand(4, 4, device=DEV)),
                lambda: F.verify_draft(ids, x.view(4, 1, 100).expand(4, 4, 100), None, torch.rand(4, 4, device=DEV), ids[:, 0].int())):
        with pytest.raises((RuntimeError, IndexError)):
            bad()


def test_a_status_of_the_library_is_an_error_with_its_text():
    p = torch.zeros(1, 1, 1 << 26, dtype=torch.bfloat16, device=DEV)
    ids = torch.zeros(1, 0, dtype=torch.int64, device=DEV)
    with pytest.raises(RuntimeError, match="exceeds the fixed maximum.*status 7"):
        torch.ops.flagos.verify_draft(ids, p, None, torch.zeros(1, 1, device=DEV))


def test_streams_and_graph_replay():
    """Each op on a side stream, and captured into a graph that is replayed on
    new inputs."""
    z, t, ids, w = make(17, 9001, 12, torch.bfloat16, 51)
    vi, vp, vq, vu, vl = drafts(5, 3, 9001, torch.float32, 52)

    def all_ops():
        return [*torch_fl.ops.topk(z, 20), *torch.ops.flagos.distill_topk(z, t, ids, 2.0),
                *torch_fl.ops.distill_topk_grad(z, t, ids, 2.0, w),
                *torch_fl.ops.verify_draft(vi, vp, vq, vu, vl)]

    want = all_ops()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = all_ops()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = all_ops()
    z2, t2, ids2, w2 = make(17, 9001, 12, torch.bfloat16, 61)
    vi2, vp2, vq2, vu2, vl2 = drafts(5, 3, 9001, torch.float32, 62)
    for a, b in zip((z, t, ids, w, vi, vp, vq, vu, vl), (z2, t2, ids2, w2, vi2, vp2, vq2, vu2, vl2)):
        a.copy_(b)
    graph.replay()
    torch.cuda.synchronize()
    fresh = all_ops()
    assert all(torch.equal(a, b) for a, b in zip(held, fresh))


def test_two_streams_at_once():
    """The ops share no state: runs that overlap on two streams give what each
    gives alone."""
    sets = []
    for n in range(2):
        z, t, ids, w = make(300, 30011, 40, torch.bfloat16, 81 + n)
        sets.append((z, t, ids, w, drafts(60, 4, 30011, torch.bfloat16, 91 + n)))

    def all_ops(z, t, ids, w, v):
        return [*torch_fl.ops.topk(z, 30), *torch_fl.ops.distill_topk_grad(z, t, ids, 2.0, w),
                torch_fl.ops.distill_topk(z, t, ids, 2.0), *torch_fl.ops.verify_draft(*v)]

    want = [all_ops(*s) for s in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for n, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[n].append(all_ops(*sets[n]))
    torch.cuda.synchronize()
    for n in range(2):
        for run in got[n]:
            assert all(torch.equal(a, b) for a, b in zip(run, want[n]))


def test_many_rows_for_few_clusters():
    """More rows than clusters are resident: the ring of stages turns many times."""
    for R, V, k, dt in ((3000, 513, 9, torch.bfloat16), (1500, 9000, 70, torch.float16),
                        (700, 20001, 100, torch.float32), (400, 40000, 30, torch.bfloat16)):
        z, t, ids, w = make(R, V, k, dt, R)
        check_distill(z, t, ids, w, 1.7, f"{R}x{V}x{k}")


def test_vocabularies_past_eight_ctas():
    """Clusters of more than 8 CTAs (131072 elements of 16 bits, 65536 of fp32)
    and rows that no cluster holds."""
    for R, V, dt in ((5, 151936, torch.bfloat16), (4, 262144, torch.float16), (4, 70000, torch.float32),
                     (3, 131072, torch.float32), (3, 262145, torch.bfloat16), (3, 131073, torch.float32)):
        check_distill(*make(R, V, 20, dt, R + V % 97), tau=1.3, what=f"{R}x{V}")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("R,V,k", [(600, 8008, 20), (300, 40003, 64), (40, 128256, 100), (9, 100, 3)])
def test_a_wait_that_runs_out_is_nan_for_the_whole_row(dtype, R, V, k):
    """With a limit of 0 a wait that finds nothing gives up: every row is then
    either whole or NaN throughout (loss, gradient), the clusters that gave up
    are counted, and the next call is as before."""
    z, t, ids, w = make(R, V, k, dtype, 97 + R)
    want = K.distill_topk_grad(z, t, ids, 2.0, w)
    before = _abi.lost_waits()
    limit = _abi.set_wait_limit(0)
    try:
        runs = [K.distill_topk_grad(z, t, ids, 2.0, w) for _ in range(3)]
        lost = _abi.lost_waits() - before
    finally:
        assert _abi.set_wait_limit(limit) == 0
    assert limit == 2_000_000_000
    nan = 0
    for loss, dz in runs:
        gone = torch.isnan(loss)
        nan += int(gone.sum())
        assert torch.isnan(dz[gone]).all()
        assert torch.equal(loss[~gone], want[0][~gone]) and torch.equal(dz[~gone], want[1][~gone])
    assert nan >= lost                                  # (a cluster has a row at least)
    # (a few hundred bytes may have come before they are first looked for: then no wait runs out)
    assert lost > 0 or z.numel() * z.element_size() < 1 << 16
    again = K.distill_topk_grad(z, t, ids, 2.0, w)
    assert torch.equal(again[0], want[0]) and torch.equal(again[1], want[1])
    assert _abi.lost_waits() == before + lost


def test_draft_model_from_teacher_to_verification():
    """As they are used: a teacher's top logits are kept, a student is trained
    on them through autograd and with the one-call gradient alike, and its
    drafts are verified against the teacher's probabilities."""
    V, H, T, k = 1200, 32, 24, 16
    g = gen(71)
    teacher_w, student_w = torch.randn(V, H, generator=g) / 4, torch.randn(V, H, generator=g) / 4
    h = torch.randn(T, H, generator=g)
    tl = (h @ teacher_w.t()).to("flagos")
    top, ids = torch_fl.ops.topk(tl, k)
    hf = h.to("flagos")
    for _ in range(3):
        w1 = student_w.to("flagos").requires_grad_()
        loss = torch_fl.ops.distill_topk(hf @ w1.t(), top, ids, 1.5)
        loss.mean().backward()
        w2 = student_w.to("flagos").requires_grad_()
        logits = hf @ w2.t()
        l2, dlogits = torch_fl.ops.distill_topk_grad(logits.detach(), top, ids, 1.5,
                                                     torch.full((), 1.0 / T, device="flagos"))
        logits.backward(dlogits)
        # the fp64 gradient of the weights through the same logits
        z = np64(logits.detach())
        _, dz, _ = ops.distill_topk_golden(z, np64(top), np64(ids).astype(np.int64), 1.5, 1.0 / T)
        ref = dz.T @ np64(h)
        # dz carries its own bound; the matrix product T + 8 roundings of its terms
        tol = bounds(logits.detach(), top, ids, 1.5, torch.full((T,), 1.0 / T))[1]
        lim = tol.T @ np.abs(np64(h)) + U * (T + 8) * (np.abs(dz).T @ np.abs(np64(h))) + 1e-12
        # (matrix products of fp32 tensors run in fp32 here: TF32 is off by default)
        assert not torch.backends.cuda.matmul.allow_tf32
        within(w1.grad, ref, lim, "autograd")
        within(w2.grad, ref, lim, "one call")
        student_w = student_w - 0.5 * w2.grad.cpu()
    n = 3
    p = torch.softmax(tl.view(6, n + 1, V), -1)
    q = torch.softmax((hf @ student_w.to("flagos").t()).view(6, n + 1, V)[:, :n], -1)
    drafted = q.argmax(-1)
    u = torch.rand(6, n + 1, generator=g).to("flagos")
    tok, acc = torch_fl.ops.verify_draft(drafted, p, q.contiguous(), u)
    gt, ga = ops.verify_draft_golden(drafted.cpu().numpy(), np64(p), np64(q), u.cpu().numpy())
    np.testing.assert_array_equal(tok.cpu().numpy(), gt)
    np.testing.assert_array_equal(acc.cpu().numpy(), ga)
