"""The operators of a training step around the matrix products, on the GPU
against 64 bits: rotary positions, the norms around a block with its gate and
residual, softmax over spans of keys, and gradient clipping.

Tolerances are carried along: `Num` holds a value in 64 bits and a bound on
how far fp32 arithmetic in the operator's order may be off it, u = 2^-24 for
each rounding; a sum of terms adds chain * u * sum |term|, chain being the
longest run of additions into one accumulator (a thread's share of the row and
the tree above it).  What is stored adds half a step of its type, and half of
the smallest subnormal.
"""

import math

import numpy as np
import pytest
import torch

import torch_fl
from torch_fl import kernels as K

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def gen(seed):
    return torch.Generator().manual_seed(seed)


def np64(t):
    return t.detach().cpu().double().numpy()


class Num:
    """A value and a bound on its error in fp32."""

    def __init__(self, v, e=0.0):
        self.v = np.asarray(v, dtype=np.float64)
        self.e = np.broadcast_to(np.asarray(e, dtype=np.float64), self.v.shape)

    def __add__(self, o):
        o = o if isinstance(o, Num) else Num(o)
        v = self.v + o.v
        return Num(v, self.e + o.e + U * np.abs(v))

    def __neg__(self):
        return Num(-self.v, self.e)

    def __sub__(self, o):
        return self + -(o if isinstance(o, Num) else Num(o))

    def __mul__(self, o):
        o = o if isinstance(o, Num) else Num(o)
        v = self.v * o.v
        return Num(v, np.abs(self.v) * o.e + np.abs(o.v) * self.e + self.e * o.e + U * np.abs(v))

    def sum(self, axis, chain):
        return Num(self.v.sum(axis, keepdims=True),
                   self.e.sum(axis, keepdims=True) + chain * U * np.abs(self.v).sum(axis, keepdims=True))

    def at(self, index):
        return Num(self.v[index], self.e[index])


def close(got, want, dtype, what=""):
    """got (a tensor of dtype) within want's bound and its own rounding."""
    f = torch.finfo(dtype)
    g = np64(got)
    half = np.maximum((np.abs(want.v) + want.e) * f.eps / 2 * 1.0001, f.tiny * f.eps * 0.5001)
    bad = np.abs(g - want.v) - want.e - half
    assert g.shape == want.v.shape and not np.isnan(g).any(), what
    if g.size == 0:
        return
    i = np.unravel_index(bad.argmax(), bad.shape)
    assert bad[i] <= 0, f"{what}: {g[i]} is not {want.v[i]} within {want.e[i]:.3e} + {half[i]:.3e} at {i}"


# --------------------------------------------------------------------- rotary
def rotary_want(x, positions, freq, scale, interleaved, inverse):
    """x [B, S, H, D], positions [B, S]."""
    turns = positions[..., None].astype(np.float64) * freq.astype(np.float64) / (2 * math.pi)
    # the fraction of a turn: fp64 products and the constant; then fp32: half a step
    # of a number below 1 (times pi), 2 steps of sincospif, one of the scale
    err = 2 * math.pi * np.abs(turns) * 2.0 ** -51 + (math.pi / 2 + 4 + 1) * U
    angle = 2 * math.pi * (turns - np.rint(turns))
    cos = Num(scale * np.cos(angle), abs(scale) * err)
    sin = Num((-1 if inverse else 1) * scale * np.sin(angle), abs(scale) * err)
    cos, sin = (Num(t.v[:, :, None], t.e[:, :, None]) for t in (cos, sin))
    n = freq.size
    a, b = (x[..., 0:2 * n:2], x[..., 1:2 * n:2]) if interleaved else (x[..., :n], x[..., n:2 * n])
    lo, hi = Num(a) * cos - Num(b) * sin, Num(b) * cos + Num(a) * sin
    out = Num(x.copy(), np.zeros_like(x))
    e = np.array(out.e)
    if interleaved:
        out.v[..., 0:2 * n:2], out.v[..., 1:2 * n:2] = lo.v, hi.v
        e[..., 0:2 * n:2], e[..., 1:2 * n:2] = lo.e, hi.e
    else:
        out.v[..., :n], out.v[..., n:2 * n] = lo.v, hi.v
        e[..., :n], e[..., n:2 * n] = lo.e, hi.e
    out.e = e
    return out


def check_rotary(q, k, positions, freq, scale=1.0, interleaved=False, inverse=False, layout="bshd", fn=None):
    dim = 2 if layout == "bshd" else 1
    fn = fn or (lambda *a: torch_fl.ops.rotary(*a, scale, interleaved, dim, inverse))
    got = fn(q, k, positions, freq)
    f = freq.cpu().numpy()
    for x, y in zip((q, k), got):
        xs = x if layout == "bshd" else x.transpose(1, 2)
        ys = y if layout == "bshd" else y.transpose(1, 2)
        pos = positions.cpu().numpy()
        pos = np.broadcast_to(pos if pos.ndim == 2 else pos[None], xs.shape[:2])
        want = rotary_want(np64(xs), pos, f, np.float32(scale), interleaved, inverse)
        assert y.dtype == x.dtype and y.shape == x.shape
        close(ys, want, x.dtype, f"{tuple(x.shape)} n={f.size} il={interleaved}")
        # what is not turned stays bit for bit
        assert torch.equal(ys[..., 2 * f.size:].cpu(), xs[..., 2 * f.size:].cpu())
    return got


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("B,S,Hq,Hk,D,n", [
    (1, 1, 1, 1, 2, 1), (2, 3, 4, 2, 8, 2), (1, 5, 3, 1, 64, 32), (8, 1, 32, 8, 128, 64), (1, 700, 32, 8, 128, 64),
    (3, 37, 5, 5, 80, 10), (1, 9, 2, 1, 96, 8), (2, 11, 16, 16, 192, 32), (1, 4, 7, 3, 6, 3), (1, 3, 2, 2, 13, 5),
    (1, 2, 1, 1, 256, 128), (1, 2, 2, 1, 2048, 1024), (1, 3, 40, 0, 64, 16),
])
def test_rotary(dtype, interleaved, B, S, Hq, Hk, D, n):
    g = gen(B * 100 + S + D)
    q = torch.randn(B, S, Hq, D, generator=g).to(dtype).to(DEV)
    k = torch.randn(B, S, Hk, D, generator=g).to(dtype).to(DEV)
    freq = (1e4 ** (-torch.arange(n, dtype=torch.float64) / n)).float().to(DEV)
    pos = torch.randint(0, 131072, (B, S), generator=g).to(DEV)
    check_rotary(q, k, pos, freq, 1.25, interleaved)
    check_rotary(q, k, pos[0].int(), freq, 1.0, interleaved, inverse=True)


@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_strides(interleaved):
    """A fused projection's views, [B, H, S, D], odd offsets, broadcast and
    strided positions, an expanded operand."""
    g = gen(5)
    B, S, H, D, n = 2, 9, 3, 32, 12
    freq = torch.rand(n, generator=g).to(DEV)
    pos = torch.randint(0, 5000, (B, 2 * S), generator=g).to(DEV)
    for dtype in TYPES:
        qkv = torch.randn(B, S, 3 * H * D + 3, generator=g).to(dtype).to(DEV)
        for off in (0, 1, 2, 3):
            q = qkv[..., off:off + H * D].view(B, S, H, D)
            k = qkv[..., H * D + off:2 * H * D + off].view(B, S, H, D)
            check_rotary(q, k, pos[:, ::2], freq, interleaved=interleaved)
            check_rotary(q.transpose(1, 2), k.transpose(1, 2), pos[:1, :S], freq, interleaved=interleaved,
                         layout="bhsd")
        one = torch.randn(B, S, 1, D, generator=g).to(dtype).to(DEV).expand(B, S, H, D)
        check_rotary(q, one, pos[0, :S], freq, interleaved=interleaved)
        turned = torch.randn(B, S, D, H, generator=g).to(dtype).to(DEV).transpose(2, 3)   # head dim strided
        check_rotary(turned, one, pos[0, :S], freq, interleaved=interleaved)


def test_rotary_far_positions():
    """Positions where an fp32 angle has lost its cosine; negative ones."""
    g = gen(6)
    freq = (1e4 ** (-torch.arange(64, dtype=torch.float64) / 64)).float().to(DEV)
    pos = torch.tensor([0, 1, -1, -131071, 1 << 20, 999999999, 1 << 31, 1 << 40, -(1 << 33)])
    q = torch.randn(1, pos.numel(), 4, 128, generator=g).to(DEV)
    check_rotary(q, q[:, :, :1], pos.to(DEV), freq)


def test_rotary_empty_and_nan():
    freq = torch.ones(4, device=DEV)
    for shape in [(0, 3, 2, 8), (2, 0, 2, 8), (2, 3, 0, 8)]:
        q, k = torch_fl.ops.rotary(torch.zeros(shape, device=DEV), torch.zeros(shape, device=DEV),
                                   torch.zeros(shape[1], dtype=torch.int64, device=DEV), freq, unsqueeze_dim=2)
        assert q.shape == k.shape == torch.Size(shape)
    x = torch.ones(1, 2, 1, 16, device=DEV)
    x[0, 0, 0, 3] = math.nan
    y, _ = torch_fl.ops.rotary(x, x, torch.arange(2, device=DEV), freq, unsqueeze_dim=2)
    assert torch.isnan(y).nonzero().tolist() == [[0, 0, 0, 3], [0, 0, 0, 7]]


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("D,n", [(64, 32), (80, 10), (24, 4)])
def test_rotary_in_place(interleaved, D, n):
    g = gen(7)
    qkv = torch.randn(2, 7, 5 * D, generator=g).bfloat16().to(DEV)
    before = qkv.clone()
    freq, pos = torch.rand(n, generator=g).to(DEV), torch.arange(7, device=DEV)
    q, k = qkv[..., :3 * D].view(2, 7, 3, D), qkv[..., 3 * D:4 * D].view(2, 7, 1, D)
    want = K.rotary(q, k, pos, freq, 1.5, interleaved, layout="bshd")
    K.rotary(q, k, pos, freq, 1.5, interleaved, layout="bshd", inplace=True)
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])
    assert torch.equal(qkv[..., 4 * D:], before[..., 4 * D:])     # the values beside them


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim", [1, 2])
def test_rotary_gradient(interleaved, dim):
    g = gen(8)
    q0, k0 = torch.randn(2, 4, 6, 16, generator=g), torch.randn(2, 4, 6, 16, generator=g)
    gq, gk = torch.randn(2, 4, 6, 16, generator=g), torch.randn(2, 4, 6, 16, generator=g)
    freq, pos = torch.rand(5, generator=g), torch.arange((6, 4)[dim - 1])
    q, k = (t.to("flagos").requires_grad_() for t in (q0, k0))
    qo, ko = torch_fl.ops.rotary(q, k, pos.to("flagos"), freq.to("flagos"), 0.7, interleaved, dim)
    dq, dk = torch.autograd.grad((qo, ko), (q, k), (gq.to("flagos"), gk.to("flagos")), create_graph=True)
    for got, grad in ((dq, gq), (dk, gk)):
        x = grad if dim == 2 else grad.transpose(1, 2)
        want = rotary_want(np64(x), np.broadcast_to(pos.numpy(), x.shape[:2]), freq.numpy(), np.float32(0.7),
                           interleaved, True)
        close(got if dim == 2 else got.transpose(1, 2), want, torch.float32)
    # linear: <R x, g> = <x, R' g>, and only one of the two asked for
    (only,) = torch.autograd.grad(torch_fl.ops.rotary(q, k, pos.to("flagos"), freq.to("flagos"), 0.7, interleaved,
                                                      dim)[1].sum(), (k,))
    assert only.shape == k.shape
    assert abs(float((qo * gq.to("flagos")).sum() - (q * dq).sum())) < 1e-3


# -------------------------------------------------------------------- sandwich
def rms(x, chain, eps):
    """1 / sqrt(mean(x^2) + eps) of the last dim: the sum's error halves under
    the root; three roundings after it."""
    s = (x * x).sum(-1, chain)
    n = x.v.shape[-1]
    m = s.v / n + eps
    r = 1 / np.sqrt(m)
    rel = 0.5 * (s.e / n + 2 * U * m) / m
    return Num(r, r * (rel / np.maximum(1 - 2 * rel, 0.5) + 3 * U))


def sandwich_want(x, res, post, pre, gate, eps, scale, off):
    chain = x.shape[-1] / 256 + 90
    rx = rms(Num(x), chain, eps)
    branch = Num(x) * (rx * scale) * (Num(post) + off)
    if gate is not None:
        branch = branch * Num(gate)
    h = branch + Num(res)
    y = h * rms(h, chain, eps) * (Num(pre) + off)
    return y, h


def sandwich_back_want(dy, dh, x, h, post, pre, gate, eps, scale, off):
    """x and the rest [rows, cols]; gate rows expanded to x's."""
    cols = x.shape[-1]
    chain, down = cols / 256 + 90, x.shape[0] + 20
    rx, rh = rms(Num(x), chain, eps), rms(Num(h), chain, eps)
    m, n = Num(h) * rh, Num(x) * rx
    d = Num(dy) * (Num(pre) + off)
    mean = (d * m).sum(-1, chain) * (1 / cols)
    g = rh * (d - m * mean)
    if dh is not None:
        g = g + Num(dh)
    gated = Num(np.ones_like(x) if gate is None else gate) * scale
    dpre = (Num(dy) * m).sum(0, down)
    each = g * n                                   # A's terms
    dpost = (each * gated).sum(0, down)
    t = g * gated * (Num(post) + off)
    dx = rx * (t - n * ((t * n).sum(-1, chain) * (1 / cols)))
    dgate_terms = each * ((Num(post) + off) * scale)
    return dx, g, dpost, dpre, dgate_terms, down


def sandwich_inputs(shape, gate, dtype, seed, off):
    g = gen(seed)
    B, S, H = shape
    x = torch.randn(B, S, H, generator=g) * (0.3 + torch.randn(H, generator=g).abs())
    res = 3 * torch.randn(B, S, H, generator=g)
    post, pre = ((1 - off + 0.2 * torch.randn(H, generator=g)) for _ in range(2))
    gs = {"none": None, "channel": (H,), "sequence": (B, 1, H), "token": (B, S, H), "first": (1, 1, H)}[gate]
    gt = None if gs is None else 0.5 * torch.randn(*gs, generator=g)
    dy, dh = torch.randn(B, S, H, generator=g), torch.randn(B, S, H, generator=g)
    return [None if t is None else t.to(dtype).to(DEV) for t in (x, res, post, pre, gt, dy, dh)]


SHAPES = [(1, 1, 1), (1, 1, 4096), (2, 3, 7), (2, 5, 64), (3, 17, 1001), (2, 40, 512), (1, 300, 2048), (4, 33, 4096),
          (1, 3, 16384), (2, 2, 20000), (5, 1, 264), (700, 2, 128)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("gate", ["none", "channel", "sequence", "token"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_sandwich(dtype, gate, shape):
    off = float(sum(shape) % 2)
    x, res, post, pre, gt, dy, dh = sandwich_inputs(shape, gate, dtype, sum(shape), off)
    y, h = torch_fl.ops.sandwich_norm(x, res, post, pre, 1e-6, gt, 0.25, off)
    gnp = None if gt is None else np64(gt)
    wy, wh = sandwich_want(np64(x), np64(res), np64(post), np64(pre), gnp, np.float32(1e-6), 0.25, off)
    close(h, wh, dtype, "h")
    close(y, wy, dtype, "y")
    got = torch.ops.flagos.sandwich_norm_backward(dy, dh, x, h, post, pre, gt, 1e-6, 0.25, off)
    rows = shape[0] * shape[1]
    flat = lambda t: np64(t).reshape(rows, -1)
    wide = None if gt is None else np.broadcast_to(gnp, x.shape).reshape(rows, -1)
    dx, g, dpost, dpre, terms, down = sandwich_back_want(flat(dy), flat(dh), flat(x), flat(h), np64(post), np64(pre),
                                                         wide, np.float32(1e-6), 0.25, off)
    close(got[1].view(rows, -1), g, dtype, "dresidual")
    close(got[0].view(rows, -1), dx, dtype, "dx")
    close(got[3][None], dpre, dtype, "dpre")
    close(got[2][None], dpost, dtype, "dpost")
    if gt is not None:
        t3 = Num(terms.v.reshape(x.shape), terms.e.reshape(x.shape))
        want = {"channel": lambda: Num(t3.v.reshape(rows, -1), t3.e.reshape(rows, -1)).sum(0, down).at(0),
                "sequence": lambda: t3.sum(1, down), "token": lambda: t3}[gate]()
        close(got[4], want, dtype, "dgate")
    # the sums have one order
    again = torch.ops.flagos.sandwich_norm_backward(dy, dh, x, h, post, pre, gt, 1e-6, 0.25, off)
    assert all(torch.equal(a, b) for a, b in zip(got, again))


@pytest.mark.parametrize("dtype", TYPES)
def test_sandwich_strided_rows_and_no_dh(dtype):
    off = 0.0
    x, res, post, pre, gt, dy, dh = sandwich_inputs((2, 9, 96), "channel", dtype, 3, off)
    wide = torch.zeros(2, 9, 200, dtype=dtype, device=DEV)
    for at in (0, 3, 8):
        xs, rs = wide[..., at:at + 96], wide.flip(0)[..., at:at + 96]
        xs.copy_(x)
        rs = rs.copy_(res)
        got = torch_fl.ops.sandwich_norm(xs, rs, post, pre, 1e-5, gt)
        want = torch_fl.ops.sandwich_norm(x, res, post, pre, 1e-5, gt)
        wy, wh = sandwich_want(np64(x), np64(res), np64(post), np64(pre), np64(gt), np.float32(1e-5), 1.0, off)
        close(got[0], wy, dtype), close(got[1], wh, dtype), close(want[0], wy, dtype)
    h = want[1]
    for d in (dy.transpose(0, 1).contiguous().transpose(0, 1), dy[:, :, :1].expand(2, 9, 96)):
        got = torch.ops.flagos.sandwich_norm_backward(d, None, x, h, post, pre, gt, 1e-5)
        flat = lambda t: np64(t).reshape(18, -1)
        dx, g, *_ = sandwich_back_want(flat(d), None, flat(x), flat(h), np64(post), np64(pre),
                                       np.broadcast_to(np64(gt), (18, 96)), np.float32(1e-5), 1.0, off)
        close(got[0].view(18, -1), dx, dtype), close(got[1].view(18, -1), g, dtype)


def test_sandwich_gate_rows_across_chunks():
    """Gate rows of every length against the chunks of the column sums."""
    for B, S in ((3, 1000), (1000, 3), (1, 3001), (37, 81), (2, 1500), (1500, 2)):
        x, res, post, pre, gt, dy, dh = sandwich_inputs((B, S, 40), "sequence", torch.float32, B, 0.0)
        h = torch_fl.ops.sandwich_norm(x, res, post, pre, 1e-6, gt)[1]
        got = torch.ops.flagos.sandwich_norm_backward(dy, dh, x, h, post, pre, gt, 1e-6)
        flat = lambda t: np64(t).reshape(B * S, -1)
        *_, terms, down = sandwich_back_want(flat(dy), flat(dh), flat(x), flat(h), np64(post), np64(pre),
                                             np.broadcast_to(np64(gt), x.shape).reshape(B * S, -1), np.float32(1e-6), 1.0, 0.0)
        close(got[4], Num(terms.v.reshape(x.shape), terms.e.reshape(x.shape)).sum(1, down), torch.float32, f"{B}x{S}")


@pytest.mark.parametrize("gate", ["none", "channel", "first", "sequence", "token"])
def test_sandwich_autograd(gate):
    """Against the formula written in torch and differentiated there, in fp64."""
    eps, scale, off = 1e-5, 0.5, 1.0
    x, res, post, pre, gt, dy, dh = (None if t is None else t.cpu() for t in
                                     sandwich_inputs((2, 5, 48), gate, torch.float32, 4, off))
    leaves = [t for t in (x, res, post, pre, gt) if t is not None]
    ref = [t.double().requires_grad_() for t in leaves]
    rx, rr, rpo, rpr = ref[:4]
    norm = lambda t: t / torch.sqrt((t * t).mean(-1, keepdim=True) + eps)
    hh = rr + scale * (ref[4] if gt is not None else 1.0) * norm(rx) * (off + rpo)
    yy = norm(hh) * (off + rpr)
    for use_y, use_h in ((True, True), (True, False), (False, True)):
        want = torch.autograd.grad((yy * dy.double()).sum() * use_y + (hh * dh.double()).sum() * use_h, ref,
                                   retain_graph=True)
        mine = [t.to("flagos").requires_grad_() for t in leaves]
        y, h = torch_fl.ops.sandwich_norm(*mine[:4], eps, mine[4] if gt is not None else None, scale, off)
        outs = [o for o, u in ((y, use_y), (h, use_h)) if u]
        grads = [t.to("flagos") for t, u in ((dy, use_y), (dh, use_h)) if u]
        got = torch.autograd.grad(outs, mine, grads)
        for a, b in zip(got, want):
            # h was rounded to fp32 before its norm's gradient (one part in 2^24 of values around 3):
            # some hundred roundings of terms around 1
            assert a.shape == b.shape and float((a.cpu().double() - b).abs().max()) < 200 * U * float(b.abs().max() + 1)


# ---------------------------------------------------------------- span softmax
def span_want(x, spans, scale, cap, slopes, positions):
    B, H, Q, n = x.shape
    key = np.arange(n)
    lo, hi = (np.clip(spans[..., i], 0, n)[:, None, :, None] for i in (0, 1))
    seen = np.broadcast_to((key >= lo) & (key < hi), x.shape)
    with np.errstate(all="ignore"):
        xs = np.where(seen, x, 0.0)
        z = xs * scale
        e = 2 * U * np.abs(z)
        if cap:
            t = np.tanh(z / cap)
            rel = 4 * U * np.abs(2 * z / cap) + 4 * U                     # of e^(2u): its argument and ex2
            z, e = cap * t, cap * ((1 - t * t) / 2 * rel + 6 * U)
        if slopes is not None:
            dist = np.abs(positions[:, None, :, None] - key)
            bias = slopes[None, :, None, None] * dist
            z, e = z - bias, e + U * np.abs(bias) + 2 * U * np.abs(z - bias)
        zm = np.where(seen, z, -np.inf)
        top = zm.max(-1, keepdims=True)
        top = np.where(np.isfinite(top), top, 0)
        p = np.where(seen, np.exp(z - top), 0.0)
        # units of log 2: the argument's conversion, the difference, ex2
        ep = p * np.expm1(np.minimum(2 * (e + np.where(seen, e, 0).max(-1, keepdims=True)) + 6 * U * (np.abs(z) + np.abs(top)), 50.0)) \
            + 4 * U * p + seen * 2.0 ** -126
        s = p.sum(-1, keepdims=True)
        es = ep.sum(-1, keepdims=True) + (n / 512 + 60) * U * s
        ok = s > 0
        y = np.where(ok, p / np.where(ok, s, 1), 0)
        rel = es / np.where(ok, s, 1)
        ey = np.where(ok, (ep + p * rel / np.maximum(1 - rel, 0.5)) / np.where(ok, s, 1) + 3 * U * y, 0)
    return Num(y, np.where(seen, ey, 0)), seen


def span_back_want(dy, y, x, seen, scale, cap):
    y, dy = np.where(seen, y, 0), np.where(seen, dy, 0)
    chain = y.shape[-1] / 512 + 60
    s = (Num(y) * Num(dy)).sum(-1, chain)
    d = Num(y) * scale * (Num(dy) - s)
    if cap:
        z = np.where(seen, x, 0) * scale / cap
        t = np.tanh(z)
        q = (1 - t) / 2
        eq = q * (1 - q) * (4 * U * np.abs(2 * z) + 4 * U) + 3 * U * q
        d = d * (Num(4 * q, 4 * eq) * Num(1 - q, eq))
    return Num(np.where(seen, d.v, 0), np.where(seen, d.e + 2.0 ** -126, 0))


def check_span(x, spans, scale=1.0, cap=None, slopes=None, positions=None, out_dtype=None, back=True, seed=0):
    B, H, Q, n = x.shape
    y = torch_fl.ops.span_softmax(x, spans, scale, cap, slopes, positions, out_dtype)
    sp = np.broadcast_to(spans.cpu().numpy().reshape(-1, Q, 2), (B, Q, 2))
    pos = np.arange(Q) + n - Q if positions is None else positions.cpu().numpy()
    pos = np.broadcast_to(pos, (B, Q)).astype(np.float64)
    sl = None if slopes is None else slopes.cpu().numpy().astype(np.float64)
    s32, c32 = float(np.float32(scale)), float(np.float32(cap or 0))
    want, seen = span_want(np64(x), sp, s32, c32, sl, pos)
    close(y, want, y.dtype, "y")
    assert not np64(y)[~seen].any()                            # exact zeros
    if back:
        dy = torch.randn(x.shape, generator=gen(seed)).to(y.dtype).to(DEV)
        dx = torch.ops.flagos.span_softmax_backward(dy, y, x, spans, scale, cap)
        assert dx.dtype == x.dtype
        close(dx, span_back_want(np64(dy), np64(y), np64(x), seen, s32, c32), x.dtype, "dx")
        assert not np64(dx)[~seen].any()
    return y


def random_spans(B, Q, n, g):
    a, b = (torch.randint(-3, n + 4, (B, Q), generator=g) for _ in range(2))
    spans = torch.stack([torch.minimum(a, b), torch.maximum(a, b)], -1)
    spans[:, ::5] = torch.tensor([0, n])
    spans[0, 0] = torch.tensor([n // 2, n // 2])                 # sees nothing
    if Q > 2:
        spans[-1, 1] = torch.tensor([n - 1, 0])                  # upside down: nothing
        spans[-1, 2] = torch.tensor([n - 1, n])                  # one key
    return spans.int().to(DEV)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cap,bias", [(None, False), (30.0, False), (None, True), (5.0, True)])
@pytest.mark.parametrize("B,H,Q,n", [
    (1, 1, 1, 1), (2, 2, 3, 5), (1, 3, 17, 64), (2, 2, 9, 255), (1, 2, 33, 511), (1, 1, 7, 1000), (2, 1, 5, 2049),
    (1, 2, 4, 4095), (1, 1, 3, 8192), (1, 1, 3, 16383), (1, 2, 2, 32768), (1, 1, 3, 40001),
])
def test_span_softmax(dtype, cap, bias, B, H, Q, n):
    g = gen(B + H + Q + n)
    x = (4 * torch.randn(B, H, Q, n, generator=g)).to(dtype).to(DEV)
    slopes = (2.0 ** -torch.arange(1, H + 1).float()).to(DEV) if bias else None
    pos = torch.randint(0, n, (B, Q), generator=g).int().to(DEV) if bias and Q % 2 else None
    spans = random_spans(B, Q, n, g)
    check_span(x, spans, 0.5, cap, slopes, pos)
    if dtype != torch.float32:
        check_span(x, spans, 0.5, cap, slopes, pos, torch.float32)


@pytest.mark.parametrize("dtype", TYPES)
def test_span_softmax_masks_of_torch(dtype):
    """attention_spans against dense masks: causal, windows, documents, a
    prefix, padding."""
    g = gen(11)
    B, H, Q = 3, 2, 45
    x = (3 * torch.randn(B, H, Q, Q, generator=g)).to(dtype)
    i, j = torch.arange(Q)[:, None], torch.arange(Q)[None]
    ids = torch.sort(torch.randint(0, 5, (B, Q), generator=g), -1).values
    same = ids[:, :, None] == ids[:, None, :]
    lens, pre = torch.tensor([45, 20, 1]), torch.tensor([7, 0, 45])
    real = (j[None] < lens[:, None, None]) & (i[None] < lens[:, None, None])
    cases = [
        (dict(), (j <= i).expand(B, Q, Q)),
        (dict(causal=False), torch.ones(B, Q, Q, dtype=torch.bool)),
        (dict(window=6), ((j <= i) & (j > i - 6)).expand(B, Q, Q)),
        (dict(causal=False, window=6), ((j - i).abs() < 6).expand(B, Q, Q)),
        (dict(documents=ids), (j <= i) & same),
        (dict(documents=ids[0], causal=False), same[:1].expand(B, Q, Q)),
        (dict(prefix=pre), (j <= i) | ((i < pre[:, None, None]) & (j < pre[:, None, None]))),
        (dict(lengths=lens, window=9), (j <= i) & (j > i - 9) & real),
        (dict(lengths=lens, documents=ids, causal=False), same & real),
    ]
    for kw, mask in cases:
        spans = torch_fl.ops.attention_spans(Q, Q, **{k: v.to(DEV) if torch.is_tensor(v) else v for k, v in kw.items()},
                                             device=DEV)
        key = torch.arange(Q, device=DEV)
        dense = (key >= spans[..., :1]) & (key < spans[..., 1:])
        assert torch.equal(dense.expand(B, Q, Q).cpu(), mask), kw
        check_span(x.to(DEV), spans, 0.7)


def test_span_softmax_special_values():
    """Anything outside a span; softmax's own rules inside it."""
    inf, nan, low = math.inf, math.nan, torch.finfo(torch.float32).min
    x = torch.full((1, 1, 8, 40), nan)
    x[..., 3:23] = torch.randn(20, generator=gen(1))
    x[0, 0, 1, :3] = inf
    x[0, 0, 2, 5] = -inf
    x[0, 0, 3, 6] = inf
    x[0, 0, 4, 7] = nan
    x[0, 0, 5, 3:23] = -inf
    x[0, 0, 6, 3:23] = low
    spans = torch.tensor([3, 23]).repeat(8, 1)
    spans[7] = torch.tensor([23, 23])
    for dtype in TYPES:
        xd = x.clamp(min=-math.inf).to(dtype)
        xd[0, 0, 6, 3:23] = torch.finfo(dtype).min
        y = torch_fl.ops.span_softmax(xd.to(DEV), spans.int().to(DEV)).cpu().double()[0, 0]
        want = torch.softmax(xd[0, 0, :, 3:23].double(), -1)
        assert not y[:, :3].any() and not y[:, 23:].any() and not y[7].any()
        for r in (3, 4, 5):
            assert torch.isnan(y[r, 3:23]).all()
        f = torch.finfo(dtype)
        ok = [0, 1, 2, 6]
        assert ((y[ok, 3:23] - want[ok]).abs() <= want[ok] * (f.eps / 2 + 100 * U) + f.tiny * f.eps).all()
    # long rows go another way
    x = torch.randn(1, 1, 4, 70000, generator=gen(2))
    x[0, 0, 1, 500] = inf
    x[0, 0, 2, 100:900] = -inf
    x[0, 0, 3, 600] = nan
    y = torch_fl.ops.span_softmax(x.to(DEV), torch.tensor([[100, 900]] * 4).int().to(DEV)).cpu()[0, 0]
    assert torch.isnan(y[1:, 100:900]).all() and not torch.isnan(y[0]).any()
    assert not y[:, :100].any() and not y[:, 900:].any()


@pytest.mark.parametrize("dtype", TYPES)
def test_span_softmax_strides(dtype):
    g = gen(12)
    wide = (2 * torch.randn(2, 3, 8, 90, generator=g)).to(dtype).to(DEV)
    spans = random_spans(2, 8, 70, g)
    for at in (0, 1, 5, 8):
        x = wide[..., at:at + 70]
        check_span(x, spans, 0.5, 20.0)
        check_span(x.transpose(0, 1).contiguous().transpose(0, 1), spans, 0.5, 20.0)
        check_span(x, spans[:1], 0.5)
    flipped = torch.stack([spans[..., 1], spans[..., 0]], -1)[..., [1, 0]]
    check_span(wide[..., :70], flipped)
    # rows far apart: offsets past 32 bits
    if dtype == torch.bfloat16:
        big = torch.empty(3 << 30, dtype=dtype, device=DEV)
        x = big.as_strided((1, 1, 3, 640), (0, 0, (3 << 30) // 2 - 640, 1))
        x.copy_(2 * torch.randn(1, 1, 3, 640, generator=g))
        check_span(x, random_spans(1, 3, 640, g), 0.5, 20.0)


def test_span_softmax_empty():
    for shape in ((0, 2, 3, 4), (2, 0, 3, 4), (2, 2, 0, 4), (2, 2, 3, 0)):
        y = torch_fl.ops.span_softmax(torch.zeros(shape, device=DEV),
                                      torch.zeros(1, shape[2], 2, dtype=torch.int32, device=DEV))
        assert y.shape == torch.Size(shape)


@pytest.mark.parametrize("cap,dtype,out", [(None, torch.float32, None), (4.0, torch.float32, None),
                                           (4.0, torch.bfloat16, torch.float32), (None, torch.bfloat16, torch.float32)])
def test_span_softmax_autograd(cap, dtype, out):
    g = gen(13)
    x0 = (2 * torch.randn(2, 3, 9, 33, generator=g)).to(dtype)
    spans, slopes = random_spans(2, 9, 33, g), torch.tensor([0.5, 0.25, 0.125])
    gy = torch.randn(2, 3, 9, 33, generator=g)
    x = x0.to("flagos").requires_grad_()
    y = torch_fl.ops.span_softmax(x, spans.cpu().to("flagos"), 0.7, cap, slopes.to("flagos"), dtype=out)
    (dx,) = torch.autograd.grad(y, x, gy.to(y.dtype).to("flagos"))
    ref = x0.double().requires_grad_()
    z = ref * 0.7
    if cap:
        z = cap * torch.tanh(z / cap)
    key = torch.arange(33)
    z = z - slopes.double()[None, :, None, None] * (torch.arange(9)[:, None] + 24 - key).abs()
    sp = spans.cpu()
    seen = ((key >= sp[:, :, :1]) & (key < sp[:, :, 1:]))[:, None].expand_as(z)
    e = torch.exp(z - z.detach().amax(-1, keepdim=True)) * seen
    s = e.sum(-1, keepdim=True)
    (want,) = torch.autograd.grad(e / torch.where(s > 0, s, 1.0), ref, gy.double())
    assert dx.dtype == dtype
    # terms around 1: some hundred roundings of fp32, and one of x's type
    tol = 200 * U + want.abs() * torch.finfo(dtype).eps / 2 * 1.001
    assert ((dx.cpu().double() - want).abs() <= tol).all()


# -------------------------------------------------------------------- clipping
def clip_want(tensors, bound, kind):
    all_ = np.concatenate([np64(t).ravel() for t in tensors]) if tensors else np.zeros(0)
    with np.errstate(all="ignore"):
        norm = np.abs(all_).max(initial=0.0) if kind == math.inf else np.sqrt(np.square(all_).sum())
        factor = bound / (norm + 1e-6)
    factor = 1.0 if factor >= 1 else factor
    return norm, factor


def check_clip(tensors, bound, kind=2.0, out=None, what=""):
    before = [t.clone() for t in tensors]
    norm, factor = clip_want(tensors, bound, kind)
    n = torch_fl.ops.grad_norm(tensors, kind)
    # squares in fp32 over 64 elements a thread, sums of positive terms
    assert abs(float(n) - norm) <= (40 * U if kind == 2.0 else U) * norm, (what, float(n), norm)
    got, n2 = torch_fl.ops.clip_grads(tensors, bound, kind, out)
    assert float(n2) == float(n) and n.dtype == torch.float32 and n.dim() == 0
    for t, b in zip(got, before):
        assert t.dtype == b.dtype and t.shape == b.shape
        want = np64(b) * factor
        close(t, Num(want, 50 * U * np.abs(want)), t.dtype, what)
    return got


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", [2.0, math.inf])
@pytest.mark.parametrize("sizes", [[1], [7], [0, 5, 0], [4096], [33, 1, 100003, 8], [64] * 33, [1001] * 129,
                                   [3] * 700, [3000001, 5]], ids=lambda s: f"{len(s)}x{s[0]}")
def test_clip(dtype, kind, sizes):
    g = gen(len(sizes) + sizes[0])
    ts = [(torch.randn(n, generator=g) * 0.01 * (1 + i % 3)).to(dtype).to(DEV) for i, n in enumerate(sizes)]
    check_clip(ts, 0.003, kind, what="clipped")
    check_clip(ts, 1e6, kind, what="within")
    out = [torch.empty_like(t) for t in ts]
    check_clip(ts, 0.003, kind, out)
    kept = [t.clone() for t in ts]
    check_clip(ts, 1e6, kind, ts)                             # in place: nothing is written
    assert all(torch.equal(a, b) for a, b in zip(ts, kept))
    check_clip(ts, 0.003, kind, ts)


def test_clip_mixed_types_offsets_and_layouts():
    g = gen(21)
    ts = []
    for i, dtype in enumerate(TYPES * 5):
        base = torch.randn(5000 + i, generator=g).to(dtype).to(DEV)
        ts.append(base[i % 9:])
    ts += [torch.randn(30, 40, generator=g).to(DEV).t(), torch.randn(4, 5, 6, generator=g).to(DEV).permute(2, 0, 1),
           torch.randn(40, 40, generator=g).to(DEV)[:, 3:17], torch.randn(3, 1, generator=g).to(DEV).expand(3, 4),
           torch.tensor(2.5, device=DEV)]
    check_clip(ts, 1.0)
    # a bucket's views, packed without gaps: other offsets than the tensors'
    bucket = torch.zeros(sum(t.numel() for t in ts[:15]) + 1, device=DEV, dtype=torch.bfloat16)
    half = [t for t in ts[:15] if t.dtype == torch.bfloat16]
    parts = list(bucket[1:1 + sum(t.numel() for t in half)].split([t.numel() for t in half]))
    check_clip(half, 0.5, out=parts)
    assert float(bucket[0]) == 0 and not bucket[1 + sum(t.numel() for t in half):].any()
    inplace = [t.clone() for t in ts[:15]] + [t.clone(memory_format=torch.preserve_format) for t in ts[15:]]
    check_clip(inplace, 0.5, out=inplace)
    sliced = torch.randn(40, 40, generator=g).to(DEV)
    kept = sliced.clone()
    torch_fl.ops.clip_grads([sliced[:, 3:17]], 0.1, out=[sliced[:, 3:17]])
    assert torch.equal(sliced[:, :3], kept[:, :3]) and torch.equal(sliced[:, 17:], kept[:, 17:])
    assert not torch.equal(sliced[:, 3:17], kept[:, 3:17])


@pytest.mark.parametrize("scale", [1e-30, 1e-22, 1e19, 1e30])
def test_clip_values_whose_squares_fp32_cannot_hold(scale):
    g = gen(22)
    for dtype in (torch.float32, torch.bfloat16):
        ts = [(torch.randn(n, generator=g) * scale).to(dtype).to(DEV) for n in (5, 70000)]
        ts.append(torch.zeros(5000, dtype=dtype, device=DEV))
        check_clip(ts, scale)
        check_clip(ts, scale, math.inf)


def test_clip_not_finite():
    """As the formula has it: NaN spreads, an infinite norm makes zeros (and
    NaN of the infinity)."""
    for kind in (2.0, math.inf):
        for bad in (math.nan, math.inf, -math.inf):
            a, b = torch.ones(5000, device=DEV), torch.ones(7, device=DEV)
            a[4321] = bad
            got, n = torch_fl.ops.clip_grads([b, a], 1.0, kind)
            want_n = torch.linalg.vector_norm(torch.cat([a, b]).cpu(), kind)
            assert torch.equal(torch.isnan(n.cpu()), torch.isnan(want_n)) and (bool(torch.isnan(n)) or float(n) == float(want_n))
            factor = (1.0 / (want_n + 1e-6)).clamp(max=1.0)
            torch.testing.assert_close(got[0].cpu(), b.cpu() * factor, equal_nan=True)
            torch.testing.assert_close(got[1].cpu(), a.cpu() * factor, equal_nan=True)
    z = torch.zeros(100, device=DEV)
    got, n = torch_fl.ops.clip_grads([z], 0.0)
    assert float(n) == 0 and not got[0].any()


def test_clip_grad_norm_of_parameters():
    ps = [torch.nn.Parameter(torch.randn(5, 7, generator=gen(i)).to("flagos")) for i in range(3)]
    for p in ps[:2]:
        p.grad = torch.randn(5, 7, generator=gen(9)).to("flagos")
    ref = [torch.nn.Parameter(torch.zeros(5, 7)) for _ in range(2)]
    for p, r in zip(ps, ref):
        r.grad = p.grad.cpu().clone()
    want = torch.nn.utils.clip_grad_norm_(ref, 0.5)
    n = torch_fl.ops.clip_grad_norm_(ps, 0.5, error_if_nonfinite=True)
    torch.testing.assert_close(n.cpu(), want, rtol=1e-6, atol=0)
    for p, r in zip(ps, ref):
        torch.testing.assert_close(p.grad.cpu(), r.grad, rtol=1e-6, atol=0)
    assert float(torch_fl.ops.clip_grad_norm_([], 1.0)) == 0.0
    ps[0].grad[0, 0] = math.inf
    kept = ps[1].grad.clone()
    with pytest.raises(RuntimeError, match="not finite"):
        torch_fl.ops.clip_grad_norm_(ps, 0.5, error_if_nonfinite=True)
    assert torch.equal(ps[1].grad.cpu(), kept.cpu())


# ------------------------------------------------------------------- refusals
def test_refusals():
    F = torch_fl.ops
    q = torch.zeros(2, 3, 4, 8, device=DEV)
    pos, freq = torch.arange(3, device=DEV), torch.ones(4, device=DEV)
    w = torch.ones(8, device=DEV)
    sp = torch.zeros(4, 2, dtype=torch.int32, device=DEV)
    bad = [
        lambda: F.rotary(q, q, pos, freq),                                # [B, H, S, D]: 4 positions
        lambda: F.rotary(q, q, pos.float(), freq, unsqueeze_dim=2),
        lambda: F.rotary(q, q, pos, freq.double(), unsqueeze_dim=2),
        lambda: F.rotary(q, q, pos, torch.ones(5, device=DEV), unsqueeze_dim=2),
        lambda: F.rotary(q, q, pos, freq[:0], unsqueeze_dim=2),
        lambda: F.rotary(q, q.bfloat16(), pos, freq, unsqueeze_dim=2),
        lambda: F.rotary(q, q[:1], pos, freq, unsqueeze_dim=2),
        lambda: F.rotary(q, q, pos, freq, unsqueeze_dim=3),
        lambda: F.rotary(q, q, pos, freq, math.nan, unsqueeze_dim=2),
        lambda: F.rotary(q, q, pos.cpu(), freq, unsqueeze_dim=2),
        lambda: F.rotary(q.double(), q.double(), pos, freq, unsqueeze_dim=2),
        lambda: F.sandwich_norm(q, q[:1], w, w, 1e-6),
        lambda: F.sandwich_norm(q, q, w[:4], w, 1e-6),
        lambda: F.sandwich_norm(q, q, w, w.half(), 1e-6),
        lambda: F.sandwich_norm(q, q, w, w, -1.0),
        lambda: F.sandwich_norm(q, q, w, w, 1e-6, torch.ones(1, 3, 1, 8, device=DEV)),   # dims inside
        lambda: F.sandwich_norm(q, q, w, w, 1e-6, torch.ones(2, 8, device=DEV)),
        lambda: F.sandwich_norm(q, q, w, w, 1e-6, w.half()),
        lambda: F.sandwich_norm(q, q, w, w, 1e-6, scale=math.inf),
        lambda: F.span_softmax(q, sp.long()),
        lambda: F.span_softmax(q, sp[:3]),
        lambda: F.span_softmax(q, sp[:, :1]),
        lambda: F.span_softmax(q, sp.expand(3, 4, 2)),
        lambda: F.span_softmax(q, sp, cap=0.0),
        lambda: F.span_softmax(q, sp, cap=-1.0),
        lambda: F.span_softmax(q, sp, cap=math.nan),
        lambda: F.span_softmax(q, sp, slopes=torch.ones(2, device=DEV)),
        lambda: F.span_softmax(q, sp, slopes=torch.ones(3, device=DEV).half()),
        lambda: F.span_softmax(q, sp, positions=torch.zeros(4, device=DEV)),
        lambda: F.span_softmax(q, sp, dtype=torch.bfloat16),
        lambda: F.span_softmax(q[0, 0, 0], sp),
        lambda: F.grad_norm([]),
        lambda: F.grad_norm([q], 1.0),
        lambda: F.grad_norm([q, pos]),
        lambda: F.clip_grads([q], -1.0),
        lambda: F.clip_grads([q], math.nan),
        lambda: F.clip_grads([q], 1.0, out=[]),
        lambda: F.clip_grads([q], 1.0, out=[q.half()]),
        lambda: F.clip_grads([q], 1.0, out=[q[:1]]),
    ]
    for i, call in enumerate(bad):
        with pytest.raises((RuntimeError, ValueError, TypeError, NotImplementedError)):
            call()
            pytest.fail(f"call {i} was taken")
    flat = torch.zeros(100, device=DEV)
    with pytest.raises(Exception):                            # an output over another part of its tensor
        F.clip_grads([flat[:50]], 1.0, out=[flat[10:60]])


def test_second_derivatives_and_tangents_are_refused():
    x = torch.randn(2, 4, 16, device="cpu").to("flagos").requires_grad_()
    w = torch.ones(16).to("flagos")
    y, h = torch_fl.ops.sandwich_norm(x, x.detach(), w, w, 1e-6)
    (g,) = torch.autograd.grad(y.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="no second derivative"):
        torch.autograd.grad(g.sum(), x)
    sp = torch_fl.ops.attention_spans(4, 16, device="flagos")
    y = torch_fl.ops.span_softmax(x, sp, cap=3.0)
    (g,) = torch.autograd.grad((y * y).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="no second derivative"):
        torch.autograd.grad(g.sum(), x)
    freq = torch.ones(4).to("flagos").requires_grad_()
    with pytest.raises(RuntimeError, match="no gradient"):
        torch_fl.ops.rotary(x[None], x[None], torch.arange(4).to("flagos"), freq, unsqueeze_dim=1)


# ------------------------------------------------------- together, as they are used
def attention_block(p, x, pos, freq, spans, slopes, mine):
    """A small decoder layer's first half and the norm before its second."""
    B, S, E = x.shape
    q = (x @ p["q"]).view(B, S, 4, E // 4)
    k = (x @ p["k"]).view(B, S, 4, E // 4)
    v = (x @ p["v"]).view(B, S, 4, E // 4).transpose(1, 2)
    if mine:
        q, k = torch_fl.ops.rotary(q, k, pos, freq, 1.1, True, unsqueeze_dim=2)
        s = q.transpose(1, 2) @ k.permute(0, 2, 3, 1)
        w = torch_fl.ops.span_softmax(s, spans, 0.3, 10.0, slopes)
        a = (w @ v).transpose(1, 2).reshape(B, S, E) @ p["o"]
        return torch_fl.ops.sandwich_norm(a, x, p["post"], p["pre"], 1e-6, p["gate"], 0.5)

    def turn(t):
        n = freq.numel()
        ang = pos.double()[:, None] * freq.double()
        c, s_ = 1.1 * torch.cos(ang)[:, None], 1.1 * torch.sin(ang)[:, None]
        e, o = t[..., 0:2 * n:2], t[..., 1:2 * n:2]
        return torch.cat([torch.stack([e * c - o * s_, o * c + e * s_], -1).flatten(-2), t[..., 2 * n:]], -1)

    q, k = turn(q), turn(k)
    z = (q.transpose(1, 2) @ k.permute(0, 2, 3, 1)) * 0.3
    z = 10.0 * torch.tanh(z / 10.0)
    key = torch.arange(S)
    z = z - slopes.double()[None, :, None, None] * (key[:, None] - key).abs()
    seen = ((key >= spans[..., :1]) & (key < spans[..., 1:]))[:, None]
    e = torch.exp(z.masked_fill(~seen, -math.inf) - z.detach().amax(-1, keepdim=True))
    t = e.sum(-1, keepdim=True)
    w = e / torch.where(t > 0, t, 1.0)
    a = (w @ v).transpose(1, 2).reshape(B, S, E) @ p["o"]
    norm = lambda t: t / torch.sqrt((t * t).mean(-1, keepdim=True) + 1e-6)
    h = x + 0.5 * p["gate"] * norm(a) * p["post"]
    return norm(h) * p["pre"], h


def test_training_step():
    """Packed documents through rotary, scores, norms; backward; clipping."""
    g = gen(31)
    B, S, E = 2, 23, 32
    p0 = {n: 0.3 * torch.randn(E, E, generator=g) for n in "qkvo"}
    p0.update(post=1 + 0.1 * torch.randn(E, generator=g), pre=1 + 0.1 * torch.randn(E, generator=g),
              gate=0.5 * torch.randn(B, 1, E, generator=g))
    x0, gy, gh = (torch.randn(B, S, E, generator=g) for _ in range(3))
    ids = torch.sort(torch.randint(0, 3, (B, S), generator=g), -1).values
    spans = torch_fl.ops.attention_spans(S, S, documents=ids, lengths=torch.tensor([S, 17]))
    pos, freq, slopes = torch.arange(S), torch.rand(3, generator=g), torch.tensor([0.5, 0.25, 0.1, 0.05])

    mine = {n: t.to("flagos").requires_grad_() for n, t in p0.items()}
    x = x0.to("flagos").requires_grad_()
    y, h = attention_block(mine, x, pos.to("flagos"), freq.to("flagos"), spans.to("flagos"), slopes.to("flagos"), True)
    torch.autograd.backward([y, h], [gy.to("flagos"), gh.to("flagos")])
    ref = {n: t.double().requires_grad_() for n, t in p0.items()}
    xr = x0.double().requires_grad_()
    yr, hr = attention_block(ref, xr, pos, freq, spans, slopes, False)
    torch.autograd.backward([yr, hr], [gy.double(), gh.double()])
    # matrix products of 32 terms and the operators in fp32: 2^-24 times a few hundred of each value's scale
    near = lambda a, b: float((a.cpu().double() - b).abs().max()) <= 1000 * U * float(b.abs().max())
    assert near(y.detach(), yr.detach()) and near(h.detach(), hr.detach()) and near(x.grad, xr.grad)
    for n in p0:
        assert near(mine[n].grad, ref[n].grad), n
    norm = torch_fl.ops.clip_grad_norm_(list(mine.values()), 1.0)
    want = torch.nn.utils.clip_grad_norm_(list(ref.values()), 1.0)
    assert abs(float(norm) - float(want)) <= 1000 * U * float(want)
    for n in p0:
        assert near(mine[n].grad, ref[n].grad), n


# -------------------------------------------------- streams, graphs, other entry points
def everything(s):
    q, k = torch_fl.ops.rotary(s["q"], s["q"], s["pos"], s["freq"], unsqueeze_dim=2)
    y, h = torch_fl.ops.sandwich_norm(s["x"], s["r"], s["w"], s["w"], 1e-6, s["gate"])
    grads = torch.ops.flagos.sandwich_norm_backward(y, h, s["x"], h, s["w"], s["w"], s["gate"], 1e-6)
    p = torch_fl.ops.span_softmax(s["s"], s["spans"], 0.5, 20.0)
    d = torch.ops.flagos.span_softmax_backward(s["s"], p, s["s"], s["spans"], 0.5, 20.0)
    c, n = torch_fl.ops.clip_grads([s["x"], s["s"], s["w"]], 0.5)
    return [q, k, y, h, *grads, p, d, *c, n]


def everything_inputs(seed):
    g = gen(seed)
    r = lambda *shape: torch.randn(*shape, generator=g).bfloat16().to(DEV)
    return {"q": r(2, 50, 4, 64), "pos": torch.randint(0, 9999, (2, 50), generator=g).to(DEV),
            "freq": torch.rand(16, generator=g).to(DEV), "x": r(2, 600, 512), "r": r(2, 600, 512), "w": r(512),
            "gate": r(2, 1, 512), "s": r(1, 4, 100, 333), "spans": random_spans(1, 100, 333, g)}


def test_graphs_replay_with_new_inputs_and_share_nothing():
    s = everything_inputs(1)
    want = [t.clone() for t in everything(s)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        everything(s)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(everything(s))
        graphs.append(g)
    for g, o in zip(graphs, outs):
        g.replay()
    torch.cuda.synchronize()
    for o in outs:
        assert all(torch.equal(a, b) for a, b in zip(o, want))
    new = everything_inputs(2)
    want = [t.clone() for t in everything(new)]
    for n in s:
        s[n].copy_(new[n])
    graphs[1].replay()
    graphs[0].replay()
    torch.cuda.synchronize()
    for o in outs:
        assert all(torch.equal(a, b) for a, b in zip(o, want))


def test_streams():
    a, b = everything_inputs(3), everything_inputs(4)
    want = [t.clone() for t in everything(a)], [t.clone() for t in everything(b)]
    torch.cuda.synchronize()
    sa, sb = torch.cuda.Stream(), torch.cuda.Stream()
    got = [None, None]
    for _ in range(3):
        with torch.cuda.stream(sa):
            got[0] = everything(a)
        with torch.cuda.stream(sb):
            got[1] = everything(b)
    torch.cuda.synchronize()
    for w, o in zip(want, got):
        assert all(torch.equal(x, y) for x, y in zip(w, o))


def test_kernels_module_agrees():
    s = everything_inputs(5)
    q, k = K.rotary(s["q"], s["q"], s["pos"], s["freq"], layout="bshd")
    y, h = K.sandwich_norm(s["x"], s["r"], s["w"], s["w"], 1e-6, s["gate"])
    grads = K.sandwich_norm_backward(y, h, s["x"], h, s["w"], s["w"], 1e-6, s["gate"])
    p = K.span_softmax(s["s"], s["spans"], 0.5, 20.0)
    d = K.span_softmax_backward(s["s"], p, s["s"], s["spans"], 0.5, 20.0)
    c, n = K.clip_grads([s["x"], s["s"], s["w"]], 0.5)
    assert float(K.grad_norm([s["x"], s["s"], s["w"]])) == float(n)
    for a, b in zip([q, k, y, h, *grads, p, d, *c, n], everything(s)):
        assert torch.equal(a, b)
    only, none = K.rotary(s["q"], None, s["pos"], s["freq"], layout="bshd")
    assert none is None and torch.equal(only, q)


def test_pdl_changes_nothing():
    s = everything_inputs(6)
    want = everything(s)
    before = torch_fl._abi.set_pdl(False)
    try:
        got = everything(s)
    finally:
        torch_fl._abi.set_pdl(before)
    assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_clip_through_the_dispatcher_and_versions():
    ts = [torch.randn(300, generator=gen(i)).to(DEV) for i in range(3)]
    want, n = torch_fl.ops.clip_grads(ts, 0.5)
    assert torch.equal(torch.ops.flagos.grad_norm(ts, 2.0), n)
    got, n2 = torch.ops.flagos.clip_grads(ts, 0.5, 2.0)
    assert torch.equal(n, n2) and all(torch.equal(a, b) for a, b in zip(got, want))
    out = [torch.empty_like(t) for t in ts]
    before = [t._version for t in out]
    assert torch.equal(torch.ops.flagos.clip_grads_out(ts, 0.5, 2.0, out), n)
    assert all(torch.equal(a, b) for a, b in zip(out, want))
    assert all(t._version > b for t, b in zip(out, before))
    with pytest.raises(RuntimeError):
        torch_fl.ops.clip_grads([ts[0], torch.zeros(3)], 1.0, out=[ts[0], torch.zeros(3)])   # on the CPU
    with pytest.raises(RuntimeError):
        torch_fl.ops.grad_norm([torch.zeros(3)])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,S,Hq,Hk,D,n", [(7, 3001, 1, 1, 80, 40), (30, 997, 2, 1, 64, 8), (1500, 13, 1, 0, 16, 4),
                                           (9000, 2, 1, 1, 24, 5), (20000, 1, 1, 1, 8, 4)])
def test_rotary_many_tokens_of_few_heads(dtype, B, S, Hq, Hk, D, n):
    g = gen(B + S)
    q, k = (torch.randn(B, S, h, D, generator=g).to(dtype).to(DEV) for h in (Hq, Hk))
    freq = (1e4 ** (-torch.arange(n, dtype=torch.float64) / n)).float().to(DEV)
    pos = torch.randint(0, 131072, (B, S), generator=g).to(DEV)
    for interleaved in (False, True):
        check_rotary(q, k, pos, freq, 1.25, interleaved)


@pytest.mark.parametrize("gate", ["none", "channel", "sequence", "token"])
@pytest.mark.parametrize("B,S,H", [(3, 700, 1001), (2, 9, 9280), (5, 60, 758), (1, 3, 33000), (300, 2, 129), (2, 150, 10248)])
def test_sandwich_rows_by_packs_and_by_elements(gate, B, S, H):
    test_sandwich(torch.float16, gate, (B, S, H))
    test_sandwich(torch.float32, gate, (B, S, H))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cap,bias", [(None, False), (20.0, True)])
def test_span_softmax_long_rows(dtype, cap, bias):
    g = gen(41)
    for n in (33000, 70001):
        x = (4 * torch.randn(1, 2, 5, n, generator=g)).to(dtype).to(DEV)
        slopes = torch.tensor([0.01, 0.001]).to(DEV) if bias else None
        check_span(x, random_spans(1, 5, n, g), 0.5, cap, slopes)
        x[0, 0, 1, n // 3:n // 2] = -math.inf                   # whole packs of nothing
        if not cap:
            y = torch_fl.ops.span_softmax(x, torch.tensor([[0, n]] * 5).int().to(DEV))
            assert not torch.isnan(y).any() and not y[0, 0, 1, n // 3:n // 2].any()
            assert abs(float(y[0, 0, 1].double().sum()) - 1) < 2.0 ** -8


def test_span_softmax_output_in_another_step():
    """Rows that begin elsewhere in a 16-byte pack than their results do."""
    g = gen(42)
    wide = (2 * torch.randn(2, 2, 6, 97, generator=g)).half().to(DEV)
    for at in range(4):
        check_span(wide[..., at:at + 90], random_spans(2, 6, 90, g), 0.5, 20.0)


@pytest.mark.parametrize("n", [40, 700, 5000, 40000])
def test_span_softmax_rows_far_from_zero(n):
    """Rows whose maximum is so far from 0 that log2 e times it has no digits
    left behind the point, or no room; the differences in a row stay exact."""
    g = gen(51)
    big = [1e3, -1e4, 1e6, -1e7, 1e9, -1e15, 1e22, -1e30, 1e37, 3e38]
    x = torch.stack([c + torch.randint(0, 9, (n,), generator=g) * max(1.0, abs(c) * 2.0 ** -23) for c in big])
    y = torch_fl.ops.span_softmax(x[None, None].to(DEV), torch.tensor([[1, n - 1]] * len(big)).int().to(DEV))[0, 0]
    want = torch.softmax(x[:, 1:n - 1].double(), -1)
    got = y[:, 1:n - 1].cpu().double()
    # scale 1: scores are exact; a difference's rounding and ex2, sums of positive terms
    assert ((got - want).abs() <= want * (n / 512 + 100) * U + 2.0 ** -126).all()


def test_span_softmax_distances_far_out():
    """Positions and keys past 2^24, where floats are whole no longer."""
    n = 64
    pos = torch.tensor([(1 << 25) + 3, -(1 << 25) - 1, 5, (1 << 31) - 1, -(1 << 31)], dtype=torch.int32)
    x = torch.zeros(1, 1, 5, n, device=DEV)
    y = torch_fl.ops.span_softmax(x, torch.tensor([[0, n]] * 5).int().to(DEV), slopes=torch.ones(1, device=DEV),
                                  positions=pos.to(DEV)).cpu().double()[0, 0]
    assert not torch.isnan(y).any()
    for r in (2,):
        want = torch.softmax(-(pos[r].double() - torch.arange(n)).abs(), -1)
        assert ((y[r] - want).abs() <= 100 * U * want + 2.0 ** -126).all()
    assert torch.allclose(y.sum(-1), torch.ones(5, dtype=torch.float64), atol=1e-5)


def test_clip_refuses_outputs_that_meet():
    a, b = torch.ones(1000, device=DEV), torch.full((1000,), 2.0, device=DEV)
    for grads, out in (([a, a], [a, a]), ([a, b], [b, a]), ([a[:500], a[400:]], [a[:500], a[400:]]),
                       ([a, b], [a, a]), ([a[:10], b], [a[5:15], b])):
        with pytest.raises(RuntimeError):
            torch_fl.ops.clip_grads(grads, 0.1, out=out)
    assert bool((a == 1).all()) and bool((b == 2).all())
    # neighbours in one buffer do not meet; one tensor may be counted twice, and clipped to new outputs
    torch_fl.ops.clip_grads([a[:500], a[500:]], 0.1, out=[a[:500], a[500:]])
    check_clip([b, b], 0.1)


def test_spans_of_documents_on_flagos():
    ids = torch.tensor([[4, 4, 4, 9, 9, 0], [1, 1, 2, 2, 2, 2]])
    kw = dict(lengths=torch.tensor([5, 6]), prefix=torch.tensor([2, 0]), window=3)
    want = torch_fl.ops.attention_spans(6, 6, documents=ids, **kw)
    got = torch_fl.ops.attention_spans(6, 6, documents=ids.to("flagos"),
                                       **{k: v.to("flagos") if torch.is_tensor(v) else v for k, v in kw.items()})
    assert got.device.type == "flagos" and torch.equal(got.cpu(), want)


@pytest.mark.parametrize("gate", ["none", "channel", "sequence", "token"])
@pytest.mark.parametrize("dtype,H", [(torch.bfloat16, 1032), (torch.float16, 4088), (torch.bfloat16, 8192),
                                     (torch.bfloat16, 16376), (torch.float32, 4104), (torch.float32, 8192)])
def test_sandwich_many_rows(dtype, H, gate):
    """Rows enough for resident CTAs that walk them."""
    rows = 4800 if H < 4000 else 7200 if H < 5000 and dtype != torch.float32 else 3000
    B, S = 6, rows // 6 + 1
    x, res, post, pre, gt, *_ = sandwich_inputs((B, S, H), gate, dtype, H, 1.0)
    y, h = torch_fl.ops.sandwich_norm(x, res, post, pre, 1e-6, gt, 0.5, 1.0)
    pick = torch.tensor([0, 1, S - 1, S, 2 * S + 3, 3 * S, B * S // 2, B * S - 2, B * S - 1])
    flat = lambda t: np64(t.reshape(B * S, H)[pick.to(DEV)])
    wide = None if gt is None else flat(gt.expand(B, S, H))
    wy, wh = sandwich_want(flat(x), flat(res), np64(post), np64(pre), wide, np.float32(1e-6), 0.5, 1.0)
    close(h.view(B * S, H)[pick.to(DEV)], wh, dtype, "h")
    close(y.view(B * S, H)[pick.to(DEV)], wy, dtype, "y")
    # every row as the same rows alone, but for the order of its sums
    y1, h1 = torch_fl.ops.sandwich_norm(x[1:2], res[1:2], post, pre, 1e-6, gt[1:2] if gt is not None and gt.dim() == 3 else gt,
                                        0.5, 1.0)
    step = torch.finfo(dtype).eps * 1.01
    assert bool(((h[1:2].float() - h1.float()).abs() <= step * h1.float().abs() + 1e-5).all())
    assert bool(((y[1:2].float() - y1.float()).abs() <= step * y1.float().abs() + 1e-5).all())


def test_dispatch_modes_see_the_ops():
    from torch.utils._python_dispatch import TorchDispatchMode

    seen = []

    class Watch(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            seen.append(func.name())
            return func(*args, **(kwargs or {}))

    s = everything_inputs(7)
    want = everything(s)
    with Watch():
        got = everything(s)
    for name in ("rotary", "sandwich_norm", "sandwich_norm_backward", "span_softmax", "span_softmax_backward"):
        assert any(f"flagos::{name}" == n.split(".")[0] for n in seen), (name, seen)
    assert all(torch.equal(a, b) for a, b in zip(want, got))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("at", [1, 2, 4, 6])
def test_sandwich_offsets(dtype, at):
    """Rows that begin one, two or four elements into a pack, forward and backward."""
    x, res, post, pre, gt, dy, dh = sandwich_inputs((3, 11, 130), "sequence", dtype, at, 1.0)
    wide = [torch.zeros(3, 11, 150, dtype=dtype, device=DEV)[..., at:at + 130].copy_(t) for t in (x, res, dy, dh)]
    y, h = torch_fl.ops.sandwich_norm(wide[0], wide[1], post, pre, 1e-6, gt, 0.5, 1.0)
    wy, wh = sandwich_want(np64(x), np64(res), np64(post), np64(pre), np64(gt), np.float32(1e-6), 0.5, 1.0)
    close(h, wh, dtype, "h"), close(y, wy, dtype, "y")
    got = torch.ops.flagos.sandwich_norm_backward(wide[2], wide[3], wide[0], h, post, pre, gt, 1e-6, 0.5, 1.0)
    flat = lambda t: np64(t).reshape(33, -1)
    dx, g, dpost, dpre, terms, down = sandwich_back_want(
        flat(dy), flat(dh), flat(x), flat(h), np64(post), np64(pre),
        np.broadcast_to(np64(gt), x.shape).reshape(33, -1), np.float32(1e-6), 0.5, 1.0)
    close(got[0].reshape(33, -1), dx, dtype, "dx"), close(got[1].reshape(33, -1), g, dtype, "dresidual")
    close(got[2][None], dpost, dtype, "dpost"), close(got[3][None], dpre, dtype, "dpre")
    close(got[4], Num(terms.v.reshape(x.shape), terms.e.reshape(x.shape)).sum(1, down), dtype, "dgate")
