"""What the C entries of the operators of a training step around the matrix
products refuse before anything is launched.  CPU only: each call here returns
its status on the host."""

import ctypes
import math

import pytest
import torch

from torch_fl import _abi

BF16, F16, F32, I32, I64 = _abi.BF16, _abi.F16, _abi.F32, _abi.I32, _abi.I64
INVALID, MISALIGNED, WORKSPACE = 1, 3, 5
Q, K, QO, KO, POS, FREQ = 1 << 20, 2 << 20, 3 << 20, 4 << 20, 5 << 20, 6 << 20


def status(name, *args):
    return getattr(_abi.lib(), name)(*args)


def rotary(q=Q, qo=QO, k=K, ko=KO, pos=POS, freq=FREQ, Hq=2, Hk=1, B=2, S=4, D=8, rot=8, dtype=BF16, pd=I32, layout="bshd",
           sq=None, sk=None, sqo=None, sko=None):
    """Strides are over (b, h, s)."""
    dense = lambda H: (S * H * D, D, H * D) if layout == "bshd" else (H * S * D, S * D, D)
    return status("fl_b200_rotary", q, qo, Hq, *(sq or dense(Hq)), *(sqo or sq or dense(Hq)), k, ko, Hk, *(sk or dense(Hk)),
                  *(sko or sk or dense(Hk)), pos, 0, 1, pd, freq, rot, 1.0, 0, 0, B, S, D, dtype, None)


P = [i << 20 for i in range(1, 20)]
FWD = dict(x=P[0], r=P[1], post=P[2], pre=P[3], gate=P[4], y=P[5], h=P[6])
BWD = dict(dy=P[0], dh=P[1], x=P[2], h=P[3], post=P[4], pre=P[5], gate=P[6], dx=P[7], dres=P[8], dpost=P[9], dpre=P[10],
           dgate=P[11], ws=P[12])


def sandwich(dtype=BF16, rows=8, cols=16, per=4, **at):
    a = {**FWD, **at}
    return status("fl_b200_sandwich_norm", a["x"], cols, a["r"], cols, a["post"], a["pre"], a["gate"], per, a["y"], a["h"],
                  rows, cols, 1e-6, 1.0, 0.0, dtype, None)


def sandwich_bwd(dtype=BF16, rows=8, cols=16, per=4, bytes_=0, **at):
    a = {**BWD, **at}
    return status("fl_b200_sandwich_norm_bwd", a["dy"], cols, a["dh"], cols, a["x"], cols, a["h"], cols, a["post"], a["pre"],
                  a["gate"], per, a["dx"], a["dres"], a["dpost"], a["dpre"], a["dgate"], rows, cols, 1e-6, 1.0, 0.0, dtype,
                  a["ws"], bytes_, None)


def span(x=P[0], out=P[1], spans=P[2], pos=P[3], slopes=P[4], rows=8, cols=16, heads=2, q=2, scale=1.0, cap=0.0, dtype=BF16,
         od=None):
    return status("fl_b200_span_softmax", x, cols, spans, 4, 2, pos, 2, 1, slopes, out, cols, rows, cols, heads, q, scale, cap,
                  dtype, dtype if od is None else od, None)


def span_bwd(dy=P[0], y=P[1], x=P[2], spans=P[3], dx=P[4], rows=8, cols=16, heads=2, q=2, scale=1.0, cap=0.0, dtype=BF16,
             yd=None):
    return status("fl_b200_span_softmax_bwd", dy, cols, y, cols, x, cols, spans, 4, 2, dx, cols, rows, cols, heads, q, scale,
                  cap, dtype if yd is None else yd, dtype, None)


def grad_norm(p=4096, norm=64, dtype=F32):
    return status("fl_b200_grad_norm", (ctypes.c_void_p * 1)(p), _abi.i64_array([10]), (ctypes.c_int * 1)(dtype), 1, 0, norm,
                  None, 0, None)


# ----------------------------------------------------------------- alignment
@pytest.mark.parametrize("call", [
    lambda: rotary(q=Q + 1), lambda: rotary(qo=QO + 1), lambda: rotary(k=K + 1), lambda: rotary(ko=KO + 1),
    lambda: rotary(q=Q + 2, dtype=F32), lambda: rotary(q=Q + 3, qo=Q + 3), lambda: rotary(freq=FREQ + 2),
    lambda: rotary(pos=POS + 2), lambda: rotary(pos=POS + 4, pd=I64),
    *[lambda n=n: sandwich(**{n: FWD[n] + 1}) for n in FWD], *[lambda n=n: sandwich(F32, **{n: FWD[n] + 2}) for n in FWD],
    *[lambda n=n: sandwich_bwd(**{n: BWD[n] + 1}) for n in BWD if n != "ws"],
    *[lambda n=n: sandwich_bwd(F32, **{n: BWD[n] + 2}) for n in BWD if n != "ws"],
    lambda: sandwich_bwd(rows=0, dpost=P[9] + 1), lambda: sandwich_bwd(F32, rows=0, dpre=P[9] + 2),
    lambda: span(x=P[0] + 1), lambda: span(out=P[1] + 1), lambda: span(out=P[1] + 2, od=F32), lambda: span(spans=P[2] + 2),
    lambda: span(pos=P[3] + 1), lambda: span(slopes=P[4] + 2),
    lambda: span_bwd(dy=P[0] + 1), lambda: span_bwd(y=P[1] + 1), lambda: span_bwd(y=P[1] + 2, yd=F32),
    lambda: span_bwd(dy=P[0] + 2, yd=F32), lambda: span_bwd(x=P[2] + 1, cap=1.0), lambda: span_bwd(spans=P[3] + 2),
    lambda: span_bwd(dx=P[4] + 1),
    lambda: grad_norm(norm=66), lambda: grad_norm(p=4098),
])
def test_addresses_inside_an_element_are_refused(call):
    """Before the kernels read or write by elements there."""
    assert call() == MISALIGNED


# ------------------------------------------------------------------- overlaps
FUSED = dict(sq=(4 * 40, 8, 40), sk=(4 * 40, 8, 40), B=2, S=4, D=8, Hq=2, Hk=1)  # [B, S, 5 heads of 8] bf16


@pytest.mark.parametrize("call", [
    lambda: rotary(qo=K),                                                # q's result over k
    lambda: rotary(qo=K + 64),
    lambda: rotary(ko=Q), lambda: rotary(ko=Q + 16 * 7),                 # k's over q, over its last head
    lambda: rotary(qo=QO, ko=QO), lambda: rotary(qo=QO, ko=QO + 16),     # the results over each other
    lambda: rotary(q=Q, qo=Q, k=Q, ko=Q), lambda: rotary(q=Q, qo=Q, k=Q + 16, ko=Q + 16),
    lambda: rotary(q=Q, qo=Q, k=Q + 16, ko=Q + 16, **FUSED),             # k is q's second head
    lambda: rotary(q=Q, qo=Q + 16, k=Q + 64, ko=Q + 64, **FUSED),        # q moved by one head
    lambda: rotary(q=Q, qo=QO, k=Q + 32, ko=QO + 16, **FUSED),
    lambda: rotary(sqo=(64, 4, 16)), lambda: rotary(q=Q, qo=Q, sq=(32, 1, 8)),  # heads of a result over each other
    lambda: rotary(q=Q, qo=Q, sq=(1, 1, 1)),
    *[lambda n=n, o=o: sandwich(**{o: FWD[n]}) for n in ("x", "r", "post", "pre", "gate") for o in ("y", "h")],
    lambda: sandwich(y=P[6] + 16), lambda: sandwich(h=P[2] + 16),
    *[lambda n=n, o=o: sandwich_bwd(**{o: BWD[n]}) for n in BWD for o in ("dx", "dres", "dpost", "dpre", "dgate")
      if n != o and n != "ws"],
    lambda: sandwich_bwd(dgate=P[7] + 32), lambda: sandwich_bwd(dpost=P[10] + 16),
])
def test_outputs_over_operands_or_each_other_are_refused(call):
    assert call() == INVALID


# ------------------------------------------------------------- caps and scales
@pytest.mark.parametrize("call", [
    *[lambda kw=kw, f=f: f(**kw) for f in (span, span_bwd) for kw in (
        dict(scale=math.inf), dict(scale=-math.inf), dict(cap=1e-40), dict(scale=1e30, cap=1e-20), dict(scale=-2e38, cap=1.0),
        dict(cap=math.inf))],
])
def test_factors_that_are_infinite_are_refused(call):
    """0 times them would be NaN."""
    assert call() == INVALID


@pytest.mark.parametrize("cap", [0.0, -1.0, 1e-60, 1e60, math.inf, math.nan])
def test_caps_that_fp32_does_not_hold_are_refused(cap):
    """One that rounds to 0 would be none."""
    from torch_fl import kernels

    x, spans = torch.zeros(1, 1, 2, 4), torch.zeros(2, 2, dtype=torch.int32)
    for call in (lambda: kernels.span_softmax(x, spans, 1.0, cap), lambda: kernels.span_softmax_backward(x, x, x, spans, 1.0, cap)):
        with pytest.raises(ValueError, match="cap"):
            call()


TOO_LARGE = 7


def test_distances_past_32_bits_are_refused():
    """A position of -2^30 is more than 2^31 from the last key of such a row."""
    wide = dict(rows=1, heads=1, q=1, cols=(1 << 30) + 8)
    assert span(**wide) == TOO_LARGE
    assert span(rows=(1 << 30) + 1, heads=1, q=(1 << 30) + 1) == TOO_LARGE


# ------------------------------------------------------------- what is not refused
def test_clipping_outputs_told_from_each_other():
    """One status each: lists whose outputs meet are refused as arguments, the
    others come as far as the workspace that is not there."""
    def clip(p, q, n=(10, 10)):
        c = len(p)
        return status("fl_b200_clip_grads", (ctypes.c_void_p * c)(*p), (ctypes.c_void_p * c)(*q), _abi.i64_array(n),
                      (ctypes.c_int * c)(*[F32] * c), c, 1.0, 0, 64, None, 0, None)

    # (without a GPU the call ends before it looks at the workspace)
    fine = WORKSPACE if torch.cuda.is_available() else clip((), (), ())
    assert fine not in (0, INVALID)
    assert clip((4096, 4096), (4096, 4096)) == INVALID
    assert clip((4096, 8192), (8192, 4096)) == INVALID
    assert clip((4096, 8192), (1 << 14, (1 << 14) + 36)) == INVALID
    assert clip((4096, 4096 + 36), (1 << 14, 4096)) == INVALID
    assert clip((4096, 4096 + 16), (1 << 14, 1 << 15)) == fine           # tensors may meet
    assert clip((4096, 8192), (1 << 14, (1 << 14) + 40)) == fine         # neighbours
    assert clip((4096, 4096 + 40), (4096, 4096 + 40)) == fine            # in place
    assert clip((4096, 4096), (1 << 14, 4096), (0, 10)) == fine          # an empty one meets nothing


def test_spans_without_keys_are_empty():
    from torch_fl import ops

    s = ops.attention_spans(2, 0)
    assert s.shape == (1, 2, 2) and bool((s[..., 0] >= s[..., 1]).all())


# ----------------------------------------------------------- arguments in Python
def test_yarn_needs_a_base_above_one():
    from torch_fl import ops

    for theta in (1.0, 0.5):
        with pytest.raises(ValueError, match="theta"):
            ops.rope_frequencies(64, theta, "yarn", 4.0, 2048)


def test_gates_of_fewer_dims_are_refused():
    from torch_fl import kernels

    with pytest.raises(ValueError, match="gate"):
        kernels._gate_rows(torch.zeros(2, 3, 4, 8), torch.zeros(1, 8))
    assert kernels._gate_rows(torch.zeros(2, 3, 4, 8), torch.zeros(2, 1, 1, 8)) == 12


@pytest.mark.parametrize("call", [sandwich, sandwich_bwd, lambda **kw: span(heads=1, q=1, slopes=None, **kw),
                                  lambda **kw: span_bwd(heads=1, q=1, **kw)])
def test_rows_whose_end_passes_31_bits_in_a_loop_are_refused(call):
    """A counter of elements that steps past 2^31 - 1 wraps around."""
    assert call(rows=1, cols=0x7fff0001) == TOO_LARGE
    assert call(rows=1, cols=0x7fffff00) == TOO_LARGE
