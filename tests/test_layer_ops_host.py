"""Host logic of the operators of a training step around the matrix products:
frequencies for long contexts, spans from masks, and the C ABI's refusals.
CPU only: nothing here launches a kernel."""

import ctypes
import math

import numpy as np
import pytest
import torch

import torch_fl
from torch_fl import _abi

BF16, F32, I32 = _abi.BF16, _abi.F32, _abi.I32


# ---------------------------------------------------------------- frequencies
def test_frequencies_default_and_linear():
    f, s = torch_fl.ops.rope_frequencies(8, 1e4)
    np.testing.assert_allclose(f.numpy(), [1, 0.1, 0.01, 0.001], rtol=2.0 ** -23)
    assert s == 1.0 and f.dtype == torch.float32
    g, _ = torch_fl.ops.rope_frequencies(8, 1e4, "linear", 4.0)
    np.testing.assert_allclose(g.numpy(), f.numpy() / 4, rtol=2.0 ** -23)


def test_frequencies_dynamic_keep_the_first_and_stretch_the_last():
    f, _ = torch_fl.ops.rope_frequencies(64, 1e4)
    short, _ = torch_fl.ops.rope_frequencies(64, 1e4, "dynamic", 2.0, 2048, 100)
    np.testing.assert_array_equal(short.numpy(), f.numpy())       # no longer than the original: unchanged
    g, _ = torch_fl.ops.rope_frequencies(64, 1e4, "dynamic", 2.0, 2048, 8192)
    assert float(g[0]) == 1.0
    # (theta r^(d/(d-2)))^(-(d-2)/d) = theta^(-(d-2)/d) / r with r = 2 * 4 - 1
    np.testing.assert_allclose(float(g[-1]), float(f[-1]) / 7, rtol=1e-6)


@pytest.mark.parametrize("method,low,high", [("yarn", 1.0, 32.0), ("llama3", 1.0, 4.0)])
def test_frequencies_by_turns(method, low, high):
    dim, theta, factor, L = 128, 5e5, 8.0, 8192
    f, _ = torch_fl.ops.rope_frequencies(dim, theta)
    g, s = torch_fl.ops.rope_frequencies(dim, theta, method, factor, L, low_turns=low, high_turns=high)
    ratio, turns = g.double() / f.double(), L * f.double() / (2 * math.pi)
    if method == "llama3":
        keep = ((turns - low) / (high - low)).clamp(0, 1)
        np.testing.assert_allclose(ratio.numpy(), (keep + (1 - keep) / factor).numpy(), rtol=1e-6)
        assert s == 1.0
    else:
        # the ramp's ends are whole indexes at or beyond the bounds
        assert (ratio[turns > high * 1.3] > 1 - 1e-6).all() and (abs(ratio[turns < low / 1.3] - 1 / factor) < 1e-6).all()
        assert (ratio.diff() <= 1e-7).all()
        assert s == pytest.approx(0.1 * math.log(factor) + 1)


@pytest.mark.parametrize("kw", [dict(dim=7), dict(dim=0), dict(dim=8, theta=0.0), dict(dim=8, factor=-1.0),
                                dict(dim=8, method="yarn"), dict(dim=2, method="dynamic", original_len=8),
                                dict(dim=8, method="llama3", original_len=8, low_turns=4.0, high_turns=1.0),
                                dict(dim=8, method="other")])
def test_frequencies_refuse(kw):
    with pytest.raises(ValueError):
        torch_fl.ops.rope_frequencies(**kw)


# ----------------------------------------------------------------------- spans
def dense(spans, k):
    key = torch.arange(k)
    return (key >= spans[..., :1]) & (key < spans[..., 1:])


def test_spans_of_a_decode_step():
    """Two new tokens after caches of different lengths, a window, padding."""
    pos = torch.tensor([[3, 4], [8, 9]])
    s = torch_fl.ops.attention_spans(2, 12, window=4, positions=pos, lengths=torch.tensor([5, 10]))
    assert s.dtype == torch.int32 and s.tolist() == [[[0, 4], [1, 5]], [[5, 9], [6, 10]]]
    s = torch_fl.ops.attention_spans(2, 12)
    assert s.tolist() == [[[0, 11], [0, 12]]]


def test_spans_of_documents_and_padding():
    ids = torch.tensor([[4, 4, 4, 9, 9, 0], [1, 1, 2, 2, 2, 2]])
    s = torch_fl.ops.attention_spans(6, 6, documents=ids, lengths=torch.tensor([5, 6]))
    same = ids[:, :, None] == ids[:, None, :]
    want = same & torch.ones(6, 6).tril().bool()
    want[0, 5] = False
    assert torch.equal(dense(s, 6), want)
    # a query outside the keys sees nothing
    s = torch_fl.ops.attention_spans(3, 6, documents=ids, positions=torch.tensor([-1, 2, 6]))
    assert (s[:, [0, 2], 0] >= s[:, [0, 2], 1]).all() and s[0, 1].tolist() == [0, 3]
    assert torch_fl.ops.attention_spans(2, 0).tolist() == [[[-2, -2], [-1, -1]]] or \
        (torch_fl.ops.attention_spans(2, 0)[..., 0] >= torch_fl.ops.attention_spans(2, 0)[..., 1]).all()


@pytest.mark.parametrize("kw", [dict(window=0), dict(documents=torch.zeros(5, dtype=torch.long)),
                                dict(positions=torch.zeros(3, dtype=torch.long))])
def test_spans_refuse(kw):
    with pytest.raises(ValueError):
        torch_fl.ops.attention_spans(4, 4, **kw)
    with pytest.raises(TypeError):
        torch_fl.ops.attention_spans(4, 4, prefix=torch.ones(1))


# ------------------------------------------------------------------- refusals
def rotary(q=4096, qo=1 << 20, Hq=2, qs=(64, 8, 16), qos=(64, 8, 16), k=None, pos=512, pd=I32, freq=256, rot=8, B=1, S=4, D=8,
           dtype=BF16, scale=1.0):
    _abi.call("fl_b200_rotary", q, qo, Hq, *qs, *qos, k, k, 0, 0, 0, 0, 0, 0, 0, pos, 0, 1, pd, freq, rot, scale, 0, 0,
              B, S, D, dtype, None)


def sandwich(x=1 << 12, r=1 << 13, y=1 << 14, h=1 << 15, rows=4, cols=8, ld=8, eps=1e-6, gate=None, per=0, dtype=BF16):
    _abi.call("fl_b200_sandwich_norm", x, ld, r, ld, 256, 512, gate, per, y, h, rows, cols, eps, 1.0, 0.0, dtype, None)


def span(x=1 << 12, out=1 << 16, spans=256, rows=8, cols=16, heads=2, q=2, cap=0.0, scale=1.0, ld=16, dtype=BF16,
         od=BF16):
    _abi.call("fl_b200_span_softmax", x, ld, spans, 4, 2, None, 0, 0, None, out, 16, rows, cols, heads, q, scale, cap,
              dtype, od, None)


def clip(p=(4096,), q=(8192,), n=(10,), dtypes=(F32,), bound=1.0, kind=0, norm=64):
    c = len(p)
    _abi.call("fl_b200_clip_grads", (ctypes.c_void_p * c)(*p), (ctypes.c_void_p * c)(*q), _abi.i64_array(n),
              (ctypes.c_int * c)(*dtypes), c, bound, kind, norm, None, 0, None)


@pytest.mark.parametrize("call,status", [
    (lambda: rotary(rot=7), 1), (lambda: rotary(rot=10), 1), (lambda: rotary(rot=0), 1), (lambda: rotary(q=None), 1),
    (lambda: rotary(freq=None), 1), (lambda: rotary(pos=None), 1), (lambda: rotary(B=-1), 1),
    (lambda: rotary(qo=4096 + 16), 1),                        # over another part of q
    (lambda: rotary(qo=4096, qos=(64, 16, 8)), 1),            # in place with other strides
    (lambda: rotary(qos=(0, 0, 0)), 1), (lambda: rotary(qs=(64, -8, 16)), 1),
    (lambda: rotary(dtype=I32), 2), (lambda: rotary(pd=F32), 2),
    (lambda: rotary(D=1 << 13, rot=1 << 12), 7), (lambda: rotary(B=1 << 20, S=1 << 20), 7),
    (lambda: sandwich(rows=-1), 1), (lambda: sandwich(x=None), 1), (lambda: sandwich(ld=4), 1),
    (lambda: sandwich(eps=-1.0), 1), (lambda: sandwich(eps=math.nan), 1), (lambda: sandwich(gate=4, per=0), 1),
    (lambda: sandwich(y=1 << 12), 1), (lambda: sandwich(h=(1 << 13) + 16), 1), (lambda: sandwich(h=(1 << 14) + 2), 1),
    (lambda: sandwich(gate=(1 << 15) + 8, per=1), 1), (lambda: sandwich(dtype=I32), 2),
    (lambda: sandwich(rows=1 << 32), 7),
    (lambda: span(rows=7), 1), (lambda: span(heads=0), 1), (lambda: span(q=0), 1), (lambda: span(spans=None), 1),
    (lambda: span(cap=-1.0), 1), (lambda: span(cap=math.nan), 1), (lambda: span(scale=math.nan), 1),
    (lambda: span(out=(1 << 12) + 8), 1), (lambda: span(ld=8), 1), (lambda: span(od=_abi.F16), 2),
    (lambda: span(dtype=I32), 2), (lambda: span(rows=1 << 32, heads=1 << 31), 7),
    (lambda: clip(bound=-1.0), 1), (lambda: clip(bound=math.nan), 1), (lambda: clip(kind=2), 1), (lambda: clip(norm=None), 1),
    (lambda: clip(p=(None,)), 1), (lambda: clip(n=(-1,)), 1), (lambda: clip(q=(4096 + 8,)), 1),
    (lambda: clip(p=(4098,)), 4 - 1), (lambda: clip(dtypes=(I32,)), 2),
])
def test_refused_on_the_host(call, status):
    with pytest.raises(_abi.FlB200Error) as ei:
        call()
    assert ei.value.status == status


def test_empty_calls_touch_nothing():
    rotary(q=None, qo=None, Hq=0)
    rotary(B=0)
    sandwich(x=None, rows=0)
    span(x=None, rows=0)
    span(x=None, cols=0)


@pytest.mark.parametrize("p,q,n", [((4096, 4096), (4096, 4096), (10, 10)), ((4096, 8192), (8192, 4096), (10, 10)),
                                   ((4096, 4096 + 16), (1 << 14, 1 << 15), (10, 10)),
                                   ((4096, 8192), (1 << 14, (1 << 14) + 36), (10, 10))])
def test_outputs_that_meet_are_refused(p, q, n):
    """The same tensor twice in place, two that swap places, outputs over each
    other; two tensors that meet are refused by the workspace only."""
    with pytest.raises(_abi.FlB200Error) as ei:
        clip(p=p, q=q, n=n, dtypes=(F32, F32))
    meets = p[0] == q[0] or p[0] == q[1] or q[1] - q[0] < 40
    assert ei.value.status == (1 if meets else 6) or (not meets and ei.value.status in (5, 6))
