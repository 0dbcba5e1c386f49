"""Tensor-level entry points of the B200 kernels (libfl_b200.so through ctypes).

Each function validates its tensors, allocates the outputs with
``torch.empty_like``-style calls on the input's device, and launches on the
current CUDA stream of that device.  Tensors may live on ``cuda`` or on the
``flagos`` PrivateUse1 device (both are plain device memory of the same GPU).
There is no CPU path: a CPU tensor is an error.

The fused-op semantics follow the HF formulas the reference runs op by op:
``rms_norm`` (transformers models/qwen3/modeling_qwen3.py:59-64),
``rope_qk`` (modeling_qwen3.py:138-169), ``swiglu`` (modeling_qwen3.py:81-82).
"""

from __future__ import annotations

import ctypes

import torch

from . import _abi

_DT = {
    torch.float32: _abi.F32,
    torch.bfloat16: _abi.BF16,
    torch.float16: _abi.F16,
    torch.int32: _abi.I32,
    torch.int64: _abi.I64,
}
_ROUND = {"fused": _abi.ROUND_FUSED, "chain": _abi.ROUND_CHAIN}


def dtype_code(t: torch.Tensor) -> int:
    try:
        return _DT[t.dtype]
    except KeyError:
        raise TypeError(f"b200 kernels do not support dtype {t.dtype}") from None


def _device_index(t: torch.Tensor) -> int:
    if t.device.type == "cpu":
        raise RuntimeError("b200 kernels need device tensors, got a CPU tensor")
    return t.device.index if t.device.index is not None else torch.cuda.current_device()


def _stream(t: torch.Tensor) -> int:
    return torch.cuda.current_stream(_device_index(t)).cuda_stream


class _on_device:
    """Make the tensor's GPU current for the launch (kernels launch there)."""

    def __init__(self, t: torch.Tensor):
        self.idx = _device_index(t)
        self.prev = None

    def __enter__(self):
        self.prev = torch.cuda.current_device()
        if self.prev != self.idx:
            torch.cuda.set_device(self.idx)

    def __exit__(self, *exc):
        if self.prev is not None and self.prev != self.idx:
            torch.cuda.set_device(self.prev)
        return False


def _rows_view(x: torch.Tensor) -> tuple[int, int, int]:
    """(rows, cols, leading stride) of x viewed as [rows, cols] over its last
    dim; requires a unit last-dim stride and rows evenly spaced."""
    if x.dim() == 0:
        return 1, 1, 1
    cols = x.shape[-1]
    rows = 1
    for s in x.shape[:-1]:
        rows *= s
    if x.stride(-1) != 1 and cols > 1:
        raise ValueError("last dim must be contiguous")
    if x.dim() == 1 or rows <= 1:
        return rows, cols, max(cols, 1)
    ld = x.stride(-2)
    # all leading dims must collapse onto one stride
    expect = ld
    for d in range(x.dim() - 2, -1, -1):
        if x.shape[d] != 1 and x.stride(d) != expect:
            raise ValueError("leading dims do not collapse to one row stride")
        expect *= x.shape[d]
    return rows, cols, ld


def _rows_or_contig(x: torch.Tensor) -> tuple[torch.Tensor, int, int, int]:
    try:
        r, c, ld = _rows_view(x)
        return x, r, c, ld
    except ValueError:
        x = x.contiguous()
        r, c, ld = _rows_view(x)
        return x, r, c, ld


# --------------------------------------------------------------------- RMSNorm
def rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float, rounding: str = "fused",
             out: torch.Tensor | None = None) -> torch.Tensor:
    x, rows, cols, ld = _rows_or_contig(x)
    if weight.dtype != x.dtype or weight.numel() != cols or not weight.is_contiguous():
        raise ValueError("weight must be a contiguous [cols] tensor of x's dtype")
    if out is None:
        out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    _, _, ldo = _rows_view(out)
    with _on_device(x):
        _abi.call("fl_b200_rms_norm_fwd", x.data_ptr(), ld, weight.data_ptr(), out.data_ptr(),
                  ldo, rows, cols, float(eps), dtype_code(x), _ROUND[rounding], _stream(x))
    return out


def add_rms_norm(x: torch.Tensor, y: torch.Tensor, weight: torch.Tensor, eps: float,
                 rounding: str = "fused", h_out: torch.Tensor | None = None,
                 out: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """h = x + y; returns (rmsnorm(h) * weight, h).  Dense tensors only."""
    if x.shape != y.shape or x.dtype != y.dtype:
        raise ValueError("x and y must match")
    x = x.contiguous()
    y = y.contiguous()
    cols = x.shape[-1]
    rows = x.numel() // cols
    h = torch.empty_like(x) if h_out is None else h_out
    o = torch.empty_like(x) if out is None else out
    with _on_device(x):
        _abi.call("fl_b200_add_rms_norm_fwd", x.data_ptr(), y.data_ptr(), h.data_ptr(),
                  weight.data_ptr(), o.data_ptr(), rows, cols, float(eps), dtype_code(x),
                  _ROUND[rounding], _stream(x))
    return o, h


# ------------------------------------------------------------------------ RoPE
def _bhsd(t: torch.Tensor, layout: str) -> tuple[int, int, int, int, tuple[int, int, int]]:
    """Sizes (B, H, S, D) and strides over (b, h, s) for a q/k tensor."""
    if t.stride(-1) != 1:
        raise ValueError("head dim must be contiguous")
    if layout == "bhsd":
        B, H, S, D = t.shape
        return B, H, S, D, (t.stride(0), t.stride(1), t.stride(2))
    if layout == "bshd":
        B, S, H, D = t.shape
        return B, H, S, D, (t.stride(0), t.stride(2), t.stride(1))
    raise ValueError(layout)


def _cos_strides(cos: torch.Tensor, B: int, S: int, D: int) -> tuple[int, int]:
    """Strides (b, s) of a cos/sin table given as [S, D], [B, S, D] or
    [B, 1, S, D] (HF unsqueezes dim 1)."""
    if cos.stride(-1) != 1:
        raise ValueError("cos/sin last dim must be contiguous")
    if cos.dim() == 4:
        cos = cos.squeeze(1)
    if cos.dim() == 2:
        if tuple(cos.shape) != (S, D):
            raise ValueError("cos/sin shape mismatch")
        return 0, cos.stride(0)
    if cos.dim() == 3:
        if cos.shape[1] != S or cos.shape[2] != D or cos.shape[0] not in (1, B):
            raise ValueError("cos/sin shape mismatch")
        return (cos.stride(0) if cos.shape[0] == B and B > 1 else 0), cos.stride(1)
    raise ValueError("cos/sin must be 2-D, 3-D or 4-D")


def rope_qk(q: torch.Tensor, k: torch.Tensor | None, cos: torch.Tensor, sin: torch.Tensor,
            layout: str = "bhsd", rounding: str = "fused", inplace: bool = False,
            q_weight: torch.Tensor | None = None, k_weight: torch.Tensor | None = None,
            eps: float = 1e-6, q_out: torch.Tensor | None = None,
            k_out: torch.Tensor | None = None):
    """q_embed, k_embed = apply_rotary_pos_emb(q, k, cos, sin); with q_weight /
    k_weight given, Qwen3's per-head RMSNorm is applied first (fused).
    Outputs go to q_out / k_out when given (same shape and layout as q / k)."""
    B, Hq, S, D, sq = _bhsd(q, layout)
    qo = q if inplace else (q_out if q_out is not None else torch.empty_like(q))
    _, _, _, _, soq = _bhsd(qo, layout)
    if k is not None:
        Bk, Hk, Sk, Dk, sk = _bhsd(k, layout)
        if (Bk, Sk, Dk) != (B, S, D) or k.dtype != q.dtype:
            raise ValueError("q and k disagree")
        ko = k if inplace else (k_out if k_out is not None else torch.empty_like(k))
        _, _, _, _, sok = _bhsd(ko, layout)
        kp, kop = k.data_ptr(), ko.data_ptr()
    else:
        Hk, sk, sok, ko, kp, kop = 0, (0, 0, 0), (0, 0, 0), None, None, None
    if cos.dtype != q.dtype or sin.dtype != q.dtype:
        raise ValueError("cos/sin dtype must match q")
    scb, scs = _cos_strides(cos, B, S, D)
    if _cos_strides(sin, B, S, D) != (scb, scs):
        raise ValueError("cos and sin must share a layout")
    with _on_device(q):
        if q_weight is None:
            _abi.call("fl_b200_rope_qk", q.data_ptr(), qo.data_ptr(), Hq, *sq, *soq,
                      kp, kop, Hk, *sk, *sok, cos.data_ptr(), sin.data_ptr(), scb, scs,
                      B, S, D, dtype_code(q), _ROUND[rounding], _stream(q))
        else:
            wk = k_weight.data_ptr() if (k is not None and k_weight is not None) else None
            _abi.call("fl_b200_rms_norm_rope", q.data_ptr(), qo.data_ptr(), Hq, *sq, *soq,
                      q_weight.data_ptr(), kp, kop, Hk, *sk, *sok, wk, cos.data_ptr(),
                      sin.data_ptr(), scb, scs, B, S, D, float(eps), dtype_code(q),
                      _ROUND[rounding], _stream(q))
    return qo, ko


# ---------------------------------------------------------------------- SwiGLU
def swiglu(gate: torch.Tensor, up: torch.Tensor, rounding: str = "fused",
           out: torch.Tensor | None = None) -> torch.Tensor:
    if gate.shape != up.shape or gate.dtype != up.dtype:
        raise ValueError("gate and up must match")
    gate, rows, cols, ldg = _rows_or_contig(gate)
    up, _, _, ldu = _rows_or_contig(up)
    if out is None:
        out = torch.empty(gate.shape, dtype=gate.dtype, device=gate.device)
    _, _, ldo = _rows_view(out)
    with _on_device(gate):
        _abi.call("fl_b200_swiglu", gate.data_ptr(), ldg, up.data_ptr(), ldu, out.data_ptr(),
                  ldo, rows, cols, dtype_code(gate), _ROUND[rounding], _stream(gate))
    return out


def swiglu_residual(gate, up, x, y, rounding: str = "fused", act_out=None, h_out=None):
    """(silu(gate) * up, x + y) in one launch.  Dense, 16-byte aligned tensors."""
    rows = gate.shape[0]
    act = torch.empty_like(gate) if act_out is None else act_out
    h = torch.empty_like(x) if h_out is None else h_out
    with _on_device(gate):
        _abi.call("fl_b200_swiglu_residual", gate.data_ptr(), up.data_ptr(), act.data_ptr(),
                  gate.numel() // rows, x.data_ptr(), y.data_ptr(), h.data_ptr(),
                  x.numel() // rows, rows, dtype_code(gate), _ROUND[rounding], _stream(gate))
    return act, h


# ---------------------------------------------------------------- elementwise
def _broadcast(a: torch.Tensor, b: torch.Tensor):
    shape = torch.broadcast_shapes(a.shape, b.shape)
    ea, eb = a.expand(shape), b.expand(shape)
    if len(shape) > 8:
        raise ValueError("at most 8 dims")
    return shape, ea.stride(), eb.stride()


def _binary_out(out, shape, a):
    if out is None:
        return torch.empty(shape, dtype=a.dtype, device=a.device)
    if tuple(out.shape) != tuple(shape) or out.dtype != a.dtype or not out.is_contiguous():
        raise ValueError("out must be a contiguous tensor of the broadcast shape and dtype")
    return out


def add(a: torch.Tensor, b: torch.Tensor, alpha: float = 1.0,
        out: torch.Tensor | None = None) -> torch.Tensor:
    if a.dtype != b.dtype:
        raise TypeError("add: operands must share a dtype (promote first)")
    shape, sa, sb = _broadcast(a, b)
    out = _binary_out(out, shape, a)
    with _on_device(a):
        _abi.call("fl_b200_add", a.data_ptr(), _abi.i64_array(sa), b.data_ptr(),
                  _abi.i64_array(sb), out.data_ptr(), _abi.i64_array(shape), len(shape),
                  float(alpha), dtype_code(a), _stream(a))
    return out


def mul(a: torch.Tensor, b: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    if a.dtype != b.dtype:
        raise TypeError("mul: operands must share a dtype (promote first)")
    shape, sa, sb = _broadcast(a, b)
    out = _binary_out(out, shape, a)
    with _on_device(a):
        _abi.call("fl_b200_mul", a.data_ptr(), _abi.i64_array(sa), b.data_ptr(),
                  _abi.i64_array(sb), out.data_ptr(), _abi.i64_array(shape), len(shape),
                  dtype_code(a), _stream(a))
    return out


def binary_scalar(a: torch.Tensor, s: float, op: str, alpha: float = 1.0) -> torch.Tensor:
    a = a.contiguous()
    out = torch.empty_like(a)
    with _on_device(a):
        _abi.call("fl_b200_binary_scalar", a.data_ptr(), float(s), out.data_ptr(), a.numel(),
                  {"add": 0, "mul": 1}[op], float(alpha), dtype_code(a), _stream(a))
    return out


def cast(x: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    x = x.contiguous()
    out = torch.empty(x.shape, dtype=dtype, device=x.device)
    with _on_device(x):
        _abi.call("fl_b200_cast", x.data_ptr(), dtype_code(x), out.data_ptr(),
                  _DT[dtype], x.numel(), _stream(x))
    return out


# --------------------------------------------------------------------- softmax
def softmax(x: torch.Tensor, dim: int = -1, out_dtype: torch.dtype | None = None,
            causal: bool = False, causal_offset: int = 0) -> torch.Tensor:
    """softmax over `dim` in fp32; out_dtype None = x.dtype (or float32 for
    half_to_float).  causal applies the mask of query row i (the second-last
    dim) over keys j <= i + causal_offset in the kernel."""
    out_dtype = out_dtype or x.dtype
    dim = dim % max(x.dim(), 1)
    if x.dim() == 0:
        return torch.ones((), dtype=out_dtype, device=x.device)
    if dim != x.dim() - 1:
        if causal:
            raise ValueError("causal softmax is over the last dim")
        xc = x.contiguous()
        outer = 1
        for s in x.shape[:dim]:
            outer *= s
        inner = 1
        for s in x.shape[dim + 1:]:
            inner *= s
        out = torch.empty(x.shape, dtype=out_dtype, device=x.device)
        with _on_device(x):
            _abi.call("fl_b200_softmax_middim", xc.data_ptr(), out.data_ptr(), outer,
                      x.shape[dim], inner, dtype_code(x), _DT[out_dtype], _stream(x))
        return out
    x, rows, cols, ld = _rows_or_contig(x)
    out = torch.empty(x.shape, dtype=out_dtype, device=x.device)
    q_len = x.shape[-2] if x.dim() >= 2 else 1
    with _on_device(x):
        _abi.call("fl_b200_softmax_lastdim", x.data_ptr(), ld, out.data_ptr(), cols, rows,
                  cols, dtype_code(x), _DT[out_dtype], int(causal), q_len,
                  int(causal_offset), _stream(x))
    return out


def _as_bhqk(x: torch.Tensor) -> torch.Tensor:
    if not 2 <= x.dim() <= 4:
        raise ValueError("x must be [Q, K], [H, Q, K] or [B, H, Q, K]")
    while x.dim() < 4:
        x = x.unsqueeze(0)
    return x


def masked_softmax(x: torch.Tensor, mask: torch.Tensor | None = None, scale: float = 1.0,
                   out_dtype: torch.dtype | None = None, rounding: str = "fused") -> torch.Tensor:
    """softmax(x * scale + mask) over the last dim, HF eager attention's tail
    (modeling_qwen3.py eager_attention_forward: scale, mask add,
    softmax(dtype=float32), cast back) in one launch.  x is [B, H, Q, K] (or
    fewer leading dims); mask has x's dtype and broadcasts to x; out_dtype
    None = x.dtype (the cast back fused), or float32."""
    out_dtype = out_dtype or x.dtype
    x4 = _as_bhqk(x)
    B, H, Q, K = x4.shape
    x4, rows, cols, ld = _rows_or_contig(x4)
    mp, sb, sh, sq = 0, 0, 0, 0
    if mask is not None:
        if mask.dtype != x.dtype:
            raise TypeError("mask must have x's dtype")
        m = mask.expand(x4.shape)
        if K > 1 and m.stride(3) != 1:
            m = m.contiguous()
        mask = m
        mp, sb, sh, sq = m.data_ptr(), m.stride(0), m.stride(1), m.stride(2)
    out = torch.empty(x4.shape, dtype=out_dtype, device=x.device)
    if out.numel():
        with _on_device(x):
            _abi.call("fl_b200_softmax_masked", x4.data_ptr(), ld, mp, sb, sh, sq,
                      out.data_ptr(), cols, rows, cols, H, Q, float(scale), dtype_code(x),
                      _DT[out_dtype], _ROUND[rounding], _stream(x))
    return out.view(x.shape)


# --------------------------------------------- the other HF formula ops
_UNARY = {"silu": _abi.UNARY_SILU, "rsqrt": _abi.UNARY_RSQRT, "neg": _abi.UNARY_NEG,
          "cos": _abi.UNARY_COS, "sin": _abi.UNARY_SIN}


def _outer(x: torch.Tensor, split: int):
    """(sizes, strides) of x's dims before `split` when its dims from `split`
    on are contiguous, else None."""
    expect = 1
    for d in range(x.dim() - 1, split - 1, -1):
        if x.size(d) != 1 and x.stride(d) != expect:
            return None
        expect *= x.size(d)
    return list(x.shape[:split]), list(x.stride()[:split])


def unary(x: torch.Tensor, op: str, exponent: float = 0.0) -> torch.Tensor:
    """silu / rsqrt / neg / cos / sin of x, or pow(x, exponent) (op "pow";
    the exponent rounded to x's dtype first, 2 and 3 as products, as the
    reference's cuda route computes them) through fl_b200_unary.  x's rows of
    the last dim may be strided (any outer dims); the result is dense."""
    if op == "pow":
        e = float(torch.tensor(exponent, dtype=x.dtype)) if x.is_floating_point() else exponent
        code = _abi.UNARY_SQUARE if e == 2.0 else (_abi.UNARY_CUBE if e == 3.0 else _abi.UNARY_POW)
    else:
        e, code = 0.0, _UNARY[op]
    view = _outer(x, x.dim() - 1) if x.dim() else ([], [])
    if view is None:
        x = x.contiguous()
        view = _outer(x, x.dim() - 1)
    sizes, strides = view
    out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    if out.numel():
        with _on_device(x):
            _abi.call("fl_b200_unary", x.data_ptr(), _abi.i64_array(sizes),
                      _abi.i64_array(strides), len(sizes), x.shape[-1] if x.dim() else 1,
                      out.data_ptr(), code, float(e), dtype_code(x), _stream(x))
    return out


def cat(tensors, dim: int = 0) -> torch.Tensor:
    """torch.cat(tensors, dim) for tensors of one dtype through fl_b200_cat
    (row blocks; each input's dims from `dim` on contiguous, any outer
    strides)."""
    t0 = tensors[0]
    d = dim % t0.dim()
    shape = list(t0.shape)
    shape[d] = sum(t.shape[d] for t in tensors)
    out = torch.empty(shape, dtype=t0.dtype, device=t0.device)
    srcs, strides, widths, keep = [], [], [], []
    for t in tensors:
        v = _outer(t, d)
        if v is None:
            t = t.contiguous()
            keep.append(t)
            v = _outer(t, d)
        srcs.append(t.data_ptr())
        strides += v[1]
        widths.append(int(torch.tensor(t.shape[d:]).prod()) if d < t.dim() else 1)
    if out.numel():
        import ctypes as C
        arr = (C.c_void_p * len(srcs))(*srcs)
        with _on_device(t0):
            _abi.call("fl_b200_cat", arr, _abi.i64_array(strides), _abi.i64_array(widths),
                      len(srcs), _abi.i64_array(shape[:d]), d, out.data_ptr(),
                      t0.element_size(), _stream(t0))
    return out


# ------------------------------------------------------------------ reductions
def _workspace(rows: int, cols: int, device) -> torch.Tensor | None:
    n = _abi.lib().fl_b200_reduce_workspace_size(rows, cols)
    if n == 0:
        return None
    return torch.empty(n, dtype=torch.uint8, device=device)


def _reduce_lastdim(name: str, x: torch.Tensor, out_dtype: torch.dtype, keepdim: bool,
                    with_out_dtype: bool = True) -> torch.Tensor:
    x, rows, cols, ld = _rows_or_contig(x)
    shape = list(x.shape[:-1]) + ([1] if keepdim else [])
    out = torch.empty(shape, dtype=out_dtype, device=x.device)
    ws = _workspace(rows, cols, x.device)
    wsp, wsn = (ws.data_ptr(), ws.numel()) if ws is not None else (None, 0)
    with _on_device(x):
        if with_out_dtype:
            _abi.call(name, x.data_ptr(), ld, rows, cols, out.data_ptr(), dtype_code(x),
                      _DT[out_dtype], wsp, wsn, _stream(x))
        else:
            _abi.call(name, x.data_ptr(), ld, rows, cols, out.data_ptr(), dtype_code(x),
                      wsp, wsn, _stream(x))
    return out


def _reduce_all(name: str, x: torch.Tensor, out_dtype: torch.dtype,
                with_out_dtype: bool = True) -> torch.Tensor:
    x = x.contiguous()
    out = torch.empty((), dtype=out_dtype, device=x.device)
    ws = _workspace(1, x.numel(), x.device)
    wsp, wsn = (ws.data_ptr(), ws.numel()) if ws is not None else (None, 0)
    with _on_device(x):
        if with_out_dtype:
            _abi.call(name, x.data_ptr(), x.numel(), out.data_ptr(), dtype_code(x),
                      _DT[out_dtype], wsp, wsn, _stream(x))
        else:
            _abi.call(name, x.data_ptr(), x.numel(), out.data_ptr(), dtype_code(x), wsp, wsn,
                      _stream(x))
    return out


def _sum_dtype(x: torch.Tensor, dtype) -> torch.dtype:
    if dtype is not None:
        return dtype
    return torch.int64 if x.dtype in (torch.int32, torch.int64) else x.dtype


def sum_lastdim(x, keepdim=False, dtype=None):
    return _reduce_lastdim("fl_b200_reduce_sum_lastdim", x, _sum_dtype(x, dtype), keepdim)


def mean_lastdim(x, keepdim=False, dtype=None):
    return _reduce_lastdim("fl_b200_reduce_mean_lastdim", x, dtype or x.dtype, keepdim)


def amax_lastdim(x, keepdim=False):
    return _reduce_lastdim("fl_b200_reduce_amax_lastdim", x, x.dtype, keepdim,
                           with_out_dtype=False)


def sum_all(x, dtype=None):
    return _reduce_all("fl_b200_reduce_sum_all", x, _sum_dtype(x, dtype))


def mean_all(x, dtype=None):
    return _reduce_all("fl_b200_reduce_mean_all", x, dtype or x.dtype)


def amax_all(x):
    return _reduce_all("fl_b200_reduce_amax_all", x, x.dtype, with_out_dtype=False)


def reduce_middim(x: torch.Tensor, dim: int, op: str, keepdim=False, dtype=None):
    x = x.contiguous()
    dim = dim % x.dim()
    outer = 1
    for s in x.shape[:dim]:
        outer *= s
    inner = 1
    for s in x.shape[dim + 1:]:
        inner *= s
    shape = list(x.shape)
    if keepdim:
        shape[dim] = 1
    else:
        shape.pop(dim)
    out_dtype = dtype or x.dtype
    out = torch.empty(shape, dtype=out_dtype, device=x.device)
    with _on_device(x):
        _abi.call("fl_b200_reduce_middim", x.data_ptr(), outer, x.shape[dim], inner,
                  out.data_ptr(), {"sum": 0, "mean": 1, "amax": 2}[op], dtype_code(x),
                  _DT[out_dtype], _stream(x))
    return out


def argmax_lastdim(x: torch.Tensor, keepdim: bool = False) -> torch.Tensor:
    x, rows, cols, ld = _rows_or_contig(x)
    shape = list(x.shape[:-1]) + ([1] if keepdim else [])
    out = torch.empty(shape, dtype=torch.int64, device=x.device)
    ws = _workspace(rows, cols, x.device)
    wsp, wsn = (ws.data_ptr(), ws.numel()) if ws is not None else (None, 0)
    with _on_device(x):
        _abi.call("fl_b200_argmax_lastdim", x.data_ptr(), ld, rows, cols, out.data_ptr(),
                  dtype_code(x), wsp, wsn, _stream(x))
    return out


def sum_i32_i64(x: torch.Tensor, full: bool) -> torch.Tensor:
    if x.dtype != torch.int32:
        raise TypeError("sum_i32_i64 takes int32")
    x, rows, cols, ld = _rows_or_contig(x)
    if full:
        x = x.contiguous()
        rows, cols, ld = 1, x.numel(), x.numel()
    out = torch.empty(() if full else x.shape[:-1], dtype=torch.int64, device=x.device)
    ws = _workspace(rows, cols, x.device)
    wsp, wsn = (ws.data_ptr(), ws.numel()) if ws is not None else (None, 0)
    with _on_device(x):
        _abi.call("fl_b200_sum_i32_i64", x.data_ptr(), ld, rows, cols, out.data_ptr(),
                  int(full), wsp, wsn, _stream(x))
    return out


# ---------------------------------- a training step around the matrix products
def _heads_like(t: torch.Tensor) -> torch.Tensor:
    """A result laid out as t where that keeps its heads whole (of overlapping
    views another dim would be innermost)."""
    o = torch.empty_like(t)
    return o if o.stride(-1) == 1 else torch.empty(t.shape, dtype=t.dtype, device=t.device)


def rotary(q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor, inv_freq: torch.Tensor,
           scale: float = 1.0, interleaved: bool = False, inverse: bool = False, layout: str = "bhsd",
           inplace: bool = False):
    """q and k turned by positions * inv_freq (no table); inplace touches the
    turned part of each head only."""
    B, Hq, S, D, sq = _bhsd(q, layout)
    ops = [t for t in (q, k, positions, inv_freq) if t is not None]
    _one_device(*ops)
    qo = q if inplace else _heads_like(q)
    soq = _bhsd(qo, layout)[4]
    Hk, sk, sok, ko = 0, (0, 0, 0), (0, 0, 0), None
    if k is not None:
        Bk, Hk, Sk, Dk, sk = _bhsd(k, layout)
        if (Bk, Sk, Dk) != (B, S, D) or k.dtype != q.dtype:
            raise ValueError("q and k disagree")
        ko = k if inplace else _heads_like(k)
        sok = _bhsd(ko, layout)[4]
    if positions.dtype not in (torch.int32, torch.int64) or positions.dim() not in (1, 2) \
            or positions.shape[-1] != S or (positions.dim() == 2 and positions.shape[0] not in (1, B)):
        raise ValueError("positions must be int32 or int64 [seq] or [batch, seq]")
    if inv_freq.dtype != torch.float32 or inv_freq.dim() != 1 or not inv_freq.is_contiguous():
        raise ValueError("inv_freq must be a contiguous float32 [n] tensor")
    spb = positions.stride(0) if positions.dim() == 2 and positions.shape[0] > 1 else 0
    with _on_device(q):
        _abi.call("fl_b200_rotary", q.data_ptr(), qo.data_ptr(), Hq, *sq, *soq,
                  None if k is None else k.data_ptr(), None if k is None else ko.data_ptr(), Hk, *sk, *sok,
                  positions.data_ptr(), spb, positions.stride(-1), _DT[positions.dtype],
                  inv_freq.data_ptr(), 2 * inv_freq.numel(), float(scale), int(interleaved), int(inverse),
                  B, S, D, dtype_code(q), _stream(q))
    return qo, ko


def _gate_rows(x: torch.Tensor, gate: torch.Tensor | None) -> int:
    """How many of x's rows share a row of the gate."""
    if gate is None or gate.dim() == 1:
        return max(1, x.shape[:-1].numel())
    d, per = x.dim() - 2, 1
    while gate.dim() == x.dim() and d >= 0 and gate.shape[d] == 1:
        per *= x.shape[d]
        d -= 1
    if gate.dim() != x.dim() or gate.shape[:d + 1] != x.shape[:d + 1] or gate.shape[-1] != x.shape[-1]:
        raise ValueError("gate must be [hidden], or x's shape with the last dims before hidden 1")
    return max(1, per)


def _sandwich_weights(x, post, pre, gate):
    for w in (post, pre):
        if w.dtype != x.dtype or w.shape != x.shape[-1:] or not w.is_contiguous():
            raise ValueError("weights must be contiguous [hidden] tensors of x's dtype")
    if gate is not None and (gate.dtype != x.dtype or gate.shape[-1:] != x.shape[-1:]):
        raise ValueError("gate must have x's dtype and hidden size")


def sandwich_norm(x: torch.Tensor, residual: torch.Tensor, post: torch.Tensor, pre: torch.Tensor, eps: float,
                  gate: torch.Tensor | None = None, scale: float = 1.0,
                  weight_offset: float = 0.0) -> tuple[torch.Tensor, torch.Tensor]:
    """(y, h): h = residual + scale * gate * rms_norm(x) * (offset + post),
    y = rms_norm(h) * (offset + pre)."""
    if x.shape != residual.shape or x.dtype != residual.dtype:
        raise ValueError("x and the residual must match")
    _sandwich_weights(x, post, pre, gate)
    _one_device(x, residual, post, pre, gate)
    per = _gate_rows(x, gate)
    gate = None if gate is None else gate.contiguous()
    shape = x.shape
    x, rows, cols, ldx = _rows_apart(x)
    residual, _, _, ldr = _rows_apart(residual)
    y, h = (torch.empty(shape, dtype=x.dtype, device=x.device) for _ in range(2))
    with _on_device(x):
        _abi.call("fl_b200_sandwich_norm", x.data_ptr(), ldx, residual.data_ptr(), ldr, post.data_ptr(),
                  pre.data_ptr(), None if gate is None else gate.data_ptr(), per, y.data_ptr(), h.data_ptr(),
                  rows, cols, float(eps), float(scale), float(weight_offset), dtype_code(x), _stream(x))
    return y, h


def sandwich_norm_backward(dy, dh, x, h, post, pre, eps: float, gate=None, scale: float = 1.0,
                           weight_offset: float = 0.0):
    """(dx, dresidual, dpost, dpre, dgate) of sandwich_norm; dh None: no
    gradient of h; dgate None without a gate."""
    for t in (dy, dh, h):
        if t is not None and (t.shape != x.shape or t.dtype != x.dtype):
            raise ValueError("dy, dh, x and h must match")
    _sandwich_weights(x, post, pre, gate)
    _one_device(x, dy, dh, h, post, pre, gate)
    per = _gate_rows(x, gate)
    gate = None if gate is None else gate.contiguous()
    shape = x.shape
    x, rows, cols, ldx = _rows_apart(x)
    h, _, _, ldh = _rows_apart(h)
    dy, _, _, ldy = _rows_apart(dy)
    ldd = 0
    if dh is not None:
        dh, _, _, ldd = _rows_apart(dh)
    dx, dres = (torch.empty(shape, dtype=x.dtype, device=x.device) for _ in range(2))
    dpost, dpre = (torch.empty(cols, dtype=x.dtype, device=x.device) for _ in range(2))
    dgate = None if gate is None else torch.empty_like(gate)
    with _on_device(x):
        nws = _abi.lib().fl_b200_sandwich_norm_bwd_workspace_size(rows, cols)
        ws = torch.empty(max(nws, 16), dtype=torch.uint8, device=x.device)
        _abi.call("fl_b200_sandwich_norm_bwd", dy.data_ptr(), ldy, None if dh is None else dh.data_ptr(), ldd,
                  x.data_ptr(), ldx, h.data_ptr(), ldh, post.data_ptr(), pre.data_ptr(),
                  None if gate is None else gate.data_ptr(), per, dx.data_ptr(), dres.data_ptr(),
                  dpost.data_ptr(), dpre.data_ptr(), None if gate is None else dgate.data_ptr(), rows, cols,
                  float(eps), float(scale), float(weight_offset), dtype_code(x), ws.data_ptr(), nws, _stream(x))
    return dx, dres, dpost, dpre, dgate


def _per_query(t: torch.Tensor, B: int, Q: int, tail: int) -> tuple[torch.Tensor, int, int]:
    u = t if tail else t.unsqueeze(-1)
    u = u.unsqueeze(0) if u.dim() == 2 else u
    if t.dtype != torch.int32 or u.dim() != 3 or u.shape[0] not in (1, B) or u.shape[1] != Q \
            or u.shape[2] != max(tail, 1):
        raise ValueError("int32 values for each query expected")
    if tail and u.stride(2) != 1:
        u = u.contiguous()
    return u, 0 if u.shape[0] == 1 else u.stride(0), u.stride(1)


def _cap(cap: float | None) -> float:
    """The cap as the kernels take it: 0 stands for none, so no cap may round to it."""
    if cap is None:
        return 0.0
    if not 0 < ctypes.c_float(cap).value <= 3e38:
        raise ValueError(f"cap must be positive and finite in float32, got {cap}")
    return float(cap)


def span_softmax(x: torch.Tensor, spans: torch.Tensor, scale: float = 1.0, cap: float | None = None,
                 slopes: torch.Tensor | None = None, positions: torch.Tensor | None = None,
                 out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """softmax of scale * x (capped, biased by distance) over each query's span
    of keys; zeros elsewhere."""
    cap = _cap(cap)
    B, H, Q, Kn = _as_bhqk(x).shape
    _one_device(x, spans, slopes, positions)
    spans, sb, sq = _per_query(spans, B, Q, 2)
    pb = pq = 0
    if positions is not None:
        positions, pb, pq = _per_query(positions, B, Q, 0)
    if slopes is not None and (slopes.dtype != torch.float32 or slopes.shape != (H,) or not slopes.is_contiguous()):
        raise ValueError("slopes must be a contiguous float32 [heads] tensor")
    out = torch.empty(x.shape, dtype=out_dtype or x.dtype, device=x.device)
    x, rows, cols, ld = _rows_apart(x)
    with _on_device(x):
        _abi.call("fl_b200_span_softmax", x.data_ptr(), ld, spans.data_ptr(), sb, sq,
                  None if positions is None else positions.data_ptr(), pb, pq,
                  None if slopes is None else slopes.data_ptr(), out.data_ptr(), cols, rows, cols, H, Q,
                  float(scale), cap, dtype_code(x), dtype_code(out), _stream(x))
    return out


def span_softmax_backward(dy: torch.Tensor, y: torch.Tensor, x: torch.Tensor, spans: torch.Tensor,
                          scale: float = 1.0, cap: float | None = None) -> torch.Tensor:
    if dy.shape != y.shape or dy.dtype != y.dtype or y.shape != x.shape:
        raise ValueError("dy, y and x must match")
    cap = _cap(cap)
    B, H, Q, Kn = _as_bhqk(y).shape
    _one_device(x, y, dy, spans)
    spans, sb, sq = _per_query(spans, B, Q, 2)
    dx = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    x, _, _, ldx = _rows_apart(x)
    dy, _, _, ldd = _rows_apart(dy)
    y, rows, cols, ldy = _rows_apart(y)
    with _on_device(y):
        _abi.call("fl_b200_span_softmax_bwd", dy.data_ptr(), ldd, y.data_ptr(), ldy, x.data_ptr(), ldx,
                  spans.data_ptr(), sb, sq, dx.data_ptr(), cols, rows, cols, H, Q, float(scale),
                  cap, dtype_code(y), dtype_code(dx), _stream(y))
    return dx


def _grad_list(tensors):
    n = len(tensors)
    if n == 0:
        raise ValueError("no tensors")
    _one_device(*tensors)
    if any(not t.is_contiguous() for t in tensors):
        raise ValueError("contiguous tensors expected")
    ptrs = (ctypes.c_void_p * n)(*[t.data_ptr() for t in tensors])
    numels = _abi.i64_array([t.numel() for t in tensors])
    dtypes = (ctypes.c_int * n)(*[dtype_code(t) for t in tensors])
    return n, ptrs, numels, dtypes


def grad_norm(tensors, max_kind: bool = False) -> torch.Tensor:
    """The norm of the tensors taken as one vector: sqrt(sum x^2), or max |x|."""
    n, ptrs, numels, dtypes = _grad_list(tensors)
    t = tensors[0]
    norm = torch.empty((), dtype=torch.float32, device=t.device)
    with _on_device(t):
        nws = _abi.lib().fl_b200_grad_norm_workspace_size(n)
        ws = torch.empty(nws, dtype=torch.uint8, device=t.device)
        _abi.call("fl_b200_grad_norm", ptrs, numels, dtypes, n, int(max_kind), norm.data_ptr(), ws.data_ptr(),
                  nws, _stream(t))
    return norm


def clip_grads(tensors, max_norm: float, max_kind: bool = False, out=None):
    """(clipped, norm): the tensors times min(1, max_norm / (norm + 1e-6))."""
    n, ptrs, numels, dtypes = _grad_list(tensors)
    out = [torch.empty_like(t) for t in tensors] if out is None else list(out)
    if len(out) != n or any(o.shape != t.shape or o.dtype != t.dtype for o, t in zip(out, tensors)):
        raise ValueError("each output must have its tensor's shape and dtype")
    _one_device(tensors[0], *out)
    outs = _grad_list(out)[1]
    t = tensors[0]
    norm = torch.empty((), dtype=torch.float32, device=t.device)
    with _on_device(t):
        nws = _abi.lib().fl_b200_grad_norm_workspace_size(n)
        ws = torch.empty(nws, dtype=torch.uint8, device=t.device)
        _abi.call("fl_b200_clip_grads", ptrs, outs, numels, dtypes, n, float(max_norm), int(max_kind),
                  norm.data_ptr(), ws.data_ptr(), nws, _stream(t))
    return out, norm


# ------------------------------------------------------ rows of the vocabulary
def _one_device(*tensors) -> None:
    """The kernels get plain pointers: every operand on the first one's GPU."""
    kept = [t for t in tensors if t is not None]
    if any(_device_index(t) != _device_index(kept[0]) for t in kept):
        raise ValueError("operands must be on one device")


def _rows_apart(x: torch.Tensor) -> tuple[torch.Tensor, int, int, int]:
    """_rows_or_contig, of a copy where rows overlap (an expanded tensor)."""
    x, rows, cols, ld = _rows_or_contig(x)
    if rows > 1 and ld < cols:
        x, rows, cols, ld = _rows_or_contig(x.contiguous())
    return x, rows, cols, ld


def topk_lastdim(x: torch.Tensor, k: int) -> tuple[torch.Tensor, torch.Tensor]:
    """(values, int64 indices) of the k largest over the last dim, descending;
    ties by ascending index, NaN above everything."""
    x, rows, cols, ld = _rows_apart(x)
    shape = list(x.shape[:-1]) + [k]
    values = torch.empty(shape, dtype=x.dtype, device=x.device)
    indices = torch.empty(shape, dtype=torch.int64, device=x.device)
    with _on_device(x):
        _abi.call("fl_b200_topk_lastdim", x.data_ptr(), ld, rows, cols, k, values.data_ptr(),
                  indices.data_ptr(), dtype_code(x), _stream(x))
    return values, indices


def topk_backward(dvalues: torch.Tensor, indices: torch.Tensor, cols: int) -> torch.Tensor:
    """dx [..., cols] of topk_lastdim's values."""
    if dvalues.shape != indices.shape or indices.dtype != torch.int64:
        raise ValueError("dvalues and int64 indices must match")
    _one_device(dvalues, indices)
    dvalues, indices = dvalues.contiguous(), indices.contiguous()
    k = dvalues.shape[-1]
    rows = dvalues.shape[:-1].numel()
    dx = torch.empty(list(dvalues.shape[:-1]) + [cols], dtype=dvalues.dtype, device=dvalues.device)
    with _on_device(dvalues):
        _abi.call("fl_b200_topk_bwd", dvalues.data_ptr(), indices.data_ptr(), dx.data_ptr(), rows,
                  cols, k, dtype_code(dvalues), _stream(dvalues))
    return dx


def _taught(logits, teacher_logits, teacher_ids):
    """Rows views of a student's logits and its teacher's lists, checked."""
    if teacher_ids.dtype not in (torch.int32, torch.int64):
        raise TypeError("teacher_ids must be int32 or int64")
    if teacher_logits.shape != teacher_ids.shape or teacher_ids.shape[:-1] != logits.shape[:-1]:
        raise ValueError("logits [..., vocab] with teacher_logits and teacher_ids [..., k] expected")
    _one_device(logits, teacher_logits, teacher_ids)
    x, rows, cols, ld = _rows_apart(logits)
    t, _, k, ld_t = _rows_or_contig(teacher_logits)
    i, _, _, ld_i = _rows_or_contig(teacher_ids)
    head = (x.data_ptr(), ld)
    lists = (t.data_ptr(), ld_t, dtype_code(t), i.data_ptr(), ld_i, dtype_code(i))
    return (x, t, i), head, lists, logits.shape[:-1].numel(), cols, k


def _row_weight(w, shape):
    """A float32 tensor that broadcasts to the loss as (tensor, pointer, row stride)."""
    if w is None:
        return None, None, 0
    if w.dtype != torch.float32:
        raise TypeError("row weights must be float32")
    w = w.expand(shape).reshape(-1)
    return w, w.data_ptr(), w.stride(0) if w.numel() > 1 else 0


def distill_topk(logits: torch.Tensor, teacher_logits: torch.Tensor, teacher_ids: torch.Tensor,
                 temperature: float = 1.0) -> tuple[torch.Tensor, torch.Tensor]:
    """(loss [...], stats [rows, 2]), both float32: temperature^2 * KL of the
    teacher's list against the student's softmax, and what the backward needs."""
    (x, *keep), head, lists, rows, cols, k = _taught(logits, teacher_logits, teacher_ids)
    loss = torch.empty(logits.shape[:-1], dtype=torch.float32, device=x.device)
    stats = torch.empty((rows, 2), dtype=torch.float32, device=x.device)
    with _on_device(x):
        _abi.call("fl_b200_distill_topk_fwd", *head, *lists, rows, cols, k, float(temperature),
                  loss.data_ptr(), stats.data_ptr(), dtype_code(x), _stream(x))
    return loss, stats


def distill_topk_backward(dloss: torch.Tensor | None, logits: torch.Tensor, stats: torch.Tensor,
                          teacher_logits: torch.Tensor, teacher_ids: torch.Tensor,
                          temperature: float = 1.0, need_logits: bool = True,
                          need_teacher: bool = False):
    """(dlogits, dteacher) from the forward's stats; None for one not needed.
    dloss broadcasts to the loss; None is 1 for every row."""
    (x, *keep), head, lists, rows, cols, k = _taught(logits, teacher_logits, teacher_ids)
    if stats.dtype != torch.float32 or tuple(stats.shape) != (rows, 2) or not stats.is_contiguous():
        raise ValueError("stats must be the forward's [rows, 2] float32 tensor")
    _one_device(x, stats, dloss)
    w, wp, ws = _row_weight(dloss, logits.shape[:-1])
    dx = torch.empty(logits.shape, dtype=x.dtype, device=x.device) if need_logits else None
    dt = torch.empty(teacher_logits.shape, dtype=teacher_logits.dtype,
                     device=x.device) if need_teacher else None
    with _on_device(x):
        _abi.call("fl_b200_distill_topk_bwd", wp, ws, *head, stats.data_ptr(), *lists,
                  dx.data_ptr() if need_logits else None, cols,
                  dt.data_ptr() if need_teacher else None, rows, cols, k, float(temperature),
                  dtype_code(x), _stream(x))
    return dx, dt


def distill_topk_grad(logits: torch.Tensor, teacher_logits: torch.Tensor, teacher_ids: torch.Tensor,
                      temperature: float = 1.0, row_weight: torch.Tensor | None = None,
                      out: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """(loss, dlogits) of sum(row_weight * loss) in one call.  out may hold the
    gradient; its rows share no memory with an operand's."""
    (x, *keep), head, lists, rows, cols, k = _taught(logits, teacher_logits, teacher_ids)
    _one_device(x, row_weight, out)
    w, wp, ws = _row_weight(row_weight, logits.shape[:-1])
    loss = torch.empty(logits.shape[:-1], dtype=torch.float32, device=x.device)
    stats = torch.empty((rows, 2), dtype=torch.float32, device=x.device)
    dx = torch.empty(logits.shape, dtype=x.dtype, device=x.device) if out is None else out
    if dx.shape != logits.shape or dx.dtype != x.dtype:
        raise ValueError("out must have the logits' shape and dtype")
    _, _, ldo = _rows_view(dx)
    with _on_device(x):
        _abi.call("fl_b200_distill_topk_grad", *head, *lists, wp, ws, rows, cols, k,
                  float(temperature), loss.data_ptr(), stats.data_ptr(), dx.data_ptr(), ldo,
                  dtype_code(x), _stream(x))
    return loss, dx


def verify_draft(draft_ids: torch.Tensor, target_probs: torch.Tensor,
                 draft_probs: torch.Tensor | None, uniform: torch.Tensor,
                 draft_lens: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """(tokens [batch, drafts + 1], accepted [batch]) of speculative sampling;
    see ops.verify_draft."""
    B, n = draft_ids.shape
    V = target_probs.shape[-1]
    if draft_ids.dtype != torch.int64 or uniform.dtype != torch.float32:
        raise TypeError("draft_ids must be int64 and uniform float32")
    if tuple(target_probs.shape) != (B, n + 1, V) or tuple(uniform.shape) != (B, n + 1):
        raise ValueError("target_probs [batch, drafts + 1, vocab] and uniform [batch, drafts + 1] expected")
    if draft_probs is not None and (tuple(draft_probs.shape) != (B, n, V)
                                    or draft_probs.dtype != target_probs.dtype):
        raise ValueError("draft_probs must be [batch, drafts, vocab] of target_probs' dtype")
    if draft_lens is not None and (tuple(draft_lens.shape) != (B,) or draft_lens.dtype != torch.int64):
        raise ValueError("draft_lens must be int64 [batch]")
    _one_device(target_probs, draft_ids, draft_probs, uniform, draft_lens)

    def unit(t):
        return t if t is None or t.shape[-1] <= 1 or t.stride(-1) == 1 else t.contiguous()

    ids, p, q, u = unit(draft_ids), unit(target_probs), unit(draft_probs), unit(uniform)
    lens = None if draft_lens is None else draft_lens.contiguous()
    tokens = torch.empty((B, n + 1), dtype=torch.int64, device=p.device)
    accepted = torch.empty((B,), dtype=torch.int64, device=p.device)
    with _on_device(p):
        _abi.call("fl_b200_verify_draft", ids.data_ptr(), ids.stride(0), p.data_ptr(), p.stride(0),
                  p.stride(1), None if q is None else q.data_ptr(), 0 if q is None else q.stride(0),
                  0 if q is None else q.stride(1), u.data_ptr(), u.stride(0),
                  None if lens is None else lens.data_ptr(), B, n, V, tokens.data_ptr(),
                  accepted.data_ptr(), dtype_code(p), _stream(p))
    return tokens, accepted


# -------------------------------------------------------------------- backward
def rms_norm_backward(dy: torch.Tensor, x: torch.Tensor, weight: torch.Tensor, eps: float,
                      need_dw: bool = True) -> tuple[torch.Tensor, torch.Tensor | None]:
    """(dx, dw) of out = weight * x * rsqrt(mean(x^2) + eps) over the last dim;
    dw is None when not need_dw.  fp32 math, deterministic dw."""
    if dy.shape != x.shape or dy.dtype != x.dtype:
        raise ValueError("dy and x must match")
    x, rows, cols, ldx = _rows_or_contig(x)
    dy, _, _, lddy = _rows_or_contig(dy)
    if weight.dtype != x.dtype or weight.numel() != cols or not weight.is_contiguous():
        raise ValueError("weight must be a contiguous [cols] tensor of x's dtype")
    dx = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    _, _, lddx = _rows_view(dx)
    dw = torch.empty(cols, dtype=x.dtype, device=x.device) if need_dw else None
    with _on_device(x):
        ws, nws = None, 0
        if need_dw:
            nws = _abi.lib().fl_b200_rms_norm_bwd_workspace_size(rows, cols)
            ws = torch.empty(max(nws, 16), dtype=torch.uint8, device=x.device) if nws else None
        _abi.call("fl_b200_rms_norm_bwd", dy.data_ptr(), lddy, x.data_ptr(), ldx,
                  weight.data_ptr(), dx.data_ptr(), lddx, dw.data_ptr() if need_dw else None,
                  rows, cols, float(eps), dtype_code(x), ws.data_ptr() if ws is not None else None,
                  nws, _stream(x))
    return dx, dw


def swiglu_backward(dout: torch.Tensor, gate: torch.Tensor,
                    up: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(dgate, dup) of out = silu(gate) * up."""
    if not (dout.shape == gate.shape == up.shape) or not (dout.dtype == gate.dtype == up.dtype):
        raise ValueError("dout, gate and up must match")
    dout, gate, up = dout.contiguous(), gate.contiguous(), up.contiguous()
    dg, du = torch.empty_like(gate), torch.empty_like(up)
    with _on_device(gate):
        _abi.call("fl_b200_swiglu_bwd", dout.data_ptr(), gate.data_ptr(), up.data_ptr(),
                  dg.data_ptr(), du.data_ptr(), gate.numel(), dtype_code(gate), _stream(gate))
    return dg, du


def silu_backward(dout: torch.Tensor, x: torch.Tensor) -> torch.Tensor:
    """d silu(x) = dout * s * (1 + x (1 - s)), s = sigmoid(x)."""
    if dout.shape != x.shape or dout.dtype != x.dtype:
        raise ValueError("dout and x must match")
    dout, x = dout.contiguous(), x.contiguous()
    dx = torch.empty_like(x)
    with _on_device(x):
        _abi.call("fl_b200_silu_bwd", dout.data_ptr(), x.data_ptr(), dx.data_ptr(), x.numel(),
                  dtype_code(x), _stream(x))
    return dx


def softmax_backward(dy: torch.Tensor, y: torch.Tensor,
                     out_dtype: torch.dtype | None = None, scale: float = 1.0) -> torch.Tensor:
    """dx = scale * y * (dy - sum(dy * y)) over the last dim; out_dtype
    defaults to y's dtype (a 16-bit dtype with fp32 dy/y: half_to_float's
    backward).  scale != 1 is the backward of masked_softmax."""
    if dy.shape != y.shape or dy.dtype != y.dtype:
        raise ValueError("dy and y must match")
    out_dtype = out_dtype or y.dtype
    if y.dim() == 0:
        return torch.zeros((), dtype=out_dtype, device=y.device)
    y, rows, cols, ldy = _rows_or_contig(y)
    dy, _, _, lddy = _rows_or_contig(dy)
    dx = torch.empty(y.shape, dtype=out_dtype, device=y.device)
    with _on_device(y):
        _abi.call("fl_b200_softmax_bwd_scaled", dy.data_ptr(), lddy, y.data_ptr(), ldy,
                  dx.data_ptr(), cols, rows, cols, float(scale), dtype_code(y), _DT[out_dtype],
                  _stream(y))
    return dx
