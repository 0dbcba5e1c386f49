"""Python entry points of the flagos:: fused ops (torch.ops.flagos.*).

They take flagos or cuda tensors and return tensors on the same device.
`rounding` is "fused" (compute in fp32, round once: within 1 ulp of the
fp32-accumulated result) or "chain" (round where the reference's op-by-op HF
chain rounds); the default comes from FLAGOS_B200_ROUNDING, else "fused".
"""

from __future__ import annotations

import math
import os

import torch

from . import _C


def default_rounding() -> str:
    r = os.environ.get("FLAGOS_B200_ROUNDING", "fused")
    if r not in ("fused", "chain"):
        raise ValueError(f"FLAGOS_B200_ROUNDING must be 'fused' or 'chain', got {r!r}")
    return r


def rms_norm(x, weight, eps: float, rounding: str | None = None):
    """weight * (x * rsqrt(mean(x^2) + eps)) over the last dim
    (transformers models/qwen3/modeling_qwen3.py:59-64)."""
    return torch.ops.flagos.rms_norm(x, weight, float(eps), rounding or default_rounding())


def add_rms_norm(x, residual, weight, eps: float, rounding: str | None = None):
    """(rms_norm(x + residual), x + residual) in one pass."""
    return torch.ops.flagos.add_rms_norm(x, residual, weight, float(eps),
                                         rounding or default_rounding())


def rope_qk(q, k, cos, sin, unsqueeze_dim: int = 1, rounding: str | None = None):
    """apply_rotary_pos_emb(q, k, cos, sin, unsqueeze_dim)
    (modeling_qwen3.py:158-181); q/k are [B,H,S,D] (unsqueeze_dim=1) or
    [B,S,H,D] (unsqueeze_dim=2), cos/sin [B,S,D] or [S,D]."""
    return torch.ops.flagos.rope_qk(q, k, cos, sin, int(unsqueeze_dim),
                                    rounding or default_rounding())


def rms_norm_rope(q, k, q_weight, k_weight, cos, sin, eps: float, unsqueeze_dim: int = 1,
                  rounding: str | None = None):
    """Qwen3's q_norm / k_norm over the head dim followed by RoPE, one pass
    (modeling_qwen3.py:248-249, 263-268)."""
    return torch.ops.flagos.rms_norm_rope(q, k, q_weight, k_weight, cos, sin, float(eps),
                                          int(unsqueeze_dim), rounding or default_rounding())


def swiglu(gate, up, rounding: str | None = None):
    """silu(gate) * up (Qwen3MLP, modeling_qwen3.py:81-82)."""
    return torch.ops.flagos.swiglu(gate, up, rounding or default_rounding())


def swiglu_residual(gate, up, x, y, rounding: str | None = None):
    """(silu(gate) * up, x + y) in one launch."""
    return torch.ops.flagos.swiglu_residual(gate, up, x, y, rounding or default_rounding())


def causal_softmax(x, offset: int = 0, dtype: torch.dtype | None = None):
    """softmax over the last dim of x [..., q_len, k_len] with the causal mask
    applied in the kernel: query i sees keys j <= i + offset; masked entries
    are exact zeros and are never read."""
    return torch.ops.flagos.causal_softmax(x, int(offset), dtype)


def masked_softmax(x, mask=None, scale: float = 1.0, dtype: torch.dtype | None = None,
                   rounding: str | None = None):
    """softmax(x * scale + mask) over the last dim in one launch: the tail of
    HF's eager attention (modeling_qwen3.py eager_attention_forward,
    `attn_weights * scaling + attention_mask`, softmax(dtype=float32), then
    `.to(query.dtype)`).  x is [B, H, Q, K] (or fewer leading dims); mask has
    x's dtype and broadcasts to x; dtype None = x's dtype (the cast back
    fused) or float32."""
    return torch.ops.flagos.masked_softmax(x, mask, float(scale), dtype,
                                           rounding or default_rounding())


# ---------------------------------- a training step around the matrix products
# (the one overload each has: a call need not look for it)
_rotary = torch.ops.flagos.rotary.default
_sandwich_norm = torch.ops.flagos.sandwich_norm.default
_span_softmax = torch.ops.flagos.span_softmax.default


def rotary(q, k, positions, inv_freq, scale: float = 1.0, interleaved: bool = False,
           unsqueeze_dim: int = 1, inverse: bool = False):
    """(q, k) with each head turned by its token's position, without a table of
    cosines: angle = position * inv_freq[i] and

        (a, b) -> scale * (a cos - b sin, b cos + a sin)

    with (a, b) = (x[i], x[i + n]) (halves) or, interleaved, (x[2i], x[2i + 1])
    (neighbours), n = len(inv_freq); elements from 2 n on stay as they are.
    q/k are [B,H,S,D] (unsqueeze_dim=1) or [B,S,H,D] (unsqueeze_dim=2) in any
    strides, positions int32 or int64 [S] or [B,S], inv_freq float32
    (`rope_frequencies`).  Angles are exact to fp64 at any position, the result
    is rounded once.  inverse turns back: with the same scale it is the
    gradient.  Differentiable in q and k, any number of times."""
    return _rotary(q, k, positions, inv_freq, float(scale), bool(interleaved), int(unsqueeze_dim),
                   bool(inverse))


def rope_frequencies(dim: int, theta: float = 1e4, method: str = "default", factor: float = 1.0,
                     original_len: int = 0, seq_len: int = 0, low_turns: float = 1.0,
                     high_turns: float = 32.0, device=None):
    """(inv_freq, scale) for `rotary`: float32 [dim / 2] and the cosines'
    factor.  f_i = theta^(-2 i / dim), and by `method`

    * "default": f_i;
    * "linear": f_i / factor (position interpolation);
    * "dynamic": theta raised to theta * (factor L / original_len - factor + 1)^(dim / (dim - 2))
      with L = max(seq_len, original_len);
    * "yarn": frequencies that turn more than high_turns times in original_len
      stay, those that turn less than low_turns times are divided by factor,
      with a linear ramp over i between; scale = 0.1 ln(factor) + 1;
    * "llama3": the same with a ramp linear in the number of turns
      (its usual bounds are 1 and 4), scale 1."""
    if dim < 2 or dim % 2:
        raise ValueError(f"dim must be even and at least 2, got {dim}")
    if not theta > 0 or not factor > 0:
        raise ValueError("theta and factor must be positive")
    half = torch.arange(0, dim, 2, dtype=torch.float64)
    freq = theta ** (-half / dim)
    scale = 1.0
    if method == "default":
        pass
    elif method == "linear":
        freq = freq / factor
    elif method in ("dynamic", "yarn", "llama3"):
        if original_len < 1:
            raise ValueError(f"{method}: original_len is needed")
        if method == "dynamic":
            if dim < 4:
                raise ValueError("dynamic: dim must be at least 4")
            ratio = factor * max(seq_len, original_len) / original_len - (factor - 1)
            freq = (theta * ratio ** (dim / (dim - 2))) ** (-half / dim)
        else:
            if not 0 < low_turns < high_turns:
                raise ValueError(f"{method}: 0 < low_turns < high_turns")
            turns = original_len * freq / (2 * math.pi)
            if method == "llama3":
                keep = ((turns - low_turns) / (high_turns - low_turns)).clamp(0, 1)
            else:
                if theta <= 1:
                    raise ValueError("yarn: theta must be above 1")

                def index(t):  # the (real) i whose frequency turns t times
                    return dim * math.log(original_len / (t * 2 * math.pi)) / (2 * math.log(theta))

                first = max(math.floor(index(high_turns)), 0)
                last = min(math.ceil(index(low_turns)), dim - 1)
                ramp = (half / 2 - first) / max(last - first, 1e-3)
                keep = 1 - ramp.clamp(0, 1)
                scale = 0.1 * math.log(factor) + 1.0 if factor > 1 else 1.0
            freq = freq * keep + freq / factor * (1 - keep)
    else:
        raise ValueError(f"unknown method {method!r}")
    return freq.float().to(device), scale


def sandwich_norm(x, residual, post_weight, pre_weight, eps: float, gate=None, scale: float = 1.0,
                  weight_offset: float = 0.0):
    """(y, h): the norm after a block, its gate and scale, the residual add and
    the norm before the next block in one pass,

        h = residual + scale * gate * rms_norm(x) * (weight_offset + post_weight)
        y = rms_norm(h) * (weight_offset + pre_weight)

    x and residual are [..., hidden]; gate is [hidden] or has x's shape with
    sizes of 1 in the last dims before hidden ([B, 1, hidden]: one for each
    sequence), None: 1.  weight_offset 1 is for weights stored as differences
    from 1.  fp32 throughout, h and y rounded once (y from h before its
    rounding).  Differentiable once in every tensor; the gradient is computed
    from x and the stored h."""
    return _sandwich_norm(x, residual, post_weight, pre_weight, gate, float(eps), float(scale),
                          float(weight_offset))


def span_softmax(x, spans, scale: float = 1.0, cap: float | None = None, slopes=None, positions=None,
                 dtype: torch.dtype | None = None):
    """softmax of attention scores x [B, H, Q, K] (or fewer leading dims) over
    each query's span of keys lo <= j < hi, int32 spans [Q, 2] or [B, Q, 2]
    (`attention_spans`): causal and window masks, packed documents, prefixes
    and padding without a mask tensor.

        z = scale * x;  z = cap * tanh(z / cap) with a cap
        z = z - slopes[h] * |positions[q] - j| with slopes, float32 [H]
        y = softmax of z over the span, 0 outside it

    positions are int32 [Q] or [B, Q], None: q + K - Q.  A query that sees
    nothing gets zeros; keys outside a span are not used, whatever they hold.
    dtype None = x's, or float32.  Differentiable once, in x."""
    return _span_softmax(x, spans, float(scale), None if cap is None else float(cap), slopes, positions,
                         dtype)


def attention_spans(q_len: int, k_len: int, causal: bool = True, window: int | None = None,
                    documents=None, prefix=None, lengths=None, positions=None, device=None):
    """int32 spans [1 or B, q_len, 2] for `span_softmax`: the keys that query i
    at positions[..., i] (int [q_len] or [B, q_len]; None: i + k_len - q_len)
    sees.

    * causal: keys up to its own; otherwise all;
    * window: of these its own and the window - 1 before it (or, not causal,
      the window - 1 after it too);
    * documents: int ids [k_len] or [B, k_len] of the keys, equal ids side by
      side: keys of its own document;
    * prefix: an int or int [B]: keys before it are seen from inside the prefix
      too;
    * lengths: int [B]: keys from there on are padding, and queries from there
      on see nothing.
    A query whose position lies outside the keys sees nothing."""
    def batch(t, cols):
        t = torch.as_tensor(t, device=device)
        if t.is_floating_point() or t.is_complex() or t.dtype == torch.bool:
            raise TypeError("whole numbers expected")
        t = t.long()
        t = t.reshape(1, -1) if t.dim() < 2 else t
        if cols is not None and t.shape[-1] != cols:
            raise ValueError(f"{cols} columns expected, got {t.shape[-1]}")
        return t

    if window is not None and window < 1:
        raise ValueError("window must be at least 1")
    for t in (documents, prefix, lengths, positions):
        if device is None and isinstance(t, torch.Tensor):
            device = t.device
    at = torch.arange(q_len, device=device)[None] + (k_len - q_len) if positions is None else batch(positions, q_len)
    lo, hi = torch.zeros_like(at), torch.full_like(at, k_len)
    if causal:
        hi = at + 1
    if prefix is not None:
        p = batch(prefix, None).reshape(-1, 1)
        hi = torch.where(at < p, torch.maximum(hi, p), hi)
    if window is not None:
        lo = torch.maximum(lo, at - (window - 1))
        if not causal:
            hi = torch.minimum(hi, at + window)
    if documents is not None and k_len:
        ids = batch(documents, k_len)
        key = torch.arange(k_len, device=device)[None]
        new = torch.ones_like(ids, dtype=torch.bool)
        new[:, 1:] = ids[:, 1:] != ids[:, :-1]
        start = torch.where(new, key, 0).cummax(-1).values
        last = torch.ones_like(new)
        last[:, :-1] = new[:, 1:]
        end = torch.where(last, key + 1, k_len).flip(-1).cummin(-1).values.flip(-1)
        rows = max(ids.shape[0], at.shape[0])
        own = at.clamp(0, k_len - 1).expand(rows, -1)
        lo = torch.maximum(lo, start.expand(rows, -1).gather(-1, own))
        hi = torch.minimum(hi, end.expand(rows, -1).gather(-1, own))
    none = (at < 0) | (at >= k_len)
    if lengths is not None:
        n = batch(lengths, None).reshape(-1, 1)
        hi = torch.minimum(hi, n)
        none = none | (at >= n)
    hi = torch.minimum(hi, torch.full_like(hi, k_len))
    lo, hi, none = torch.broadcast_tensors(lo, hi, none)
    hi = torch.where(none, lo, torch.maximum(lo, hi))
    return torch.stack([lo, hi], -1).int()


def _grads(tensors):
    return [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)


# Lists of tensors go to the extension without the dispatcher (24 us for 128
# tensors, 42 us through it), except where a dispatch mode is to see the op.
_watched = torch._C._len_torch_dispatch_stack


def grad_norm(grads, norm_type: float = 2.0):
    """The norm of all tensors of a list taken as one vector (2, or inf for the
    largest magnitude): float32, on the device, in two launches.  Types may be
    mixed; squares that fp32 cannot hold are added in fp64."""
    grads = _grads(grads)
    if _watched():
        return torch.ops.flagos.grad_norm(grads, float(norm_type))
    return _C._grad_norm(grads, float(norm_type))


def clip_grads(grads, max_norm: float, norm_type: float = 2.0, out=None):
    """(clipped, norm): every tensor of the list times
    min(1, max_norm / (norm + 1e-6)), and the norm before, in two launches.
    `out`: tensors of the same shapes and types to write to (a bucket's views,
    say, or the gradients themselves), of which no two share memory; a list
    that names one tensor twice cannot be clipped in place.  Not
    differentiable."""
    grads = _grads(grads)
    if out is None:
        return torch.ops.flagos.clip_grads(grads, float(max_norm), float(norm_type))
    out = _grads(out)
    if _watched():
        return out, torch.ops.flagos.clip_grads_out(grads, float(max_norm), float(norm_type), out)
    return out, _C._clip_grads_out(grads, float(max_norm), float(norm_type), out)


def clip_grad_norm_(parameters, max_norm: float, norm_type: float = 2.0, error_if_nonfinite: bool = False):
    """torch.nn.utils.clip_grad_norm_ on the device, for dense gradients of one
    GPU and norms 2 and inf: clips the parameters' gradients in place and
    returns their norm; the host does not wait, except with
    error_if_nonfinite."""
    if isinstance(parameters, torch.Tensor):
        parameters = [parameters]
    grads = [p.grad for p in parameters if p.grad is not None]
    if not grads:
        return torch.tensor(0.0)
    if error_if_nonfinite and not math.isfinite(float(grad_norm(grads, norm_type))):
        raise RuntimeError(f"the norm of order {norm_type} of the gradients is not finite: nothing was clipped")
    return clip_grads(grads, max_norm, norm_type, out=grads)[1]


# ---------------------------------------------------- rows of the vocabulary
def topk(x, k: int):
    """(values, indices) of the k <= 1024 largest elements over the last dim,
    descending; equal values (-0 and +0 among them) by ascending index, NaN
    above everything, so there is one right answer.  Gradient: dvalues at the
    indices, which can be differentiated again."""
    return torch.ops.flagos.topk(x, int(k))


def distill_topk(logits, teacher_logits, teacher_ids, temperature: float = 1.0):
    """The distillation loss of each row, float32 [...]:

        temperature^2 * KL(softmax(teacher_logits / temperature) ||
                           softmax(logits / temperature)[teacher_ids])

    for a student's logits [..., vocab] and the k <= 1024 logits [..., k] that
    were kept of a teacher (`topk`), with their token ids (int32 or int64).
    The teacher's softmax is over its list; entries whose id lies outside
    [0, vocab) (-1, say) are absent, and a row without any has loss 0 and zero
    gradients whatever its logits hold.  Repeated ids add.  Differentiable once
    in logits and in teacher_logits (a second derivative raises, and so do
    forward mode and torch.func's transforms of gradients); the gradient is computed from the saved
    logits, which the forward and the backward read once each;
    `distill_topk_grad` reads them once for both."""
    return torch.ops.flagos.distill_topk(logits, teacher_logits, teacher_ids, float(temperature))[0]


def distill_topk_grad(logits, teacher_logits, teacher_ids, temperature: float = 1.0,
                      row_weight=None):
    """(loss, dlogits): `distill_topk`'s loss of each row, and the gradient of
    sum(row_weight * loss) with respect to the logits, in one call, for
    training loops whose row weights are known beforehand (1 / tokens, a loss
    mask, a loss scale).  row_weight is float32 and broadcasts to the loss;
    None weighs every row 1.  Not differentiable: hand dlogits on with
    `logits.backward(dlogits)`."""
    return torch.ops.flagos.distill_topk_grad(logits, teacher_logits, teacher_ids,
                                              float(temperature), row_weight)


def verify_draft(draft_ids, target_probs, draft_probs, uniform, draft_lens=None):
    """Speculative sampling's verification: (tokens, accepted), int64
    [batch, drafts + 1] and [batch].

    draft_ids [batch, drafts] are the drafted tokens, draft_lens [batch] how
    many of them each sequence has (None: all), target_probs
    [batch, drafts + 1, vocab] the target's probabilities at each and after
    the last, draft_probs [batch, drafts, vocab] the draft model's (None:
    drafts that come without, as looked-up ones do), uniform
    [batch, drafts + 1] float32 numbers in [0, 1).  Token i is kept while
    uniform[i] * q(token) < p(token); the next is drawn with uniform[drafts]
    from max(p - q, 0) at the first token turned down, else from the target's
    row after the last.  tokens holds the kept ones, the drawn one, then -1;
    accepted how many were kept.  The draw is exact in 36-bit fixed point, so
    it does not depend on the order of any sum."""
    return torch.ops.flagos.verify_draft(draft_ids, target_probs, draft_probs, uniform, draft_lens)
