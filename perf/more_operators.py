"""The operators of a training step around a decoder's matrix products, in the forms that newer
decoders give them, and in those that serving gives them.

    rotary    query and key heads turned by their tokens' positions: halves or neighbours, the whole
              head or its first part, frequencies scaled for long contexts; and the gradient
    sandwich  the norm after a block, its gate and scale, the residual add and the norm before the
              next block in one; and the gradients
    span      softmax of attention scores over each query's span of keys (causal, a window, packed
              documents, a prefix), scores capped by a tanh or biased by distance; and the gradient
    clip      the norm of all gradients, and the gradients clipped to it

`run` computes the plain forms with elementary torch operations; with `own` set it makes the calls
a user makes of torch_fl.
"""

import math
import os
import sys

import torch

own = False

EPS = 1e-6
_TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_BYTES = {"bf16": 2, "f16": 2, "f32": 4}


def listed():
    return [
        # one decode step of a small batch in a long context: launch latency
        {"name": "rotary_decode", "kind": "rotary", "batch": 8, "tokens": 1, "heads": 32, "kv_heads": 8, "head": 128, "turned": 128, "neighbours": False, "stretch": 4.0, "reach": 131072, "back": False, "type": "bf16"},
        # a prefill, or the forward of a training batch
        {"name": "rotary_batch", "kind": "rotary", "batch": 16, "tokens": 4096, "heads": 32, "kv_heads": 8, "head": 128, "turned": 128, "neighbours": False, "stretch": 1.0, "reach": 4096, "back": False, "type": "bf16"},
        # the backward of heads of which a part is turned, neighbours together, over an odd length
        {"name": "rotary_back_part", "kind": "rotary", "batch": 3, "tokens": 2731, "heads": 16, "kv_heads": 16, "head": 192, "turned": 64, "neighbours": True, "stretch": 1.0, "reach": 2731, "back": True, "type": "f32"},
        # one decode step: launch latency
        {"name": "sandwich_decode", "kind": "sandwich", "batch": 8, "tokens": 1, "hidden": 4096, "gate": "none", "scale": 1.0, "offset": 1.0, "back": False, "type": "bf16"},
        # the forward of a large batch with a learned gate for each channel
        {"name": "sandwich_batch", "kind": "sandwich", "batch": 8, "tokens": 8192, "hidden": 4096, "gate": "channel", "scale": 0.25, "offset": 0.0, "back": False, "type": "bf16"},
        # a training step, forward and backward, with a gate for each sequence (conditioning)
        {"name": "sandwich_train", "kind": "sandwich", "batch": 8, "tokens": 4096, "hidden": 4096, "gate": "sequence", "scale": 1.0, "offset": 0.0, "back": True, "type": "bf16"},
        # a decode step over a cache: sequences of different lengths, a bias by distance
        {"name": "span_decode", "kind": "span", "batch": 16, "heads": 32, "queries": 1, "keys": 8192, "mask": "causal", "window": 0, "padded": True, "cap": 0.0, "bias": True, "back": False, "type": "bf16"},
        # the forward of packed training documents, capped scores
        {"name": "span_documents", "kind": "span", "batch": 8, "heads": 32, "queries": 2048, "keys": 2048, "mask": "documents", "window": 0, "padded": False, "cap": 50.0, "bias": False, "back": False, "type": "bf16"},
        # a training step, forward and backward, over a prefix and odd lengths, padded rows
        {"name": "span_train_odd", "kind": "span", "batch": 4, "heads": 12, "queries": 1531, "keys": 1531, "mask": "prefix", "window": 0, "padded": True, "cap": 30.0, "bias": True, "back": True, "type": "f16"},
        # the gradients of low-rank adapters: many small tensors, launch latency
        {"name": "clip_adapters", "kind": "clip", "layers": 16, "hidden": 2048, "inner": 0, "rank": 16, "vocab": 0, "clip": True, "norm": 2.0, "type": "f32"},
        # the gradients of two decoder layers and an embedding
        {"name": "clip_layers", "kind": "clip", "layers": 2, "hidden": 4096, "inner": 14336, "rank": 0, "vocab": 128256, "clip": True, "norm": 2.0, "type": "bf16"},
        # gradients of odd sizes under a loss scale
        {"name": "clip_odd", "kind": "clip", "layers": 24, "hidden": 1001, "inner": 2731, "rank": 0, "vocab": 32003, "clip": True, "norm": 2.0, "type": "f16"},
    ]


def draw(rng):
    def spread(lo, hi):
        return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))

    kind = rng.choice(["rotary", "sandwich", "span", "clip"])
    type_ = rng.choice(["bf16", "f16", "f32"])
    size = _BYTES[type_]
    if kind == "rotary":
        head = rng.choice([64, 80, 96, 128, 192, 256])
        turned = head if rng.random() < 0.5 else max(2, head * rng.choice([1, 2, 3]) // 4 // 2 * 2)
        kv_heads = spread(1, 16)
        heads = kv_heads * spread(1, 8)
        most = 65536 * 40 * 128 * 2 // ((heads + kv_heads) * head * size)
        tokens = spread(1, min(8192, most))
        return {"kind": kind, "batch": spread(1, max(1, min(64, most // tokens))), "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "head": head, "turned": turned,
                "neighbours": rng.random() < 0.5, "stretch": rng.choice([1.0, 1.0, 4.0, 32.0]), "reach": max(tokens, spread(1024, 1000000)), "back": rng.random() < 0.4, "type": type_}
    if kind == "sandwich":
        hidden = spread(256, 16384)
        if rng.random() < 0.75:
            hidden = hidden // 64 * 64
        back = rng.random() < 0.5
        most = (32768 if back else 65536) * 4096 * 2 // (hidden * size)
        tokens = spread(1, min(8192, most))
        return {"kind": kind, "batch": spread(1, max(1, min(64, most // tokens))), "tokens": tokens, "hidden": hidden, "gate": rng.choice(["none", "channel", "sequence", "token"]),
                "scale": rng.choice([1.0, 0.25, 0.5]), "offset": rng.choice([0.0, 1.0]), "back": back, "type": type_}
    if kind == "span":
        heads, back = spread(1, 32), rng.random() < 0.5
        mask = rng.choice(["causal", "documents", "prefix"])
        most = (8 if back else 16) * 32 * 2048 * 2048 // size
        if mask == "causal" and rng.random() < 0.5:
            queries, keys = spread(1, 16), spread(64, 65536)
        else:
            queries = keys = spread(16, 4096)
            if rng.random() < 0.5:
                queries = keys = max(16, keys // 8 * 8)
        return {"kind": kind, "batch": spread(1, max(1, min(64, most // (heads * queries * keys)))), "heads": heads, "queries": min(queries, keys), "keys": keys, "mask": mask,
                "window": rng.choice([0, 0, max(1, keys // 5)]) if mask == "causal" else 0, "padded": rng.random() < 0.5, "cap": rng.choice([0.0, 20.0, 50.0]), "bias": rng.random() < 0.5, "back": back, "type": type_}
    if rng.random() < 0.5:
        return {"kind": kind, "layers": spread(1, 48), "hidden": spread(128, 8192), "inner": 0, "rank": spread(1, 64), "vocab": 0, "clip": rng.random() < 0.7, "norm": rng.choice([2.0, 2.0, math.inf]), "type": type_}
    hidden = spread(64, 4096)
    inner = int(hidden * rng.choice([2.5, 2.73, 3.5]))
    layer = hidden * (3 * inner + 4 * hidden)
    most = 900000000 // layer // (size // 2)
    return {"kind": kind, "layers": spread(1, max(1, min(64, most))), "hidden": hidden, "inner": inner, "rank": 0, "vocab": spread(64, max(64, min(128256, 50000000 // hidden))), "clip": rng.random() < 0.7,
            "norm": rng.choice([2.0, 2.0, math.inf]), "type": type_}


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _shapes(case):
    """The gradients' shapes, in a program's order."""
    n, i, r = case["hidden"], case["inner"], case["rank"]
    shapes = [(case["vocab"], n)] if case["vocab"] else []
    for _ in range(case["layers"]):
        if r:
            shapes += [(r, n), (n, r)] * 4                       # adapters of four projections
        else:
            kv = max(1, n // 4)
            shapes += [(n,), (n, n), (kv, n), (kv, n), (n, n), (n,), (i, n), (i, n), (n, i)]
    return shapes


def prepare(case, seed):
    g = _generator(seed)
    type_, kind = _TYPES[case["type"]], case["kind"]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    def whole(lo, hi, *shape):
        return torch.randint(lo, hi, shape, generator=g, device="cuda")

    if kind == "rotary":
        batch, tokens, half = case["batch"], case["tokens"], case["turned"] // 2
        q = normal(batch, tokens, case["heads"], case["head"]).to(type_)
        k = normal(batch, tokens, case["kv_heads"], case["head"]).to(type_)
        # each sequence goes on from where it stands; frequencies of a base of 1e4, the slow ones
        # stretched for a longer context and the fast ones kept, with a ramp between them
        start = whole(0, max(1, case["reach"] - tokens + 1), batch, 1)
        positions = start + torch.arange(tokens, device="cuda")
        fast = 1e4 ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half)
        turns = fast * 4096 / (2 * math.pi)
        ramp = ((turns - 1) / 31).clamp(0, 1)
        freq = fast * ramp + fast / case["stretch"] * (1 - ramp)
        return {"case": case, "q": q, "k": k, "positions": positions, "freq": freq.float(), "scale": 1.0 + 0.1 * math.log(case["stretch"])}

    if kind == "sandwich":
        batch, tokens, hidden = case["batch"], case["tokens"], case["hidden"]
        s = {"case": case}
        s["x"] = (normal(batch, tokens, hidden) * (0.3 + normal(1, 1, hidden).abs())).to(type_)
        s["residual"] = normal(batch, tokens, hidden).mul_(3.0).to(type_)
        s["post"] = (1.0 - case["offset"] + 0.2 * normal(hidden)).to(type_)
        s["pre"] = (1.0 - case["offset"] + 0.2 * normal(hidden)).to(type_)
        shape = {"none": None, "channel": (hidden,), "sequence": (batch, 1, hidden), "token": (batch, tokens, hidden)}[case["gate"]]
        s["gate"] = None if shape is None else (0.5 * normal(*shape)).to(type_)
        if case["back"]:
            s["dy"] = normal(batch, tokens, hidden).mul_(0.01).to(type_)
            s["dh"] = normal(batch, tokens, hidden).mul_(0.01).to(type_)
        return s

    if kind == "span":
        batch, heads, queries, keys = case["batch"], case["heads"], case["queries"], case["keys"]
        # lengths of padded sequences: the rows of a decode step end where their sequence does, a
        # training batch's rows behind the end see nothing
        ends = torch.full((batch, 1), keys, device="cuda")
        if case["padded"]:
            ends = whole(max(queries, keys // 4 if queries < keys else 3 * keys // 4), keys + 1, batch, 1)
        at = torch.arange(queries, device="cuda").expand(batch, queries)
        if queries < keys:
            at = at + ends - queries
        lo, hi = torch.zeros_like(at), at + 1
        if case["mask"] == "documents":
            cuts = torch.sort(whole(1, max(2, keys), batch, 7), -1).values
            cuts = torch.cat([torch.zeros_like(cuts[:, :1]), cuts], -1)
            lo = torch.where(cuts[:, None] <= at[..., None], cuts[:, None], 0).amax(-1)
        elif case["mask"] == "prefix":
            hi = torch.maximum(hi, whole(1, max(2, keys // 2), batch, 1))
        if case["window"]:
            lo = torch.maximum(lo, at - case["window"] + 1)
        hi = torch.where(at < ends, torch.minimum(hi, ends), lo)
        s = {"case": case, "spans": torch.stack([lo, hi], -1).int(), "positions": at.int()}
        s["x"] = normal(batch, heads, queries, keys).mul_(12.0 if case["cap"] else 6.0).to(type_)
        s["scale"] = 0.5
        s["slopes"] = 2.0 ** (-8.0 * torch.arange(1, heads + 1, device="cuda") / heads) if case["bias"] else None
        if case["back"]:
            s["dy"] = normal(batch, heads, queries, keys).mul_(0.1).to(type_)
        return s

    # gradients of layers differ in size, and half precision has a loss scale; the bound is some
    # two fifths of their norm, so that clipping does work; clipped gradients go to one bucket
    shapes, step = _shapes(case), 0.064 if case["type"] == "f16" else 1e-3
    grads = [(normal(*shape).mul_(step * (1 + i % 5))).to(type_) for i, shape in enumerate(shapes)]
    s = {"case": case, "grads": grads}
    if case["norm"] == math.inf:
        s["bound"] = 7.0 * step
    else:
        s["bound"] = 0.4 * step * math.sqrt(sum((1 + i % 5) ** 2 * t.numel() for i, t in enumerate(grads)))
    if case["clip"]:
        room = [-(-t.numel() // 64) * 64 for t in grads]
        s["bucket"] = torch.zeros(sum(room), device="cuda", dtype=type_)
        s["out"] = [part[: t.numel()].view(t.shape) for part, t in zip(s["bucket"].split(room), grads)]
    return s


# ------------------------------------------------------------------------------------- plain forms
def _turn(x, cos, sin, turned, neighbours):
    a = x[..., :turned].float()
    cos, sin = cos[:, :, None], sin[:, :, None]
    if neighbours:
        even, odd = a[..., 0::2], a[..., 1::2]
        a = torch.stack([even * cos - odd * sin, odd * cos + even * sin], -1).flatten(-2)
    else:
        low, high = a[..., : turned // 2], a[..., turned // 2:]
        a = torch.cat([low * cos - high * sin, high * cos + low * sin], -1)
    return torch.cat([a.to(x.dtype), x[..., turned:]], -1)


def _rotary(s):
    case = s["case"]
    angle = s["positions"][..., None].double() * s["freq"].double()
    cos, sin = (torch.cos(angle) * s["scale"]).float(), (torch.sin(angle) * s["scale"]).float()
    if case["back"]:
        sin = -sin
    return {"q": _turn(s["q"], cos, sin, case["turned"], case["neighbours"]), "k": _turn(s["k"], cos, sin, case["turned"], case["neighbours"])}


def _sandwich(s):
    case = s["case"]
    x, post, pre = s["x"].float(), s["post"].float() + case["offset"], s["pre"].float() + case["offset"]
    gate = case["scale"] if s["gate"] is None else case["scale"] * s["gate"].float()
    rx = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
    n = x * rx
    h = s["residual"].float() + gate * (n * post)
    y = h * torch.rsqrt((h * h).mean(-1, keepdim=True) + EPS) * pre
    out = {"y": y.to(s["x"].dtype), "h": h.to(s["x"].dtype)}
    if case["back"]:
        del y, h
        # the gradients take h as it was stored
        h, dy = out["h"].float(), s["dy"].float()
        rh = torch.rsqrt((h * h).mean(-1, keepdim=True) + EPS)
        m = h * rh
        out["dpre"] = (dy * m).flatten(0, 1).sum(0).to(s["pre"].dtype)
        dy = dy * pre
        dh = s["dh"].float() + rh * (dy - m * (dy * m).mean(-1, keepdim=True))
        del dy, m, h
        out["dresidual"] = dh.to(s["x"].dtype)
        if s["gate"] is not None:
            dgate = dh * (n * post) * case["scale"]
            dims = [d for d in range(3) if s["gate"].dim() == 1 and d < 2 or s["gate"].dim() == 3 and s["gate"].shape[d] != dgate.shape[d]]
            if dims:
                dgate = dgate.sum(dims, keepdim=s["gate"].dim() == 3)
            out["dgate"] = dgate.to(s["gate"].dtype)
            del dgate
        dh = dh * gate
        out["dpost"] = (dh * n).flatten(0, 1).sum(0).to(s["post"].dtype)
        dh = dh * post
        out["dx"] = (rx * (dh - n * (dh * n).mean(-1, keepdim=True))).to(s["x"].dtype)
    return out


def _span(s):
    case, spans = s["case"], s["spans"][:, None]
    key = torch.arange(case["keys"], device="cuda", dtype=torch.int32)
    seen = (key >= spans[..., :1]) & (key < spans[..., 1:])
    z = s["x"].float() * s["scale"]
    t = None
    if case["cap"]:
        t = torch.tanh(z / case["cap"])
        z = case["cap"] * t
    if s["slopes"] is not None:
        z = z - s["slopes"][:, None, None] * (s["positions"][:, None, :, None] - key).abs()
    z = z.masked_fill_(~seen, -math.inf)
    top = z.amax(-1, keepdim=True)
    e = torch.exp(z - torch.where(top > -math.inf, top, 0.0))
    del z
    total = e.sum(-1, keepdim=True)
    y = e / torch.where(total > 0, total, 1.0)
    del e
    out = {"y": y.to(s["x"].dtype)}
    if case["back"]:
        # the gradient takes y as it was stored
        y, dy = out["y"].float(), s["dy"].float()
        dx = s["scale"] * y * (dy - (y * dy).sum(-1, keepdim=True))
        if t is not None:
            dx = dx * (1 - t * t)
        out["dx"] = dx.to(s["x"].dtype)
    return out


def _clip(s):
    case = s["case"]
    if case["norm"] == math.inf:
        norm = torch.stack([t.abs().amax() for t in s["grads"]]).amax().double()
    else:
        norm = torch.stack([t.float().square().sum(dtype=torch.float64) for t in s["grads"]]).sum().sqrt()
    out = {"norm": norm.float()}
    if case["clip"]:
        factor = (s["bound"] / (norm + 1e-6)).clamp(max=1.0).float()
        for t, into in zip(s["grads"], s["out"]):
            into.copy_(t.float() * factor)
        out["clipped"] = s["bucket"]
    return out


def _plain(s):
    return {"rotary": _rotary, "sandwich": _sandwich, "span": _span, "clip": _clip}[s["case"]["kind"]](s)


# ------------------------------------------------------------------------------------- torch_fl
def _package():
    if "torch_fl" not in sys.modules:
        sys.path.insert(0, os.path.join(os.getcwd(), "pytorch-plugin-fl_b200"))
    import torch_fl

    return torch_fl


def _calls(s):
    fl, case = _package(), s["case"]
    kind = case["kind"]
    if kind == "rotary":
        # the gradient is the turn back, as autograd calls it
        q, k = fl.ops.rotary(s["q"], s["k"], s["positions"], s["freq"], scale=s["scale"], interleaved=case["neighbours"], unsqueeze_dim=2, inverse=case["back"])
        return {"q": q, "k": k}
    if kind == "sandwich":
        y, h = fl.ops.sandwich_norm(s["x"], s["residual"], s["post"], s["pre"], EPS, gate=s["gate"], scale=case["scale"], weight_offset=case["offset"])
        out = {"y": y, "h": h}
        if case["back"]:
            dx, dresidual, dpost, dpre, dgate = torch.ops.flagos.sandwich_norm_backward(s["dy"], s["dh"], s["x"], h, s["post"], s["pre"], s["gate"], EPS, case["scale"], case["offset"])
            out.update(dpre=dpre, dresidual=dresidual)
            if s["gate"] is not None:
                out["dgate"] = dgate
            out.update(dpost=dpost, dx=dx)
        return out
    if kind == "span":
        y = fl.ops.span_softmax(s["x"], s["spans"], scale=s["scale"], cap=case["cap"] or None, slopes=s["slopes"], positions=s["positions"])
        out = {"y": y}
        if case["back"]:
            out["dx"] = torch.ops.flagos.span_softmax_backward(s["dy"], y, s["x"], s["spans"], s["scale"], case["cap"] or None)
        return out
    if case["clip"]:
        _, norm = fl.ops.clip_grads(s["grads"], s["bound"], norm_type=case["norm"], out=s["out"])
        return {"norm": norm, "clipped": s["bucket"]}
    return {"norm": fl.ops.grad_norm(s["grads"], norm_type=case["norm"])}


def run(state):
    if own:
        return _calls(state)
    return _plain(state)


# ------------------------------------------------------------------------------------- what it takes
def _seen(case):
    """Keys in the spans of one head and sequence, in the mean over what prepare() draws."""
    q, k = case["queries"], case["keys"]
    share = (5 / 8 if q < k else 7 / 8) if case["padded"] else 1.0
    if q < k:
        n = q * k * share
    elif case["mask"] == "documents":
        n = k * k / 9
    elif case["mask"] == "prefix":
        n = k * k / 2 * share * share + k * k / 24
    else:
        n = k * k / 2 * share * share
    if case["window"]:
        n = min(n, q * case["window"])
    return n


def work(case):
    size, kind = _BYTES[case["type"]], case["kind"]
    if kind == "rotary":
        tokens = case["batch"] * case["tokens"]
        heads = case["heads"] + case["kv_heads"]
        return {"bytes": tokens * (2 * heads * case["head"] * size + 8) + case["turned"] * 2, "flops": tokens * heads * case["turned"] * 3}
    if kind == "sandwich":
        rows, hidden = case["batch"] * case["tokens"], case["hidden"]
        gate = {"none": 0, "channel": 1, "sequence": case["batch"], "token": rows}[case["gate"]]
        if case["back"]:
            return {"bytes": (8 * rows + 2 * gate + 4) * hidden * size, "flops": rows * hidden * 30}
        return {"bytes": (4 * rows + gate + 2) * hidden * size, "flops": rows * hidden * 9}
    if kind == "span":
        maps = case["batch"] * case["heads"]
        full, seen = case["queries"] * case["keys"], _seen(case)
        passes = 2 if case["back"] else 1
        return {"bytes": int(maps * (full + seen) * size * passes + case["batch"] * case["queries"] * 12), "flops": int(maps * seen * 8 * passes)}
    n = sum(math.prod(shape) for shape in _shapes(case))
    return {"bytes": n * size * (2 if case["clip"] else 1) + 4, "flops": n * (3 if case["clip"] else 2)}


# ------------------------------------------------------------------------------------- 64 bits
def _exact_rotary(s):
    case, half = s["case"], s["case"]["turned"] // 2
    angle = torch.einsum("bt,f->btf", s["positions"].double(), s["freq"].double())
    turn = torch.polar(torch.full_like(angle, s["scale"]), -angle if case["back"] else angle)
    out = {}
    for name in ("q", "k"):
        wide = s[name].double()
        for b in range(wide.shape[0]):
            part = wide[b, ..., : 2 * half]
            pairs = part.unflatten(-1, (half, 2)) if case["neighbours"] else part.unflatten(-1, (2, half)).transpose(-1, -2)
            pairs = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn[b, :, None])
            wide[b, ..., : 2 * half] = (pairs if case["neighbours"] else pairs.transpose(-1, -2)).flatten(-2)
        out[name] = wide
    return out


def _exact_sandwich(s):
    case, type_ = s["case"], s["x"].dtype
    batch, tokens, hidden = s["x"].shape
    post, pre = s["post"].double() + case["offset"], s["pre"].double() + case["offset"]
    out = {"y": [], "h": []}
    if case["back"]:
        out.update(dpre=0.0, dresidual=[])
        if s["gate"] is not None:
            out["dgate"] = [] if case["gate"] != "channel" else 0.0
        out.update(dpost=0.0, dx=[])
    for b in range(batch):
        x, gate = s["x"][b].double(), torch.full((1, hidden), case["scale"], device="cuda", dtype=torch.float64)
        if s["gate"] is not None:
            gate = gate * (s["gate"] if case["gate"] == "channel" else s["gate"][b]).double()
        root = torch.sqrt(x.pow(2).sum(-1, keepdim=True) / hidden + EPS)
        normed = x / root
        h = s["residual"][b].double() + gate * post * normed
        out["h"].append(h)
        out["y"].append(pre * h / torch.sqrt(h.pow(2).sum(-1, keepdim=True) / hidden + EPS))
        if not case["back"]:
            continue
        held, dy = h.to(type_).double(), s["dy"][b].double()
        root_h = torch.sqrt(held.pow(2).sum(-1, keepdim=True) / hidden + EPS)
        out["dpre"] = out["dpre"] + (dy * held / root_h).sum(0)
        along = (dy * pre * held).sum(-1, keepdim=True) / hidden
        dh = s["dh"][b].double() + dy * pre / root_h - held * along / root_h.pow(3)
        out["dresidual"].append(dh)
        each = dh * normed
        out["dpost"] = out["dpost"] + (each * gate).sum(0)
        if s["gate"] is not None:
            dgate = each * post * case["scale"]
            if case["gate"] == "channel":
                out["dgate"] = out["dgate"] + dgate.sum(0)
            else:
                out["dgate"].append(dgate.sum(0, keepdim=True) if case["gate"] == "sequence" else dgate)
        along = (dh * gate * post * x).sum(-1, keepdim=True) / hidden
        out["dx"].append(dh * gate * post / root - x * along / root.pow(3))
    return {name: torch.stack(v) if isinstance(v, list) else v for name, v in out.items()}


def _exact_span(s):
    case = s["case"]
    out = {"y": []}
    if case["back"]:
        out["dx"] = []
    key = torch.arange(case["keys"], device="cuda")
    for b in range(case["batch"]):
        first, last = s["spans"][b, :, 0].long(), s["spans"][b, :, 1].long()
        outside = (key[None] < first[:, None]) | (key[None] >= last[:, None])
        for name in out:
            out[name].append([])
        for head in range(case["heads"]):
            score = s["x"][b, head].double() * s["scale"]
            slope = None
            if case["cap"]:
                tanh = torch.tanh(score / case["cap"])
                score, slope = tanh * case["cap"], 1 - tanh.pow(2)
            if s["slopes"] is not None:
                score = score - s["slopes"][head].double() * (key[None] - s["positions"][b, :, None].long()).abs()
            y = torch.softmax(score.masked_fill(outside, -math.inf), -1).masked_fill(outside, 0.0)
            out["y"][-1].append(y)
            if case["back"]:
                held, dy = y.to(s["x"].dtype).double(), s["dy"][b, head].double()
                dx = held * (dy - (held * dy).sum(-1, keepdim=True)) * s["scale"]
                out["dx"][-1].append(dx if slope is None else dx * slope)
        for name in out:
            out[name][-1] = torch.stack(out[name][-1])
    return {name: torch.stack(v) for name, v in out.items()}


def _exact_clip(s):
    case = s["case"]
    if case["norm"] == math.inf:
        norm = max(float(t.abs().max()) for t in s["grads"])
    else:
        norm = math.sqrt(math.fsum(float(torch.linalg.vector_norm(t, dtype=torch.float64)) ** 2 for t in s["grads"]))
    out = {"norm": torch.tensor(norm, dtype=torch.float64, device="cuda")}
    if case["clip"]:
        out["clipped"] = torch.zeros_like(s["bucket"], dtype=torch.float64)
        for t, into in zip(s["grads"], s["out"]):
            at = into.storage_offset()
            out["clipped"][at : at + t.numel()] = t.flatten().double() * min(1.0, s["bound"] / (norm + 1e-6))
    return out


def exact(case, seed):
    """What run() returns, from the definitions in 64 bits."""
    s = prepare(case, seed)
    return {"rotary": _exact_rotary, "sandwich": _exact_sandwich, "span": _exact_span, "clip": _exact_clip}[case["kind"]](s)
