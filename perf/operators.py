"""The vocabulary-row operators of a draft model's life: its target's top logits, the distillation
loss on them with its gradient, and the verification of the tokens it drafts.

    topk    the k largest of each row, descending, ties to the lowest index
    loss    KL(teacher's top logits || student), one value a row
    grad    that loss and its gradient with respect to the student's logits, in one call
    train   the loss, then its gradients with respect to the student's and the teacher's logits, as
            autograd calls them
    verify  drafted tokens against the target's probabilities, from given uniform numbers

`run` computes the plain forms with elementary torch operations; with `own` set it makes the calls
a user makes of torch_fl.
"""

import math
import os
import sys

import numpy as np
import torch

own = False

GRID = 2.0 ** 36          # probabilities are held as whole multiples of 1 / GRID when one is sampled
STEPS = 2 ** 24           # steps of a float32 uniform number
_TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_BYTES = {"bf16": 2, "f16": 2, "f32": 4}


def listed():
    return [
        # the top candidates of one decode step of a small batch: launch latency
        {"name": "topk_decode", "kind": "topk", "rows": 4, "vocab": 32000, "k": 8, "type": "bf16"},
        # a reranker's candidates in float32, rows that no 16-byte boundary begins
        {"name": "topk_odd_f32", "kind": "topk", "rows": 333, "vocab": 40003, "k": 50, "type": "f32"},
        # a teacher's top logits over a batch of training tokens, to be kept for distillation
        {"name": "topk_teacher", "kind": "topk", "rows": 4096, "vocab": 128256, "k": 64, "type": "bf16"},
        # evaluation of a small student on a few rows, float32 logits
        {"name": "loss_small_f32", "kind": "loss", "rows": 32, "vocab": 32000, "k": 16, "type": "f32", "temperature": 1.0},
        # evaluation over a training batch with a large vocabulary
        {"name": "loss_batch", "kind": "loss", "rows": 8192, "vocab": 128256, "k": 64, "type": "bf16", "temperature": 2.0},
        # a training step that asks for loss and gradient at once
        {"name": "grad_batch", "kind": "grad", "rows": 2048, "vocab": 128256, "k": 64, "type": "bf16", "temperature": 2.0},
        # the same with an odd vocabulary, masked entries at its end, and loss scaling
        {"name": "grad_odd_f16", "kind": "grad", "rows": 1001, "vocab": 40003, "k": 33, "type": "f16", "temperature": 1.5},
        # a training step through autograd: forward, then backward, teacher's gradient too
        {"name": "train_batch", "kind": "train", "rows": 4096, "vocab": 65536, "k": 32, "type": "bf16", "temperature": 1.0},
        # the same in float32 for a few odd rows
        {"name": "train_odd_f32", "kind": "train", "rows": 63, "vocab": 32001, "k": 7, "type": "f32", "temperature": 4.0},
        # one user's drafted tokens: launch latency
        {"name": "verify_one", "kind": "verify", "batch": 1, "drafts": 4, "vocab": 32000, "type": "f32", "draft_probs": True},
        # a serving batch whose draft model gives its probabilities
        {"name": "verify_batch", "kind": "verify", "batch": 256, "drafts": 5, "vocab": 128256, "type": "f32", "draft_probs": True},
        # drafts looked up in the prompt: no probabilities come with them
        {"name": "verify_lookup", "kind": "verify", "batch": 97, "drafts": 7, "vocab": 40003, "type": "bf16", "draft_probs": False},
    ]


def draw(rng):
    def spread(lo, hi):
        return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))

    kind = rng.choice(["topk", "loss", "grad", "train", "verify"])
    type_ = rng.choice(["bf16", "f16", "f32"])
    vocab = spread(1000, 131072)
    if rng.random() < 0.5:
        vocab = max(1000, vocab // 8 * 8)
    if kind == "verify":
        drafts = rng.randint(1, 16)
        most = 256 * 6 * 128256 * 4 // ((drafts + 1) * vocab * _BYTES[type_])
        return {"kind": kind, "batch": spread(1, max(1, min(256, most))), "drafts": drafts, "vocab": vocab, "type": type_, "draft_probs": rng.random() < 0.6}
    most = {"topk": 4096, "loss": 8192, "grad": 2048, "train": 2048}[kind] * 128256 * 2 // (vocab * _BYTES[type_])
    case = {"kind": kind, "rows": spread(1, max(1, min(8192, most))), "vocab": vocab, "k": spread(1, 256), "type": type_}
    if kind != "topk":
        case["temperature"] = rng.choice([0.7, 1.0, 1.5, 2.0, 4.0])
    return case


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def prepare(case, seed):
    g = _generator(seed)
    type_, vocab = _TYPES[case["type"]], case["vocab"]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    def uniform(*shape):
        return torch.rand(*shape, generator=g, device="cuda")

    def whole(lo, hi, *shape):
        return torch.randint(lo, hi, shape, generator=g, device="cuda")

    if case["kind"] == "topk":
        # a bulk of unlikely tokens; 16-bit logits tie often
        x = normal(case["rows"], vocab).mul_(2.5).to(type_)
        return {"case": case, "x": x}

    if case["kind"] == "verify":
        batch, drafts = case["batch"], case["drafts"]
        logits = normal(batch, drafts + 1, vocab).mul_(3.0)
        p = torch.softmax(logits, -1)
        if case["draft_probs"]:
            # a draft model near its target; its tokens are drawn from its own probabilities
            q = torch.softmax(logits[:, :drafts] + 0.35 * normal(batch, drafts, vocab), -1)
            race = q / -torch.log(uniform(batch, drafts, vocab).clamp_(1e-7, 1 - 1e-7))
            ids = race.argmax(-1)
            q = q.to(type_)
        else:
            # looked-up tokens: often the likeliest, else any
            q = None
            scaled = torch.softmax(2.0 * logits, -1)
            p = scaled
            ids = torch.where(uniform(batch, drafts) < 0.8, p[:, :drafts].argmax(-1), whole(0, vocab, batch, drafts))
        lens = torch.where(uniform(batch) < 0.75, torch.full((batch,), drafts, device="cuda"), whole(0, drafts + 1, batch))
        return {"case": case, "ids": ids, "p": p.to(type_), "q": q, "u": uniform(batch, drafts + 1), "lens": lens}

    rows, k = case["rows"], case["k"]
    # teacher: k distinct tokens a row with descending logits
    step = whole(1, max(2, vocab // k), rows, 1)
    ids = (whole(0, vocab, rows, 1) + step * torch.arange(k, device="cuda")) % vocab
    teacher = 14.0 - torch.cumsum(0.35 * -torch.log(uniform(rows, k).clamp_(1e-6, 1.0)), -1)
    # the student knows most of what the teacher does
    x = normal(rows, vocab).mul_(2.0)
    x.scatter_(1, ids, teacher + 0.7 * normal(rows, k))
    if vocab % 2:
        x[:, vocab - min(13, vocab // 4):] = -math.inf      # padded vocabulary
        ids = torch.where(ids < vocab - min(13, vocab // 4), ids, -1)
    # lists cut short, and padding tokens without a teacher
    held = torch.where(uniform(rows, 1) < 0.8, torch.full((rows, 1), k, device="cuda"), whole(1, k + 1, rows, 1))
    live = uniform(rows, 1) >= 0.04
    live[0] = True
    ids = torch.where((torch.arange(k, device="cuda") < held) & live, ids, -1)
    weight = (live / live.sum().clamp(min=1)).float().view(rows)
    if case["type"] == "f16":
        weight = weight * 1024.0                            # loss scaling
    return {"case": case, "x": x.to(type_), "teacher": teacher.to(type_), "ids": ids, "weight": weight}


# ------------------------------------------------------------------------------------- plain forms
def _order(x):
    """int32 keys whose order is that of float32 values (x has no NaN; -0 counts as 0)."""
    bits = (x + 0.0).view(torch.int32)
    return torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits)


def _topk(s):
    x, k = s["x"], s["case"]["k"]
    vocab = x.shape[-1]
    back = torch.arange(vocab - 1, -1, -1, device=x.device)
    keys = _order(x.float()).long() * 2 ** 32 + back          # distinct: ties go to the lowest index
    index = vocab - 1 - (torch.topk(keys, min(k, vocab), dim=-1).values & (2 ** 32 - 1))
    return {"values": torch.gather(x, -1, index), "indices": index}


def _distill(s, student=False, teacher=False):
    tau, vocab = s["case"]["temperature"], s["x"].shape[-1]
    z = s["x"].float() / tau
    e = torch.exp(z - z.amax(-1, keepdim=True))
    total = e.sum(-1, keepdim=True)
    held = (s["ids"] >= 0) & (s["ids"] < vocab)
    at = torch.where(held, s["ids"], 0)
    t = torch.where(held, s["teacher"].float() / tau, -math.inf)
    top = t.amax(-1, keepdim=True)
    live = top > -math.inf
    t = t - torch.where(live, top, 0.0)
    et = torch.exp(t)
    sum_t = et.sum(-1, keepdim=True)
    p = torch.where(live, et / sum_t, 0.0)
    log_q = torch.gather(z, -1, at) - z.amax(-1, keepdim=True) - torch.log(total)
    gap = torch.where(p > 0, t - torch.log(sum_t) - log_q, 0.0)
    kl = (p * gap).sum(-1, keepdim=True)
    out = {"loss": (tau * tau * kl).squeeze(-1)}
    by = s["weight"][:, None] * tau
    if student:
        d = torch.where(live, e / total, 0.0)
        d.scatter_add_(-1, at, -p)
        out["dlogits"] = (d * by).to(s["x"].dtype)
    if teacher:
        out["dteacher"] = (by * p * (gap - kl)).to(s["teacher"].dtype)
    return out


def _fixed(p):
    """Probabilities as whole multiples of 2^-36, clamped to [0, 1]."""
    return torch.round(torch.nan_to_num(p.double(), nan=0.0).clamp(0, 1) * GRID).long()


def _verify(s):
    ids, p, q, u = s["ids"], s["p"], s["q"], s["u"]
    batch, drafts = ids.shape
    vocab = p.shape[-1]
    place = torch.arange(drafts, device=ids.device)
    known = (ids >= 0) & (ids < vocab)
    at = torch.where(known, ids, 0)[..., None]
    pt = torch.gather(p[:, :drafts], -1, at)[..., 0].double()
    qt = torch.ones_like(pt) if q is None else torch.gather(q, -1, at)[..., 0].double()
    lens = s["lens"].clamp(0, drafts)
    ok = known & (u[:, :drafts].double() * qt < pt) & (place < lens[:, None])
    count = torch.cumprod(ok.long(), -1).sum(-1)
    row = torch.arange(batch, device=ids.device)
    base = _fixed(p[row, count])
    cut = count < lens                                        # a draft was turned down
    last = torch.clamp(count, max=drafts - 1)
    if q is None:
        out = torch.zeros_like(base).scatter_(-1, at[row, last], 1) > 0
        rest = torch.where(out & known[row, last][:, None], 0, base)
    else:
        rest = (base - _fixed(q[row, last])).clamp(min=0)
    rest = torch.where(cut[:, None] & (rest.sum(-1, keepdim=True) > 0), rest, base)
    run_ = torch.cumsum(rest, -1)
    sum_ = run_[:, -1]
    t = torch.floor(u[:, drafts].double().clamp(0, 1) * STEPS).long().clamp(max=STEPS - 1)
    mark = t * (sum_ // STEPS) + t * (sum_ % STEPS) // STEPS
    token = torch.where(sum_ > 0, (run_ <= mark[:, None]).sum(-1), -1)
    place = torch.arange(drafts + 1, device=ids.device)
    padded = torch.cat([ids, torch.full_like(ids[:, :1], -1)], -1)
    tokens = torch.where(place < count[:, None], padded, -1)
    return {"tokens": torch.where(place == count[:, None], token[:, None], tokens), "accepted": count}


def _plain(s):
    kind = s["case"]["kind"]
    if kind == "topk":
        return _topk(s)
    if kind == "verify":
        return _verify(s)
    return _distill(s, student=kind != "loss", teacher=kind == "train")


# ------------------------------------------------------------------------------------- torch_fl
def _package():
    if "torch_fl" not in sys.modules:
        sys.path.insert(0, os.path.join(os.getcwd(), "pytorch-plugin-fl_b200"))
    import torch_fl

    return torch_fl


def _calls(s):
    fl, case = _package(), s["case"]
    kind = case["kind"]
    if kind == "topk":
        values, indices = fl.ops.topk(s["x"], min(case["k"], s["x"].shape[-1]))
        return {"values": values, "indices": indices}
    if kind == "verify":
        tokens, accepted = fl.ops.verify_draft(s["ids"], s["p"], s["q"], s["u"], s["lens"])
        return {"tokens": tokens, "accepted": accepted}
    if kind == "loss":
        return {"loss": fl.ops.distill_topk(s["x"], s["teacher"], s["ids"], case["temperature"])}
    if kind == "grad":
        loss, dlogits = fl.ops.distill_topk_grad(s["x"], s["teacher"], s["ids"], case["temperature"], s["weight"])
        return {"loss": loss, "dlogits": dlogits}
    loss, stats = torch.ops.flagos.distill_topk(s["x"], s["teacher"], s["ids"], case["temperature"])
    dlogits, dteacher = torch.ops.flagos.distill_topk_backward(s["weight"], s["x"], stats, s["teacher"], s["ids"], case["temperature"], True, True)
    return {"loss": loss, "dlogits": dlogits, "dteacher": dteacher}


def run(state):
    if own:
        return _calls(state)
    return _plain(state)


# ------------------------------------------------------------------------------------- what it takes
def work(case):
    size, kind = _BYTES[case["type"]], case["kind"]
    vocab = case["vocab"]
    if kind == "verify":
        batch, drafts = case["batch"], case["drafts"]
        # one row of the target a sequence; the draft's too where a token was turned down (for the
        # drafts of prepare() about half the sequences); the drafted tokens' own entries
        row = vocab * (1.5 if case["draft_probs"] else 1.0)
        return {"bytes": int(batch * (row * size + drafts * (8 + 4 + 2 * size) + 8 * (drafts + 1) + 16)), "flops": int(batch * vocab * 4)}
    rows, k = case["rows"], min(case["k"], vocab)
    if kind == "topk":
        return {"bytes": rows * (vocab * size + k * (size + 8)), "flops": rows * vocab}
    taught = rows * case["k"] * (size + 8)
    if kind == "loss":
        return {"bytes": rows * (vocab * size + 4) + taught, "flops": rows * vocab * 4}
    more = rows * case["k"] * size if kind == "train" else 0
    return {"bytes": rows * (2 * vocab * size + 8) + taught + more, "flops": rows * vocab * 7}


# ------------------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    """What run() returns, from the definitions in 64 bits."""
    s = prepare(case, seed)
    if case["kind"] == "topk":
        values, indices = [], []
        for part in s["x"].split(256):
            wide = part.double()
            order = torch.sort(wide, dim=-1, descending=True, stable=True)
            values.append(order.values[:, : case["k"]])
            indices.append(order.indices[:, : case["k"]])
        return {"values": torch.cat(values), "indices": torch.cat(indices)}
    if case["kind"] == "verify":
        return _exact_verify(s)
    tau = case["temperature"]
    loss, dlogits, dteacher = [], [], []
    for r in range(0, case["rows"], 512):
        z = s["x"][r:r + 512].double() / tau
        ids, t, w = s["ids"][r:r + 512], s["teacher"][r:r + 512].double() / tau, s["weight"][r:r + 512, None].double()
        log_s = z - torch.logsumexp(z, -1, keepdim=True)
        held = ids >= 0
        some = held.any(-1, keepdim=True)
        t = t.masked_fill(~held, -math.inf)
        log_p = (t - torch.logsumexp(t, -1, keepdim=True)).masked_fill(~held, 0.0)
        p = torch.exp(log_p).masked_fill(~held, 0.0)
        apart = (log_p - torch.gather(log_s, -1, ids.clamp(min=0))).masked_fill(~held, 0.0)
        kl = (p * apart).sum(-1, keepdim=True)
        loss.append((tau ** 2 * kl)[:, 0])
        if case["kind"] == "loss":
            continue
        target = torch.zeros_like(z).scatter_add_(-1, ids.clamp(min=0), p)
        dlogits.append(torch.where(some, (torch.exp(log_s) - target) * tau * w, 0.0))
        dteacher.append(tau * w * p * (apart - kl))
    out = {"loss": torch.cat(loss)}
    if case["kind"] != "loss":
        out["dlogits"] = torch.cat(dlogits)
    if case["kind"] == "train":
        out["dteacher"] = torch.cat(dteacher)
    return out


def _exact_verify(s):
    ids, u, lens = s["ids"].cpu().numpy(), s["u"].cpu().numpy().astype(np.float64), s["lens"].cpu().numpy()
    batch, drafts = ids.shape
    tokens, accepted = np.full((batch, drafts + 1), -1, np.int64), np.zeros(batch, np.int64)
    for b in range(batch):
        n = 0
        while n < lens[b]:
            x = int(ids[b, n])
            p = float(s["p"][b, n, x])
            q = 1.0 if s["q"] is None else float(s["q"][b, n, x])
            if not u[b, n] * q < p:
                break
            tokens[b, n] = x
            n += 1
        accepted[b] = n
        p = np.rint(s["p"][b, n].cpu().double().numpy() * GRID).astype(np.int64)
        weights = p
        if n < lens[b]:
            if s["q"] is None:
                weights = p.copy()
                weights[ids[b, n]] = 0
            else:
                weights = np.maximum(p - np.rint(s["q"][b, n].cpu().double().numpy() * GRID).astype(np.int64), 0)
            if not weights.any():
                weights = p
        sums = np.cumsum(weights)
        mark = int(u[b, drafts] * STEPS) * int(sums[-1]) // STEPS
        tokens[b, n] = np.searchsorted(sums, mark, side="right")
    return {"tokens": torch.from_numpy(tokens), "accepted": torch.from_numpy(accepted)}
