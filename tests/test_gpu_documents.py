"""The documents' examples that use the operators of a training step around the
matrix products, run as they stand there."""

import os
import re

import pytest
import torch

import torch_fl
from torch_fl import kernels as K

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def example(name):
    with open(os.path.join(ROOT, name)) as f:
        blocks = re.findall(r"```python\n(.*?)```", f.read(), re.S)
    (block,) = [b for b in blocks if "rope_frequencies" in b]
    # (patches transformers for the whole process)
    return "\n".join(line for line in block.splitlines() if "enable_hf_fused_ops" not in line)


def hands(dev, dtype=torch.bfloat16):
    """What a program has in hand before the examples' lines."""
    g = torch.Generator().manual_seed(1)
    B, S, H, D, hidden, V = 2, 24, 4, 128, 256, 1000
    r = lambda *s: torch.randn(*s, generator=g).to(dtype).to(dev)
    p = lambda *s: torch.softmax(torch.randn(*s, generator=g), -1).to(dev)
    model = torch.nn.Linear(8, 8).to(dev)
    for t in model.parameters():
        t.grad = torch.ones_like(t)
    docs = torch.sort(torch.randint(0, 3, (B, S), generator=g), -1).values.to(dev)
    return dict(torch=torch, torch_fl=torch_fl, K=K, B=B, S=S, D=D, q=r(B, S, H, D), k=r(B, S, 1, D),
                positions=torch.arange(S).to(dev), doc_ids=docs, lens=torch.tensor([S, S - 5]).to(dev),
                scores=r(B, H, S, S), attn_out=r(B, S, hidden), attn=r(B, S, hidden), h=r(B, S, hidden),
                post_w=r(hidden), pre_w=r(hidden), post=r(hidden), pre=r(hidden), gate=r(B, 1, hidden), model=model,
                grads=[r(30, 7), r(5)], teacher_logits=r(6, V), student_logits=r(6, V),
                draft_ids=torch.randint(0, V, (B, 3), generator=g).to(dev), p_draft=p(B, 3, V), p_target=p(B, 4, V),
                uniform=torch.rand(B, 4, generator=g).to(dev))


def test_readme():
    n = hands("flagos")
    before = n["q"].clone()
    exec(example("README.md"), n)
    assert n["q"].shape == before.shape and not torch.equal(n["q"], before)
    assert n["w"].shape == n["scores"].shape and n["spans"].shape == (2, 24, 2)
    assert n["y"].shape == n["h"].shape == n["attn_out"].shape
    assert abs(float(n["norm"]) - 72 ** 0.5) < 1e-5


def test_integration():
    n = hands("cuda")
    before, heads = n["q"].clone(), n["q"]
    exec(example("INTEGRATION.md"), n)
    assert n["q"] is heads and torch.equal(heads[..., 64:], before[..., 64:]) and not torch.equal(heads, before)
    assert n["w"].shape == n["scores"].shape and n["y"].shape == n["attn"].shape
    assert n["clipped"][0] is n["grads"][0] and float(n["norm"]) > 1
