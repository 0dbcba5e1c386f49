"""The vocabulary-row operators without a GPU: the 64-bit oracle against
finite differences and by its own distribution, and the host-side refusals of
the C ABI (nothing here launches a kernel)."""

import os
import subprocess
import sys

import numpy as np
import pytest

from oracle import ops
from torch_fl import _abi

INVALID, DTYPE, MISALIGNED, TOO_LARGE = 1, 2, 3, 7


def _case(R=3, V=11, k=4, seed=0, repeat=False):
    g = np.random.default_rng(seed)
    z, t = 2 * g.standard_normal((R, V)), 2 * g.standard_normal((R, k))
    ids = np.stack([g.permutation(V)[:k] for _ in range(R)])
    if repeat:
        ids[0, 1] = ids[0, 0]
        ids[1, 2] = -1
    return z, t, ids


@pytest.mark.parametrize("tau", [0.7, 1.0, 3.0])
@pytest.mark.parametrize("repeat", [False, True])
def test_oracle_gradient_matches_differences(tau, repeat):
    z, t, ids = _case(repeat=repeat)
    w = np.array([1.0, 0.5, -2.0])
    _, dz, dt = ops.distill_topk_golden(z, t, ids, tau, w)
    h = 1e-5

    def total(zz, tt):
        return (w * ops.distill_topk_golden(zz, tt, ids, tau)[0]).sum()

    # central differences: error h^2 |f'''| / 6 < 1e-9 here, plus 2^-52 |f| / h
    for a, grad, first in ((z, dz, True), (t, dt, False)):
        for i in np.ndindex(a.shape):
            up, dn = a.copy(), a.copy()
            up[i] += h
            dn[i] -= h
            d = (total(up, t) - total(dn, t)) if first else (total(z, up) - total(z, dn))
            assert abs(d / (2 * h) - grad[i]) < 1e-8, (first, i)


def test_oracle_loss_is_zero_for_a_student_equal_to_a_full_teacher():
    z, _, _ = _case(R=2, V=6)
    ids = np.tile(np.arange(6), (2, 1))
    loss, dz, dt = ops.distill_topk_golden(z, z, ids, 1.3)
    assert np.all(np.abs(loss) < 1e-14) and np.all(np.abs(dz) < 1e-14) and np.all(np.abs(dt) < 1e-14)


def test_oracle_verification_samples_the_target():
    """Kept or redrawn, the first token is distributed as the target's: over a
    grid of uniform numbers each token's share is p within the grid's step."""
    p, q = np.array([0.5, 0.3, 0.2, 0.0]), np.array([0.2, 0.2, 0.5, 0.1])
    n = 200
    grid = (np.arange(n) + 0.5) / n
    share = np.zeros(4)
    for x in range(4):
        ids = np.full((n * n, 1), x)
        u = np.stack(np.meshgrid(grid, grid), -1).reshape(-1, 2)
        pp = np.broadcast_to(p, (n * n, 2, 4))
        tok, _ = ops.verify_draft_golden(ids, pp, np.broadcast_to(q, (n * n, 1, 4)), u)
        share += q[x] * np.bincount(tok[:, 0], minlength=4) / (n * n)
    assert np.all(np.abs(share - p) < 2.0 / n), share


def test_oracle_topk_order():
    x = np.array([[1.0, np.nan, 3.0, 3.0, -np.inf, np.inf, np.nan, -0.0, 0.0]])
    v, i = ops.topk_golden(x, 9)
    assert i.tolist() == [[1, 6, 5, 2, 3, 0, 7, 8, 4]]
    assert np.isnan(v[0, :2]).all() and v[0, 2] == np.inf and v[0, 8] == -np.inf


def _topk(x=16, ld=8, rows=2, cols=8, k=4, v=16, i=16, dtype=1):
    return lambda: _abi.call("fl_b200_topk_lastdim", x, ld, rows, cols, k, v, i, dtype, None)


def _fwd(x=16, ld=8, t=16, t_dtype=1, ids=16, ids_dtype=4, rows=2, cols=8, k=4, tau=1.0, loss=16,
         stats=16, dtype=1):
    return lambda: _abi.call("fl_b200_distill_topk_fwd", x, ld, t, 4, t_dtype, ids, 4, ids_dtype,
                             rows, cols, k, tau, loss, stats, dtype, None)


def _bwd(stride=1, x=32, ld_dx=8, tau=1.0, dtype=1, stats=16, t_dtype=1, k=4):
    return lambda: _abi.call("fl_b200_distill_topk_bwd", 16, stride, x, 8, stats, 16, 4, t_dtype, 16,
                             4, 4, 16, ld_dx, None, 2, 8, k, tau, dtype, None)


def _grad(dx=16, k=4, tau=1.0, ld_dx=8):
    return lambda: _abi.call("fl_b200_distill_topk_grad", 32, 8, 16, 4, 1, 16, 4, 4, None, 0, 2, 8, k,
                             tau, 16, 16, dx, ld_dx, 1, None)


def _verify(ids=16, p=16, u=16, batch=2, drafts=3, vocab=8, tokens=16, acc=16, dtype=0, stride=8):
    return lambda: _abi.call("fl_b200_verify_draft", ids, 3, p, 4 * stride, stride, None, 0, 0, u, 4,
                             None, batch, drafts, vocab, tokens, acc, dtype, None)


@pytest.mark.parametrize("call,status", [
    (_topk(k=9), INVALID), (_topk(k=-1), INVALID), (_topk(rows=-1), INVALID),
    (_topk(x=None), INVALID), (_topk(v=None), INVALID), (_topk(i=None), INVALID),
    (_topk(ld=7), INVALID), (_topk(dtype=3), DTYPE), (_topk(dtype=9), DTYPE),
    (_topk(cols=4096, ld=4096, k=1025), TOO_LARGE), (_topk(rows=1 << 31), TOO_LARGE),
    (_topk(cols=1 << 31, ld=1 << 31), TOO_LARGE),
    (lambda: _abi.call("fl_b200_topk_bwd", None, 16, 16, 2, 8, 4, 1, None), INVALID),
    (lambda: _abi.call("fl_b200_topk_bwd", 16, 16, 16, 2, 3, 4, 1, None), INVALID),
    (lambda: _abi.call("fl_b200_topk_bwd", 16, 16, 16, 2, 8, 4, 4, None), DTYPE),
    (_fwd(x=None), INVALID), (_fwd(t=None), INVALID), (_fwd(ids=None), INVALID),
    (_fwd(loss=None), INVALID), (_fwd(stats=None), INVALID), (_fwd(stats=20), MISALIGNED),
    (_fwd(tau=0.0), INVALID), (_fwd(tau=-1.0), INVALID), (_fwd(tau=float("nan")), INVALID),
    (_fwd(tau=float("inf")), INVALID), (_fwd(rows=-1), INVALID), (_fwd(cols=0, ld=0), INVALID),
    (_fwd(ld=7), INVALID), (_fwd(k=-1), INVALID), (_fwd(k=1025), TOO_LARGE),
    (_fwd(dtype=4), DTYPE), (_fwd(t_dtype=3), DTYPE), (_fwd(ids_dtype=0), DTYPE),
    (_bwd(stride=-1), INVALID), (_bwd(x=16), INVALID), (_bwd(ld_dx=7), INVALID), (_bwd(tau=0.0), INVALID),
    (_bwd(dtype=3), DTYPE), (_bwd(stats=None), INVALID), (_bwd(stats=12), MISALIGNED),
    (_bwd(t_dtype=4), DTYPE), (_bwd(k=1025), TOO_LARGE),
    (_grad(dx=None), INVALID), (_grad(k=1025), TOO_LARGE), (_grad(tau=-2.0), INVALID),
    (_grad(ld_dx=7), INVALID), (_grad(dx=32), INVALID), (_fwd(tau=1e-38), INVALID),
    (_verify(ids=None), INVALID), (_verify(p=None), INVALID), (_verify(u=None), INVALID),
    (_verify(tokens=None), INVALID), (_verify(acc=None), INVALID), (_verify(vocab=0), INVALID),
    (_verify(batch=-1), INVALID), (_verify(drafts=-1), INVALID), (_verify(dtype=4), DTYPE),
    (_verify(stride=-8), INVALID), (_verify(vocab=1 << 26), TOO_LARGE),
])
def test_bad_arguments_are_refused_on_the_host(call, status):
    with pytest.raises(_abi.FlB200Error) as e:
        call()
    assert e.value.status == status


def _apart(grad=True, **at):
    """A call over 4 rows of 8 bf16 logits, 2 teacher entries a row, each operand
    in a 4 KB page of its own but where `at` puts it."""
    names = ("logits", "teacher", "ids", "weight", "loss", "stats", "dlogits", "dteacher")
    p = {n: 0x100000 + 0x1000 * i for i, n in enumerate(names)} | at
    if grad:
        return lambda: _abi.call("fl_b200_distill_topk_grad", p["logits"], 8, p["teacher"], 2, 1, p["ids"], 2, 4,
                                 p["weight"], 1, 4, 8, 2, 1.0, p["loss"], p["stats"], p["dlogits"], 8, 1, None)
    return lambda: _abi.call("fl_b200_distill_topk_bwd", p["weight"], 1, p["logits"], 8, p["stats"], p["teacher"], 2,
                             1, p["ids"], 2, 4, p["dlogits"], 8, p["dteacher"], 4, 8, 2, 1.0, 1, None)


@pytest.mark.parametrize("call", [
    _apart(dlogits=0x100000), _apart(dlogits=0x100010), _apart(dlogits=0x100000 - 48), _apart(dlogits=0x10003e),
    _apart(dlogits=0x101000 - 60), _apart(dlogits=0x102030), _apart(dlogits=0x103008), _apart(dlogits=0x104000),
    _apart(dlogits=0x105010), _apart(loss=0x10000c), _apart(stats=0x102008), _apart(loss=0x103000),
    _apart(False, dlogits=0x100010), _apart(False, dlogits=0x100000 - 16), _apart(False, dlogits=0x101004),
    _apart(False, dteacher=0x101000), _apart(False, dteacher=0x10003e), _apart(False, dteacher=0x105004),
    _apart(False, dteacher=0x106020), _apart(False, dteacher=0x103000), _apart(False, dlogits=0x102000),
])
def test_results_that_overlap_an_operand_are_refused(call):
    """Rows are read and stored in no order: a result that shares memory with an
    operand, at whatever offset, is a race."""
    with pytest.raises(_abi.FlB200Error) as e:
        call()
    assert e.value.status == INVALID


def test_tensor_entry_points_refuse_before_they_launch():
    """K.*: shapes, types and CPU tensors are refused on the host."""
    import torch

    from torch_fl import kernels as K

    x, t, ids = torch.zeros(4, 100), torch.zeros(4, 3), torch.zeros(4, 3, dtype=torch.int64)
    p, u = torch.zeros(4, 4, 100), torch.zeros(4, 4)
    for bad in (lambda: K.topk_lastdim(x, 2), lambda: K.topk_backward(t, ids, 100),
                lambda: K.topk_backward(t, ids.int(), 100), lambda: K.distill_topk(x, t, ids),
                lambda: K.distill_topk(x, t, ids.float()), lambda: K.distill_topk(x, t[:3], ids[:3]),
                lambda: K.distill_topk_grad(x, t, ids, 1.0, out=x), lambda: K.verify_draft(ids, p, None, u),
                lambda: K.verify_draft(ids.int(), p, None, u), lambda: K.verify_draft(ids, p[:, :3], None, u),
                lambda: K.verify_draft(ids, p, p, u), lambda: K.verify_draft(ids, p, None, u[:, :2]),
                lambda: K.verify_draft(ids, p, None, u, ids[0])):
        with pytest.raises((RuntimeError, ValueError, TypeError)):
            bad()


def test_empty_work_is_a_no_op():
    _topk(rows=0, x=None, v=None, i=None)()
    _topk(k=0, v=None, i=None)()
    _fwd(rows=0, x=None, t=None, ids=None, loss=None, stats=None)()
    _verify(batch=0, ids=None, p=None, u=None, tokens=None, acc=None)()
    _abi.call("fl_b200_topk_bwd", None, None, None, 0, 8, 4, 1, None)
    _abi.call("fl_b200_distill_topk_bwd", None, 0, None, 0, None, None, 0, 1, None, 0, 4, None, 0, None,
              0, 8, 4, 1.0, 1, None)
    _abi.call("fl_b200_distill_topk_grad", None, 0, None, 0, 1, None, 0, 4, None, 0, 0, 8, 4, 1.0, None,
              None, None, 0, 1, None)


def test_the_wait_limit_is_clamped_and_comes_back():
    first = _abi.set_wait_limit(-5)
    assert first == 2_000_000_000
    assert _abi.set_wait_limit(1 << 40) == 0
    assert _abi.set_wait_limit(first) == 2_000_000_000


def test_a_message_with_numbers_is_an_error_not_a_crash():
    """Native checks whose message holds integers raise (in a child process:
    they once ended it)."""
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "pytorch-plugin-fl_b200")
    code = ("import torch_fl\nfrom torch_fl import _C\n"
            "try:\n    _C._set_device(99)\nexcept RuntimeError as e:\n    print('raised', e)\n")
    r = subprocess.run([sys.executable, "-c", code], env=dict(os.environ, PYTHONPATH=pkg),
                       capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "raised flagos: invalid device index 99" in r.stdout, (r.returncode, r.stdout, r.stderr[-300:])
