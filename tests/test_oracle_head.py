"""CPU: the float64 definition of the head losses (oracle/head_loss.py) against
autograd, against differences, and at rows that do not count."""
import math

import pytest
import torch

from oracle import head_loss as oh


def _case(rows=5, dim=6, vocab=11, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, dim, generator=g, dtype=torch.float64)
    w = torch.randn(vocab, dim, generator=g, dtype=torch.float64)
    return g, x, w


def _targets(op, g, rows, vocab, T):
    if op == "ce":
        t = torch.randint(0, vocab, (rows,), generator=g)
        t[1] = -100
        return oh.ce_target(t, vocab)
    ids = torch.randint(0, vocab, (rows, 4), generator=g)
    ids[0, 1] = ids[0, 0]         # the same id twice
    ids[1] = -1                   # no entry
    ids[2, 3] = -1
    y = torch.randn(rows, 4, generator=g, dtype=torch.float64) * 3
    y[3, 0] = -math.inf
    return oh.distill_target(ids, y, vocab, T)


@pytest.mark.parametrize("op,T", [("ce", 1.0), ("distill", 1.0), ("distill", 2.5)])
def test_gradients_are_those_of_autograd_and_of_differences(op, T):
    g, x, w = _case()
    keep, p, plogp = _targets(op, g, 5, 11, T)
    grad = torch.rand(5, generator=g, dtype=torch.float64) + 0.5
    loss, lse, dx, dw = oh.head_loss(x, w, keep, p, plogp, 0.7, T, grad)
    xa, wa = x.clone().requires_grad_(), w.clone().requires_grad_()
    logq = torch.log_softmax(0.7 / T * (xa @ wa.T), 1)
    want = T * T * (plogp - (p * logq).sum(1)) * keep
    torch.testing.assert_close(loss, want.detach(), rtol=0, atol=1e-12)
    (want * grad).sum().backward()
    torch.testing.assert_close(dx, xa.grad, rtol=0, atol=1e-12)
    torch.testing.assert_close(dw, wa.grad, rtol=0, atol=1e-12)
    h = 1e-5
    for t, d in ((x, dx), (w, dw)):
        for at in ((0, 0), (2, 3), (4, 5)):
            v = float(t[at])
            t[at] = v + h
            up = (oh.head_loss(x, w, keep, p, plogp, 0.7, T)[0] * grad).sum()
            t[at] = v - h
            dn = (oh.head_loss(x, w, keep, p, plogp, 0.7, T)[0] * grad).sum()
            t[at] = v
            # differences of a smooth function: h^2 and rounding / h
            assert abs(float(up - dn) / (2 * h) - float(d[at])) < 1e-8


def test_rows_that_do_not_count():
    g, x, w = _case()
    x[1] = math.nan
    for op in ("ce", "distill"):
        keep, p, plogp = _targets(op, g, 5, 11, 1.0)
        out = oh.head_loss(x, w, keep, p, plogp)
        assert not bool(keep[1]) and all(bool(torch.isfinite(o).all()) for o in out)
        assert float(out[0][1]) == 0.0 and float(out[1][1]) == 0.0 and float(out[2][1].abs().sum()) == 0.0


def test_distillation_of_one_entry_is_cross_entropy():
    g, x, w = _case()
    t = torch.randint(0, 11, (5,), generator=g)
    a = oh.head_loss(x, w, *oh.ce_target(t, 11))
    b = oh.head_loss(x, w, *oh.distill_target(t[:, None], torch.zeros(5, 1), 11, 1.0))
    for u, v in zip(a, b):
        torch.testing.assert_close(u, v, rtol=0, atol=1e-12)


def test_a_student_like_its_teacher_has_no_loss():
    """With every id an entry and the teacher's logits the student's own, the
    divergence is zero and so are the gradients."""
    g, x, w = _case()
    T = 3.0
    z = x @ w.T
    ids = torch.arange(11).repeat(5, 1)
    loss, _, dx, dw = oh.head_loss(x, w, *oh.distill_target(ids, z, 11, T), 1.0, T)
    for v in (loss, dx, dw):
        assert float(v.abs().max()) < 1e-12


def test_null_context_is_refused_before_anything_else():
    import neural_engine_b200 as ne
    lib = ne.load_library()
    assert lib.ne_head_alloc(None, 1, 8, 8, 0) == 1
    assert lib.ne_head_ce_fwd(None, None, None, None, None) == 1
    assert lib.ne_head_ce_bwd(None, None, None, None, None, None) == 1
    assert lib.ne_head_distill_fwd(None, None, None, None, None) == 1
    assert lib.ne_head_distill_bwd(None, None, None, None, None, None) == 1
    assert lib.ne_lmhead_distill_fwd_bwd(None, None, 0.0, None) == 8
