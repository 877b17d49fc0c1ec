"""GPU: the head losses in use -- a distillation micro-step through the per-layer
entry points, scoring and training of one head together, against float64.

Tolerances of the micro-step are those of the training step it is a variant of
(bf16 products and attention against float64 autograd): loss 2e-3 relative,
gradients 3e-2 relative L2 per tensor.
"""
import functools

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from oracle import head_loss as oh  # noqa: E402
from oracle import model as om  # noqa: E402
from oracle import train as ot  # noqa: E402
from tests.test_gpu_train import GRAD_REL, LOSS_REL, _cfg, _compare_grads, _engine  # noqa: E402

pytestmark = pytest.mark.gpu


def _model(seed, B, S):
    cfg = _cfg(qk_norm=True, theta=1e6, eps=1e-6)
    layers, rf, emb, qk = om.init_weights(cfg, seed=seed, std=0.08, bf16=True)
    layers, rf, qk = om.random_gains(cfg, layers, rf, qk)
    tok = om.prompt_tokens(cfg.vocab, S + 1, seed + 1, batch=B)
    return cfg, (layers, rf, emb, qk), tok, _engine(cfg, layers, rf, emb, qk, B, S)


def _teacher(cfg, rows, K, seed):
    g = torch.Generator().manual_seed(seed)
    ids = torch.stack([torch.randperm(cfg.vocab, generator=g)[:K] for _ in range(rows)]).to(torch.int32)
    ids[torch.rand(rows, K, generator=g) < 0.2] = -1
    ids[3] = -1
    return ids, torch.randn(rows, K, generator=g) * 2


def _micro_step(e, cfg, tok, classifier):
    d_tok = torch.tensor(tok, dtype=torch.int32, device="cuda")
    d_loss = torch.zeros(1, device="cuda")
    torch.cuda.synchronize()
    e.embed_fwd(d_tok.data_ptr())
    for l in range(cfg.n_layers):
        e.attn_fwd(l)
        e.ffn_fwd(l)
    classifier(d_loss.data_ptr())
    for l in reversed(range(cfg.n_layers)):
        e.ffn_bwd(l)
        e.attn_bwd(l)
    e.embed_bwd()
    e.sync()
    return float(d_loss.item())


@pytest.mark.parametrize("hard", [0.0, 0.3])
@pytest.mark.parametrize("B,S", [(2, 64), (1, 320)])
def test_distillation_micro_step(hard, B, S):
    K, T = 24, 2.0
    cfg, w, tok, e = _model(71, B, S)
    ids, y = _teacher(cfg, B * S, K, 5)
    d_ids, d_y = ids.cuda(), y.cuda()
    e.head_alloc(B * S, cfg.dim, cfg.vocab, K)
    loss = _micro_step(e, cfg, tok, lambda p: e.lmhead_distill_fwd_bwd(
        d_ids.data_ptr(), d_y.data_ptr(), K, T, hard, p))
    fn = functools.partial(ot.distill_loss, ids=ids, teacher=y, temperature=T, hard=hard)
    ref, g = ot.loss_and_grads(cfg, *w, tok, loss_fn=fn)
    assert abs(loss - ref) <= LOSS_REL * ref, (loss, ref)
    _compare_grads(cfg, e.get_grads(), g)
    e.close()


def test_hard_targets_alone_are_the_cross_entropy_step():
    """hard_weight 1 without a teacher: the same step as ne_lmhead_ce_fwd_bwd, up to
    the bf16 rounding of its dz on both sides (2^-8 of each, summed in fp32)."""
    B, S = 2, 128
    cfg, _, tok, a = _model(81, B, S)
    _, _, _, b = _model(81, B, S)
    a.head_alloc(B * S, cfg.dim, cfg.vocab)
    la = _micro_step(a, cfg, tok, lambda p: a.lmhead_distill_fwd_bwd(hard_weight=1.0, d_loss=p))
    lb = _micro_step(b, cfg, tok, b.lmhead_ce_fwd_bwd)
    assert abs(la - lb) <= 2e-6 * lb, (la, lb)
    ga, gb = a.get_grads(), b.get_grads()
    for L in range(cfg.n_layers):
        for k in ga["layers"][L]:
            x, y = ga["layers"][L][k], gb["layers"][L][k]
            # the rounding of dz, and of every bf16 gradient after it
            assert np.linalg.norm(x - y) <= GRAD_REL / 2 * np.linalg.norm(y), (L, k)
    assert np.linalg.norm(ga["embed"] - gb["embed"]) <= GRAD_REL / 2 * np.linalg.norm(gb["embed"])
    a.close()
    b.close()


def test_accumulates_like_a_micro_step_and_leaves_the_loss_out_when_not_asked():
    B, S, K = 1, 64, 8
    cfg, _, tok, e = _model(91, B, S)
    ids, y = _teacher(cfg, B * S, K, 6)
    d_ids, d_y = ids.cuda(), y.cuda()
    e.head_alloc(B * S, cfg.dim, cfg.vocab, K)
    step = lambda p: e.lmhead_distill_fwd_bwd(d_ids.data_ptr(), d_y.data_ptr(), K, 1.0, 0.5, None)  # noqa: E731
    _micro_step(e, cfg, tok, step)
    one = e.get_grads()["embed"].copy()
    _micro_step(e, cfg, tok, step)
    two = e.get_grads()["embed"]
    # twice the gradient: fp32 adds, 2^-22 of the sum's size each, a few hundred of them
    assert np.linalg.norm(two - 2 * one) <= 1e-4 * np.linalg.norm(one)
    e.close()


def test_refusals():
    import neural_engine_b200 as ne
    cfg, _, tok, e = _model(95, 1, 64)
    d = torch.zeros(64, 4, dtype=torch.int32, device="cuda")
    y = torch.zeros(64, 4, device="cuda")

    def refused(status, *a, **k):
        with pytest.raises(ne.NeError) as err:
            e.lmhead_distill_fwd_bwd(*a, **k)
        assert err.value.status == status, err.value

    refused(8, d.data_ptr(), y.data_ptr(), 4)                 # no head_alloc
    e.head_alloc(63, cfg.dim, cfg.vocab, 4)
    refused(8, d.data_ptr(), y.data_ptr(), 4)                 # too few rows
    e.head_alloc(64, cfg.dim, cfg.vocab, 4)
    for h in (-0.1, 1.1, float("nan")):
        refused(1, d.data_ptr(), y.data_ptr(), 4, hard_weight=h)
    refused(1, hard_weight=0.5)                               # no teacher
    refused(1, d.data_ptr(), None, 4)
    refused(1, d.data_ptr(), y.data_ptr(), 0)
    refused(1, d.data_ptr(), y.data_ptr(), 4, temperature=0.0)
    refused(8, d.data_ptr(), y.data_ptr(), 5)
    e.train_set_vocab_map(np.arange(100))
    refused(8, d.data_ptr(), y.data_ptr(), 4)
    e.close()
    e = ne.Engine(ne.ModelConfig(1, 128, 256, 2, 2, 64, 256))
    refused(8, d.data_ptr(), y.data_ptr(), 4)                 # no training workspace
    e.close()


def test_scoring_and_both_losses_of_one_head():
    """What a distillation loop does with a head: cross entropy and distillation of
    the same batch, gradients of both in one fp32 dw, then the log-probability of
    one token at a time, which has to agree with the batch's."""
    import neural_engine_b200 as ne
    rows, dim, vocab, K, T = 333, 136, 1111, 9, 1.5
    e = ne.Engine(ne.ModelConfig(1, 128, 256, 2, 2, 64, 256))
    e.head_alloc(rows, dim, vocab, K)
    g = torch.Generator().manual_seed(3)
    x = torch.randn(rows, dim, generator=g).to(torch.bfloat16)
    w = (torch.randn(vocab, dim, generator=g) * 0.2).to(torch.bfloat16)
    tgt = torch.randint(0, vocab, (rows,), generator=g).to(torch.int32)
    tgt[::5] = -1
    ids = torch.randint(0, vocab, (rows, K), generator=g).to(torch.int32)
    ids[::7] = -1
    y = torch.randn(rows, K, generator=g)
    gc, gd = torch.rand(rows, generator=g), torch.rand(rows, generator=g)
    d = {k: v.cuda() for k, v in dict(x=x, w=w, tgt=tgt, ids=ids, y=y, gc=gc, gd=gd).items()}
    f = lambda *s: torch.zeros(*s, device="cuda")  # noqa: E731
    lc, ld, sc, sd, dw, dxc, dxd = f(rows), f(rows), f(rows), f(rows), f(vocab, dim), f(rows, dim), f(rows, dim)
    one_loss, one_lse = f(rows), f(rows)
    torch.cuda.synchronize()
    h = dict(x=d["x"].data_ptr(), w=d["w"].data_ptr(), rows=rows, dim=dim, vocab=vocab)
    kd = dict(ids=d["ids"].data_ptr(), teacher=d["y"].data_ptr(), topk=K, temperature=T)
    e.head_ce_fwd(**h, target=d["tgt"].data_ptr(), loss=lc.data_ptr(), lse=sc.data_ptr())
    e.head_distill_fwd(**h, **kd, loss=ld.data_ptr(), lse=sd.data_ptr())
    e.head_ce_bwd(**h, target=d["tgt"].data_ptr(), lse=sc.data_ptr(), grad=d["gc"].data_ptr(),
                  dx=dxc.data_ptr(), dw=dw.data_ptr(), dx_f32=True, dw_f32=True)
    e.head_distill_bwd(**h, **kd, lse=sd.data_ptr(), grad=d["gd"].data_ptr(), dx=dxd.data_ptr(),
                       dw=dw.data_ptr(), dx_f32=True, dw_f32=True)
    for i in range(0, rows, 29):
        e.head_ce_fwd(**dict(h, x=d["x"][i].data_ptr(), rows=1), target=d["tgt"][i:].data_ptr(),
                      loss=one_loss[i:].data_ptr(), lse=one_lse[i:].data_ptr())
    e.sync()
    tc = oh.ce_target(tgt, vocab)
    td = oh.distill_target(ids, y, vocab, T)
    wc = oh.head_loss(x, w, *tc, grad=gc)
    wd = oh.head_loss(x, w, *td, temperature=T, grad=gd)
    bc = oh.bounds(x, w, tc[0], tc[1], grad=gc)
    bd = oh.bounds(x, w, td[0], td[1], temperature=T, grad=gd)
    for got, ref, b in ((lc, wc[0], bc[0]), (ld, wd[0], bd[0]), (sc, wc[1], bc[1]), (sd, wd[1], bd[1])):
        assert float((got.cpu().double() - ref).abs().max()) <= b
    for got, ref, b in ((dxc, wc[2], bc[2]), (dxd, wd[2], bd[2]), (dw, wc[3] + wd[3], bc[3] + bd[3])):
        assert float(((got.cpu().double() - ref).abs() - b - 2.0 ** -22 * ref.abs() - 1e-30).max()) <= 0
    at = torch.arange(0, rows, 29)
    assert float((one_loss.cpu()[at].double() - wc[0][at]).abs().max()) <= bc[0]
    assert float((one_lse.cpu()[at].double() - wc[1][at]).abs().max()) <= bc[1]
    e.close()
