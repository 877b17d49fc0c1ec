"""GPU: the head losses (ne_head_ce_*, ne_head_distill_*) against their float64
definition (oracle/head_loss.py).

Tolerances are oracle.head_loss.bounds, entry by entry, worked out there from
the steps that round; bf16 outputs add half a step, 2^-8 of their size.
"""
import math

import pytest

torch = pytest.importorskip("torch")

from oracle import head_loss as oh  # noqa: E402

pytestmark = pytest.mark.gpu

NAN = float("nan")


@pytest.fixture(scope="module")
def eng():
    import neural_engine_b200 as ne
    e = ne.Engine(ne.ModelConfig(1, 128, 256, 2, 2, 64, 256))
    yield e
    e.close()


class Head:
    """One call's inputs on both sides; pad: extra columns behind every row."""

    def __init__(self, rows, dim, vocab, seed=0, pad=0, scale=1.0, spread=2.0):
        self.g = g = torch.Generator().manual_seed(seed)
        self.rows, self.dim, self.vocab, self.pad, self.scale = rows, dim, vocab, pad, scale
        self.x = torch.randn(rows, dim, generator=g).to(torch.bfloat16)
        self.w = (torch.randn(vocab, dim, generator=g) * (spread / math.sqrt(dim))).to(torch.bfloat16)
        self.grad = torch.rand(rows, generator=g) - 0.25
        self.T = 1.0

    def ce(self, masked=0.0):
        self.target = torch.randint(0, self.vocab, (self.rows,), generator=self.g).to(torch.int32)
        out = torch.rand(self.rows, generator=self.g) < masked
        self.target[out] = -100
        self.fwd, self.bwd, self.topk = "head_ce_fwd", "head_ce_bwd", 0
        self.args = lambda: dict(target=self.d_target.data_ptr())
        return self

    def distill(self, K, T=1.0, ragged=True, masked=0.0):
        g = self.g
        self.T, self.topk = T, K
        self.ids = torch.randint(0, self.vocab, (self.rows, K), generator=g).to(torch.int32)
        self.teacher = torch.randn(self.rows, K, generator=g) * 3
        if ragged:
            self.ids[torch.rand(self.rows, K, generator=g) < 0.3] = -1
        self.ids[torch.rand(self.rows, generator=g) < masked] = -1
        self.fwd, self.bwd = "head_distill_fwd", "head_distill_bwd"
        self.args = lambda: dict(ids=self.d_ids.data_ptr(), teacher=self.d_teacher.data_ptr(),
                                 topk=K, temperature=T)
        return self

    def targets(self):
        if self.topk:
            return oh.distill_target(self.ids, self.teacher, self.vocab, self.T)
        return oh.ce_target(self.target, self.vocab)

    def _wide(self, t, fill):
        w = torch.full((t.shape[0], self.dim + self.pad), fill, dtype=t.dtype)
        w[:, :self.dim] = t
        return w.cuda()

    def upload(self):
        self.d_x, self.d_w = self._wide(self.x, NAN), self._wide(self.w, NAN)
        if self.topk:
            self.d_ids, self.d_teacher = self.ids.cuda(), self.teacher.cuda()
        else:
            self.d_target = self.target.cuda()
        self.d_grad = self.grad.cuda()
        n = self.rows + 3   # rows behind the last one stay as they are
        self.loss, self.lse = (torch.full((n,), 7.0, device="cuda") for _ in range(2))
        ld = self.dim + self.pad
        self.dx = torch.full((n, ld), 7.0, dtype=torch.bfloat16, device="cuda")
        self.dw = torch.full((self.vocab + 3, ld), 7.0, dtype=torch.bfloat16, device="cuda")
        self.dx32 = torch.full((n, ld), 7.0, device="cuda")
        self.dw32 = torch.full((self.vocab + 3, ld), 7.0, device="cuda")
        torch.cuda.synchronize()

    def head(self):
        ld = self.dim + self.pad
        return dict(x=self.d_x.data_ptr(), w=self.d_w.data_ptr(), rows=self.rows, dim=self.dim,
                    vocab=self.vocab, scale=self.scale, ldx=ld, ldw=ld)

    def forward(self, e):
        getattr(e, self.fwd)(**self.head(), **self.args(), loss=self.loss.data_ptr(),
                             lse=self.lse.data_ptr())

    def backward(self, e, f32=False, dx=True, dw=True, grad=True):
        ld = self.dim + self.pad
        a, b = (self.dx32, self.dw32) if f32 else (self.dx, self.dw)
        getattr(e, self.bwd)(**self.head(), **self.args(), lse=self.lse.data_ptr(),
                             grad=self.d_grad.data_ptr() if grad else None,
                             dx=a.data_ptr() if dx else None, dw=b.data_ptr() if dw else None,
                             lddx=ld, lddw=ld, dx_f32=f32, dw_f32=f32)

    def run(self, e):
        self.upload()
        e.head_alloc(self.rows, self.dim, self.vocab, self.topk)
        self.forward(e)
        self.backward(e)
        self.backward(e, f32=True)
        e.sync()
        return self

    def check(self):
        keep, p, plogp = self.targets()
        k = dict(scale=self.scale, temperature=self.T, grad=self.grad)
        want = oh.head_loss(self.x, self.w, keep, p, plogp, **k)
        # with up to 64 rows that count dz is kept in two bf16 parts
        tol = oh.bounds(self.x, self.w, keep, p, **k, dz_step=2.0 ** (-16 if int(keep.sum()) <= 64 else -8))
        R, V, D = self.rows, self.vocab, self.dim
        for name, got, ref, b in (("loss", self.loss, want[0], tol[0]), ("lse", self.lse, want[1], tol[1])):
            got = got.cpu().double()
            assert bool((got[R:] == 7.0).all()), f"{name}: behind the last row"
            assert bool((got[:R][~keep] == 0.0).all()), f"{name}: left-out rows"
            err = float((got[:R] - ref).abs().max())
            assert err <= b, f"{name}: {err:.3e} > {b:.3e}"
        for name, got, n, ref, b, base, half in (
                ("dx", self.dx, R, want[2], tol[2], 0.0, 2.0 ** -8),
                ("dw", self.dw, V, want[3], tol[3], 0.0, 2.0 ** -8),
                ("dx32", self.dx32, R, want[2], tol[2], 0.0, 2.0 ** -23),
                ("dw32", self.dw32, V, want[3], tol[3], 7.0, 2.0 ** -22)):   # added to sevens
            got = got.cpu().double()
            assert bool((got[n:] == 7.0).all()) and bool((got[:, D:] == 7.0).all()), f"{name}: outside"
            ref = ref + base
            over = (got[:n, :D] - ref).abs() - (b + half * (ref.abs() + b) + 1e-30)
            assert bool(torch.isfinite(got[:n, :D]).all()) and float(over.max()) <= 0, \
                f"{name}: {float(over.max()):.3e} over, worst of {float((got[:n, :D] - ref).abs().max()):.3e}"
        assert bool((self.dx[:R].cpu()[~keep][:, :D] == 0).all())


SIZES = [(1, 8, 1), (1, 64, 37), (2, 768, 1000), (7, 72, 257), (64, 128, 64), (65, 64, 300),
         (128, 136, 511), (129, 64, 513), (200, 264, 1023), (511, 72, 777), (512, 64, 512),
         (513, 80, 2049), (700, 520, 1300)]


@pytest.mark.parametrize("rows,dim,vocab", SIZES)
def test_cross_entropy(eng, rows, dim, vocab):
    Head(rows, dim, vocab, seed=rows + vocab).ce().run(eng).check()


@pytest.mark.parametrize("rows,dim,vocab", SIZES)
@pytest.mark.parametrize("K,T", [(1, 1.0), (13, 2.0), (70, 0.5)])
def test_distillation(eng, rows, dim, vocab, K, T):
    Head(rows, dim, vocab, seed=rows + vocab + K).distill(K, T).run(eng).check()


@pytest.mark.parametrize("masked", [0.1, 0.5, 0.95, 1.0])
@pytest.mark.parametrize("rows", [1, 33, 128, 130, 600])
def test_left_out_rows_reach_nothing(eng, rows, masked):
    """Masked rows of every share, all of them among it, hold NaN and infinity."""
    for h in (Head(rows, 64, 333, seed=rows).ce(masked), Head(rows, 64, 333, seed=rows).distill(5, 1.5, masked=masked)):
        keep = h.targets()[0]
        bad = torch.nonzero(~keep)[:, 0]
        h.x[bad[::2]] = NAN
        h.x[bad[1::2]] = math.inf
        h.grad[bad] = NAN
        h.run(eng)
        h.grad[bad] = 0.0
        h.check()


def test_exactly_64_and_128_rows_count(eng):
    """The packed rows end at a block's edge: nothing stale is summed into dw."""
    for n in (64, 128, 256):
        h = Head(300, 64, 300, seed=n).ce()
        h.target[n:] = -1
        Head(300, 64, 300, seed=1, spread=50.0).ce().run(eng)   # leaves large values in the workspace
        h.run(eng).check()


@pytest.mark.parametrize("pad,scale", [(8, 1.0), (40, 0.25), (0, 3.0)])
def test_strides_and_scale(eng, pad, scale):
    Head(150, 72, 700, seed=pad, pad=pad, scale=scale).ce(0.2).run(eng).check()
    Head(9, 72, 700, seed=pad, pad=pad, scale=scale).distill(9, 2.0).run(eng).check()


def test_large_logits(eng):
    """Logits in the thousands, of both signs: the running maximum carries them."""
    for s in (1, 200):
        Head(s, 256, 1500, seed=3, spread=600.0).ce().run(eng).check()
    h = Head(200, 256, 1500, seed=4, spread=600.0).ce()
    h.x = -h.x.abs()
    h.w = h.w.abs()
    h.run(eng).check()


@pytest.mark.parametrize("rows", [3, 200, 600])
def test_long_sums(eng, rows):
    """Dims beyond 2048, whole and not in the lengths the sum is taken in: the
    bound's term per column is held to 1536 of them there."""
    for dim in (2056, 4096):
        h = Head(rows, dim, 520, seed=dim).ce(0.1).run(eng)
        h.check()
        keep, p, plogp = h.targets()
        want = oh.head_loss(h.x, h.w, keep, p, plogp)
        # 4.8e-10 a column of 1536, and of the other roundings 2^-22 each of the
        # logits' sum, its logarithm and the change of base
        size = float(want[1].abs().max())
        assert float((h.lse[:rows].cpu().double() - want[1]).abs().max()) <= (1536 * 4.8e-10 + 3 * 2.0 ** -22) * size


@pytest.mark.parametrize("rows", [128, 300])
@pytest.mark.parametrize("dim", [512, 2048, 4096])
def test_no_bias_from_accumulating(eng, rows, dim):
    """With one id lse is the logit.  An accumulator that truncates loses half a
    step of its partial sum in each of dim / 16 additions: of an evenly growing
    sum ln 2 / 32 * 2^-24 per column (of at most 2048 columns, longer sums are
    split).  On average less than half of that may be missing or added."""
    g = torch.Generator().manual_seed(20 + dim)
    w = torch.randn(1, dim, generator=g).to(torch.bfloat16)
    x = (0.3 * w.float() + torch.randn(rows, dim, generator=g)).to(torch.bfloat16)
    z = (x.double() @ w.double().T)[:, 0]
    d_x, d_w, t = x.cuda(), w.cuda(), torch.zeros(rows, dtype=torch.int32, device="cuda")
    loss, lse = torch.empty(2, rows, device="cuda")
    torch.cuda.synchronize()
    eng.head_alloc(rows, dim, 1)
    eng.head_ce_fwd(x=d_x.data_ptr(), w=d_w.data_ptr(), rows=rows, dim=dim, vocab=1, target=t.data_ptr(),
                    loss=loss.data_ptr(), lse=lse.data_ptr())
    eng.sync()
    slope = float(((lse.cpu().double() - z) * z).sum() / (z * z).sum())
    assert abs(slope) < 0.5 * math.log(2) / 32 * 2.0 ** -24 * min(dim, 2048)


def test_teacher_entries(eng):
    """Repeats, -inf, ids in any order, NaN and infinity behind absent ids, 256 entries."""
    h = Head(6, 64, 90, seed=5).distill(256, 1.0, ragged=False)
    h.ids[1, :] = 17                          # one id, 256 times
    h.teacher[2, ::2] = -math.inf
    h.ids[3, 1:] = -1
    h.teacher[3, 1::2], h.teacher[3, 2::2] = NAN, math.inf
    h.teacher[4, :] = -math.inf               # no entry at all
    h.ids[5] = torch.arange(256).flip(0) % 90
    h.teacher[5] *= 40                        # probabilities that underflow
    h.run(eng).check()


@pytest.mark.parametrize("f32", [False, True])
def test_one_gradient_alone(eng, f32):
    h = Head(140, 64, 600, seed=6).ce(0.3)
    h.run(eng)
    both = [t.clone() for t in ((h.dx32, h.dw32) if f32 else (h.dx, h.dw))]
    for k in range(2):
        h.upload()
        h.forward(eng)
        h.backward(eng, f32=f32, dx=k == 0, dw=k == 1)
        eng.sync()
        got = (h.dx32, h.dw32) if f32 else (h.dx, h.dw)
        assert torch.equal(got[k], both[k])
        assert bool((got[1 - k] == 7.0).all())


def test_ones_where_no_row_gradient_is_given(eng):
    h = Head(40, 64, 100, seed=7).ce()
    h.upload()
    eng.head_alloc(40, 64, 100)
    h.forward(eng)
    h.backward(eng, grad=False)
    h.backward(eng, grad=False, f32=True)
    eng.sync()
    h.grad = torch.ones(40)
    h.check()


def test_several_pieces_of_the_vocabulary(eng):
    """Rows and ids enough that dz does not fit one piece."""
    h = Head(2000, 64, 20001, seed=8, scale=0.5).ce(0.4)
    h.run(eng)
    keep, p, plogp = h.targets()
    k = dict(scale=0.5, grad=h.grad)
    loss, lse, dx, dw = oh.head_loss(h.x, h.w, keep, p, plogp, **k)
    tol = oh.bounds(h.x, h.w, keep, p, **k)
    for got, ref, b, half in ((h.loss[:2000], loss, tol[0], 0), (h.lse[:2000], lse, tol[1], 0),
                              (h.dx[:2000], dx, tol[2], 2.0 ** -8), (h.dw[:20001], dw, tol[3], 2.0 ** -8)):
        over = (got.cpu().double() - ref).abs() - (b + half * (ref.abs() + b))
        assert float(over.max()) <= 0


@pytest.mark.parametrize("rows", [8192, 8193, 20011])
def test_many_rows(eng, rows):
    """Rows beyond 8192 are packed several groups a block."""
    h = Head(rows, 64, 130, seed=rows).ce(0.5)
    h.target[5000:7500] = -7          # whole groups without a row that counts
    h.run(eng).check()
    Head(rows, 64, 130, seed=rows).distill(3, masked=0.6).run(eng).check()


def test_two_contexts_at_once():
    """Two contexts' passes enqueued on their streams together: neither's units
    wait for CTAs that the other keeps off the SMs."""
    import neural_engine_b200 as ne
    es = [ne.Engine(ne.ModelConfig(1, 128, 256, 2, 2, 64, 256)) for _ in range(2)]
    hs = [Head(1500, 136, 9001, seed=21).ce(0.2), Head(700, 264, 12000, seed=22).distill(11, 2.0)]
    for e, h in zip(es, hs):
        h.upload()
        e.head_alloc(h.rows, h.dim, h.vocab, h.topk)
    for _ in range(8):
        for e, h in zip(es, hs):
            h.forward(e)
            h.backward(e)
    for e in es:
        e.sync()
    got = [[t.clone() for t in (h.loss, h.lse, h.dx, h.dw)] for h in hs]
    for e, h, a in zip(es, hs, got):
        h.upload()
        h.forward(e)
        h.backward(e)
        e.sync()
        for u, v in zip(a, (h.loss, h.lse, h.dx, h.dw)):
            assert torch.equal(u, v)
        e.close()


def test_the_same_bits_every_time(eng):
    for h in (Head(700, 136, 3001, seed=9).ce(0.3), Head(700, 136, 3001, seed=9).distill(20, 2.0)):
        h.run(eng)
        a = [t.clone() for t in (h.loss, h.lse, h.dx, h.dw, h.dx32, h.dw32)]
        h.run(eng)
        for u, v in zip(a, (h.loss, h.lse, h.dx, h.dw, h.dx32, h.dw32)):
            assert torch.equal(u, v)


def test_no_rows(eng):
    h = Head(1, 64, 50, seed=10).ce()
    h.upload()
    h.rows = 0
    h.forward(eng)
    h.backward(eng)
    h.backward(eng, f32=True)
    eng.sync()
    assert bool((h.loss == 7.0).all()) and bool((h.dx == 7.0).all()) and bool((h.dw32 == 7.0).all())
    assert bool((h.dw[:50] == 0.0).all()) and bool((h.dw[50:] == 7.0).all())


def test_empty_arrays_have_no_address(eng):
    """With rows 0 the arrays of rows are NULL; dw of no rows is still written."""
    eng.head_alloc(1, 64, 50, 4)
    w = torch.zeros(50, 64, dtype=torch.bfloat16, device="cuda")
    dw = torch.full((50, 64), 7.0, dtype=torch.bfloat16, device="cuda")
    x = torch.empty(0, 64, dtype=torch.bfloat16, device="cuda")
    t = torch.empty(0, 4, dtype=torch.int32, device="cuda")
    f = torch.empty(0, device="cuda")
    assert x.data_ptr() == t.data_ptr() == f.data_ptr() == 0
    torch.cuda.synchronize()
    head = dict(x=x.data_ptr(), w=w.data_ptr(), rows=0, dim=64, vocab=50)
    kd = dict(head, ids=t.data_ptr(), teacher=f.data_ptr(), topk=4, lse=f.data_ptr())
    eng.head_ce_fwd(**head, target=t.data_ptr(), loss=f.data_ptr(), lse=f.data_ptr())
    eng.head_distill_fwd(**kd, loss=f.data_ptr())
    eng.head_ce_bwd(**head, target=t.data_ptr(), lse=f.data_ptr(), dx=x.data_ptr())
    eng.head_distill_bwd(**kd, grad=f.data_ptr(), dx=x.data_ptr())
    eng.sync()
    assert bool((dw == 7.0).all())
    eng.head_ce_bwd(**head, target=t.data_ptr(), lse=f.data_ptr(), dx=x.data_ptr(), dw=dw.data_ptr())
    eng.sync()
    assert bool((dw == 0.0).all())


def test_captured_and_replayed(eng):
    """Two graphs that share the context's workspaces, replayed in turn with new
    inputs, give what eager calls give."""
    hs = [Head(300, 64, 1000, seed=11).ce(0.5), Head(20, 64, 700, seed=12).distill(12, 2.0)]
    eng.head_alloc(300, 64, 1000, 12)
    st = torch.cuda.ExternalStream(eng.stream_ptr)
    graphs = []
    for h in hs:
        h.upload()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            h.forward(eng)
            h.backward(eng)
        graphs.append(g)
    for h in hs:   # other values in the same buffers
        h.x = torch.randn(h.rows, h.dim, generator=h.g).to(torch.bfloat16)
        h.d_x.copy_(h.x)
    hs[0].target = hs[0].target.flip(0).contiguous()
    hs[0].d_target.copy_(hs[0].target)
    torch.cuda.synchronize()
    for _ in range(2):
        for g in graphs:
            with torch.cuda.stream(st):
                g.replay()
    eng.sync()
    got = [[t.clone() for t in (h.loss, h.lse, h.dx, h.dw)] for h in hs]
    for h, a in zip(hs, got):
        h.run(eng).check()
        for u, v in zip(a, (h.loss, h.lse, h.dx, h.dw)):
            assert torch.equal(u, v)


def test_ids_past_the_vocabulary_are_absent_and_reported():
    import neural_engine_b200 as ne
    for op in ("ce", "distill"):
        for rows in (5, 200):
            e = ne.Engine(ne.ModelConfig(1, 128, 256, 2, 2, 64, 256))
            h = Head(rows, 64, 100, seed=13)
            h = h.ce() if op == "ce" else h.distill(3, ragged=False)
            if op == "ce":
                h.target[3] = 100
            else:
                h.ids[3, 1] = 2 ** 31 - 1
            with pytest.raises(ne.NeError) as err:
                h.run(e)
            assert err.value.status == 9
            h.check()
            e.close()


def test_refusals():
    import neural_engine_b200 as ne
    eng = ne.Engine(ne.ModelConfig(1, 128, 256, 2, 2, 64, 256))
    h = Head(4, 64, 100, seed=14).ce()
    h.upload()
    eng.head_alloc(4, 64, 100, 4)
    t = torch.zeros(4, 4, dtype=torch.int32, device="cuda")
    y = torch.zeros(4, 4, device="cuda")
    ok = dict(h.head(), target=h.d_target.data_ptr(), loss=h.loss.data_ptr(), lse=h.lse.data_ptr())
    back = {k: v for k, v in ok.items() if k != "loss"} | dict(dx=h.dx.data_ptr(), dw=h.dw.data_ptr())
    kd = {k: v for k, v in ok.items() if k != "target"} | dict(
        ids=t.data_ptr(), teacher=y.data_ptr(), topk=4, temperature=1.0)
    kdb = {k: v for k, v in kd.items() if k != "loss"} | dict(dx=h.dx.data_ptr(), dw=h.dw.data_ptr())

    def refused(status, fn, base, **kw):
        with pytest.raises(ne.NeError) as err:
            fn(**dict(base, **kw))
        assert err.value.status == status, err.value

    for fn, base in ((eng.head_ce_fwd, ok), (eng.head_ce_bwd, back), (eng.head_distill_fwd, kd),
                     (eng.head_distill_bwd, kdb)):
        for kw in (dict(x=None), dict(w=None), dict(lse=None), dict(rows=-1), dict(dim=0), dict(vocab=0),
                   dict(ldx=56), dict(ldw=68), dict(x=h.d_x.data_ptr() + 2), dict(w=h.d_w.data_ptr() + 8),
                   dict(scale=0.0), dict(scale=-1.0), dict(scale=NAN), dict(scale=math.inf)):
            refused(1, fn, base, **kw)
        refused(7, fn, base, dim=60, ldx=64, ldw=64)
        for kw in (dict(rows=2 ** 30), dict(vocab=2 ** 30), dict(dim=2 ** 20, ldx=2 ** 20, ldw=2 ** 20)):
            refused(8, fn, base, **kw)
    for kw in (dict(target=None), dict(loss=None)):
        refused(1, eng.head_ce_fwd, ok, **kw)
    for fn, base in ((eng.head_ce_bwd, back), (eng.head_distill_bwd, kdb)):
        for kw in (dict(dx=None, dw=None), dict(lddx=56), dict(lddw=68), dict(dx=h.dx.data_ptr() + 4),
                   dict(dw=h.dw.data_ptr() + 2)):
            refused(1, fn, base, **kw)
    for fn, base in ((eng.head_distill_fwd, kd), (eng.head_distill_bwd, kdb)):
        for kw in (dict(ids=None), dict(teacher=None), dict(topk=0), dict(topk=-3), dict(temperature=0.0),
                   dict(temperature=NAN), dict(temperature=-1.0), dict(temperature=1e-45),
                   dict(temperature=1e30)):
            refused(1, fn, base, **kw)
        refused(7, fn, base, topk=257)
        refused(8, fn, base, topk=256)
    for kw in ((0, 64, 10, 0), (1, 0, 10, 0), (1, 64, 0, 0), (1, 64, 10, -1)):
        with pytest.raises(ne.NeError) as err:
            eng.head_alloc(*kw)
        assert err.value.status == 1
    for kw in ((1, 60, 10, 0), (1, 64, 10, 257), (2 ** 23, 64, 10, 0)):
        with pytest.raises(ne.NeError) as err:
            eng.head_alloc(*kw)
        assert err.value.status == 7
    e2 = ne.Engine(ne.ModelConfig(1, 128, 256, 2, 2, 64, 256))
    refused(8, e2.head_ce_fwd, ok)
    refused(8, e2.head_distill_fwd, kd)
    e2.close()
    eng.sync()
    assert bool((h.loss == 7.0).all()) and bool((h.dw == 7.0).all())   # nothing was enqueued
    eng.close()


def test_factors_past_the_range_are_refused(eng):
    """scale / T and scale * T have to be numbers of fp32 other than 0."""
    import neural_engine_b200 as ne
    h = Head(4, 64, 100, seed=15).distill(4, 2.0)
    h.upload()
    eng.head_alloc(4, 64, 100, 4)
    for scale, T in ((1e-30, 1e18), (1e30, 1e15)):
        h.scale, h.T = scale, T
        with pytest.raises(ne.NeError) as err:
            eng.head_distill_fwd(**h.head(), ids=h.d_ids.data_ptr(), teacher=h.d_teacher.data_ptr(), topk=4,
                                 temperature=T, loss=h.loss.data_ptr(), lse=h.lse.data_ptr())
        assert err.value.status == 1


def test_room_that_cannot_be_had():
    """A size out of range is refused; one that memory cannot hold leaves the
    context without workspaces and otherwise as it was."""
    import neural_engine_b200 as ne
    eng = ne.Engine(ne.ModelConfig(1, 128, 256, 2, 2, 64, 256))
    for kw in ((1, 2 ** 28 + 8, 10, 0), (1, 64, 2 ** 28 + 1, 0)):
        with pytest.raises(ne.NeError) as err:
            eng.head_alloc(*kw)
        assert err.value.status == 7
    h = Head(4, 64, 100, seed=16).ce()
    h.run(eng).check()
    with pytest.raises(ne.NeError) as err:   # the pairs of the rows alone are 94 TB
        eng.head_alloc(2 ** 22, 64, 2 ** 28, 0)
    assert err.value.status == 3
    with pytest.raises(ne.NeError) as err:
        h.forward(eng)
    assert err.value.status == 8
    h.run(eng).check()
    eng.close()
