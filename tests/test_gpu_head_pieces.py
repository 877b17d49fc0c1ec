"""GPU: the head losses' backward pass over several pieces of the vocabulary,
against the float64 definition (oracle/head_loss.py, run on the GPU).

The sizes are held against the plan that the host makes (`plan`, worked out from
the budgets in csrc/head_loss.cu): more pieces than there are buffers of dz, a
last piece of another size, dx in slabs of its own and added up from piece to
piece, one CTA a tile and pairs, rows that stand twice.  Tolerances are
oracle.head_loss.bounds; outputs in bf16 add half a step, 2^-8 of their size, in
fp32 2^-23 and, where they are added to what was there, 2^-22.
"""
import math
import os
import re

import pytest

torch = pytest.importorskip("torch")

from oracle import head_loss as oh  # noqa: E402
from tests.test_gpu_head_loss import Head  # noqa: E402

pytestmark = pytest.mark.gpu

SRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                   "neural_engine_b200", "csrc", "head_loss.cu")
BUFFERS = 3   # of dz


def _budget(name):
    with open(SRC) as f:
        m = re.search(r"constexpr size_t %s = (\d+)u << 20;" % name, f.read())
    return int(m.group(1)) << 20


def plan(rows, dim, vocab, sms):
    """(pieces, ids a piece, own slabs): head_plan of csrc/head_loss.cu."""
    up = lambda n, to: -(-n // to) * to  # noqa: E731
    rows64 = max(up(rows, 64), 128)
    cg = 2 if rows64 > 128 else 1
    room = max(256, _budget("kPieceBytes") // 2 // rows64 // 256 * 256)
    pieces = -(-vocab // room)
    piece = up(-(-vocab // pieces), 256)
    pieces = -(-vocab // piece)
    m_tiles, d_tiles, kb = -(-rows64 // (128 * cg)), -(-dim // 256), piece / 64
    load = m_tiles * d_tiles * kb + piece // (128 * cg) * d_tiles * max(9.0, rows64 / 64)
    slabs = max(1, _budget("kSlabBytes") // (rows64 * dim * 4))
    want = max(1, min(math.ceil(kb / max(8.0, load / (sms // cg) / 2)), slabs))
    splits = -(-piece // up(-(-piece // want), 256))
    return pieces, piece, splits * pieces <= slabs


class Pieces(Head):
    def exact(self):
        keep, p, plogp = (t.cuda() for t in self.targets())
        x, w, k = self.x.cuda(), self.w.cuda(), dict(scale=self.scale, temperature=self.T, grad=self.grad.cuda())
        with torch.device("cuda"):
            want = oh.head_loss(x, w, keep, p, plogp, **k)
            step = 2.0 ** (-16 if int(keep.sum()) <= 64 else -8)
            return want, oh.bounds(x, w, keep, p, **k, dz_step=step)

    def hold(self, dx=True, dw=True, f32=False):
        """What was asked for is within its bounds, what was not is as it was."""
        (loss, lse, wx, ww), (b_loss, b_lse, b_dx, b_dw) = self.exact()
        R, V, D = self.rows, self.vocab, self.dim
        assert float((self.loss[:R].double() - loss).abs().max()) <= b_loss
        assert float((self.lse[:R].double() - lse).abs().max()) <= b_lse
        outs = ((self.dx32 if f32 else self.dx, R, wx, b_dx, dx, 0.0, 2.0 ** (-23 if f32 else -8)),
                (self.dw32 if f32 else self.dw, V, ww, b_dw, dw, 7.0 if f32 else 0.0, 2.0 ** (-22 if f32 else -8)))
        for got, n, ref, b, asked, base, half in outs:
            if not asked:
                assert bool((got == 7.0).all())
                continue
            assert bool((got[n:] == 7.0).all()) and bool((got[:, D:] == 7.0).all())
            ref = ref + base
            over = (got[:n, :D].double() - ref).abs() - (b + half * (ref.abs() + b) + 1e-30)
            assert bool(torch.isfinite(got[:n, :D]).all()) and float(over.max()) <= 0


@pytest.fixture(scope="module")
def eng():
    import neural_engine_b200 as ne
    e = ne.Engine(ne.ModelConfig(1, 128, 256, 2, 2, 64, 256))
    yield e
    e.close()


def _reaches(rows, dim, vocab, own):
    pieces, piece, has = plan(rows, dim, vocab, torch.cuda.get_device_properties(0).multi_processor_count)
    assert pieces > BUFFERS and vocab % piece and has is own, (pieces, piece, has)


def _pass(e, h, f32=False, dx=True, dw=True):
    h.upload()
    e.head_alloc(h.rows, h.dim, h.vocab, h.topk)
    h.forward(e)
    h.backward(e, f32=f32, dx=dx, dw=dw)
    e.sync()
    return [t.clone() for t in (h.loss, h.lse, h.dx, h.dw, h.dx32, h.dw32)]


# 5 pieces; dim 64: dx of each piece in slabs of its own, dim 520: added up
MANY = [(16384, 64, 16500, True), (16384, 520, 16500, False)]


@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("rows,dim,vocab,own", MANY)
def test_cross_entropy(eng, rows, dim, vocab, own, f32):
    _reaches(rows, dim, vocab, own)
    h = Pieces(rows, dim, vocab, seed=dim, scale=0.5).ce(0.3)
    a = _pass(eng, h, f32)
    h.hold(f32=f32)
    for _ in range(3):   # the same bits, whichever pair a unit went to
        for u, v in zip(a, _pass(eng, h, f32)):
            assert torch.equal(u, v)


@pytest.mark.parametrize("rows,dim,vocab,own", MANY)
def test_distillation(eng, rows, dim, vocab, own):
    _reaches(rows, dim, vocab, own)
    h = Pieces(rows, dim, vocab, seed=dim + 1).distill(3, 2.0, masked=0.4)
    _pass(eng, h)
    h.hold()


@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("alone", ["dx", "dw"])
@pytest.mark.parametrize("rows,dim,vocab,own", MANY)
def test_one_gradient_alone(eng, rows, dim, vocab, own, alone, f32):
    _reaches(rows, dim, vocab, own)
    h = Pieces(rows, dim, vocab, seed=dim + 2).ce(0.3)
    both = _pass(eng, h, f32)
    one = _pass(eng, h, f32, dx=alone == "dx", dw=alone == "dw")
    at = (2 if alone == "dx" else 3) + 2 * f32
    for k in range(2, 6):
        assert torch.equal(one[k], both[k]) if k == at else bool((one[k] == 7.0).all())


@pytest.mark.parametrize("counted", [0, 1, 40, 64, 65])
@pytest.mark.parametrize("rows,dim,vocab,own", MANY)
def test_few_of_many_rows_count(eng, rows, dim, vocab, own, counted):
    _reaches(rows, dim, vocab, own)
    h = Pieces(rows, dim, vocab, seed=counted + dim).ce()
    out = torch.randperm(rows, generator=h.g)[counted:]
    h.target[out] = -100
    h.x[out] = math.nan
    h.grad[out] = math.nan
    _pass(eng, h)
    h.grad[out] = 0.0
    h.hold()


@pytest.mark.parametrize("rows", [5, 64, 65, 128])
def test_few_rows_of_a_huge_vocabulary(rows):
    """One CTA a tile, more pieces than buffers."""
    import neural_engine_b200 as ne
    vocab = 3 * (_budget("kPieceBytes") // 2 // 128) + 70000
    assert plan(rows, 8, vocab, torch.cuda.get_device_properties(0).multi_processor_count)[0] > BUFFERS
    e = ne.Engine(ne.ModelConfig(1, 128, 256, 2, 2, 64, 256))
    for f32 in (False, True):
        h = Pieces(rows, 8, vocab, seed=rows).ce(0.1)
        _pass(e, h, f32)
        h.hold(f32=f32)
    e.close()
