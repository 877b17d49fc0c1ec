"""GPU: the head losses where sums are taken in runs and a block has several tiles,
against the float64 definition on the GPU (tolerances: oracle.head_loss.bounds).

The forward pass splits a sum beyond 384 columns, the backward pass one beyond 1024
products (dim, rows that count, ids of a split); an accumulator serves every other
run, so odd and even numbers of runs a tile both have to come round.
"""
import pytest

torch = pytest.importorskip("torch")

from tests.test_gpu_head_pieces import Pieces  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def eng():
    import neural_engine_b200 as ne
    e = ne.Engine(ne.ModelConfig(1, 128, 256, 2, 2, 64, 256))
    yield e
    e.close()


def _pass(e, h, f32):
    h.upload()
    e.head_alloc(h.rows, h.dim, h.vocab, h.topk)
    h.forward(e)
    h.backward(e, f32=f32)
    e.sync()
    return [t.clone() for t in (h.loss, h.lse, h.dx, h.dw, h.dx32, h.dw32)]


# one CTA a tile, one pair's tile of rows, packed rows; 2 and 3 runs a logit
@pytest.mark.parametrize("dim", [448, 1000])
@pytest.mark.parametrize("rows", [1, 100, 200, 300])
def test_runs_over_several_tiles(eng, rows, dim):
    h = Pieces(rows, dim, 80001, seed=rows + dim, scale=0.5).ce(0.2 if rows > 1 else 0.0)
    _pass(eng, h, False)
    h.hold()
    h = Pieces(rows, dim, 80001, seed=rows + dim + 1, pad=8).distill(5, 2.0, masked=0.2 if rows > 1 else 0.0)
    _pass(eng, h, True)
    h.hold(f32=True)


# logits of 18 k-blocks, dx over splits of many, dw over 33 and 17 k-blocks of rows
@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("rows,dim,vocab", [(2100, 1104, 9001), (1030, 328, 40000), (40, 2056, 30001), (128, 1160, 12345)])
def test_runs_of_the_backward_pass(eng, rows, dim, vocab, f32):
    h = Pieces(rows, dim, vocab, seed=rows).ce(0.0)
    a = _pass(eng, h, f32)
    h.hold(f32=f32)
    for u, v in zip(a, _pass(eng, h, f32)):
        assert torch.equal(u, v)
