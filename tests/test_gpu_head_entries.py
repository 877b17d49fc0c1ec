"""GPU: a teacher's entries at the edges of what the head losses allow, against
the float64 definition (tolerances: oracle.head_loss.bounds).
"""
import math

import pytest

torch = pytest.importorskip("torch")

from tests.test_gpu_head_loss import Head  # noqa: E402

pytestmark = pytest.mark.gpu

INT_MAX = 2 ** 31 - 1


@pytest.fixture()
def eng():
    import neural_engine_b200 as ne
    e = ne.Engine(ne.ModelConfig(1, 128, 256, 2, 2, 64, 256))
    yield e
    e.close()


@pytest.mark.parametrize("rows", [5, 300])
def test_ids_behind_a_logit_of_minus_infinity_are_not_looked_at(eng, rows):
    """Entries padded with -inf and any id are absent, and nothing is reported."""
    h = Head(rows, 64, 100, seed=rows).distill(6, 2.0, ragged=False)
    for k, i in enumerate((100, 101, INT_MAX, -1, -2 ** 31)):
        h.ids[k::5, 1 + k:] = i
        h.teacher[k::5, 1 + k:] = -math.inf
    h.ids[3], h.teacher[3] = INT_MAX, -math.inf   # no entry at all
    h.run(eng).check()


LOWEST = torch.finfo(torch.float32).min


@pytest.mark.parametrize("T", [0.01, 0.5, 1.0, 3.0])
def test_logits_at_the_ends_of_the_range(eng, T):
    """A finite logit is an entry however small the temperature: logits / T may pass
    the range of fp32, their differences from the row's largest decide."""
    h = Head(8, 64, 100, seed=3).distill(5, T, ragged=False)
    h.teacher[0] = LOWEST                       # every entry alike: a fifth each
    h.teacher[1, 1:] = LOWEST                   # one entry has it all
    h.teacher[2] = -LOWEST                      # a fifth each again
    h.teacher[3] = torch.tensor([3e38, 2.9e38, 3e38, -3e38, LOWEST])
    h.teacher[4] = torch.tensor([-3e38, -2.9e38, LOWEST, -math.inf, -2.9e38])
    h.teacher[5] = 0.0
    h.teacher[6, ::2] = LOWEST
    h.run(eng).check()


def test_temperatures_whose_square_passes_the_range_are_refused(eng):
    """T^2 is a factor of the loss: at T = 1e-21 it is 0 in fp32, and the loss, of the
    order of T times the logits, was too."""
    import neural_engine_b200 as ne
    h = Head(4, 64, 100, seed=15).distill(4, 2.0)
    h.upload()
    eng.head_alloc(4, 64, 100, 4)
    for T in (1e-21, 5e-20, 2e19):
        h.T = T
        kd = dict(h.head(), ids=h.d_ids.data_ptr(), teacher=h.d_teacher.data_ptr(), topk=4, temperature=T,
                  lse=h.lse.data_ptr())
        for call in (lambda: eng.head_distill_fwd(**kd, loss=h.loss.data_ptr()),
                     lambda: eng.head_distill_bwd(**kd, dx=h.dx.data_ptr(), dw=h.dw.data_ptr())):
            with pytest.raises(ne.NeError) as err:
                call()
            assert err.value.status == 1
    eng.sync()
    assert bool((h.loss == 7.0).all()) and bool((h.dw == 7.0).all())
    Head(4, 64, 100, seed=16).distill(4, 2e-6).run(eng)   # far from it
