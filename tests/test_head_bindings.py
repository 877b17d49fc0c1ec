"""CPU: sizes that a C int does not hold are refused by the head losses' bindings,
before the library is called (ctypes would keep their low 32 bits)."""
import ctypes

import numpy as np
import pytest

import neural_engine_b200 as ne


class _Untouched:
    def __getattr__(self, name):
        def called(*a):
            raise AssertionError(f"{name} was called")
        return called


@pytest.fixture()
def eng():
    e = ne.Engine.__new__(ne.Engine)
    e.lib, e._ctx = _Untouched(), ctypes.c_void_p()
    return e


@pytest.mark.parametrize("n", [2 ** 31, 2 ** 32 + 5, -2 ** 31 - 1, 2 ** 64 + 1])
def test_sizes_past_32_bits_are_refused(eng, n):
    head = dict(x=16, w=16, rows=4, dim=64, vocab=100, lse=16)
    ce, kd = dict(head, target=16), dict(head, ids=16, teacher=16, topk=4)
    calls = [(f, base, k) for f, base in (
        (lambda **a: eng.head_ce_fwd(loss=16, **a), ce), (lambda **a: eng.head_ce_bwd(dx=16, **a), ce),
        (lambda **a: eng.head_distill_fwd(loss=16, **a), kd), (lambda **a: eng.head_distill_bwd(dx=16, **a), kd))
        for k in ("rows", "dim", "vocab", "topk") if k in base]
    calls += [(eng.head_alloc, dict(max_rows=4, max_dim=64, max_vocab=100, max_topk=4), k)
              for k in ("max_rows", "max_dim", "max_vocab", "max_topk")]
    calls.append((eng.lmhead_distill_fwd_bwd, dict(ids=16, teacher=16, topk=4), "topk"))
    for f, base, k in calls:
        with pytest.raises(ne.NeError) as err:
            f(**dict(base, **{k: n}))
        assert err.value.status == 1 and k in str(err.value)


def test_sizes_of_other_integer_types():
    d = ne.Engine._head(16, 32, np.int64(3), np.int32(64), np.uint8(100), 1.0, 0, 0)
    assert (d.rows, d.dim, d.vocab, d.ldx, d.ldw) == (3, 64, 100, 64, 64)
