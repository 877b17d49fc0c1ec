"""GPU: what rounding dz to bf16 takes from a row's target is put back in dx and dw.

The logits are all 0 and there are 512 ids, so softmax is 2^-9, which bf16 holds, and
dz at the target is a (2^-9 - 1), which it does not: rounded it is off by 2^-9 of its
size.  The row gradients a are numbers of a few bits.
"""
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

V = 512
ROWS_PUT_BACK = 32   # of each 32 ids, in dw


@pytest.fixture(scope="module")
def eng():
    import neural_engine_b200 as ne
    e = ne.Engine(ne.ModelConfig(1, 128, 256, 2, 2, 64, 256))
    yield e
    e.close()


class Case:
    def __init__(self, rows, dim, K, seed):
        g = self.g = torch.Generator().manual_seed(seed)
        self.rows, self.dim, self.K = rows, dim, K
        self.values = torch.randn(max(rows, V), dim, generator=g).to(torch.bfloat16)
        self.grad = torch.tensor([1.0, -0.75, 0.625, 2.5])[torch.randint(0, 4, (rows,), generator=g)]
        self.target = torch.randint(0, V, (rows,), generator=g).to(torch.int32)
        self.target[torch.rand(rows, generator=g) < 0.1] = -1

    def entries(self):
        """A teacher that is sure of its last entry; the others, of logit -200, have
        probability 0."""
        ids = torch.randint(0, V, (self.rows, self.K), generator=self.g).to(torch.int32)
        ids[:, -1] = self.target
        ids[self.target < 0] = -1
        y = torch.full((self.rows, self.K), -200.0)
        y[:, -1] = 3.0
        return ids, y

    def run(self, eng, dx, f32):
        """dx with x = 0, or dw with w = 0: (what came, the formula in float64)."""
        a, t = self.grad.cuda(), self.target.cuda()
        keep = t >= 0
        zero = torch.zeros(V if not dx else self.rows, self.dim, dtype=torch.bfloat16, device="cuda")
        some = self.values[:V if dx else self.rows].cuda()
        x, w = (zero, some) if dx else (some, zero)
        loss, lse = torch.empty(2, self.rows, device="cuda")
        out = torch.zeros(x.shape if dx else w.shape, dtype=torch.float32 if f32 else torch.bfloat16, device="cuda")
        if self.K:
            ids, y = (v.cuda() for v in self.entries())
            want = dict(ids=ids.data_ptr(), teacher=y.data_ptr(), topk=self.K)
            fwd, bwd = eng.head_distill_fwd, eng.head_distill_bwd
        else:
            want, fwd, bwd = dict(target=t.data_ptr()), eng.head_ce_fwd, eng.head_ce_bwd
        torch.cuda.synchronize()
        eng.head_alloc(self.rows, self.dim, V, self.K)
        head = dict(x=x.data_ptr(), w=w.data_ptr(), rows=self.rows, dim=self.dim, vocab=V, lse=lse.data_ptr(), **want)
        fwd(**head, loss=loss.data_ptr())
        bwd(**head, grad=a.data_ptr(), **{"dx" if dx else "dw": out.data_ptr(), "dx_f32" if dx else "dw_f32": f32})
        eng.sync()
        dz = torch.full((self.rows, V), 2.0 ** -9, dtype=torch.float64, device="cuda")
        dz[torch.arange(self.rows, device="cuda"), t.long().clamp_min(0)] -= 1.0
        dz = torch.where(keep[:, None], dz * a.double()[:, None], 0.0)
        full = dz @ some.double() if dx else dz.T @ some.double()
        # fp32 sums of at most 1024 products, in steps of 16 that lose 5.25 * 2^-23 each
        # (test_gpu_head_sums.py); the exponential at the target 2^-22 of 2^-9, its
        # logit's shift 2^-21 of it, and the subtraction 2^-24
        mag = dz.abs() @ some.double().abs() if dx else dz.abs().T @ some.double().abs()
        return out.double(), full, (64 * 5.25 + 4) * 2.0 ** -23 * mag


@pytest.mark.parametrize("f32", [True, False])
@pytest.mark.parametrize("K", [0, 1, 3, 4])
@pytest.mark.parametrize("rows,dim", [(80, 64), (129, 200), (300, 72), (300, 520)])
def test_targets_are_as_exact_as_the_rest(eng, rows, dim, K, f32):
    c = Case(rows, dim, K, rows + dim + K)
    count = torch.bincount((c.target[c.target >= 0] // 32).long(), minlength=V // 32)
    assert int(count.max()) <= ROWS_PUT_BACK and int((c.target >= 0).sum()) > 64
    for dx in (True, False):
        got, ref, b = c.run(eng, dx, f32)
        if not f32:
            b = b + 2.0 ** -8 * ref.abs()
        assert bool(((got - ref).abs() <= b).all()), float(((got - ref).abs() - b).max())


def test_many_rows_of_few_ids_keep_the_rounding_in_dw(eng):
    """More rows than the list of 32 ids holds: dw is then off by the rounding of dz,
    2^-9 of each target's, and dx is not; the same bits every time all the same."""
    c = Case(500, 136, 0, 5)
    c.target = torch.randint(0, 40, (500,), generator=c.g).to(torch.int32)
    got, ref, b = c.run(eng, True, True)
    assert bool(((got - ref).abs() <= b).all())
    got, ref, b = c.run(eng, False, True)
    own = torch.zeros(V, 136, dtype=torch.float64, device="cuda")
    own.index_add_(0, c.target.long().cuda(),
                   (c.values[:500].double() * c.grad.double()[:, None]).abs().cuda())
    assert bool(((got - ref).abs() <= b + 2.0 ** -9 * own).all())
    for _ in range(3):
        assert torch.equal(got, c.run(eng, False, True)[0])
