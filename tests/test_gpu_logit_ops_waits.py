"""What follows a device wait of the losses' kernel that gives up: the calls end, the rows are NaN, the host is told, and the
next call is as if nothing had been.

The waits are made to run out by their limit: one thread block of each row is told that its own did, and the others of the
row then miss what it would have sent.  Nothing faults, and every wait is bounded.
"""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

OK, ETIMEOUT = 0, 5
NONE = 0xFFFFFFFF


@pytest.fixture
def waits(gpu_pkg):
    L = gpu_pkg.lib()
    assert gpu_pkg.logit_ops_status() == OK
    yield L.bs_debug_logit_ops_waits
    L.bs_debug_logit_ops_waits(0, NONE, 0)
    gpu_pkg.logit_ops_status()


SIZES = [(40, 1000, torch.float32), (700, 8000, torch.bfloat16), (150, 40000, torch.float32), (300, 128256, torch.bfloat16),
         (60, 256000, torch.float32)]


@pytest.mark.parametrize("op", ["policy", "slots", "tail"])
@pytest.mark.parametrize("grad", [True, False], ids=["grad", "loss alone"])
@pytest.mark.parametrize("rows,vocab,dtype", SIZES, ids=str)
@pytest.mark.parametrize("rank,row", [(0, 0), (1, 0), (0, 3), (1, 2)])
def test_a_wait_that_gives_up(gpu_pkg, waits, op, grad, rows, vocab, dtype, rank, row):
    g = torch.Generator(device="cuda").manual_seed(211)
    x = torch.randn(rows, vocab, generator=g, device="cuda").to(dtype)
    t = torch.randint(0, vocab, (rows,), generator=g, device="cuda").int()
    w = torch.rand(rows, generator=g, device="cuda") + 0.5
    w[::7] = 0.0
    one = torch.ones(rows, device="cuda")
    tl, ids = torch.topk(x.float(), 20, dim=1)
    lse = torch.logsumexp(x.float(), 1) + 0.1

    def call():
        if op == "policy":
            return gpu_pkg.policy_loss(x, t, -9 * one, one, None, w, grad=grad)
        return gpu_pkg.distill_loss(x, ids.int(), tl, lse if op == "tail" else None, w, grad=grad)

    want = call()
    assert gpu_pkg.logit_ops_status() == OK
    waits(2_000_000, rank, row)      # a millisecond
    got = call()
    status = gpu_pkg.logit_ops_status()
    waits(0, NONE, 0)
    lost = got.row_losses.isnan()
    if status == OK:                 # no row has such a block, or no block that many rows
        assert torch.equal(got.row_losses, want.row_losses) and (rank == 1 or row > 0)
        if grad:
            assert torch.equal(got.grad, want.grad)
    else:
        assert status == ETIMEOUT
        assert bool(lost.any()) and bool(got.loss.isnan())
        assert not bool(lost[::7].any()) and not bool(got.row_losses[::7].any())     # left-out rows are zeros all the same
        assert torch.equal(got.row_losses[~lost], want.row_losses[~lost])
        if row == 0:
            assert bool(lost[w != 0].all())
        if grad:
            same = (got.grad == want.grad) | got.grad.isnan()
            assert bool(same.all()) and not bool(got.grad[::7].any())
            assert bool(got.grad[lost].isnan().any(1).all())
    # the next call starts clean
    again = call()
    assert gpu_pkg.logit_ops_status() == OK
    assert torch.equal(again.row_losses, want.row_losses) and torch.equal(again.loss, want.loss)
    if grad:
        assert torch.equal(again.grad, want.grad)
