"""The vocabulary-row operators as parts of a user's program: autograd around them, ids of every type, streams of other
devices, batches that go through the same blocks in place."""
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("call", ["logprobs", "policy", "distill"])
def test_a_gradient_over_logits_that_autograd_saved(gpu_pkg, call):
    # a z-loss saves the logits; with the gradient written over them its backward has to raise, not to go by the gradient
    head = torch.randn(64, 4, device="cuda", requires_grad=True)
    logits = torch.randn(3, 4, device="cuda") @ head.t()
    z_loss = logits.logsumexp(-1).square().mean()
    x = logits.detach()
    t = torch.arange(3, dtype=torch.int32, device="cuda")
    one = torch.ones(3, device="cuda")
    before = logits._version
    if call == "logprobs":
        gpu_pkg.token_logprobs_grad(x, t, gpu_pkg.token_logprobs(x, t), one, out=x)
    elif call == "policy":
        gpu_pkg.policy_loss(x, t, -one, one, out=x)
    else:
        gpu_pkg.distill_loss(x, t[:, None], one[:, None], out=x)
    assert logits._version == before + 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        z_loss.backward()
    # without a gradient nothing is written, and a buffer of one's own is no concern of the logits
    logits = torch.randn(3, 4, device="cuda") @ head.t()
    z_loss = logits.logsumexp(-1).square().mean()
    x = logits.detach()
    gpu_pkg.policy_loss(x, t, -one, one, grad=False, out=x)
    gpu_pkg.policy_loss(x, t, -one, one, out=torch.empty_like(x))
    z_loss.backward()
    assert head.grad is not None and bool(torch.isfinite(head.grad).all())
    # one row, 1-D
    row = torch.randn(40, device="cuda")
    v = row._version
    gpu_pkg.policy_loss(row, t[:1], -one[:1], one[:1], out=row)
    assert row._version == v + 1


def test_a_gradient_over_inference_tensors(gpu_pkg):
    with torch.inference_mode():
        x = torch.randn(3, 40, device="cuda")
    t, one = torch.arange(3, dtype=torch.int32, device="cuda"), torch.ones(3, device="cuda")
    want = gpu_pkg.policy_loss(x, t, -one, one).grad
    assert torch.equal(gpu_pkg.policy_loss(x, t, -one, one, out=x).grad, want)


@pytest.mark.parametrize("dtype", [torch.int8, torch.uint8, torch.int16, torch.uint16, torch.int64, torch.uint32, torch.uint64], ids=str)
def test_ids_of_every_type(gpu_pkg, dtype):
    x = torch.randn(4, 100, device="cuda")
    want = gpu_pkg.token_logprobs(x, torch.tensor([5, 99, 0, -1], dtype=torch.int32, device="cuda")).logprobs
    # an id that no vocabulary holds leaves its row out, and is not cut down to one that it holds
    far = {torch.int8: -1, torch.uint8: 200, torch.int16: -1, torch.uint16: 65535, torch.int64: 2**32 + 5, torch.uint32: 2**32 - 1,
           torch.uint64: 2**32 + 5}[dtype]
    for other in (far, 2**63 + 7) if dtype == torch.uint64 else (far,):
        ids = torch.tensor([5, 99, 0, other], dtype=dtype).cuda()
        assert torch.equal(gpu_pkg.token_logprobs(x, ids).logprobs, want), other


def test_a_stream_of_another_device_is_refused(gpu_pkg):
    class Elsewhere(torch.cuda.Stream):
        device = property(lambda self: torch.device("cuda", 1))

    x, t, one = torch.randn(3, 40, device="cuda"), torch.arange(3, dtype=torch.int32, device="cuda"), torch.ones(3, device="cuda")
    s = Elsewhere()
    for call in (lambda: gpu_pkg.token_logprobs(x, t, stream=s), lambda: gpu_pkg.top_logits(x, 2, stream=s),
                 lambda: gpu_pkg.policy_loss(x, t, one, one, stream=s), lambda: gpu_pkg.distill_loss(x, t[:, None], one[:, None], stream=s)):
        with pytest.raises(ValueError, match="device"):
            call()


@pytest.mark.parametrize("vocab", [7, 5000, 128256])
def test_a_row_without_a_distribution(gpu_pkg, vocab):
    # all masked: lse is -inf as a logsumexp, and whoever takes the row for a teacher with a tail gets NaN, not zeros
    x = torch.randn(3, vocab, device="cuda")
    x[1] = -math.inf
    top = gpu_pkg.top_logits(x, 5)
    assert torch.equal(top.lse == -math.inf, torch.tensor([False, True, False], device="cuda"))
    assert top.ids[1].tolist() == [0, 1, 2, 3, 4] and bool((top.logits[1] == -math.inf).all())
    t = torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda")
    lp = gpu_pkg.token_logprobs(x, t)
    assert lp.logprobs.isnan().tolist() == [False, True, False] and lp.entropy.isnan().tolist() == [False, True, False]
    y = torch.randn(3, vocab, device="cuda")
    w = torch.ones(3, device="cuda")
    r = gpu_pkg.distill_loss(y, top.ids, top.logits, top.lse, w)
    assert r.row_losses.isnan().tolist() == [False, True, False] and bool(r.grad[1].isnan().all())
    assert not bool(r.grad[0].isnan().any()) and not bool(r.grad[2].isnan().any())
    assert float(gpu_pkg.distill_loss(y, top.ids, top.logits, None, w).row_losses[1]) == 0.0
    w[1] = 0.0
    r = gpu_pkg.distill_loss(y, top.ids, top.logits, top.lse, w)
    assert bool(torch.isfinite(r.loss)) and not bool(r.grad[1].any()) and float(r.row_losses[1]) == 0.0


def test_soft_caps_at_the_ends_of_f32(gpu_pkg):
    # no cap is refused but NaN and infinity; 1 / cap is past f32 for the smallest
    x = torch.tensor([[0.0, 1.0, -1.0, 30.0, math.inf, -math.inf, 1e-42, -0.0]], device="cuda")
    one = torch.ones(1, device="cuda")
    for cap in (1e-45, 1e-40, 1.5e-38, 1e-30, 1e30, 3e38):
        top = gpu_pkg.top_logits(x, 8, final_logit_softcapping=cap)
        c = float(torch.tensor(cap, dtype=torch.float32))
        want = c * torch.tanh(x.double() / c).gather(1, top.ids.long())
        want = torch.where(x.gather(1, top.ids.long()).isinf(), torch.sign(want) * c, want)
        assert bool(((top.logits.double() - want).abs() <= 4 * 2.0**-24 * want.abs() + 2.0**-148).all()), (cap, top.logits, want)
        t = torch.zeros(1, dtype=torch.int32, device="cuda")
        r = gpu_pkg.token_logprobs(x, t, final_logit_softcapping=cap)
        if cap < 1.0:      # eight equal ones, as far as exp can tell
            assert abs(float(r.logprobs) + math.log(8.0)) <= 8 * 2.0**-24
            g = gpu_pkg.token_logprobs_grad(x, t, r, one, final_logit_softcapping=cap)
            assert bool(torch.isfinite(g).all()) and abs(float(g[0, 0]) - 0.875) <= 8 * 2.0**-24


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("rows,vocab,ld,cap", [(1500, 1031, 1031, 0.0), (900, 8192, 8192, 0.0), (500, 40003, 40003, 0.0), (300, 128256, 128256, 0.0),
                                               (60, 256000, 256001, 0.0), (20, 600000, 600000, 0.0), (300, 40003, 40003, 2.0),
                                               (20, 600000, 600000, 2.0)])
def test_gradients_over_the_logits_of_many_rows(gpu_pkg, dtype, rows, vocab, ld, cap):
    """The gradient in place, rows going one after the other through the same blocks: what is loaded ahead (rows, tokens,
    single elements, a teacher's logits) is read before another block writes over it, rows that do not fit on chip and
    logits above a soft-cap are read again by whoever writes there.  The same bits as into a buffer of its own."""
    off = 1 if ld % 8 else 0
    g = torch.Generator(device="cuda").manual_seed(221)
    base = torch.zeros(off + rows * ld, dtype=dtype, device="cuda")
    src = 3.0 * torch.randn(rows, vocab, generator=g, device="cuda")

    def fresh():
        x = base[off:].view(rows, ld)[:, :vocab]
        x.copy_(src)
        return x

    x = fresh()
    t = torch.randint(0, vocab, (rows,), generator=g, device="cuda").int()
    t[::11] = 0                                    # single elements before and behind the chunks
    t[5::11] = vocab - 1
    t[torch.rand(rows, generator=g, device="cuda") < 0.1] = -1
    w = torch.rand(rows, generator=g, device="cuda") + 0.5
    w[torch.rand(rows, generator=g, device="cuda") < 0.2] = 0.0
    w[rows // 3:rows // 2] = 0.0
    one = torch.ones(rows, device="cuda")
    tl, ids = torch.topk(src + torch.randn(rows, vocab, generator=g, device="cuda"), 40, dim=1)
    ids = ids.int()
    ids[::5, 1] = ids[::5, 0]                      # an id twice
    ids[3::7] = -1                                 # no teacher
    ids[2::9, 4] = vocab - 1
    lse = torch.logsumexp(src, 1) + 0.1
    calls = {
        "policy": lambda x, out: gpu_pkg.policy_loss(x, t, -9 * one, one, -9 * one, w, kl_coef=0.01, entropy_coef=0.01,
                                                     final_logit_softcapping=cap, out=out),
        "slots": lambda x, out: gpu_pkg.distill_loss(x, ids, tl, None, w, final_logit_softcapping=cap, out=out),
        "tail": lambda x, out: gpu_pkg.distill_loss(x, ids, tl, lse, w, final_logit_softcapping=cap, out=out),
    }
    for name, call in calls.items():
        # (a buffer whose rows are aligned like the logits': a kernel's writes do not depend on it, its sums on the logits)
        want = call(x, None)
        for _ in range(2):
            y = fresh()
            got = call(y, y)
            assert torch.equal(got.row_losses, want.row_losses), name
            assert torch.equal(y, want.grad), (name, int((y != want.grad).sum()))
        x = fresh()
