"""What the vocabulary-row operators work out of a row's sums, where little of it is left: ratios near 1, a KL near 0,
probabilities near 1, losses whose terms cancel.

The rows are such that their f32 sums are exact (all terms are powers of two), so that the scalars' own arithmetic shows.
EPS = 2^-24 is half a step of f32.
"""
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

EPS = 2.0**-24


def relative(got, want, tol, what=""):
    got, want = got.double().cpu(), torch.as_tensor(want, dtype=torch.float64).cpu()
    err = ((got - want).abs() / want.abs()).max()
    assert float(err) <= tol, (what, float(err), tol)


@pytest.mark.parametrize("vocab", [1, 2, 64, 4096, 131072])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_policy_scalars(gpu_pkg, vocab, dtype):
    # equal logits: every term is 2^0, S = vocab without rounding, lp = -ln vocab to 64 bits; each output is rounded once
    steps = torch.tensor([1e-6, 1e-5, 1e-4, 1e-3, 0.01, 0.1, 0.5, -1e-5, -1e-3, -0.1, -0.5], dtype=torch.float64)
    rows = len(steps)
    x = torch.full((rows, vocab), 1.5, dtype=dtype, device="cuda")
    t = torch.arange(rows, dtype=torch.int32, device="cuda") % vocab
    lp = -math.log(vocab)
    old, ref = (lp - steps).float(), (lp + steps).float()
    adv = torch.linspace(-2.0, 2.0, rows, dtype=torch.float64).float()
    adv[rows // 2] = 0.25
    for klc in (0.0, 0.1):
        got = gpu_pkg.policy_loss(x, t, old.cuda(), adv.cuda(), ref.cuda(), None, clip_low=0.75, clip_high=0.75, kl_coef=klc,
                                  temperature=0.7)
        ratio = (lp - old.double()).exp()
        d = ref.double() - lp
        some = d != 0          # (a reference that rounds to lp itself has a KL of 0)
        kl = torch.expm1(d) - d
        # the KL's own cancellation: 64-bit roundings of d (16 of them) over d^2 / 2
        tol = EPS + 2.0**-49 * (1 + abs(lp)) / d[some].abs().min()
        relative(got.kl[some.cuda()], kl[some], float(tol), "kl")
        rows_want = -ratio * adv.double() + float(np.float32(klc)) * kl
        relative(got.row_losses, rows_want, 1.01 * EPS, "rows")


@pytest.mark.parametrize("gap", [6, 10, 13])
@pytest.mark.parametrize("vocab", [2, 9, 20011])
def test_gradient_at_a_likely_token(gpu_pkg, gap, vocab):
    """1 - p of a token with p near 1."""
    # 1 / T is ln 2 to f32, so that d is a whole number and S = 1 + 2^-gap without rounding.  What k = 1 leaves off m log2 e
    # (below 2^-24) is corrected to first order.
    T = float(np.float32(1.0 / math.log(2.0)))
    x = torch.full((3, vocab), -math.inf, device="cuda")
    x[:, 0] = 2.0
    x[:, vocab - 1] = 2.0 - gap
    t = torch.zeros(3, dtype=torch.int32, device="cuda")
    rest = math.exp(-gap / T)
    p_other = rest / (1.0 + rest)
    w = torch.tensor([1.0, -0.5, 0.25], device="cuda")
    r = gpu_pkg.token_logprobs(x, t, temperature=T)
    relative(r.logprobs, [-math.log1p(rest)] * 3, 2 * EPS, "logprobs")
    g = gpu_pkg.token_logprobs_grad(x, t, r, w, None, temperature=T)
    # the normaliser's f32 in stats, the result's rounding, and one to spare
    relative(g[:, 0], w.double().cpu() * p_other / T, 3 * EPS, "gradient of the log-probability")
    old = torch.full((3,), float(-math.log1p(rest)), device="cuda")
    ratio = (-math.log1p(rest) - old.double().cpu()).exp()
    p = gpu_pkg.policy_loss(x, t, old, torch.ones(3, device="cuda"), None, w, temperature=T)
    relative(p.grad[:, 0], -ratio * w.double().cpu() * p_other / T, 3 * EPS, "gradient of the policy loss")


def uniform_distill(vocab, ids, tl, lse, T, w):
    """Loss and gradient of one equal-logits row, 64 bits, from the f32 inputs."""
    logp = -math.log(vocab)
    u = tl.double() / T
    logq = u - torch.logsumexp(u, 0) if lse is None else u - float(lse)
    q = logq.exp()
    loss = (q * (logq - logp)).sum()
    p = 1.0 / vocab
    grad = torch.full((vocab,), p, dtype=torch.float64)
    if lse is not None:
        qr, pr = 1 - q.sum(), (vocab - len(ids)) / vocab
        loss = loss + qr * (qr.log() - math.log(pr))
        grad = grad - qr / pr * p
        grad[ids.long()] = p
    grad[ids.long()] -= q
    return loss, w * grad / T


@pytest.mark.parametrize("vocab,K", [(64, 64), (4096, 8), (4096, 130), (131072, 1024)])
@pytest.mark.parametrize("tail", [False, True], ids=["slots", "tail"])
@pytest.mark.parametrize("near", [1e-1, 1e-3])
def test_student_near_its_teacher(gpu_pkg, vocab, K, tail, near):
    # equal logits again, and a teacher whose shares differ from the student's by `near`.  With T = 1 and 2 nothing but
    # the inputs is rounded before the results.  The loss is near^2 / 2 of the named mass in size, worked out from terms of
    # q |log q|: some 2^-50 of their sum beside the rounding.
    if tail and K == vocab:
        pytest.skip("no rest")
    g = torch.Generator().manual_seed(171)
    for T in (1.0, 2.0):
        x = torch.full((2, vocab), -0.75, device="cuda")
        ids = torch.randperm(vocab, generator=g)[:K].int()
        tl = near * torch.randn(K, generator=g)
        lse = torch.tensor(math.log(vocab) + near).float() if tail else None
        w = 0.5
        want, grad = uniform_distill(vocab, ids, tl, lse, T, w)
        both = lambda v: torch.stack([v, v]).cuda()  # noqa: E731
        got = gpu_pkg.distill_loss(x, both(ids), both(tl), both(lse) if tail else None, torch.full((2,), w, device="cuda"),
                                   temperature=T)
        big = max(1.0, math.log(vocab))
        relative(got.row_losses, [want] * 2, EPS + 2.0**-50 * big / float(want), "rows")
        at = ids.long()
        # p - q in 64 bits: one rounding, and 2^-50 of p over the difference
        few = grad[at].abs() > 1e-9 / vocab
        relative(got.grad[:, at.cuda()][0][few.cuda()], grad[at][few],
                 1.01 * EPS + 2.0**-48 / vocab / float(grad[at][few].abs().min()), "named tokens")
        rest = torch.ones(vocab, dtype=torch.bool)
        rest[at] = False
        if rest.any():
            # 2^l of l = -log2 S: l rounded twice to f32 (2 |l| EPS ln 2), ex2 2^-22, the coefficient and the result; the
            # coefficient's 64 bits lose 2^-50 over 1 - q_rest / p_rest
            l2s = math.log2(vocab)
            tol = EPS * (2 * l2s * math.log(2.0) + 4 + 2) + (2.0**-50 * vocab / float(grad[rest].abs().min()) / vocab if tail else 0)
            relative(got.grad[:, rest.cuda()], grad[rest].expand(2, -1), tol, "rest")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("gap", [60.0, 90.0, 104.0, 200.0, 2000.0, -200.0])
@pytest.mark.parametrize("vocab,off", [(40, 0), (5001, 1), (128256, 3)])
def test_rest_far_below_the_teacher(gpu_pkg, dtype, gap, vocab, off):
    """The tail's outcome where the student gives it e^-gap of a named token (or, below zero, the named ones that)."""
    g = torch.Generator(device="cuda").manual_seed(181)
    rows, K = 3, 7
    x = torch.zeros(off + rows * vocab, dtype=dtype, device="cuda")[off:].view(rows, vocab)
    x.copy_(torch.randn(rows, vocab, generator=g, device="cuda"))
    ids = torch.stack([torch.randperm(vocab, generator=g, device="cuda")[:K] for _ in range(rows)]).int()
    ids[0, 0], ids[0, 1] = 0, vocab - 1        # (single elements before and behind the 16-byte chunks, where there are)
    for i in range(rows):
        x[i, ids[i].long()] = (gap + 3.0 * torch.randn(K, generator=g, device="cuda")).to(dtype)
    ids[1, 3] = ids[1, 2]                      # one twice
    ids[2, 5] = -1
    tl = torch.randn(rows, K, generator=g, device="cuda")
    lse = torch.logsumexp(tl, 1) + 0.5
    w = torch.tensor([1.0, 0.5, 0.25], device="cuda")
    got = gpu_pkg.distill_loss(x, ids, tl, lse, w)
    v = x.double().requires_grad_()
    valid = ids >= 0
    at = ids.long().clamp_min(0)
    q = torch.where(valid, (tl.double() - lse.double()[:, None]).exp(), 0.0)
    logp = torch.log_softmax(v, 1)
    inside = torch.zeros(rows, vocab, dtype=torch.bool, device="cuda")
    for i in range(rows):
        inside[i, at[i][valid[i]]] = True
    qr = 1 - q.sum(1)
    lr = torch.logsumexp(logp.masked_fill(inside, -math.inf), 1)
    L = torch.where(valid, q * (q.clamp_min(1e-300).log() - logp.gather(1, at)), 0.0).sum(1) + qr * (qr.log() - lr)
    (L * w).sum().backward()
    # logits of one side differ by at most R; a term of its sum carries 3 R ln 2 EPS and 4 EPS, is rescaled at most 8 times,
    # and is one of vocab / 128 + 32 a thread and its fold adds
    R = 12.0 * 1.4427
    delta = EPS * (9 * (3 * R + 4) + vocab / 128 + 32)
    tol_L = delta + 2 * EPS * L.abs()
    assert bool(((got.row_losses.double() - L).abs() <= tol_L).all()), (got.row_losses, L)
    size = w[:, None] * torch.where(inside, (logp.exp() + q.sum(1, keepdim=True)), (logp - lr[:, None]).exp())
    half = torch.finfo(dtype).eps / 2
    # (2^l is 0 below 2^-126: a named token that takes another's place leaves its logit in the rest, and the others there
    # have shares near e^-gap; half of f16's least step is 2^-25)
    tol = 3 * delta * size + 1.01 * half * v.grad.abs() + (2.0**-25 if dtype == torch.float16 else 2.0**-126)
    bad = (got.grad.double() - v.grad).abs() > tol
    assert not bool(bad.any()), (int(bad.sum()), got.grad.double()[bad][:5], v.grad[bad][:5])


def test_no_rest_is_left_out(gpu_pkg):
    # all of the rest masked: the outcome that the student cannot give is left out, whatever share the teacher gives it
    x = torch.full((2, 300), -math.inf, device="cuda")
    ids = torch.tensor([[3, 299, 150], [0, 1, 2]], dtype=torch.int32, device="cuda")
    x[0, ids[0].long()] = torch.tensor([1.0, 2.0, -1.0], device="cuda")
    x[1, ids[1].long()] = torch.tensor([500.0, 2.0, -1.0], device="cuda")
    tl = torch.tensor([[0.5, 0.0, 0.25], [0.5, 0.0, 0.25]], device="cuda")
    lse = torch.logsumexp(tl, 1) + 0.5
    got = gpu_pkg.distill_loss(x, ids, tl, lse, torch.ones(2, device="cuda"))
    q = (tl - lse[:, None]).double().exp()
    logp = torch.log_softmax(x.double(), 1).gather(1, ids.long())
    want = (q * (q.log() - logp)).sum(1)
    assert bool(((got.row_losses - want).abs() <= 8 * EPS * (1 + want.abs())).all())
    grad = (logp.exp() * q.sum(1, keepdim=True) - q)
    assert bool(((got.grad.gather(1, ids.long()) - grad).abs() <= 8 * EPS).all())
    rest = got.grad.scatter(1, ids.long(), 0.0)
    assert not bool(rest.any()) and bool(torch.isfinite(rest).all())


@pytest.mark.parametrize("cap", [30.0, 20.0, 50.0, 0.37, 1000.0])
def test_soft_cap_is_as_exact_as_tanh(gpu_pkg, cap):
    """c(v) is within 4 half steps of cap tanh(v / cap), 0.8 of one in the mean, and off to no side, as cap * tanhf(v / cap) is."""
    # top_logits returns c(v) itself.  Half steps, |v| <= cap: the argument's product and 1 / cap 2, squared 5, felt by c at
    # 0.23 at most; v y and the polynomial 3, on 0.31 of c; the last step 1: 3.3.  Beyond: the exponential 5 and its
    # quotient 4, on 0.31 of c; the last step 1: 3.8.
    cap32 = float(np.float32(cap))
    g = torch.Generator(device="cuda").manual_seed(191)
    for lo, hi, dtype in ((0.0, 0.5, torch.float32), (0.0, 1.0, torch.float32), (0.9, 1.5, torch.float32), (1.0, 9.0, torch.float32),
                          (0.0, 1.0, torch.bfloat16)):
        v = (lo + (hi - lo) * torch.rand(64, 1024, generator=g, device="cuda")) * cap32
        v = (v * torch.where(torch.rand(v.shape, generator=g, device="cuda") < 0.5, -1.0, 1.0)).to(dtype)
        got = gpu_pkg.top_logits(v, 1024, final_logit_softcapping=cap)
        c = got.logits.double()
        want = cap32 * torch.tanh(v.double().gather(1, got.ids.long()) / cap32)
        some = want != 0
        off = ((c - want) / want)[some] / EPS
        f32 = (cap32 * torch.tanh(v.float().gather(1, got.ids.long()) / cap32)).double()
        plain = ((f32 - want) / want)[some] / EPS
        assert float(off.abs().max()) <= 4.0, (lo, hi, float(off.abs().max()))
        assert float(off.square().mean().sqrt()) <= 1.15 * float(plain.square().mean().sqrt()), (lo, hi)
        if dtype == torch.float32 and hi <= 1.0:
            assert abs(float(off.mean())) <= 0.3, (lo, hi, float(off.mean()))
        x = torch.tensor([[math.inf, -math.inf, 0.0, 1e30, -1e30]], device="cuda")
        assert gpu_pkg.top_logits(x, 5, final_logit_softcapping=cap).logits.tolist() == [[cap32, cap32, 0.0, -cap32, -cap32]]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("vocab,off", [(64, 0), (1003, 1), (40000, 3)])
def test_gradient_where_the_soft_cap_saturates(gpu_pkg, dtype, vocab, off):
    """Each gradient element holds its own bits where the slope 1 / cosh^2(v / cap) is small, up to 8 cap."""
    cap, rows = 4.0, 4
    g = torch.Generator(device="cuda").manual_seed(201)
    x = torch.zeros(off + rows * vocab, dtype=dtype, device="cuda")[off:].view(rows, vocab)
    x.copy_(cap * 16.0 * (torch.rand(rows, vocab, generator=g, device="cuda") - 0.5))
    t = torch.tensor([0, vocab - 1, vocab // 2, 3], dtype=torch.int32, device="cuda")
    x[0, 0], x[1, vocab - 1], x[2, vocab // 2], x[3, 3] = 7.5 * cap, -7.5 * cap, 0.99 * cap, 4.0 * cap
    v = x.double()
    slope = 1 / torch.cosh(v / cap) ** 2
    z = cap * torch.tanh(v / cap)
    logp = torch.log_softmax(z, 1)
    p, H = logp.exp(), -(logp.exp() * logp).sum(1, keepdim=True)
    hot = torch.zeros_like(p).scatter_(1, t.long()[:, None], 1.0)
    # a term of the sum: d up to 8 log2(e) = 11.6, 3 R EPS; ex2 4; c off by 4 half steps of cap at most, twice; 8 rescalings
    delta = EPS * (9 * (3 * 11.6 + 4 + 8 * cap) + vocab / 128 + 32)
    w = torch.tensor([1.0, 0.5, -2.0, 1.0], device="cuda")
    wd = w.double()[:, None]
    half, tiny = torch.finfo(dtype).eps / 2, (2.0**-25 if dtype == torch.float16 else 2.0**-126)

    def check(got, pre, size, what):
        # the slope: t twice (4 half steps each) on at most 0.58 of it, over 0.42; beyond, the exponent's rounding (18 at
        # 9 cap, 16 here), the exponential's 4 and the quotient's 4, twice: 30 half steps with the products
        out = pre * slope
        tol = slope * (delta * size + 40 * EPS * size) + 1.01 * half * out.abs() + tiny
        bad = (got.double() - out).abs() > tol
        assert not bool(bad.any()), (what, int(bad.sum()), got.double()[bad][:4], out[bad][:4])

    r = gpu_pkg.token_logprobs(x, t, final_logit_softcapping=cap)
    got = gpu_pkg.token_logprobs_grad(x, t, r, w, 0.25 * w, final_logit_softcapping=cap)
    size = wd.abs() * (hot + p + 0.25 * p * (3 * logp.abs() + 3 * H + 3))
    check(got, wd * (hot - p) - 0.25 * wd * p * (logp + H), size, "log-probabilities")
    lp = (hot * logp).sum(1)
    got = gpu_pkg.policy_loss(x, t, lp.float(), torch.ones(rows, device="cuda"), None, w, final_logit_softcapping=cap).grad
    ratio = (lp - lp.float().double()).exp()[:, None]
    check(got, -wd * ratio * (hot - p), 3 * wd.abs() * (hot + p), "policy")
    ids = torch.stack([torch.randperm(vocab, generator=g, device="cuda")[:9] for _ in range(rows)]).int()
    ids[0, 0], ids[1, 0] = 0, vocab - 1
    ids[0, 1:][ids[0, 1:] == 0] = -1
    ids[1, 1:][ids[1, 1:] == vocab - 1] = -1
    tl = torch.randn(rows, 9, generator=g, device="cuda")
    lse = torch.logsumexp(tl, 1) + 0.7
    valid = ids >= 0
    for tail in (None, lse):
        got = gpu_pkg.distill_loss(x, ids, tl, tail, w, final_logit_softcapping=cap).grad
        u = torch.where(valid, tl.double(), -math.inf)
        q = torch.softmax(u, 1) if tail is None else torch.where(valid, (u - tail.double()[:, None]).exp(), 0.0)
        spread = torch.zeros_like(p).scatter_add_(1, ids.long().clamp_min(0), torch.where(valid, q, 0.0))
        factor, big = torch.ones_like(p), torch.ones_like(p)
        if tail is not None:
            inside = torch.zeros_like(p).scatter_add_(1, ids.long().clamp_min(0), valid.double()) > 0
            qr = 1 - q.sum(1, keepdim=True)
            pr = torch.where(inside, 0.0, p).sum(1, keepdim=True)
            factor = torch.where(inside, 1.0, 1 - qr / pr)
            big = torch.where(inside, 1.0, 1 + qr / pr)
        check(got, wd * (p * factor - spread), 3 * wd.abs() * (p * big + spread), ("distillation", tail is not None))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("rows", [1, 600])
def test_small_terms_beside_a_large_one(gpu_pkg, dtype, rows):
    # one term of 1 and 131071 of 2^-25, which one by one round away against it (the row holds 3.9e-3 of them)
    vocab, T = 131072, float(np.float32(1.0 / math.log(2.0)))
    x = torch.full((rows, vocab), -25.0, dtype=dtype, device="cuda")
    at = torch.arange(rows, device="cuda") * 211 % vocab
    x[torch.arange(rows, device="cuda"), at] = 0.0
    want = -math.log1p((vocab - 1) * math.exp(-25.0 / T))
    # at most 16 terms that share a step with the large one are lost; then one rounding for each of the sum's folds: 5
    # between a warp's lanes, 4 between warps, 3 between blocks, and the last chunk steps
    tol = 16 * 2.0**-25 + 16 * EPS
    r = gpu_pkg.token_logprobs(x, at.int(), temperature=T)
    assert float((r.logprobs.double() - want).abs().max()) <= tol
    top = gpu_pkg.top_logits(x, 3, temperature=T)
    assert float((top.lse.double() + want).abs().max()) <= tol
    one = torch.ones(rows, device="cuda")
    p = gpu_pkg.policy_loss(x, at.int(), 0 * one, one, None, one, temperature=T)
    assert float((p.logprobs.double() - want).abs().max()) <= tol


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("rows,vocab", [(1, 131072), (3, 40000), (600, 131072), (700, 8192)])
def test_a_very_likely_token(gpu_pkg, dtype, rows, vocab):
    """ln S of S = 1 + some 1e-5: what the fold of a row's sums would round away beside the 1."""
    # d is a whole number and every term a power of two, as above; the small ones keep off the elements that the large one's
    # thread would sum by itself (the first chunk of each step), where they meet it in f32
    T = float(np.float32(1.0 / math.log(2.0)))
    at = [p for p in range(100, vocab, 53) if min(p % 1024, p % 2048, p % 2560, p % 4096) >= 16][:500]
    x = torch.full((rows, vocab), -math.inf, dtype=dtype, device="cuda")
    x[:, 0] = 0.0
    x[:, at] = -25.0
    want = math.log1p(len(at) * math.exp(-25.0 / T))
    t = torch.zeros(rows, dtype=torch.int32, device="cuda")
    one = torch.ones(rows, device="cuda")
    # the result's rounding, 64 bits before it; the correction of k's rounding goes to first order
    relative(gpu_pkg.token_logprobs(x, t, temperature=T).logprobs, [-want] * rows, 2 * EPS, "log-probability")
    # (without the entropy's sum there is no correction: k is off by half a step at most, which a term of d = -25 feels
    # 25 ln 2 = 17.4 times)
    relative(gpu_pkg.top_logits(x, 3, temperature=T).lse, [want] * rows, (2 + 17.4) * EPS, "lse")
    p = gpu_pkg.policy_loss(x, t, 0 * one, one, None, one, temperature=T)
    relative(p.logprobs, [-want] * rows, 2 * EPS, "log-probability of the policy loss")
