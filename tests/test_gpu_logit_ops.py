"""The vocabulary-row operators on the GPU against plain implementations in 64 bits.

Tolerances count roundings.  EPS = 2^-24 is half a step of f32.  With
d_j = (c_j - M) k in base 2, R = max |d_j| over the terms that count (those of
2^-150 and more), a term 2^d carries at most 3 R EPS from d (k, difference,
product) and 4 EPS from ex2.approx (2^-22); with a soft-cap c_j is off by at
most 12 EPS cap (two sums of positive terms, 3 EPS each; their fit, 1; the
argument, 1; three products and the reciprocal's unit, 4), so d by 18 EPS cap m.
A term is rescaled at most 8 times on its way into the sum (each time like a
term), and added in at most V / 128 steps of a thread and 32 between threads.
So log p and ln S are off by at most

    delta = EPS (9 (3 R + 4 + 18 cap m) + V / 128 + 32),

a probability by delta relative, the entropy by 2 delta (H + 2); the soft-cap's
slope 1 - (c / cap)^2 by 24 EPS, and the gradient's products by 16 EPS more.
"""
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

EPS = 2.0**-24
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
HALF = {"f32": 2.0**-24, "bf16": 2.0**-8, "f16": 2.0**-11}   # half a step, relative
TINY = {"f32": 2.0**-126, "bf16": 2.0**-126, "f16": 2.0**-25}  # flushed or half the least step


def make(rows, vocab, dtype, seed, ld=None, off=0, scale=3.0):
    """rows x vocab logits as a view into a larger buffer of a sentinel."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    ld = ld or vocab
    buf = torch.full((off + rows * ld + 64,), 77.0, dtype=TYPES[dtype], device="cuda")
    x = buf[off:off + rows * ld].view(rows, ld)[:, :vocab]
    v = scale * torch.randn(rows, vocab, generator=g, device="cuda")
    v[:, torch.randint(0, vocab, (4,), generator=g, device="cuda")] += 8.0
    x.copy_(v)
    return x, buf


class Ref:
    """64-bit values of rows of logits."""

    def __init__(self, x, T=1.0, cap=0.0, scale=1.0):
        v = x.double()
        self.m = 1.0 / (scale * T)
        c = cap * torch.tanh(v / cap) if cap else v
        self.slope = 1 - torch.tanh(v / cap) ** 2 if cap else torch.ones_like(v)
        z = c * self.m
        self.c, self.z = c, z
        self.lse = torch.logsumexp(z, 1)
        self.logp = z - self.lse[:, None]
        self.p = self.logp.exp()
        self.H = -(self.p * self.logp.clamp_min(-1e30)).sum(1)
        d = ((z.amax(1, keepdim=True) - z) * 1.4426950408889634).clamp_max(150.0)
        R = d.amax(1)
        self.delta = EPS * (9 * (3 * R + 4 + 18 * cap * self.m) + x.shape[1] / 128 + 32)
        self.tol_H = 2 * self.delta * (self.H + 2)

    def token(self, t):
        t = t.long()
        live = (t >= 0) & (t < self.z.shape[1])
        at = torch.where(live, t, 0)
        lp = self.logp.gather(1, at[:, None])[:, 0]
        hot = torch.zeros_like(self.p).scatter_(1, at[:, None], 1.0)
        return live, lp, hot

    def lp_tol(self, lp):
        return self.delta + 3 * EPS * lp.abs()   # the token's own difference, and the result's rounding

    def grad(self, dtype, hot, g, h, dg=0.0):
        """(gradient, its tolerance) from d/d logprob = g and d/d entropy = h."""
        col = lambda v: torch.as_tensor(v, dtype=torch.float64, device="cuda").expand(self.H.shape)[:, None]  # noqa: E731
        g, h, dg = col(g), col(h), col(dg)
        H, tol_H, delta = self.H[:, None], self.tol_H[:, None], self.delta[:, None]
        lp = self.logp.clamp_min(-1e3)
        pre = self.m * (g * (hot - self.p) - h * self.p * (lp + H))
        size = self.m * (g.abs() * (hot + self.p) + h.abs() * self.p * (lp.abs() + H.abs()))
        err = self.m * (g.abs() * self.p * delta + dg * (hot + self.p)
                        + h.abs() * self.p * (delta * (lp.abs() + H.abs() + 1) + tol_H)) + 40 * EPS * size
        out = pre * self.slope
        return out, err + HALF[dtype] * (out.abs() + err) + TINY[dtype]


def near(got, want, tol, what=""):
    got = got.double()
    bad = ~((got - want).abs() <= tol)
    assert not bool(bad.any()), (what, int(bad.sum()), float(((got - want).abs() / tol).nan_to_num(1e9).max()))


SHAPES = [  # rows, vocab, ld, offset in elements
    (1, 1, 1, 0), (3, 2, 2, 1), (2, 7, 9, 3), (5, 8, 8, 0), (4, 31, 33, 5), (3, 1000, 1000, 0), (37, 1025, 1025, 2),
    (2, 32003, 32003, 1), (6, 32000, 32768, 0), (150, 4099, 4100, 0), (1, 128256, 128256, 0), (3, 151936, 151936, 7),
    (2, 256000, 256000, 0), (1, 300001, 300001, 0), (9, 40000, 40000, 0), (17, 16385, 16385, 3),
]
T07 = float(np.float32(0.7))   # the C ABI takes the temperature as f32
FACTORS = [dict(T=1.0, cap=0.0, scale=1.0), dict(T=T07, cap=30.0, scale=2.0)]


def how(f):
    return dict(temperature=f["T"], final_logit_softcapping=f["cap"], logit_scale=f["scale"])


def tokens_for(rows, vocab, seed):
    t = torch.from_numpy(np.random.default_rng(seed).integers(0, vocab, rows).astype(np.int32)).cuda()
    if rows > 2:
        t[1] = -1
    return t


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("f", FACTORS, ids=["plain", "capped"])
def test_token_logprobs_and_gradient(gpu_pkg, dtype, shape, f):
    rows, vocab, ld, off = shape
    x, buf = make(rows, vocab, dtype, 1, ld, off)
    before = buf.clone()
    t = tokens_for(rows, vocab, 2)
    r = gpu_pkg.token_logprobs(x, t, **how(f))
    ref = Ref(x, **f)
    live, lp, hot = ref.token(t)
    near(r.logprobs, torch.where(live, lp, 0.0), ref.lp_tol(lp), "logprobs")
    near(r.entropy, torch.where(live, ref.H, 0.0), ref.tol_H, "entropy")
    g = torch.Generator(device="cuda").manual_seed(3)
    gl, gh = torch.randn(rows, generator=g, device="cuda"), torch.randn(rows, generator=g, device="cuda")
    for a, b in ((gl, gh), (gl, None), (None, gh)):
        got = gpu_pkg.token_logprobs_grad(x, t, r, a, b, **how(f))
        want, tol = ref.grad(dtype, hot, 0.0 if a is None else a.double(), 0.0 if b is None else b.double())
        assert got.dtype == x.dtype
        near(got, torch.where(live[:, None], want, 0.0), tol, "grad")
    # into a larger buffer, at another alignment: nothing beside the rows is written
    obuf = torch.full((rows * (vocab + 5) + 9,), 55.0, dtype=x.dtype, device="cuda")
    out = obuf[3:3 + rows * (vocab + 5)].view(rows, vocab + 5)[:, :vocab]
    again = gpu_pkg.token_logprobs_grad(x, t, r, gl, gh, out=out, **how(f))
    assert again.data_ptr() == out.data_ptr()
    assert torch.equal(out, gpu_pkg.token_logprobs_grad(x, t, r, gl, gh, **how(f)))
    mask = torch.ones_like(obuf, dtype=torch.bool)
    mask[3:3 + rows * (vocab + 5)].view(rows, vocab + 5)[:, :vocab] = False
    assert bool((obuf[mask] == 55.0).all())
    assert torch.equal(buf, before)


def policy_ref(ref, dtype, t, old, adv, rlp, w, lo, hi, klc, entc):
    live, lp, hot = ref.token(t)
    live = live & (w != 0)
    A, w = adv.double(), w.double()
    r = (lp - old.double()).exp()
    L = -torch.minimum(r * A, r.clamp(1 - lo, 1 + hi) * A)
    clipped = ((A > 0) & (r > 1 + hi)) | ((A < 0) & (r < 1 - lo))
    g = torch.where(clipped, 0.0, -r * A)
    size = r * A.abs()
    kl = torch.zeros_like(lp)
    tol_kl = kl
    tlp = ref.lp_tol(lp) + 2 * EPS
    if rlp is not None:
        d = rlp.double() - lp
        kl = torch.expm1(d) - d
        tol_kl = (torch.expm1(d).abs() + 4 * EPS) * (tlp + 4 * EPS) + EPS * kl + tlp**2
        L = L + klc * kl
        g = g - klc * torch.expm1(d)
        size = size + klc * (d.exp() + 1)
    L = L - entc * ref.H
    tol_L = (size * 2 + 1) * 2 * tlp + klc * tol_kl + entc * ref.tol_H + 4 * EPS * (L.abs() + size)
    zero = lambda v: torch.where(live, v, 0.0)  # noqa: E731
    grad, tol_g = ref.grad(dtype, hot, zero(g * w), zero(-entc * w), zero(w.abs() * size * 2 * tlp))
    return dict(live=live, L=zero(L), tol_L=tol_L, lp=zero(lp), H=zero(ref.H), kl=zero(kl), tol_kl=tol_kl, tlp=tlp,
                loss=(zero(L) * w).sum(), tol_loss=(tol_L * w.abs()).sum() + EPS * (zero(L) * w).sum().abs(),
                grad=torch.where(live[:, None], grad, 0.0), tol_g=tol_g)


def policy_inputs(ref, t, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rows = t.shape[0]
    _, lp, _ = ref.token(t)
    d = 0.3 * torch.randn(rows, generator=g, device="cuda").double()
    for edge in (math.log(0.9), math.log(1.3)):   # off the corners, where the gradient jumps
        d = torch.where((d - edge).abs() < 1e-3, edge + 2e-3, d)
    old = (lp - d).float()
    rlp = (lp + 0.3 * torch.randn(rows, generator=g, device="cuda")).float()
    adv = torch.randn(rows, generator=g, device="cuda")
    w = torch.rand(rows, generator=g, device="cuda") + 0.5
    if rows > 3:
        w[2] = 0.0
    return old, adv, rlp, w


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("f", FACTORS, ids=["plain", "capped"])
def test_policy_loss(gpu_pkg, dtype, shape, f):
    rows, vocab, ld, off = shape
    x, _ = make(rows, vocab, dtype, 11, ld, off)
    t = tokens_for(rows, vocab, 12)
    ref = Ref(x, **f)
    old, adv, rlp, w = policy_inputs(ref, t, 13)
    for klc, entc, weights in ((0.0, 0.0, None), (0.1, 0.0, w), (0.05, 0.02, w)):
        got = gpu_pkg.policy_loss(x, t, old, adv, rlp if klc else None, weights, clip_low=0.1, clip_high=0.3,
                                  kl_coef=klc, entropy_coef=entc, **how(f))
        ww = torch.full((rows,), 1.0 / rows, device="cuda") if weights is None else weights
        want = policy_ref(ref, dtype, t, old, adv, rlp if klc else None, ww, 0.1, 0.3, klc, entc)
        near(got.logprobs, want["lp"], want["tlp"], "logprobs")
        near(got.entropy, want["H"], ref.tol_H, "entropy")
        near(got.kl, want["kl"], want["tol_kl"], "kl")
        near(got.row_losses, want["L"], want["tol_L"], "rows")
        near(got.loss, want["loss"], want["tol_loss"] + 2 * EPS * (want["L"].abs() * ww.double()).sum(), "loss")
        near(got.grad, want["grad"], want["tol_g"], "grad")
        no = gpu_pkg.policy_loss(x, t, old, adv, rlp if klc else None, weights, clip_low=0.1, clip_high=0.3,
                                 kl_coef=klc, entropy_coef=entc, grad=False, **how(f))
        assert no.grad is None and abs(float(no.loss) - float(got.loss)) <= 2 * float(want["tol_loss"]) + 1e-12


def distill_ref(ref, dtype, ids, tl, tlse, w, T):
    V = ref.z.shape[1]
    ids = ids.long()
    valid = (ids >= 0) & (ids < V)
    at = torch.where(valid, ids, 0)
    u = torch.where(valid, tl.double() / T, -math.inf)
    live = valid.any(1) & (w != 0)
    w = w.double()
    if tlse is None:
        live = live & (u.amax(1) > -math.inf)
        q = torch.softmax(u, 1)
    else:
        q = torch.exp(u - tlse.double()[:, None])
    q = torch.where(valid, q, 0.0)
    lp = ref.logp.gather(1, at)
    L = torch.where(q > 0, q * (q.log() - lp), 0.0).sum(1)
    # a share is off by 8 EPS (exponent's rounding, expf, the division) and by the f32 of its 64-bit exponent, |u - ref| EPS
    dq = (8 + torch.where(q > 0, q.log(), 0.0).abs()) * EPS
    tol_L = torch.where(q > 0, q * (dq * (2 + q.log().abs() + lp.abs()) + ref.delta[:, None] + 3 * EPS * lp.abs()), 0.0).sum(1)
    spread = torch.zeros_like(ref.p).scatter_add_(1, at, q)
    spread_err = torch.zeros_like(ref.p).scatter_add_(1, at, q * dq)
    Q = q.sum(1)
    factor = Q[:, None].expand(ref.p.shape)
    err_f = ((q * dq).sum(1) + 4 * EPS)[:, None].expand(ref.p.shape)
    if tlse is not None:
        inside = torch.zeros_like(ref.p, dtype=torch.bool)
        inside.scatter_(1, at, valid) if bool(valid.all()) else [inside[i].index_fill_(0, at[i][valid[i]], True) for i in range(len(at))]
        rest = torch.where(inside, 0.0, ref.p).sum(1)
        qr = (1 - Q).clamp_min(0.0)
        has = (qr > 0) & (rest > 0)
        dqr = (q * dq).sum(1) + 2 * EPS   # absolute
        lr = torch.where(has, qr.clamp_min(1e-300).log() - rest.clamp_min(1e-300).log(), 0.0)
        L = L + torch.where(has, qr * lr, 0.0)
        tol_L = tol_L + dqr * (2 + lr.abs() + torch.log(1 / (qr + dqr))) + qr * 2 * ref.delta + qr * 3 * EPS * lr.abs()
        ratio = torch.where(has, qr / rest.clamp_min(1e-300), 0.0)
        err_r = torch.where(rest > 0, dqr / rest.clamp_min(1e-300), 0.0) + ratio * 2 * ref.delta
        factor = factor + torch.where(has, qr, 0.0)[:, None] - torch.where(inside, 0.0, ratio[:, None])
        err_f = err_f + dqr[:, None] + torch.where(inside, 0.0, err_r[:, None])
    mw = ref.m * w[:, None]
    pre = mw * (ref.p * factor - spread)
    err = mw.abs() * (ref.p * (factor.abs() * ref.delta[:, None] + err_f) + spread_err) \
        + 40 * EPS * mw.abs() * (ref.p * factor.abs() + spread)
    out = torch.where(live[:, None], pre * ref.slope, 0.0)
    tol = err + HALF[dtype] * (out.abs() + err) + TINY[dtype]
    L = torch.where(live, L, 0.0)
    tol_L = tol_L + 4 * EPS * L.abs() + 1e-30
    return dict(L=L, tol_L=tol_L, loss=(L * w).sum(), tol_loss=(tol_L * w.abs()).sum() + 2 * EPS * (L * w).abs().sum(),
                grad=out, tol_g=tol)


def teacher_for(x, K, seed, T):
    g = torch.Generator(device="cuda").manual_seed(seed)
    y = x.float() + torch.randn(x.shape, generator=g, device="cuda")
    tl, ids = torch.topk(y, K, dim=1)
    lse = torch.logsumexp(y.double() / T, 1).float()
    w = torch.rand(x.shape[0], generator=g, device="cuda") + 0.5
    if x.shape[0] > 3:
        w[2] = 0.0
    return tl, ids.int(), lse, w


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("f", FACTORS, ids=["plain", "capped"])
@pytest.mark.parametrize("tail", [False, True], ids=["slots", "tail"])
def test_distill_loss(gpu_pkg, dtype, shape, f, tail):
    rows, vocab, ld, off = shape
    x, _ = make(rows, vocab, dtype, 21, ld, off)
    ref = Ref(x, **f)
    for K in sorted({1, min(vocab, 5), min(vocab, 64), min(vocab, 1000)}):
        tl, ids, lse, w = teacher_for(x, K, 22, f["T"])
        if K >= 5:   # empty slots, one slot without a share, a row without a teacher
            ids[0, 3], tl[0, 3] = -1, float("nan")
            tl[0, 2] = -math.inf
            if rows > 4:
                ids[3, :] = vocab
                ids[4, 1] = 2**31 - 1
        got = gpu_pkg.distill_loss(x, ids, tl, lse if tail else None, w, **how(f))
        want = distill_ref(ref, dtype, ids, tl, lse if tail else None, w, f["T"])
        near(got.row_losses, want["L"], want["tol_L"], ("rows", K))
        near(got.loss, want["loss"], want["tol_loss"], ("loss", K))
        near(got.grad, want["grad"], want["tol_g"], ("grad", K))
        no = gpu_pkg.distill_loss(x, ids, tl, lse if tail else None, w, grad=False, **how(f))
        assert no.grad is None
        near(no.loss, want["loss"], want["tol_loss"], ("loss alone", K))


@pytest.mark.parametrize("tail", [False, True], ids=["slots", "tail"])
def test_distill_same_id_twice(gpu_pkg, tail):
    x, _ = make(3, 500, "f32", 31)
    ref = Ref(x)
    ids = torch.tensor([[7, 9, 7, 7, 30], [499, 499, 0, 0, 1], [4, 4, 4, 4, 4]], dtype=torch.int32, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(32)
    tl = torch.randn(3, 5, generator=g, device="cuda")
    lse = torch.logsumexp(tl, 1) + 0.5
    w = torch.ones(3, device="cuda")
    got = gpu_pkg.distill_loss(x, ids, tl, lse if tail else None, w)
    want = distill_ref(ref, "f32", ids, tl, lse if tail else None, w, 1.0)
    near(got.row_losses, want["L"], want["tol_L"], "rows")
    near(got.grad, want["grad"], want["tol_g"], "grad")
    again = gpu_pkg.distill_loss(x, ids, tl, lse if tail else None, w)
    assert torch.equal(again.grad, got.grad)


def test_distill_teacher_covers_the_vocabulary(gpu_pkg):
    # nothing is left for the rest: the outcome is left out, whatever 1 - sum q rounds to
    x, _ = make(4, 64, "f32", 33)
    y, _ = make(4, 64, "f32", 34)
    top = gpu_pkg.top_logits(y, 64)
    w = torch.ones(4, device="cuda")
    got = gpu_pkg.distill_loss(x, top.ids, top.logits, top.lse, w)
    want = distill_ref(Ref(x), "f32", top.ids, top.logits, top.lse, w, 1.0)
    near(got.row_losses, want["L"], want["tol_L"], "rows")
    near(got.grad, want["grad"], want["tol_g"], "grad")
    # a teacher all of whose logits are -inf gives no share
    bad = torch.full_like(top.logits, -math.inf)
    none = gpu_pkg.distill_loss(x, top.ids, bad, None, w)
    assert float(none.loss) == 0.0 and not bool(none.grad.any()) and not bool(none.row_losses.any())


def top_ref(x, k):
    """Stable sort on the host: NaN below -inf, the lower id first among equals."""
    v = x.float().cpu().numpy()
    key = np.where(np.isnan(v), -np.inf, v).astype(np.float64)
    nan = np.isnan(v)
    ids = np.stack([np.lexsort((np.arange(v.shape[1]), -key[i], nan[i]))[:k] for i in range(v.shape[0])])
    return ids, np.take_along_axis(v, ids, 1)


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("f", FACTORS, ids=["plain", "capped"])
def test_top_logits(gpu_pkg, dtype, shape, f):
    rows, vocab, ld, off = shape
    x, _ = make(rows, vocab, dtype, 41, ld, off)
    ref = Ref(x, **f)
    ids, _ = top_ref(x, min(vocab, 1024))
    for k in sorted({1, min(vocab, 2), min(vocab, 20), min(vocab, 64), min(vocab, 257), min(vocab, 1024)}):
        got = gpu_pkg.top_logits(x, k, **how(f))
        assert np.array_equal(got.ids.cpu().numpy(), ids[:, :k]), k
        want = (ref.c / f["scale"]).gather(1, got.ids.long())
        if f["cap"] == 0.0 and f["scale"] == 1.0:
            assert torch.equal(got.logits.double(), want)
        else:
            near(got.logits, want, 14 * EPS * f["cap"] / f["scale"], "logits")
        near(got.lse, ref.lse, ref.delta + 3 * EPS * ref.lse.abs() + 3 * EPS * ref.z.amax(1).abs(), "lse")


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("vocab", [5, 700, 32003, 128256])
def test_top_logits_ties_and_odd_values(gpu_pkg, dtype, vocab):
    low = torch.finfo(TYPES[dtype]).min
    g = torch.Generator(device="cuda").manual_seed(51)
    rows = [torch.full((vocab,), 1.25), torch.full((vocab,), -math.inf), torch.full((vocab,), low),
            torch.randint(0, 3, (vocab,)).float(), torch.zeros(vocab), torch.full((vocab,), float("nan")),
            torch.randn(vocab).round() * 0.5]
    x = torch.stack(rows).cuda()
    x[4, ::3] = -0.0                                     # +0 and -0 are equal
    x[6, torch.randint(0, vocab, (vocab // 4 + 1,), generator=g, device="cuda")] = float("nan")
    x[6, vocab // 2] = math.inf
    x[1, vocab - 1] = low
    x = x.to(TYPES[dtype])
    for k in sorted({1, min(vocab, 3), min(vocab, 100), min(vocab, 1024)}):
        got = gpu_pkg.top_logits(x, k)
        ids, vals = top_ref(x, k)
        assert np.array_equal(got.ids.cpu().numpy(), ids), k
        assert np.array_equal(got.logits.cpu().numpy(), vals, equal_nan=True), k
    lse = gpu_pkg.top_logits(x, 1).lse.double()
    want = torch.logsumexp(x.double(), 1)
    assert torch.equal(lse.isnan(), torch.tensor([0, 0, 0, 0, 0, 1, 1], device="cuda").bool())
    tol = EPS * (9 * 22 * 3 + vocab / 128 + 32) + 3 * EPS * want.abs()
    near(lse[:5], want[:5], tol[:5], "lse")


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("vocab", [9000, 50001, 128256])
def test_top_logits_hard_rows(gpu_pkg, dtype, vocab):
    g = torch.Generator(device="cuda").manual_seed(55)
    x = torch.randn(6, vocab, generator=g, device="cuda")
    x[0, torch.arange(vocab, device="cuda") % 997 != 5] = -math.inf      # fewer tokens left than wanted
    x[1] = torch.arange(vocab, device="cuda").float() / 64.0             # the largest side by side
    x[2] = -torch.arange(vocab, device="cuda").float().div(700).floor()  # long runs of equal ones
    x[3] = -20.0 - x[3].abs() * 1e-3                                     # all below zero, close together
    x[4, vocab // 2:vocab // 2 + 3000] += 50.0
    x[5] = x[5] * 1e-30
    x = x.to(TYPES[dtype])
    for k in (1, 50, 700, 1024):
        got = gpu_pkg.top_logits(x, k)
        ids, vals = top_ref(x, k)
        assert np.array_equal(got.ids.cpu().numpy(), ids), k
        assert np.array_equal(got.logits.cpu().numpy(), vals), k


def test_masked_logits(gpu_pkg):
    """-inf and the type's lowest value as masks; a row that the mask empties; NaN and +inf."""
    for dtype in TYPES:
        low = torch.finfo(TYPES[dtype]).min
        x, _ = make(8, 5000, dtype, 61)
        x[0, 100:] = -math.inf
        x[1, 100:] = low
        x[2, :] = low                    # uniform
        x[3, :] = -math.inf              # no distribution
        x[4, 17] = float("nan")
        x[5, 17] = math.inf
        x[6, 1:] = -math.inf             # one token left
        x[7, :] = float("nan")           # left out below: never looked at
        t = torch.tensor([50, 50, 4999, 3, 3, 3, 0, -1], dtype=torch.int32, device="cuda")
        r = gpu_pkg.token_logprobs(x, t)
        ref = Ref(torch.where(torch.isfinite(x), x, x).clone())
        assert r.logprobs.isnan().tolist() == [False, False, False, True, True, True, False, False]
        assert r.entropy.isnan().tolist() == [False, False, False, True, True, True, False, False]
        tol = 1500 * EPS   # delta at R = 40
        want = ref.logp.gather(1, t.clamp_min(0).long()[:, None])[:, 0]
        for i in (0, 1):
            assert abs(float(r.logprobs[i]) - float(want[i])) <= tol
        assert abs(float(r.logprobs[2]) + math.log(5000)) <= tol and abs(float(r.entropy[2]) - math.log(5000)) <= 2 * tol * 11
        assert float(r.logprobs[6]) == 0.0 and float(r.entropy[6]) == 0.0
        assert float(r.logprobs[7]) == 0.0 and float(r.entropy[7]) == 0.0
        one = torch.ones(8, device="cuda")
        for gr in (gpu_pkg.token_logprobs_grad(x, t, r, one, 0.5 * one),
                   gpu_pkg.policy_loss(x, t, r.logprobs.nan_to_num(0.0), -one, None, one, entropy_coef=-0.5).grad):
            for i in (0, 1, 6):
                assert bool(torch.isfinite(gr[i]).all()), i
                assert not bool(gr[i, 100:].any())
            for i in (3, 4, 5):
                assert bool(gr[i].isnan().any()), i
            assert not bool(gr[7].any()) and not bool(gr[7].isnan().any())
        p = gpu_pkg.policy_loss(x, t, r.logprobs.nan_to_num(0.0), one, None, one)
        assert p.row_losses.isnan().tolist() == [False, False, False, True, True, True, False, False]
        assert bool(p.loss.isnan())
        w = one.clone()
        w[3:6] = 0.0                     # rows of weight 0 stay out of everything
        p = gpu_pkg.policy_loss(x, t, r.logprobs.nan_to_num(0.0), one, None, w)
        assert bool(torch.isfinite(p.loss)) and bool(torch.isfinite(p.grad).all())
        d = gpu_pkg.distill_loss(x, torch.arange(4, dtype=torch.int32, device="cuda").repeat(8, 1),
                                 torch.zeros(8, 4, device="cuda"), None, torch.cat([w[:7], w[3:4]]))
        assert bool(torch.isfinite(d.grad[:6]).all()) and not bool(d.grad[3:6].any()) and not bool(d.grad[7].any())


def test_largest_vocabulary(gpu_pkg):
    V = gpu_pkg.logit_ops.MAX_VOCAB
    x, _ = make(2, V, "f32", 65)
    ref = Ref(x)
    t = torch.tensor([V - 1, 5], dtype=torch.int32, device="cuda")
    _, lp, hot = ref.token(t)
    r = gpu_pkg.token_logprobs(x, t)
    near(r.logprobs, lp, ref.lp_tol(lp), "logprobs")
    top = gpu_pkg.top_logits(x, 1024)
    assert np.array_equal(top.ids.cpu().numpy(), top_ref(x, 1024)[0])
    w = torch.ones(2, device="cuda")
    for lse in (None, top.lse):
        got = gpu_pkg.distill_loss(x, top.ids, top.logits, lse, w)
        want = distill_ref(ref, "f32", top.ids, top.logits, lse, w, 1.0)
        near(got.grad, want["grad"], want["tol_g"], "grad")
    old, adv, rlp, _ = policy_inputs(ref, t, 66)
    got = gpu_pkg.policy_loss(x, t, old, adv, rlp, w, clip_low=0.1, clip_high=0.3, kl_coef=0.1, entropy_coef=0.01)
    want = policy_ref(ref, "f32", t, old, adv, rlp, w, 0.1, 0.3, 0.1, 0.01)
    near(got.grad, want["grad"], want["tol_g"], "grad")


def test_rows_past_32_bits(gpu_pkg):
    # element offsets above 2^32: rows of a large stride, the last one checked
    rows, vocab, ld = 3, 1000, (1 << 31) + 8
    buf = torch.zeros((rows - 1) * ld + vocab, dtype=torch.bfloat16, device="cuda")
    x = buf.as_strided((rows, vocab), (ld, 1))
    src, _ = make(rows, vocab, "bf16", 67)
    x.copy_(src)
    t = torch.tensor([1, 2, 3], dtype=torch.int32, device="cuda")
    a, b = gpu_pkg.token_logprobs(x, t), gpu_pkg.token_logprobs(src, t)
    assert torch.equal(a.logprobs, b.logprobs)
    one = torch.ones(rows, device="cuda")
    assert torch.equal(gpu_pkg.token_logprobs_grad(x, t, a, one, one), gpu_pkg.token_logprobs_grad(src, t, b, one, one))
    p, q = gpu_pkg.top_logits(x, 10), gpu_pkg.top_logits(src, 10)
    assert torch.equal(p.ids, q.ids)
    want = gpu_pkg.policy_loss(src, t, a.logprobs, one)
    got = gpu_pkg.policy_loss(x, t, a.logprobs, one, out=x)
    assert got.grad.data_ptr() == x.data_ptr() and torch.equal(x, want.grad)


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("vocab", [1001, 128256])
def test_gradient_over_the_logits(gpu_pkg, dtype, vocab):
    x, _ = make(9, vocab, dtype, 71)
    t = tokens_for(9, vocab, 72)
    old, adv, rlp, w = policy_inputs(Ref(x), t, 73)
    want = gpu_pkg.policy_loss(x, t, old, adv, rlp, w, kl_coef=0.1, entropy_coef=0.01)
    y = x.clone()
    got = gpu_pkg.policy_loss(y, t, old, adv, rlp, w, kl_coef=0.1, entropy_coef=0.01, out=y)
    assert torch.equal(y, want.grad) and torch.equal(got.row_losses, want.row_losses)
    tl, ids, lse, w = teacher_for(x, 50, 74, 1.0)
    for s in (None, lse):
        want, y = gpu_pkg.distill_loss(x, ids, tl, s, w), x.clone()
        gpu_pkg.distill_loss(y, ids, tl, s, w, out=y)
        assert torch.equal(y, want.grad)
    r, one = gpu_pkg.token_logprobs(x, t), torch.ones(9, device="cuda")
    want, y = gpu_pkg.token_logprobs_grad(x, t, r, one, one), x.clone()
    gpu_pkg.token_logprobs_grad(y, t, r, one, one, out=y)
    assert torch.equal(y, want)


def differences(loss, x, at, h=2.0**-5):
    """Central differences with one step of extrapolation, in the loss's own arithmetic."""
    out = []
    for i, j in at:
        d = []
        for step in (h, 2 * h):
            v = []
            for s in (step, -step):
                y = x.clone()
                y[i, j] += s
                v.append(float(loss(y)))
            d.append((v[0] - v[1]) / (2 * step))
        out.append((4 * d[0] - d[1]) / 3)
    return out


def test_gradients_against_differences(gpu_pkg):
    # 5-point differences at h = 2^-5: truncation h^4/30 |f^(5)| < 1e-6 for these losses (a softmax's derivatives
    # are below 10 there); f32 losses of size 1 with an error of delta ~ 2e-6 at worst give 3 delta / h ~ 2e-4
    x, _ = make(3, 40, "f32", 81, scale=1.0)
    t = torch.tensor([3, 39, 0], dtype=torch.int32, device="cuda")
    ref = Ref(x, 0.9, 20.0)
    old, adv, rlp, _ = policy_inputs(ref, t, 82)
    w = torch.tensor([1.0, 0.5, 0.25], device="cuda")
    f = dict(temperature=0.9, final_logit_softcapping=20.0)
    tl, ids, lse, _ = teacher_for(x, 6, 83, 0.9)
    at = [(0, 3), (0, 10), (1, 39), (2, 0), (2, 21)] + [(1, int(ids[1, 2])), (0, int(ids[0, 0]))]

    def logprob_sum(y):
        r = gpu_pkg.token_logprobs(y, t, **f)
        return (w.double() * (r.logprobs.double() - 0.3 * r.entropy.double())).sum()

    cases = {
        "policy": (lambda y, **k: gpu_pkg.policy_loss(y, t, old, adv, rlp, w, clip_low=5.0, clip_high=5.0, kl_coef=0.2,
                                                      entropy_coef=0.05, **f, **k)),
        "slots": (lambda y, **k: gpu_pkg.distill_loss(y, ids, tl, None, w, **f, **k)),
        "tail": (lambda y, **k: gpu_pkg.distill_loss(y, ids, tl, lse, w, **f, **k)),
    }
    for name, call in cases.items():
        g = call(x).grad
        for (i, j), d in zip(at, differences(lambda y: call(y, grad=False).row_losses.double() @ w.double(), x, at)):
            assert abs(float(g[i, j]) - d) <= 3e-4, (name, i, j)
    g = gpu_pkg.token_logprobs_grad(x, t, gpu_pkg.token_logprobs(x, t, **f), w, -0.3 * w, **f)
    for (i, j), d in zip(at, differences(logprob_sum, x, at)):
        assert abs(float(g[i, j]) - d) <= 3e-4, ("logprobs", i, j)


def test_inputs_in_other_forms(gpu_pkg):
    x, _ = make(6, 1003, "bf16", 91)
    t32 = tokens_for(6, 1003, 92)
    t64 = t32.long()
    t64[1] = -100
    t64[3] = 2**32 + 5        # no id: int32 would wrap it to 5
    want32 = t32.clone()
    want32[3] = -1
    a, b = gpu_pkg.token_logprobs(x, t64), gpu_pkg.token_logprobs(x, want32)
    assert torch.equal(a.logprobs, b.logprobs) and float(a.logprobs[3]) == 0.0
    wide = torch.stack([t32, t32], 1)[:, 0]               # a strided column
    assert torch.equal(gpu_pkg.token_logprobs(x, wide).logprobs, gpu_pkg.token_logprobs(x, t32).logprobs)
    one = gpu_pkg.token_logprobs(x[0], t32[:1])           # one row, 1-D
    assert torch.equal(one.logprobs, gpu_pkg.token_logprobs(x[:1], t32[:1]).logprobs)
    old, adv = torch.zeros(6, device="cuda"), torch.ones(6, device="cuda")
    p = gpu_pkg.policy_loss(x, t32, old.double(), adv.half())
    assert torch.equal(p.grad, gpu_pkg.policy_loss(x, t32, old, adv).grad)
    assert gpu_pkg.policy_loss(x[0], t32[:1], old[:1], adv[:1]).grad.shape == (1003,)
    e = x[:0]
    assert gpu_pkg.token_logprobs(e, t32[:0]).logprobs.shape == (0,)
    z = gpu_pkg.policy_loss(e, t32[:0], old[:0], adv[:0])
    assert float(z.loss) == 0.0 and z.grad.shape == (0, 1003)
    z = gpu_pkg.distill_loss(e, t32[:0, None], old[:0, None])
    assert float(z.loss) == 0.0 and z.grad.shape == (0, 1003)
    assert gpu_pkg.top_logits(e, 3).ids.shape == (0, 3)


def test_refusals_on_device(gpu_pkg):
    x, _ = make(4, 50, "f32", 95)
    t, f = tokens_for(4, 50, 96), torch.zeros(4, device="cuda")
    r = gpu_pkg.token_logprobs(x, t)
    bad = [
        lambda: gpu_pkg.token_logprobs(x.double(), t), lambda: gpu_pkg.token_logprobs(x.t(), t),
        lambda: gpu_pkg.token_logprobs(x[:1].expand(4, 50), t), lambda: gpu_pkg.token_logprobs(x, t[:3]),
        lambda: gpu_pkg.token_logprobs(x, f), lambda: gpu_pkg.token_logprobs(x, t.cpu()),
        lambda: gpu_pkg.token_logprobs(x[None], t), lambda: gpu_pkg.token_logprobs(x[:, :0], t),
        lambda: gpu_pkg.token_logprobs_grad(x, t, r), lambda: gpu_pkg.token_logprobs_grad(x, t, r, f[:2]),
        lambda: gpu_pkg.token_logprobs_grad(x, t, r, f, out=torch.empty(4, 50, device="cuda", dtype=torch.half)),
        lambda: gpu_pkg.token_logprobs_grad(x[:3], t[:3], gpu_pkg.token_logprobs(x[:3], t[:3]), f[:3], out=x[1:]),
        lambda: gpu_pkg.top_logits(x, 0), lambda: gpu_pkg.top_logits(x, 51),
        lambda: gpu_pkg.distill_loss(x, t, f), lambda: gpu_pkg.distill_loss(x, t[:, None], f),
        lambda: gpu_pkg.distill_loss(x, t[:, None], f[:, None], f[:2]),
        lambda: gpu_pkg.policy_loss(x, t, f, f, kl_coef=0.1), lambda: gpu_pkg.policy_loss(x, t, f, f, weights=f[:2]),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was not refused")
    with pytest.raises(gpu_pkg.SamplerError):
        gpu_pkg.token_logprobs(x, t, temperature=0.0)
    with pytest.raises(gpu_pkg.SamplerError):
        gpu_pkg.policy_loss(x, t, f, f, clip_low=-1.0)


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("rows,vocab,ld", [(4000, 1031, 1031), (2500, 4096, 4096), (700, 40003, 40003), (400, 128256, 128256),
                                           (90, 256000, 256001)])
def test_many_rows(gpu_pkg, dtype, rows, vocab, ld):
    """Long runs of rows through the same thread blocks, left-out rows scattered and in runs among them."""
    x, _ = make(rows, vocab, dtype, 131, ld, 1 if ld % 8 else 0)
    g = torch.Generator(device="cuda").manual_seed(132)
    t = torch.randint(0, vocab, (rows,), generator=g, device="cuda").int()
    t[torch.rand(rows, generator=g, device="cuda") < 0.1] = -1
    ref = Ref(x)
    old, adv, rlp, w = policy_inputs(ref, t, 133)
    w[torch.rand(rows, generator=g, device="cuda") < 0.2] = 0.0
    w[rows // 3:rows // 3 + rows // 5] = 0.0
    got = gpu_pkg.policy_loss(x, t, old, adv, rlp, w, clip_low=0.1, clip_high=0.3, kl_coef=0.1, entropy_coef=0.01)
    want = policy_ref(ref, dtype, t, old, adv, rlp, w, 0.1, 0.3, 0.1, 0.01)
    near(got.row_losses, want["L"], want["tol_L"], "rows")
    near(got.loss, want["loss"], want["tol_loss"] + 2 * EPS * (want["L"].abs() * w.double()).sum(), "loss")
    near(got.grad, want["grad"], want["tol_g"], "grad")
    no = gpu_pkg.policy_loss(x, t, old, adv, rlp, w, clip_low=0.1, clip_high=0.3, kl_coef=0.1, entropy_coef=0.01, grad=False)
    near(no.row_losses, want["L"], want["tol_L"], "rows without a gradient")
    del got, no, want
    r = gpu_pkg.token_logprobs(x, t)
    live, lp, hot = ref.token(t)
    near(r.logprobs, torch.where(live, lp, 0.0), ref.lp_tol(lp), "logprobs")
    del hot
    for K in (7, 150):
        tl, ids, lse, _ = teacher_for(x, K, 134, 1.0)
        ids[torch.rand(rows, generator=g, device="cuda") < 0.1] = -1      # no teacher
        ids[::5, 1] = ids[::5, 0]                                         # an id twice
        for s in (None, lse):
            got = gpu_pkg.distill_loss(x, ids, tl, s, w)
            want = distill_ref(ref, dtype, ids, tl, s, w, 1.0)
            near(got.row_losses, want["L"], want["tol_L"], ("rows", K))
            near(got.grad, want["grad"], want["tol_g"], ("grad", K))
            no = gpu_pkg.distill_loss(x, ids, tl, s, w, grad=False)
            near(no.row_losses, want["L"], want["tol_L"], ("rows without a gradient", K))
    top = gpu_pkg.top_logits(x, 9)
    at = torch.linspace(0, rows - 1, 20).long().cuda()
    assert np.array_equal(top.ids[at].cpu().numpy(), top_ref(x[at], 9)[0])


def run_all(pkg, x, t, old, adv, rlp, w, ids, tl, lse, stream=None):
    """The operators together, as an update uses them."""
    r = pkg.token_logprobs(x, t, stream=stream)
    g = pkg.token_logprobs_grad(x, t, r, w, w, stream=stream)
    top = pkg.top_logits(x, 33, stream=stream)
    p = pkg.policy_loss(x, t, old, adv, rlp, w, kl_coef=0.1, entropy_coef=0.01, stream=stream)
    d = pkg.distill_loss(x, ids, tl, lse, w, stream=stream)
    return [r.logprobs, r.entropy, g, top.logits, top.ids, top.lse, p.loss, p.kl, p.grad, d.loss, d.grad]


def all_inputs(rows, vocab, dtype, seed):
    x, _ = make(rows, vocab, dtype, seed)
    t = tokens_for(rows, vocab, seed + 1)
    old, adv, rlp, w = policy_inputs(Ref(x), t, seed + 2)
    tl, ids, lse, _ = teacher_for(x, 40, seed + 3, 1.0)
    return [x, t, old, adv, rlp, w, ids, tl, lse]


def test_streams_and_graphs(gpu_pkg):
    ins = all_inputs(12, 32003, "bf16", 101)
    want = [v.clone() for v in run_all(gpu_pkg, *ins)]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    for form in (s, s.cuda_stream):
        got = run_all(gpu_pkg, *ins, stream=form)
        s.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    # two graphs captured from the same inputs, replayed at once on two streams, while eager calls run
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs = run_all(gpu_pkg, *ins)
        graphs.append((g, outs, torch.cuda.Stream()))
    other = all_inputs(12, 32003, "bf16", 202)
    want2 = [v.clone() for v in run_all(gpu_pkg, *other)]
    for a, b in zip(ins, other):
        a.copy_(b)                      # replayed graphs read the new values
    torch.cuda.synchronize()
    for _ in range(5):
        for g, _, st in graphs:
            with torch.cuda.stream(st):
                g.replay()
        eager = run_all(gpu_pkg, *other)
    torch.cuda.synchronize()
    for outs in [o for _, o, _ in graphs] + [eager]:
        assert all(torch.equal(a, b) for a, b in zip(outs, want2))


FIRST_CALL = """
import sys, torch
sys.path.insert(0, {root!r})
import __graft_entry__ as g
pkg = g.load_package()
x = torch.randn(40, 20000, device="cuda", dtype=torch.bfloat16)
t = torch.arange(40, device="cuda", dtype=torch.int32)
f = torch.full((40,), 0.02, device="cuda")
ids = torch.arange(4, device="cuda", dtype=torch.int32).repeat(40, 1)
tl = torch.randn(40, 4, device="cuda")
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
def run():
    r = pkg.token_logprobs(x, t)
    return [pkg.token_logprobs_grad(x, t, r, f, f), pkg.top_logits(x, 5).ids, pkg.policy_loss(x, t, f, f, f, f, kl_coef=0.1).grad,
            pkg.distill_loss(x, ids, tl, None, f).grad]
with torch.cuda.graph(graph):
    outs = run()
graph.replay()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(outs, run()))
print("captured")
"""


def test_first_call_may_be_captured(gpu_pkg):
    import subprocess
    import sys
    root = gpu_pkg.build.ROOT
    r = subprocess.run([sys.executable, "-c", FIRST_CALL.format(root=root)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "captured" in r.stdout, r.stderr[-2000:]


def test_calls_from_two_threads(gpu_pkg):
    import threading
    ins = [all_inputs(30, 32003, "bf16", 141), all_inputs(30, 32003, "bf16", 151)]
    want = [[v.clone() for v in run_all(gpu_pkg, *i)] for i in ins]
    torch.cuda.synchronize()
    bad = []

    def work(k):
        s = torch.cuda.Stream()
        for _ in range(20):
            got = run_all(gpu_pkg, *ins[k], stream=s)
            s.synchronize()
            if not all(torch.equal(a, b) for a, b in zip(got, want[k])):
                bad.append(k)

    threads = [threading.Thread(target=work, args=(k,)) for k in (0, 1)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


def test_same_call_same_bits(gpu_pkg):
    ins = all_inputs(300, 20011, "f32", 111)
    a = run_all(gpu_pkg, *ins)
    for _ in range(3):
        assert all(torch.equal(u, v) for u, v in zip(a, run_all(gpu_pkg, *ins)))


def test_sampler_path(gpu_pkg):
    """Draw, score the drawn tokens with the sampler's own factors, train on them and on a teacher's top logits."""
    rows, vocab = 16, 32003
    x, _ = make(rows, vocab, "f32", 121)
    s = gpu_pkg.Sampler(gpu_pkg.SamplerConfig(temperature=0.7, top_k=40, repetition_penalty=1.0), batch=rows, vocab=vocab)
    s.set_logit_prologue(30.0, 2.0)
    t = s.sample(x)
    r = s.token_logprobs(x, t)
    ref = Ref(x, float(np.float32(0.7)), 30.0, 2.0)
    _, lp, hot = ref.token(t)
    near(r.logprobs, lp, ref.lp_tol(lp) + EPS, "logprobs")
    f = dict(temperature=0.7, final_logit_softcapping=30.0, logit_scale=2.0)
    top = gpu_pkg.top_logits(x, 40, **f)
    assert bool((top.ids == t[:, None]).any(1).all())       # top-k 40 drew every token
    adv = torch.ones(rows, device="cuda")
    p = gpu_pkg.policy_loss(x, t, r.logprobs, adv, **f)
    # (two calls that split the row differently: each within lp_tol of the exact value)
    two = 2 * (ref.lp_tol(lp) + EPS)
    near(p.logprobs, r.logprobs.double(), two, "logprobs of the two calls")
    # the ratio's log is the 64-bit log-probability minus the other call's in f32: at most `two` and a rounding,
    # EPS |lp|; then expf's two units in the last place (4 EPS) and the product's rounding
    near(p.row_losses, -torch.ones_like(adv).double(), two + EPS * (lp.abs() + 6), "on-policy rows")
    d = gpu_pkg.distill_loss(x, top.ids, top.logits, top.lse, **f)   # the student is the teacher
    tol = distill_ref(ref, "f32", top.ids, top.logits, top.lse, adv / rows, float(np.float32(0.7)))
    near(d.row_losses, tol["L"], tol["tol_L"] + EPS * 64, "itself")
    # through a model: the LM head's gradient from the loss's
    head = torch.randn(vocab, 8, device="cuda", requires_grad=True)
    h = torch.randn(rows, 8, device="cuda")
    logits = h @ head.t()
    p = gpu_pkg.policy_loss(logits, t, r.logprobs, adv, entropy_coef=0.01)
    logits.backward(p.grad)
    assert torch.equal(head.grad, p.grad.t() @ h) or torch.allclose(head.grad, p.grad.t() @ h, rtol=1e-5, atol=1e-7)
    s.close()
