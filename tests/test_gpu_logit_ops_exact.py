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
