"""CPU checks of the vocabulary-row operators: what they refuse, at the C ABI
and in the Python mirror (no GPU is touched by a refused call)."""
import ctypes

import pytest

torch = pytest.importorskip("torch")

OK, EINVAL, ENOTSUP = 0, 1, 6
P = ctypes.c_void_p(4096)   # a pointer that no refused call follows


def desc(pkg, **over):
    f = dict(data=4096, ld=100, rows=4, vocab=100, dtype=0, temperature=1.0, final_logit_softcapping=0.0,
             logit_scale=1.0)
    f.update(over)
    return ctypes.byref(pkg.logit_ops.BsLogits(*(f[n] for n, _ in pkg.logit_ops.BsLogits._fields_)))


def calls(pkg, d):
    """Every entry point with otherwise valid arguments."""
    L = pkg.lib()
    cfg = ctypes.byref(pkg.logit_ops.BsPolicyConfig(0.2, 0.2, 0.0, 0.0))
    return {
        "logprobs": lambda: L.bs_token_logprobs(d, P, P, P, P, None),
        "grad": lambda: L.bs_token_logprobs_grad(d, P, P, P, P, None, P, 100, None),
        "top": lambda: L.bs_top_logits(d, 5, P, P, P, P, 1 << 20, None),
        "distill": lambda: L.bs_distill_loss(d, P, P, None, 3, None, P, P, P, 100, None),
        "policy": lambda: L.bs_policy_loss(d, P, P, P, None, None, cfg, P, P, None, None, None, P, 100, None),
    }


BAD = {
    "null data": dict(data=None), "vocab 0": dict(vocab=0), "rows overlap": dict(ld=99), "type": dict(dtype=3),
    "vocabulary too large": dict(vocab=1048577, ld=1048577), "misaligned": dict(data=4098),
    "T 0": dict(temperature=0.0), "T < 0": dict(temperature=-1.0), "T NaN": dict(temperature=float("nan")),
    "T inf": dict(temperature=float("inf")), "T tiny": dict(temperature=1e-45), "T huge": dict(temperature=3e38, logit_scale=1e10),
    "cap NaN": dict(final_logit_softcapping=float("nan")), "cap inf": dict(final_logit_softcapping=float("inf")),
    "scale < 0": dict(logit_scale=-2.0), "scale NaN": dict(logit_scale=float("nan")), "too many rows": dict(rows=2**31),
}


@pytest.mark.parametrize("why", sorted(BAD))
def test_descriptor_refusals(pkg, why):
    for name, call in calls(pkg, desc(pkg, **BAD[why])).items():
        assert call() == EINVAL, name


def test_argument_refusals(pkg):
    L = pkg.lib()
    d = desc(pkg)
    cfg = lambda *a: ctypes.byref(pkg.logit_ops.BsPolicyConfig(*a))  # noqa: E731
    good = cfg(0.2, 0.2, 0.0, 0.0)
    nan, inf = float("nan"), float("inf")
    odd = ctypes.c_void_p(4098)
    assert L.bs_token_logprobs(None, P, P, P, P, None) == EINVAL
    assert L.bs_token_logprobs(d, None, P, P, P, None) == EINVAL
    assert L.bs_token_logprobs(d, P, None, P, P, None) == EINVAL
    assert L.bs_token_logprobs(d, P, P, P, ctypes.c_void_p(4100), None) == EINVAL
    g = L.bs_token_logprobs_grad
    assert g(d, P, P, P, None, None, P, 100, None) == EINVAL        # no gradient comes in
    assert g(d, P, P, None, None, P, P, 100, None) == EINVAL        # the entropy's needs the entropy
    assert g(d, P, None, P, P, None, P, 100, None) == EINVAL
    assert g(d, P, P, P, P, None, None, 100, None) == EINVAL
    assert g(d, P, P, P, P, None, P, 99, None) == EINVAL
    assert g(d, P, P, P, P, None, odd, 100, None) == EINVAL
    assert L.bs_top_logits(d, 0, P, P, P, P, 1 << 20, None) == EINVAL
    assert L.bs_top_logits(d, 101, P, P, P, P, 1 << 20, None) == EINVAL
    assert L.bs_top_logits(desc(pkg, vocab=5000, ld=5000), 1025, P, P, P, P, 1 << 20, None) == ENOTSUP
    assert L.bs_top_logits(d, 5, None, P, P, P, 1 << 20, None) == EINVAL
    need = L.bs_top_logits_workspace(d)
    assert need > 0
    assert L.bs_top_logits(d, 5, P, P, P, None, need, None) == EINVAL
    assert L.bs_top_logits(d, 5, P, P, P, P, need - 1, None) == EINVAL
    assert L.bs_top_logits(d, 5, P, P, P, ctypes.c_void_p(4104), need, None) == EINVAL
    f = L.bs_distill_loss
    assert f(d, P, P, None, 0, None, P, P, P, 100, None) == EINVAL
    assert f(d, P, P, None, 1025, None, P, P, P, 100, None) == ENOTSUP
    assert f(d, None, P, None, 3, None, P, P, P, 100, None) == EINVAL
    assert f(d, P, None, None, 3, None, P, P, P, 100, None) == EINVAL
    assert f(d, P, P, None, 3, None, None, P, P, 100, None) == EINVAL
    assert f(d, P, P, None, 3, None, P, None, P, 100, None) == EINVAL
    assert f(d, P, P, None, 3, None, P, P, P, 99, None) == EINVAL
    q = L.bs_policy_loss
    assert q(d, P, P, P, None, None, None, P, P, None, None, None, P, 100, None) == EINVAL
    assert q(d, None, P, P, None, None, good, P, P, None, None, None, P, 100, None) == EINVAL
    assert q(d, P, None, P, None, None, good, P, P, None, None, None, P, 100, None) == EINVAL
    assert q(d, P, P, None, None, None, good, P, P, None, None, None, P, 100, None) == EINVAL
    assert q(d, P, P, P, None, None, good, None, P, None, None, None, P, 100, None) == EINVAL
    assert q(d, P, P, P, None, None, good, P, None, None, None, None, P, 100, None) == EINVAL
    assert q(d, P, P, P, None, None, good, P, P, None, None, None, P, 99, None) == EINVAL
    for bad in ((-0.1, 0.2, 0, 0), (0.2, -0.1, 0, 0), (nan, 0.2, 0, 0), (0.2, 0.2, inf, 0), (0.2, 0.2, 0, nan)):
        assert q(d, P, P, P, P, None, cfg(*bad), P, P, None, None, None, P, 100, None) == EINVAL, bad
    assert q(d, P, P, P, None, None, cfg(0.2, 0.2, 0.1, 0.0), P, P, None, None, None, P, 100, None) == EINVAL


def test_no_rows_need_no_device(pkg):
    d = desc(pkg, rows=0, data=None)
    L = pkg.lib()
    assert L.bs_token_logprobs(d, None, None, None, None, None) == OK
    assert L.bs_token_logprobs_grad(d, None, None, None, None, None, None, 0, None) == OK
    assert L.bs_top_logits(d, 5, None, None, None, None, 0, None) == OK


def test_python_refuses_host_tensors(pkg):
    x, t = torch.zeros(2, 8), torch.zeros(2, dtype=torch.int32)
    f = torch.zeros(2)
    for call in (lambda: pkg.token_logprobs(x, t), lambda: pkg.top_logits(x, 1),
                 lambda: pkg.distill_loss(x, t[:, None], f[:, None]), lambda: pkg.policy_loss(x, t, f, f),
                 lambda: pkg.token_logprobs(x.numpy(), t)):
        with pytest.raises(ValueError):
            call()


def test_structs_match_the_header(pkg):
    o = pkg.logit_ops
    assert ctypes.sizeof(o.BsLogits) == 40 and o.BsLogits.rows.offset == 16 and o.BsLogits.logit_scale.offset == 36
    assert ctypes.sizeof(o.BsPolicyConfig) == 16
    text = open(pkg.build.ROOT + "/include/b200_sampler.h").read()
    assert f"#define BS_MAX_VOCAB {o.MAX_VOCAB}" in text and f"#define BS_MAX_TOP {o.MAX_TOP}" in text
