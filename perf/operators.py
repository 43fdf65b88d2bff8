"""The vocabulary-row operators beside the sampler: what is measured, and their plain forms.

An operator takes rows of logits v (rows x vocab; float32, bfloat16 or float16) as the LM head leaves them.  With
the logit prologue and the temperature that the sampler draws with,

    z_j = c(v_j) / (logit_scale T),  c(v) = cap tanh(v / cap) where a soft-cap is set, else v,
    p_j = exp(z_j - lse),            lse = log sum_j exp(z_j),

the operators are

* ``logprobs``  the log-probability of a row's token and the row's entropy; backward: the logits' gradient from
                the gradients of both.  A token outside the vocabulary (-1: padding) leaves its row out (zeros).
* ``top``       the k largest logits of a row with their ids (ties: the lowest id first) and the row's lse.
* ``distill``   the divergence of the student's row from a teacher's top logits, with the logits' gradient.  The
                teacher is renormalised over its top ids, or (``tail``) the rest of the vocabulary is one more
                outcome, whose mass follows from the teacher's lse.
* ``policy``    the clipped policy loss with a KL term towards a reference model and an entropy bonus, with the
                logits' gradient.

``run`` computes the plain forms with elementary torch operations, or (``own``) calls the library.
"""
import importlib.util
import math
import os
import sys

import torch

own = False

_DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_BYTES = {"f32": 4, "bf16": 2, "f16": 2}
_MOST = 2 * 4096 * 128256  # bytes of the largest listed case's logits


def _ops():
    """The library (its directory name contains a dot, so it is loaded by path)."""
    if "llama_zig_b200" not in sys.modules:
        here = os.path.join(os.getcwd(), "llama.zig_b200")
        spec = importlib.util.spec_from_file_location("llama_zig_b200", os.path.join(here, "__init__.py"),
                                                      submodule_search_locations=[here])
        mod = importlib.util.module_from_spec(spec)
        sys.modules["llama_zig_b200"] = mod
        spec.loader.exec_module(mod)
    return sys.modules["llama_zig_b200"]


def _case(name, op, rows, vocab, dtype, temperature=1.0, softcap=0.0, pad=0.0, **more):
    c = dict(op=op, rows=rows, vocab=vocab, dtype=dtype, temperature=temperature, softcap=softcap, pad=pad, **more)
    return dict(c, name=name) if name else c


def listed():
    return [
        # a decode step at batch 1 that reports its token's log-probability (sizes of the single-row sampler)
        _case("logprobs_decode", "logprobs", 1, 128256, "f32", 0.8, backward=False),
        # the batched sampler's step with log-probabilities
        _case("logprobs_batch", "logprobs", 256, 128256, "f32", 0.7, backward=False),
        # a training step through log-probabilities and entropies, padded sequences
        _case("logprobs_train", "logprobs", 2048, 151936, "bf16", 1.0, pad=0.125, backward=True),
        # the twenty best tokens of a handful of requests, a vocabulary of odd size
        _case("top_serve", "top", 5, 32003, "f16", 1.0, k=20),
        # a teacher's top logits over the batched sampler's sizes
        _case("top_teacher", "top", 256, 128256, "f32", 1.0, k=64),
        # a teacher with a very large vocabulary and many kept logits
        _case("top_large", "top", 1024, 256000, "bf16", 2.0, k=256),
        # a small student's step, odd sizes
        _case("distill_small", "distill", 37, 32003, "f32", 2.0, k=16, tail=False),
        # a student's training step on a padded batch
        _case("distill_train", "distill", 2048, 128256, "bf16", 1.0, pad=0.25, k=64, tail=False),
        # a student with soft-capped logits and a very large vocabulary, the teacher's tail as one outcome
        _case("distill_tail", "distill", 512, 256000, "f32", 2.0, softcap=30.0, k=128, tail=True),
        # the smallest update: one minibatch of a small model
        _case("policy_small", "policy", 64, 32000, "f32", 1.0, kl=0.0, entropy=0.0),
        # an update on a padded minibatch with a KL term
        _case("policy_train", "policy", 4096, 128256, "bf16", 1.0, pad=0.125, kl=0.04, entropy=0.0),
        # an update of a policy that drew at a temperature, with every term, an odd number of tokens
        _case("policy_full", "policy", 777, 151936, "f32", 0.7, kl=0.1, entropy=0.01),
    ]


def draw(rng):
    def spread(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["logprobs", "top", "distill", "policy"])
    vocab = rng.choice([spread(1000, 256000), spread(1000, 256000), 128256, 151936, 256000])
    dtype = rng.choice(["f32", "bf16", "f16"])
    rows = spread(1, min(8192, _MOST // (vocab * _BYTES[dtype])))
    temperature = rng.choice([1.0, round(rng.uniform(0.5, 2.0), 2)])
    softcap = rng.choice([0.0, 0.0, 0.0, 30.0])
    pad = rng.choice([0.0, round(rng.uniform(0.05, 0.5), 3)])
    if op == "logprobs":
        return _case(None, op, rows, vocab, dtype, temperature, softcap, pad, backward=rng.random() < 0.5)
    if op == "top":  # a sort of whole rows is the dear part of its plain form
        rows = min(rows, max(1, _MOST // 4 // vocab))
        return _case(None, op, rows, vocab, dtype, temperature, softcap, k=spread(1, 512))
    if op == "distill":
        return _case(None, op, rows, vocab, dtype, temperature, softcap, pad, k=spread(1, 256), tail=rng.random() < 0.5)
    return _case(None, op, rows, vocab, dtype, temperature, softcap, pad, kl=rng.choice([0.0, 0.04, 0.1]),
                 entropy=rng.choice([0.0, 0.01]))


def _padded(case):
    return int(case["rows"] * case["pad"])


def _scores64(v, case):
    """z of some rows, in 64 bits."""
    v = v.double()
    if case["softcap"]:
        v = case["softcap"] * torch.tanh(v / case["softcap"])
    return v / case["temperature"]


def _blocks(rows, vocab):
    """Rows in blocks of at most 2^26 logits."""
    step = max(1, (1 << 26) // vocab)
    return [slice(r, min(rows, r + step)) for r in range(0, rows, step)]


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    rows, vocab, dtype = case["rows"], case["vocab"], _DTYPES[case["dtype"]]
    rand = lambda *s: torch.rand(*s, generator=g, device="cuda")  # noqa: E731
    randn = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    # a broad bulk and a few likely tokens, as the sampler's workloads have them
    logits = torch.empty(rows, vocab, dtype=dtype, device="cuda")
    tokens = torch.empty(rows, dtype=torch.int32, device="cuda")
    lp = torch.empty(rows, dtype=torch.float64, device="cuda")
    teacher = {k: [] for k in ("ids", "logits", "lse")}
    for b in _blocks(rows, vocab):
        n = b.stop - b.start
        x = 3.0 * randn(n, vocab)
        at = torch.randint(0, vocab, (n, 16), generator=g, device="cuda")
        x.scatter_(1, at, x.gather(1, at) + 5.0 + 10.0 * rand(n, 16))
        logits[b] = x.to(dtype)
        if case["op"] in ("logprobs", "policy"):  # tokens drawn from the rows' own distribution
            z = _scores64(logits[b], case)
            t = (z.float() - torch.log(-torch.log(rand(n, vocab).clamp_(1e-30, 1 - 2**-24)))).argmax(1)
            tokens[b] = t.int()
            lp[b] = z.gather(1, t[:, None])[:, 0] - torch.logsumexp(z, 1)
        if case["op"] == "distill":  # a teacher that mostly agrees with the student
            x += randn(n, vocab)
            v, i = torch.topk(x, case["k"], dim=1)
            teacher["ids"].append(i.int())
            teacher["logits"].append(v)
            teacher["lse"].append(torch.logsumexp(x.double() / case["temperature"], 1).float())
    s = {"case": dict(case), "logits": logits, "tokens": tokens}
    pad = torch.randperm(rows, generator=g, device="cuda")[: _padded(case)]
    weights = torch.full((rows,), 1.0 / max(1, rows - _padded(case)), device="cuda")
    weights[pad] = 0.0
    if case["op"] == "logprobs":
        tokens[pad] = -1
        s["d_logprobs"], s["d_entropy"] = randn(rows) / rows, 0.1 * randn(rows) / rows
    if case["op"] == "distill":
        s |= {"teacher_" + k: torch.cat(v) for k, v in teacher.items()}
        if not case["tail"]:  # some teachers kept fewer
            kept = torch.randint(max(1, case["k"] // 2), case["k"] + 1, (rows, 1), generator=g, device="cuda")
            s["teacher_ids"][torch.arange(case["k"], device="cuda") >= kept] = -1
        s["weights"] = weights
    if case["op"] == "policy":
        # the policy that drew the tokens is some updates old; ratios are kept off the clip's two corners, where
        # the gradient jumps
        d = 0.2 * randn(rows).double()
        for edge in (math.log(0.8), math.log(1.2)):
            d = torch.where((d - edge).abs() < 1e-4, d + 3e-4, d)
        s["old_logprobs"] = (lp - d).float()
        s["ref_logprobs"] = (lp + 0.3 * randn(rows)).float()
        s["advantages"] = randn(rows)
        s["weights"] = weights
    return s


def work(case):
    rows, vocab, size = case["rows"], case["vocab"], _BYTES[case["dtype"]]
    live = rows - _padded(case)
    op = case["op"]
    if op == "logprobs":
        b, n = live * vocab * size + rows * 12, 6 * live * vocab
        if case["backward"]:  # the gradient needs the row's normaliser first: one read and one write at the least
            b, n = b + rows * vocab * size + rows * 8, n + 6 * live * vocab
        return {"bytes": b, "flops": n}
    if op == "top":
        return {"bytes": rows * vocab * size + rows * (8 * case["k"] + 4), "flops": 5 * rows * vocab}
    row = 8 * case["k"] + 12 if op == "distill" else 36
    return {"bytes": live * vocab * size + rows * (vocab * size + row), "flops": 12 * live * vocab}


# ---- plain forms ---------------------------------------------------------------------------------------------------


def _scores(s):
    """(z, dz/dv) in 32 bits."""
    c = s["case"]
    v = s["logits"].float()
    slope = 1.0 / c["temperature"]
    if c["softcap"]:
        th = torch.tanh(v / c["softcap"])
        v, slope = c["softcap"] * th, slope * (1 - th * th)
    return v / c["temperature"], slope


def _softmax(z):
    """(z - max, exp(z - max), its sum, log of the sum in 64 bits), rows by columns."""
    d = z - z.amax(1, keepdim=True)
    e = torch.exp(d)
    total = e.sum(1, keepdim=True)
    return d, e, total, torch.log(total.double())


def _token_rows(s):
    z, slope = _scores(s)
    d, e, total, log_total = _softmax(z)
    t = s["tokens"].long()
    live = (t >= 0) & (t < z.shape[1])
    t = torch.where(live, t, 0)[:, None]
    lp = torch.where(live, (d.gather(1, t).double() - log_total)[:, 0], 0.0)
    logp = d - log_total.float()
    p = e / total
    entropy = torch.where(live, -(p * logp).sum(1), 0.0)
    return live, t, lp, entropy, p, logp, slope


def _token_grad(s, live, t, p, logp, entropy, slope, d_lp, d_entropy):
    """The logits' gradient from those of a row's log-probability and entropy (both zero where a row is left out)."""
    out = p * (-d_lp[:, None] - d_entropy[:, None] * (logp + entropy[:, None]))
    out.scatter_(1, t, out.gather(1, t) + d_lp[:, None])
    out *= slope
    return torch.where(live[:, None], out, 0.0).to(s["logits"].dtype)


def _plain_logprobs(s):
    live, t, lp, entropy, p, logp, slope = _token_rows(s)
    out = {"logprobs": lp.float(), "entropy": entropy}
    if s["case"]["backward"]:
        out["grad"] = _token_grad(s, live, t, p, logp, entropy, slope, s["d_logprobs"], s["d_entropy"])
    return out


def _plain_top(s):
    k = s["case"]["k"]
    values, ids = torch.sort(s["logits"], dim=1, descending=True, stable=True)
    values, ids = values[:, :k].float(), ids[:, :k].int()
    cap = s["case"]["softcap"]
    if cap:
        values = cap * torch.tanh(values / cap)
    z, _ = _scores(s)
    lse = z.amax(1).double() + _softmax(z)[3][:, 0]
    return {"logits": values, "ids": ids, "lse": lse.float()}


def _plain_distill(s):
    c = s["case"]
    z, slope = _scores(s)
    d, e, total, log_total = _softmax(z)
    ids, w = s["teacher_ids"].long(), s["weights"]
    valid = (ids >= 0) & (ids < z.shape[1])
    at = torch.where(valid, ids, 0)
    u = torch.where(valid, s["teacher_logits"].double() / c["temperature"], -math.inf)
    live = valid.any(1) & (w != 0)
    if c["tail"]:
        q = torch.exp(u - s["teacher_lse"].double()[:, None])
    else:
        q = torch.exp(u - u.amax(1, keepdim=True))
        q = q / q.sum(1, keepdim=True)
    lp = d.gather(1, at).double() - log_total
    rows = torch.where(valid & (q > 0), q * (torch.log(q) - lp), 0.0).sum(1)
    mass, rest_share = q.sum(1), None
    if c["tail"]:
        top = torch.zeros_like(e, dtype=torch.bool).scatter_(1, at, valid)
        rest = torch.where(top, 0.0, e).sum(1).double()
        q_rest = (1 - mass).clamp_min(0.0)
        has = (rest > 0) & (q_rest > 0)
        p_rest = rest / total[:, 0]
        rows = rows + torch.where(has, q_rest * (torch.log(q_rest) - torch.log(p_rest)), 0.0)
        mass = mass + torch.where(has, q_rest, 0.0)
        rest_share = torch.where(has, q_rest / p_rest, 0.0).float()[:, None]
    factor = mass.float()[:, None]
    if c["tail"]:
        factor = factor - torch.where(top, 0.0, rest_share)
    grad = e / total * factor
    grad.scatter_add_(1, at, torch.where(valid, -q, 0.0).float())
    grad = torch.where(live[:, None], grad * slope * w[:, None], 0.0).to(s["logits"].dtype)
    rows = torch.where(live, rows, 0.0)
    return {"loss": (rows * w).sum().float(), "row_losses": rows.float(), "grad": grad}


def _plain_policy(s):
    c = s["case"]
    live, t, lp, entropy, p, logp, slope = _token_rows(s)
    w, a = s["weights"], s["advantages"].double()
    live = live & (w != 0)
    ratio = torch.exp(lp - s["old_logprobs"].double())
    rows = -torch.minimum(ratio * a, ratio.clamp(0.8, 1.2) * a)
    clipped = ((a > 0) & (ratio > 1.2)) | ((a < 0) & (ratio < 0.8))
    d_lp = torch.where(clipped, 0.0, -ratio * a)
    kl = torch.zeros_like(lp)
    if c["kl"]:
        d = s["ref_logprobs"].double() - lp
        kl = torch.expm1(d) - d
        rows = rows + c["kl"] * kl
        d_lp = d_lp - c["kl"] * torch.expm1(d)
    rows = torch.where(live, rows - c["entropy"] * entropy, 0.0)
    d_lp = torch.where(live, d_lp * w, 0.0).float()
    d_entropy = torch.where(live, -c["entropy"] * w, 0.0)
    zero = lambda v: torch.where(live, v, 0.0).float()  # noqa: E731
    return {"loss": (rows * w).sum().float(), "row_losses": rows.float(), "logprobs": zero(lp), "entropy": zero(entropy),
            "kl": zero(kl), "grad": _token_grad(s, live, t, p, logp, entropy, slope, d_lp, d_entropy)}


_PLAIN = {"logprobs": _plain_logprobs, "top": _plain_top, "distill": _plain_distill, "policy": _plain_policy}


# ---- the library's calls -------------------------------------------------------------------------------------------


def _own(s):
    c, ops = s["case"], _ops()
    how = {"temperature": c["temperature"], "final_logit_softcapping": c["softcap"]}
    if c["op"] == "logprobs":
        r = ops.token_logprobs(s["logits"], s["tokens"], **how)
        out = {"logprobs": r.logprobs, "entropy": r.entropy}
        if c["backward"]:
            out["grad"] = ops.token_logprobs_grad(s["logits"], s["tokens"], r, s["d_logprobs"], s["d_entropy"], **how)
        return out
    if c["op"] == "top":
        r = ops.top_logits(s["logits"], c["k"], **how)
        return {"logits": r.logits, "ids": r.ids, "lse": r.lse}
    if c["op"] == "distill":
        r = ops.distill_loss(s["logits"], s["teacher_ids"], s["teacher_logits"], s["teacher_lse"] if c["tail"] else None,
                             s["weights"], **how)
        return {"loss": r.loss, "row_losses": r.row_losses, "grad": r.grad}
    r = ops.policy_loss(s["logits"], s["tokens"], s["old_logprobs"], s["advantages"],
                        s["ref_logprobs"] if c["kl"] else None, s["weights"], clip_low=0.2, clip_high=0.2, kl_coef=c["kl"],
                        entropy_coef=c["entropy"], **how)
    return {"loss": r.loss, "row_losses": r.row_losses, "logprobs": r.logprobs, "entropy": r.entropy, "kl": r.kl,
            "grad": r.grad}


def run(state):
    return _own(state) if own else _PLAIN[state["case"]["op"]](state)


# ---- the definition in 64 bits -------------------------------------------------------------------------------------


def _exact_block(s, b):
    """The rows of one block: outputs by name, the block's share of the loss under "loss"."""
    c = s["case"]
    v = s["logits"][b].double().requires_grad_(c["op"] != "top")
    logp = torch.log_softmax(_scores64(v, c), 1)
    if c["op"] == "top":
        # one whole number that orders by value, then by the lower id
        bits = (s["logits"][b].float() + 0.0).view(torch.int32).long()
        order = torch.where(bits < 0, -1 - (bits & 0x7FFFFFFF), bits)
        key = order * (1 << 24) + ((1 << 24) - 1 - torch.arange(v.shape[1], device="cuda"))
        ids = torch.topk(key, c["k"], dim=1).indices
        z = _scores64(v, c)
        return {"logits": z.gather(1, ids) * c["temperature"], "ids": ids.int(), "lse": torch.logsumexp(z, 1)}
    entropy = -(logp.exp() * logp).sum(1)
    if c["op"] in ("logprobs", "policy"):
        t = s["tokens"][b].long()
        live = t >= 0
        lp = logp.gather(1, t.clamp_min(0)[:, None])[:, 0]
    if c["op"] == "logprobs":
        out = {"logprobs": lp * live, "entropy": entropy * live}
        if c["backward"]:
            score = (out["logprobs"] * s["d_logprobs"][b].double() + out["entropy"] * s["d_entropy"][b].double()).sum()
            out["grad"] = torch.autograd.grad(score, v)[0]
        return {k: x.detach() for k, x in out.items()}
    w = s["weights"][b].double()
    if c["op"] == "policy":
        a = s["advantages"][b].double()
        ratio = (lp - s["old_logprobs"][b].double()).exp()
        rows = -torch.min(ratio * a, torch.clamp(ratio, 0.8, 1.2) * a) - c["entropy"] * entropy
        kl = torch.zeros_like(lp)
        if c["kl"]:
            d = s["ref_logprobs"][b].double() - lp
            kl = d.exp() - 1 - d
            rows = rows + c["kl"] * kl
        live = (w != 0).double()
        out = {"row_losses": rows * live, "logprobs": lp * live, "entropy": entropy * live, "kl": kl * live}
    else:
        ids = s["teacher_ids"][b].long()
        valid = ids >= 0
        u = s["teacher_logits"][b].double() / c["temperature"]
        q = (u - s["teacher_lse"][b].double()[:, None]).exp() if c["tail"] else torch.softmax(u.masked_fill(~valid, -1e300), 1)
        lq = torch.log(q.clamp_min(1e-300))
        rows = (q * valid * (lq - logp.gather(1, ids.clamp_min(0)))).sum(1)
        if c["tail"]:
            inside = torch.zeros(v.shape, device="cuda", dtype=torch.bool).scatter_(1, ids, True)
            q_rest = (1 - q.sum(1)).clamp_min(0.0)
            lp_rest = torch.logsumexp(logp.masked_fill(inside, -math.inf), 1)
            rows = rows + torch.where(q_rest > 0, q_rest * (torch.log(q_rest.clamp_min(1e-300)) - lp_rest), 0.0)
        out = {"row_losses": rows * (w != 0)}
    out["loss"] = (out["row_losses"] * w).sum()
    out["grad"] = torch.autograd.grad(out["loss"], v)[0]
    return {k: x.detach() for k, x in out.items()}


def exact(case, seed):
    s = prepare(case, seed)
    got = [_exact_block(s, b) for b in _blocks(case["rows"], case["vocab"])]
    out = {k: sum(g[k] for g in got) if k == "loss" else torch.cat([g[k] for g in got]) for k in got[0]}
    return out
