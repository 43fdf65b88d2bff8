"""Operators on rows of logits beside the sampler, over the C ABI.

What a caller of :class:`Sampler` does with the same rows: the log-probability
of the drawn tokens (:func:`token_logprobs`, with its gradient
:func:`token_logprobs_grad`), the best tokens of a row (:func:`top_logits`),
and the losses that train a model on drawn tokens (:func:`policy_loss`) or on
another model's top logits (:func:`distill_loss`).

All take CUDA logits (float32, bfloat16 or float16; rows x vocab with unit
column stride, or one row) and see a row through the sampler's logit prologue
and temperature: ``z = c(v) / (logit_scale * temperature)``, ``c`` the soft-cap
``cap * tanh(v / cap)`` where ``final_logit_softcapping > 0``.  The two losses
return the logits' gradient from the same call (``logits.backward(r.grad)``
carries it on into a model); nothing here records an autograd graph, so every
call can be captured in a CUDA graph.  Results are stream-ordered and live on
``stream`` (default: the current stream of the logits' device).
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple, Optional

from . import sampler as _s

MAX_VOCAB = 1048576   # BS_MAX_VOCAB
MAX_TOP = 1024        # BS_MAX_TOP


class BsLogits(ctypes.Structure):
    """bs_logits."""

    _fields_ = [
        ("data", ctypes.c_void_p),
        ("ld", ctypes.c_size_t),
        ("rows", ctypes.c_uint32),
        ("vocab", ctypes.c_uint32),
        ("dtype", ctypes.c_uint32),
        ("temperature", ctypes.c_float),
        ("final_logit_softcapping", ctypes.c_float),
        ("logit_scale", ctypes.c_float),
    ]


class BsPolicyConfig(ctypes.Structure):
    """bs_policy_config."""

    _fields_ = [
        ("clip_low", ctypes.c_float),
        ("clip_high", ctypes.c_float),
        ("kl_coef", ctypes.c_float),
        ("entropy_coef", ctypes.c_float),
    ]


class TokenLogprobs(NamedTuple):
    logprobs: "torch.Tensor"    # rows: log-probability of the row's token
    entropy: "torch.Tensor"     # rows
    stats: "torch.Tensor"       # rows x 2: max of c(v), log sum exp(z - max z)


class TopLogits(NamedTuple):
    logits: "torch.Tensor"      # rows x k: c(v) / logit_scale, falling
    ids: "torch.Tensor"         # rows x k, int32
    lse: "torch.Tensor"         # rows: log sum exp(z)


class DistillLoss(NamedTuple):
    loss: "torch.Tensor"        # sum of weights * row_losses
    row_losses: "torch.Tensor"  # rows
    grad: Optional["torch.Tensor"]


class PolicyLoss(NamedTuple):
    loss: "torch.Tensor"
    row_losses: "torch.Tensor"  # rows
    logprobs: "torch.Tensor"    # rows
    entropy: "torch.Tensor"     # rows
    kl: "torch.Tensor"          # rows: exp(d) - d - 1, d = ref - logprob (zeros without ref_logprobs)
    grad: Optional["torch.Tensor"]


torch = None      # imported by the first call: the rest of the package does without
_dtypes = {}      # torch types -> bs_dtype


def _import_torch():
    global torch
    import torch as t
    _dtypes.update({t.float32: 0, t.bfloat16: 1, t.float16: 2})
    torch = t


def _raw_stream(index):
    """The current stream of a device, as a pointer."""
    fast = getattr(torch._C, "_cuda_getCurrentRawStream", None)
    return fast(index) if fast is not None else torch.cuda.current_stream(index).cuda_stream


class _Rows:
    """Checked logits of one call: the descriptor, and where to run."""

    def __init__(self, logits, temperature, softcap, logit_scale, stream):
        if torch is None:
            _import_torch()
        x = logits
        if not isinstance(x, torch.Tensor) or not x.is_cuda or x.dtype not in _dtypes:
            raise ValueError("logits must be a CUDA tensor of float32, bfloat16 or float16")
        if x.dim() == 1:
            x = x.unsqueeze(0)
        if x.dim() != 2 or x.shape[1] == 0 or (x.stride(1) != 1 and x.shape[1] > 1):
            raise ValueError("logits must be rows x vocab with unit column stride")
        self.rows, self.vocab = x.shape
        ld = x.stride(0) if self.rows > 1 else self.vocab
        if ld < self.vocab:
            raise ValueError("rows of logits overlap")
        if self.vocab > MAX_VOCAB:
            raise ValueError(f"vocab is at most {MAX_VOCAB}")
        self.x, self.ld, self.device = x, ld, x.device
        self.desc = BsLogits(x.data_ptr(), ld, self.rows, self.vocab, _dtypes[x.dtype], temperature, softcap,
                             logit_scale)
        self._stream = stream

    def run(self, call):
        """``call(stream)`` with the logits' device and the caller's stream
        current: results are allocated on the stream that writes them."""
        s, index = self._stream, self.device.index
        if s is None:
            if torch.cuda.current_device() == index:
                return call(_raw_stream(index))
            with torch.cuda.device(index):
                return call(_raw_stream(index))
        with torch.cuda.device(index):
            if isinstance(s, torch.cuda.Stream):
                if s.device != self.device:
                    raise ValueError("stream must be of the logits' device")
            else:
                ptr = int(getattr(s, "cuda_stream", s))
                s = torch.cuda.ExternalStream(ptr, device=self.device) if ptr else torch.cuda.default_stream()
            with torch.cuda.stream(s):
                return call(s.cuda_stream)

    def floats(self, t, what, shape=None):
        """A float32 input on the logits' device, packed."""
        shape = (self.rows,) if shape is None else shape
        if isinstance(t, torch.Tensor) and t.dtype is torch.float32 and t.device == self.device and t.shape == shape \
                and t.is_contiguous():
            return t
        if not isinstance(t, torch.Tensor) or t.device != self.device or not t.is_floating_point():
            raise ValueError(f"{what} must be a floating tensor on the logits' device")
        if tuple(t.shape) != shape and not (shape == (1,) and t.dim() == 0):
            raise ValueError(f"{what} must have shape {shape}")
        if t.dtype != torch.float32:
            t = t.float()
        return t.contiguous()

    def ids(self, t, what, shape=None):
        """Token ids as packed int32; an id that int32 cannot hold is outside
        every vocabulary and becomes -1."""
        shape = (self.rows,) if shape is None else shape
        if isinstance(t, torch.Tensor) and t.dtype is torch.int32 and t.device == self.device and t.shape == shape \
                and t.is_contiguous():
            return t
        if not isinstance(t, torch.Tensor) or t.device != self.device or t.is_floating_point() or t.is_complex() \
                or t.dtype == torch.bool:
            raise ValueError(f"{what} must be an integer tensor on the logits' device")
        if tuple(t.shape) != shape and not (shape == (1,) and t.dim() == 0):
            raise ValueError(f"{what} must have shape {shape}")
        if t.dtype == torch.uint64:
            t = t.to(torch.int64)   # (2^63 and above become negative)
        if t.dtype == torch.int64:
            t = torch.where((t >= 0) & (t < 2**31), t, -1)
        if t.dtype not in (torch.int32, torch.uint32):
            t = t.to(torch.int32)
        return t.contiguous()

    def grad_out(self, out):
        """(tensor, row stride) of the gradient."""
        if out is None:
            if self.ld == self.vocab and self.rows > 1:
                return torch.empty_like(self.x), self.vocab
            g = torch.empty((self.rows, self.vocab), dtype=self.x.dtype, device=self.device)
            return g, self.vocab
        g = out.unsqueeze(0) if isinstance(out, torch.Tensor) and out.dim() == 1 else out
        if not isinstance(g, torch.Tensor) or g.dtype != self.x.dtype or g.device != self.device \
                or tuple(g.shape) != (self.rows, self.vocab) or (g.stride(1) != 1 and self.vocab > 1):
            raise ValueError("out must be like the logits, with unit column stride")
        ld = g.stride(0) if self.rows > 1 else self.vocab
        if ld < self.vocab:
            raise ValueError("rows of out overlap")
        if self.rows and (g.data_ptr() != self.x.data_ptr() or ld != self.ld):
            size = g.element_size()
            a0, b0 = g.data_ptr(), self.x.data_ptr()
            a1 = a0 + ((self.rows - 1) * ld + self.vocab) * size
            b1 = b0 + ((self.rows - 1) * self.ld + self.vocab) * size
            if a0 < b1 and b0 < a1:
                raise ValueError("out overlaps the logits without being them")
        return g, ld

    def empty(self, *shape):
        return torch.empty(*shape, dtype=torch.float32, device=self.device)


def _ptr(t):
    return None if t is None else t.data_ptr()


def _like(logits, grad):
    return grad[0] if grad is not None and logits.dim() == 1 else grad


def _written(out):
    """Tells autograd that the kernel wrote over the caller's tensor, as an
    in-place operation of torch's does: a backward that saved its old values
    raises, and does not go by the new ones."""
    if out is not None and not out.is_inference():   # (these have no version)
        torch.autograd.graph.increment_version(out)


def logit_ops_status(device=None) -> int:
    """BS_ETIMEOUT if a bounded device wait of one of these operators gave up on
    the device since the last such call, else BS_OK (bs_logit_ops_status).
    Waits for the device."""
    if torch is None:
        _import_torch()
    with torch.cuda.device(device):
        return _s.lib().bs_logit_ops_status()


def token_logprobs(logits, tokens, *, temperature: float = 1.0, final_logit_softcapping: float = 0.0,
                   logit_scale: float = 1.0, stream=None) -> TokenLogprobs:
    """Log-probability of each row's token and the row's entropy (bs_token_logprobs).

    ``tokens``: rows ids; a row whose id is outside the vocabulary (-1, -100,
    the sampler's 0xFFFFFFFF) is left out: zeros.  ``stats`` is what
    :func:`token_logprobs_grad` needs.
    """
    r = _Rows(logits, temperature, final_logit_softcapping, logit_scale, stream)

    def call(st):
        t = r.ids(tokens, "tokens")
        lp = r.empty(r.rows)
        ent, stats = torch.empty_like(lp), r.empty(r.rows, 2)
        _s._check(_s.lib().bs_token_logprobs(ctypes.byref(r.desc), t.data_ptr(), lp.data_ptr(), ent.data_ptr(),
                                             stats.data_ptr(), st), "bs_token_logprobs")
        return TokenLogprobs(lp, ent, stats)

    return r.run(call)


def token_logprobs_grad(logits, tokens, fwd: TokenLogprobs, grad_logprobs=None, grad_entropy=None, *,
                        temperature: float = 1.0, final_logit_softcapping: float = 0.0, logit_scale: float = 1.0,
                        out=None, stream=None):
    """The logits' gradient from those of ``fwd.logprobs`` and ``fwd.entropy``
    (bs_token_logprobs_grad); ``fwd`` is :func:`token_logprobs` of the same
    logits, tokens and factors.  ``out`` may be the logits themselves."""
    r = _Rows(logits, temperature, final_logit_softcapping, logit_scale, stream)
    if grad_logprobs is None and grad_entropy is None:
        raise ValueError("neither grad_logprobs nor grad_entropy is given")

    def call(st):
        t = r.ids(tokens, "tokens")
        stats, ent = r.floats(fwd.stats, "fwd.stats", (r.rows, 2)), r.floats(fwd.entropy, "fwd.entropy")
        gl = None if grad_logprobs is None else r.floats(grad_logprobs, "grad_logprobs")
        gh = None if grad_entropy is None else r.floats(grad_entropy, "grad_entropy")
        g, ld = r.grad_out(out)
        _s._check(_s.lib().bs_token_logprobs_grad(ctypes.byref(r.desc), t.data_ptr(), stats.data_ptr(), ent.data_ptr(),
                                                  _ptr(gl), _ptr(gh), g.data_ptr(), ld, st), "bs_token_logprobs_grad")
        _written(out)
        return _like(logits, g)

    return r.run(call)


def top_logits(logits, k: int, *, temperature: float = 1.0, final_logit_softcapping: float = 0.0,
               logit_scale: float = 1.0, stream=None) -> TopLogits:
    """The k largest logits of each row in falling order (the lowest id first
    among equals) with their ids, and the row's normaliser (bs_top_logits).
    ``logits / temperature - lse[:, None]`` are their log-probabilities.  A row
    all of -inf has an lse of -inf."""
    r = _Rows(logits, temperature, final_logit_softcapping, logit_scale, stream)
    if not 1 <= int(k) <= min(r.vocab, MAX_TOP):
        raise ValueError(f"k must be between 1 and the vocabulary (and {MAX_TOP})")
    def call(st):
        values, lse = r.empty(r.rows, k), r.empty(r.rows)
        ids = torch.empty(r.rows, k, dtype=torch.int32, device=r.device)
        L, d = _s.lib(), ctypes.byref(r.desc)
        size = L.bs_top_logits_workspace(d)
        work = r.empty(size // 4)
        _s._check(L.bs_top_logits(d, k, values.data_ptr(), ids.data_ptr(), lse.data_ptr(), work.data_ptr(), size, st),
                  "bs_top_logits")
        return TopLogits(values, ids, lse)

    return r.run(call)


def distill_loss(logits, teacher_ids, teacher_logits, teacher_lse=None, weights=None, *, temperature: float = 1.0,
                 final_logit_softcapping: float = 0.0, logit_scale: float = 1.0, grad: bool = True, out=None,
                 stream=None) -> DistillLoss:
    """Divergence of the student's rows from a teacher's top logits, with the
    gradient of the weighted sum (bs_distill_loss).

    ``teacher_ids`` and ``teacher_logits`` (rows x K, as :func:`top_logits`
    returns them; ids outside the vocabulary are empty slots).  Without
    ``teacher_lse`` the teacher is renormalised over its slots; with it
    (:func:`top_logits` at the same temperature) the rest of the vocabulary is
    one more outcome.  ``weights``: rows (default: the mean); a row of weight 0
    is left out.  ``out``: where the gradient goes (may be the logits).
    """
    r = _Rows(logits, temperature, final_logit_softcapping, logit_scale, stream)
    if teacher_ids.dim() == 1 and logits.dim() == 1:
        teacher_ids, teacher_logits = teacher_ids.unsqueeze(0), teacher_logits.unsqueeze(0)
    if teacher_ids.dim() != 2 or not 1 <= teacher_ids.shape[1] <= MAX_TOP:
        raise ValueError(f"teacher_ids must be rows x K with K between 1 and {MAX_TOP}")
    shape = (r.rows, teacher_ids.shape[1])

    def call(st):
        ids, tl = r.ids(teacher_ids, "teacher_ids", shape), r.floats(teacher_logits, "teacher_logits", shape)
        lse = None if teacher_lse is None else r.floats(teacher_lse, "teacher_lse")
        w = None if weights is None else r.floats(weights, "weights")
        g, ld = r.grad_out(out) if grad else (None, 0)
        rows = r.empty(r.rows)
        loss = rows.new_empty(())
        _s._check(_s.lib().bs_distill_loss(ctypes.byref(r.desc), ids.data_ptr(), tl.data_ptr(), _ptr(lse), shape[1],
                                           _ptr(w), loss.data_ptr(), rows.data_ptr(), _ptr(g), ld, st),
                  "bs_distill_loss")
        if grad:
            _written(out)
        return DistillLoss(loss, rows, _like(logits, g))

    return r.run(call)


def policy_loss(logits, tokens, old_logprobs, advantages, ref_logprobs=None, weights=None, *, clip_low: float = 0.2,
                clip_high: float = 0.2, kl_coef: float = 0.0, entropy_coef: float = 0.0, temperature: float = 1.0,
                final_logit_softcapping: float = 0.0, logit_scale: float = 1.0, grad: bool = True, out=None,
                stream=None) -> PolicyLoss:
    """Clipped policy loss of the rows' tokens with a KL term towards
    ``ref_logprobs`` and an entropy bonus, and the gradient of the weighted
    sum (bs_policy_loss):

        L = -min(r A, clip(r, 1 - clip_low, 1 + clip_high) A) + kl_coef (exp(d) - d - 1) - entropy_coef H,
        r = exp(lp - old_logprobs), d = ref_logprobs - lp, A = advantages.

    ``weights``: rows (default: the mean); a row of weight 0, or whose token
    is outside the vocabulary, is left out.  ``out``: where the gradient goes
    (may be the logits).
    """
    r = _Rows(logits, temperature, final_logit_softcapping, logit_scale, stream)
    if kl_coef != 0.0 and ref_logprobs is None:
        raise ValueError("kl_coef needs ref_logprobs")
    cfg = BsPolicyConfig(clip_low, clip_high, kl_coef, entropy_coef)

    def call(st):
        t = r.ids(tokens, "tokens")
        old, adv = r.floats(old_logprobs, "old_logprobs"), r.floats(advantages, "advantages")
        ref = None if ref_logprobs is None else r.floats(ref_logprobs, "ref_logprobs")
        w = None if weights is None else r.floats(weights, "weights")
        g, ld = r.grad_out(out) if grad else (None, 0)
        n = r.rows
        buf = r.empty(4 * n + 1)
        p = buf.data_ptr()
        _s._check(_s.lib().bs_policy_loss(ctypes.byref(r.desc), t.data_ptr(), old.data_ptr(), adv.data_ptr(), _ptr(ref),
                                          _ptr(w), ctypes.byref(cfg), p + 16 * n, p, p + 4 * n, p + 8 * n, p + 12 * n,
                                          _ptr(g), ld, st), "bs_policy_loss")
        if grad:
            _written(out)
        rows, lp, ent, kl, loss = buf.split_with_sizes((n, n, n, n, 1))
        return PolicyLoss(loss.squeeze(0), rows, lp, ent, kl, _like(logits, g))

    return r.run(call)
