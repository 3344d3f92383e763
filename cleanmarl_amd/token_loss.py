"""Losses of policies whose action is a token: log-probabilities, the clipped policy loss, the preference loss.

The learners of this package train networks whose logits never leave the fused kernels (<= 64 actions).  A policy that is the caller's own
model hands its logits over instead: ``[..., vocab]`` of any float type, thousands of columns.  Each ``*_fwd_bwd`` call returns the
statistics AND the gradient of the logits (cleanmarl/mappo_multienvs.py:527-582 on tokens), which goes into the model with
``logits.backward(result.dlogits)``.  Everything runs on the current HIP stream of the logits' device; nothing synchronises.

Rows with a negative token (padding), weight 0 or no available column are left out: log-probability, entropy and gradient 0, not counted.
"""
import ctypes as C
from typing import NamedTuple, Optional

import torch

from . import _native as N

_DTYPES = {torch.float32: N.DTYPE_F32, torch.float16: N.DTYPE_F16, torch.bfloat16: N.DTYPE_BF16}
_KINDS = {"sigmoid": 0, "squared": 1}


class TokenLogProb(NamedTuple):
    logp: torch.Tensor                      # like token, fp32
    entropy: Optional[torch.Tensor] = None  # like token, fp32
    keep: Optional[torch.Tensor] = None     # what token_logprob_bwd needs of the softmax


class PolicyLoss(NamedTuple):
    stats: torch.Tensor    # [8] weighted sums, slots N.STAT_* (N.STAT_LOSS is the loss)
    dlogits: torch.Tensor  # like logits
    logp: torch.Tensor     # like token, fp32


class PreferenceLoss(NamedTuple):
    stats: torch.Tensor     # [8] sums over the pairs, slots N.PREF_*
    dlogits: torch.Tensor   # like logits
    margin: torch.Tensor    # [pairs]
    seq_logp: torch.Tensor  # [2 * pairs]


def _row_stride(t, what):
    """Elements between the rows of a [..., n] tensor whose leading axes collapse into one without a copy."""
    n = t.shape[-1]
    if n > 1 and t.stride(-1) != 1:
        raise ValueError(f"{what}: the last axis must be contiguous, got strides {tuple(t.stride())}")
    axes = [(s, d) for s, d in zip(t.shape[:-1], t.stride()[:-1]) if s != 1]
    if not axes or t.numel() == 0:
        return n
    for (_, outer), (size, inner) in zip(axes, axes[1:]):
        if outer != size * inner:
            raise ValueError(f"{what}: the leading axes of shape {tuple(t.shape)} with strides {tuple(t.stride())} are not one axis of rows; make it contiguous")
    return axes[-1][1]


def _vector(t, token, what, dtype=torch.float32):
    if t is None:
        return None
    if t.dtype != dtype or t.shape != token.shape or t.device != token.device or not t.is_contiguous():
        raise ValueError(f"{what}: need a contiguous {dtype} tensor of shape {tuple(token.shape)} on {token.device}, got {t.dtype} {tuple(t.shape)} on {t.device}")
    return t


def _rows(logits, token, avail, temperature):
    if logits.device.type != "cuda":
        raise ValueError(f"logits are on {logits.device}: the kernels have no CPU form")
    if logits.dtype not in _DTYPES:
        raise ValueError(f"logits: float32, float16 or bfloat16, got {logits.dtype}")
    if logits.dim() < 1 or logits.shape[-1] < 1 or token.shape != logits.shape[:-1]:
        raise ValueError(f"token: need shape {tuple(logits.shape[:-1])} for logits {tuple(logits.shape)}, got {tuple(token.shape)}")
    if token.dtype not in (torch.int32, torch.int64) or token.device != logits.device or not token.is_contiguous():
        raise ValueError(f"token: need a contiguous int32 or int64 tensor on {logits.device}, got {token.dtype} on {token.device}")
    ld, av, av_ld = _row_stride(logits, "logits"), None, 0
    if avail is not None:
        if avail.dtype not in (torch.uint8, torch.bool) or avail.shape != logits.shape or avail.device != logits.device:
            raise ValueError(f"avail: need uint8 or bool of shape {tuple(logits.shape)} on {logits.device}, got {avail.dtype} {tuple(avail.shape)} on {avail.device}")
        av, av_ld = avail.data_ptr(), _row_stride(avail, "avail")
    return N.TokenRows(logits.data_ptr(), ld, av, av_ld, token.data_ptr(), token.numel(), logits.shape[-1], _DTYPES[logits.dtype],
                       token.element_size(), 0, float(temperature))


def _grad(out, logits):
    """The tensor that receives the gradient and its row stride; ``out`` may be the logits themselves."""
    if out is None:
        out = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
    elif out.dtype != logits.dtype or out.shape != logits.shape or out.device != logits.device:
        raise ValueError(f"out: need {logits.dtype} {tuple(logits.shape)} on {logits.device}, got {out.dtype} {tuple(out.shape)} on {out.device}")
    return out, _row_stride(out, "out")


def _workspace(nbytes, device):
    return torch.empty(max(int(nbytes), 16), dtype=torch.uint8, device=device)


def token_logprob(logits, token, avail=None, temperature=1.0, entropy=False, keep=False):
    """log softmax(logits / temperature)[token] of every row, and its entropy; ``keep=True`` for a later token_logprob_bwd.

    Replaces Categorical(logits).log_prob / .entropy (cleanmarl/mappo_multienvs.py:172-176, 549-550): one pass over the logits."""
    rows = _rows(logits, token, avail, temperature)
    lib = N.load()
    with torch.cuda.device(logits.device):
        new = lambda *shape: torch.empty(shape, dtype=torch.float32, device=logits.device)  # noqa: E731
        r = TokenLogProb(new(*token.shape), new(*token.shape) if entropy else None, new(*token.shape, 2) if keep else None)
        ws = _workspace(lib.cm_token_workspace_bytes(rows.rows, rows.vocab), logits.device)
        N.check(lib.cm_token_logprob(C.byref(rows), N.ptr(r.logp), N.ptr(r.entropy), N.ptr(r.keep), N.ptr(ws), ws.numel(), N.stream_ptr()), "cm_token_logprob")
    return r


def token_logprob_bwd(logits, token, forward, d_logp, d_entropy=None, avail=None, temperature=1.0, out=None):
    """Gradient of sum(d_logp * logp + d_entropy * entropy) with respect to the logits.

    ``forward``: what token_logprob(..., keep=True) returned for the same logits, token, avail and temperature.  ``out``: where the
    gradient goes; the logits themselves are allowed."""
    rows = _rows(logits, token, avail, temperature)
    if forward.keep is None or forward.keep.shape != (*token.shape, 2) or forward.keep.device != logits.device or not forward.keep.is_contiguous():
        raise ValueError("forward: need the result of token_logprob(..., keep=True) for these rows")
    if d_entropy is not None and forward.entropy is None:
        raise ValueError("d_entropy: the forward call has to compute the entropy (entropy=True)")
    _vector(d_logp, token, "d_logp")
    _vector(d_entropy, token, "d_entropy")
    H = _vector(forward.entropy, token, "forward.entropy") if d_entropy is not None else None
    lib = N.load()
    with torch.cuda.device(logits.device):
        out, ld = _grad(out, logits)
        N.check(lib.cm_token_logprob_bwd(C.byref(rows), N.ptr(forward.keep), N.ptr(H), N.ptr(d_logp), N.ptr(d_entropy), N.ptr(out), ld, N.stream_ptr()),
                "cm_token_logprob_bwd")
    return out


def policy_loss_fwd_bwd(logits, token, logp_old, adv, logp_ref=None, weight=None, avail=None, temperature=1.0, clip_low=0.2, clip_high=0.2,
                        kl_coef=0.0, entropy_coef=0.0, out=None):
    """Clipped policy loss with a KL term, forward and backward in one call (cleanmarl/mappo_multienvs.py:536-582 on tokens).

    loss = sum weight * (-min(adv rho, adv clip(rho, 1 - clip_low, 1 + clip_high)) - entropy_coef H + kl_coef (e^d - d - 1)),
    rho = exp(logp - logp_old), d = logp_ref - logp.  ``weight`` carries mask and normalisation (None: ones).  All per-row tensors have
    token's shape.  ``out``: where the gradient goes; the logits themselves are allowed."""
    rows = _rows(logits, token, avail, temperature)
    for t, what in ((logp_old, "logp_old"), (adv, "adv"), (logp_ref, "logp_ref"), (weight, "weight")):
        _vector(t, token, what)
    lib = N.load()
    with torch.cuda.device(logits.device):
        out, ld = _grad(out, logits)
        f32 = dict(dtype=torch.float32, device=logits.device)
        stats, logp = torch.empty(N.NUM_STATS, **f32), torch.empty(token.shape, **f32)
        ws = _workspace(lib.cm_token_workspace_bytes(rows.rows, rows.vocab), logits.device)
        N.check(lib.cm_token_policy_fwd_bwd(C.byref(rows), N.ptr(logp_old), N.ptr(adv), N.ptr(logp_ref), N.ptr(weight), clip_low, clip_high, kl_coef,
                                            entropy_coef, N.ptr(out), ld, N.ptr(logp), N.ptr(stats), N.ptr(ws), ws.numel(), N.stream_ptr()),
                "cm_token_policy_fwd_bwd")
    return PolicyLoss(stats, out, logp)


def preference_loss_fwd_bwd(logits, token, seq_start, logp_ref, beta=0.1, label_smoothing=0.0, kind="sigmoid", scale=None, avail=None,
                            temperature=1.0, out=None):
    """Preference loss on paired log ratios, forward and backward in one call.

    ``logits`` [rows, vocab]: the packed rows of 2P sequences, the P chosen answers first, then the P rejected ones; sequence q has the rows
    ``seq_start[q]:seq_start[q + 1]`` (int32, on the device).  Tokens that are not part of an answer are negative.  ``logp_ref`` [2P]: the
    reference policy's sums.  ``scale``: factor of the gradient, 1/P (the mean over the pairs) by default.  Rows outside all sequences of
    ``out`` are not written (zeros in a tensor that is made here)."""
    rows = _rows(logits, token, avail, temperature)
    if logits.dim() != 2:
        raise ValueError(f"logits: need [rows, vocab], got {tuple(logits.shape)}")
    if kind not in _KINDS:
        raise ValueError(f"kind: one of {sorted(_KINDS)}, got {kind!r}")
    n = seq_start.numel()
    if seq_start.dtype != torch.int32 or seq_start.dim() != 1 or n < 3 or n % 2 == 0 or seq_start.device != logits.device or not seq_start.is_contiguous():
        raise ValueError(f"seq_start: need a contiguous int32 tensor of 2 * pairs + 1 starts on {logits.device}, got {seq_start.dtype} {tuple(seq_start.shape)} on {seq_start.device}")
    pairs = n // 2
    if logp_ref.dtype != torch.float32 or logp_ref.shape != (2 * pairs,) or logp_ref.device != logits.device or not logp_ref.is_contiguous():
        raise ValueError(f"logp_ref: need float32 [{2 * pairs}] on {logits.device}, got {logp_ref.dtype} {tuple(logp_ref.shape)} on {logp_ref.device}")
    lib = N.load()
    with torch.cuda.device(logits.device):
        if out is None:
            out = torch.zeros_like(logits, memory_format=torch.contiguous_format)
        out, ld = _grad(out, logits)
        f32 = dict(dtype=torch.float32, device=logits.device)
        stats, margin, seq_logp = torch.empty(N.NUM_STATS, **f32), torch.empty(pairs, **f32), torch.empty(2 * pairs, **f32)
        ws = _workspace(lib.cm_preference_workspace_bytes(rows.rows, rows.vocab, pairs), logits.device)
        N.check(lib.cm_preference_fwd_bwd(C.byref(rows), N.ptr(seq_start), pairs, N.ptr(logp_ref), beta, label_smoothing, _KINDS[kind],
                                          1.0 / pairs if scale is None else scale, N.ptr(out), ld, N.ptr(margin), N.ptr(seq_logp), N.ptr(stats),
                                          N.ptr(ws), ws.numel(), N.stream_ptr()), "cm_preference_fwd_bwd")
    return PreferenceLoss(stats, out, margin, seq_logp)
