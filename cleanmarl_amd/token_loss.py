"""Losses of policies whose action is a token: log-probabilities, the clipped policy loss, the preference loss.

The learners of this package train networks whose logits never leave the fused kernels (<= 64 actions).  A policy that is the caller's own
model hands its logits over instead: ``[..., vocab]`` of any float type, thousands of columns.  Each ``*_fwd_bwd`` call returns the
statistics AND the gradient of the logits (cleanmarl/mappo_multienvs.py:527-582 on tokens), which goes into the model with
``logits.backward(result.dlogits)``.  ``out=`` over the logits counts as an in-place operation on them: a model whose last
operation saved its output for its backward pass (tanh, a softmax) raises then.  Everything runs on the current HIP stream of the logits' device; nothing synchronises.

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
    if t.is_contiguous():
        return n
    if n > 1 and t.stride(-1) != 1:
        raise ValueError(f"{what}: the last axis must be contiguous, got strides {tuple(t.stride())}")
    axes = [(s, d) for s, d in zip(t.shape[:-1], t.stride()[:-1]) if s != 1]
    if not axes or t.numel() == 0:
        return n
    for (_, outer), (size, inner) in zip(axes, axes[1:]):
        if outer != size * inner:
            raise ValueError(f"{what}: the leading axes of shape {tuple(t.shape)} with strides {tuple(t.stride())} are not one axis of rows; make it contiguous")
    return axes[-1][1]


def _vector(t, token, what):
    """Address of an optional fp32 value per row."""
    if t is None:
        return None
    if t.dtype is not torch.float32 or t.shape != token.shape or t.device != token.device or not t.is_contiguous():
        raise ValueError(f"{what}: need a contiguous float32 tensor of shape {tuple(token.shape)} on {token.device}, got {t.dtype} {tuple(t.shape)} on {t.device}")
    return t.data_ptr()


def _rows(logits, token, avail, temperature):
    device, shape = logits.device, logits.shape
    if device.type != "cuda":
        raise ValueError(f"logits are on {device}: the kernels have no CPU form")
    dtype = _DTYPES.get(logits.dtype)
    if dtype is None:
        raise ValueError(f"logits: float32, float16 or bfloat16, got {logits.dtype}")
    if not shape or shape[-1] < 1 or token.shape != shape[:-1]:
        raise ValueError(f"token: need shape {tuple(shape[:-1])} for logits {tuple(shape)}, got {tuple(token.shape)}")
    width = 8 if token.dtype is torch.int64 else 4 if token.dtype is torch.int32 else 0
    if not width or token.device != device or not token.is_contiguous():
        raise ValueError(f"token: need a contiguous int32 or int64 tensor on {device}, got {token.dtype} on {token.device}")
    av, av_ld = None, 0
    if avail is not None:
        if avail.dtype not in (torch.uint8, torch.bool) or avail.shape != shape or avail.device != device:
            raise ValueError(f"avail: need uint8 or bool of shape {tuple(shape)} on {device}, got {avail.dtype} {tuple(avail.shape)} on {avail.device}")
        av, av_ld = avail.data_ptr(), _row_stride(avail, "avail")
    return N.TokenRows(logits.data_ptr(), _row_stride(logits, "logits"), av, av_ld, token.data_ptr(), token.numel(), shape[-1], dtype, width, 0, temperature)


def _grad(out, logits):
    """The tensor that receives the gradient and its row stride; ``out`` may be the logits themselves."""
    if out is None:
        return torch.empty_like(logits, memory_format=torch.contiguous_format), logits.shape[-1]
    if out.dtype != logits.dtype or out.shape != logits.shape or out.device != logits.device:
        raise ValueError(f"out: need {logits.dtype} {tuple(logits.shape)} on {logits.device}, got {out.dtype} {tuple(out.shape)} on {out.device}")
    return out, _row_stride(out, "out")


def _wrote(out, given):
    """The gradient is in `out`; where that is the caller's (`given`), a graph that saved it -- it may lie over the logits -- has to notice."""
    if given is not None:
        torch.autograd.graph.increment_version(given)
    return out


def _workspace(nbytes, device):
    return torch.empty(max(nbytes, 16), dtype=torch.uint8, device=device)


def token_logprob(logits, token, avail=None, temperature=1.0, entropy=False, keep=False):
    """log softmax(logits / temperature)[token] of every row, and its entropy; ``keep=True`` for a later token_logprob_bwd.

    Replaces Categorical(logits).log_prob / .entropy (cleanmarl/mappo_multienvs.py:172-176, 549-550): one pass over the logits."""
    rows = _rows(logits, token, avail, temperature)
    lib, device, index = N.load(), logits.device, logits.get_device()
    with N.on_device(index):
        logp = torch.empty(token.shape, dtype=torch.float32, device=device)
        H = torch.empty(token.shape, dtype=torch.float32, device=device) if entropy else None
        kept = torch.empty((*token.shape, 2), dtype=torch.float32, device=device) if keep else None
        nbytes = lib.cm_token_workspace_bytes(rows.rows, rows.vocab)
        ws = _workspace(nbytes, device)
        N.check(lib.cm_token_logprob(C.byref(rows), logp.data_ptr(), None if H is None else H.data_ptr(), None if kept is None else kept.data_ptr(),
                                     ws.data_ptr(), nbytes, N.raw_stream(index)), "cm_token_logprob")
    return TokenLogProb(logp, H, kept)


def token_logprob_bwd(logits, token, forward, d_logp, d_entropy=None, avail=None, temperature=1.0, out=None):
    """Gradient of sum(d_logp * logp + d_entropy * entropy) with respect to the logits.

    ``forward``: what token_logprob(..., keep=True) returned for the same logits, token, avail and temperature.  ``out``: where the
    gradient goes; the logits themselves are allowed."""
    rows = _rows(logits, token, avail, temperature)
    kept = forward.keep
    if kept is None or kept.dtype is not torch.float32 or kept.shape != (*token.shape, 2) or kept.device != logits.device or not kept.is_contiguous():
        raise ValueError("forward: need the result of token_logprob(..., keep=True) for these rows")
    if d_entropy is not None and forward.entropy is None:
        raise ValueError("d_entropy: the forward call has to compute the entropy (entropy=True)")
    dl, dh = _vector(d_logp, token, "d_logp"), _vector(d_entropy, token, "d_entropy")
    H = _vector(forward.entropy, token, "forward.entropy") if d_entropy is not None else None
    lib, index = N.load(), logits.get_device()
    with N.on_device(index):
        d, ld = _grad(out, logits)
        N.check(lib.cm_token_logprob_bwd(C.byref(rows), kept.data_ptr(), H, dl, dh, d.data_ptr(), ld, N.raw_stream(index)), "cm_token_logprob_bwd")
    return _wrote(d, out)


def policy_loss_fwd_bwd(logits, token, logp_old, adv, logp_ref=None, weight=None, avail=None, temperature=1.0, clip_low=0.2, clip_high=0.2,
                        kl_coef=0.0, entropy_coef=0.0, out=None):
    """Clipped policy loss with a KL term, forward and backward in one call (cleanmarl/mappo_multienvs.py:536-582 on tokens).

    loss = sum weight * (-min(adv rho, adv clip(rho, 1 - clip_low, 1 + clip_high)) - entropy_coef H + kl_coef (e^d - d - 1)),
    rho = exp(logp - logp_old), d = logp_ref - logp.  ``weight`` carries mask and normalisation (None: ones).  All per-row tensors have
    token's shape.  ``out``: where the gradient goes; the logits themselves are allowed."""
    rows = _rows(logits, token, avail, temperature)
    old, ad = _vector(logp_old, token, "logp_old"), _vector(adv, token, "adv")
    ref, w = _vector(logp_ref, token, "logp_ref"), _vector(weight, token, "weight")
    lib, device, index = N.load(), logits.device, logits.get_device()
    with N.on_device(index):
        d, ld = _grad(out, logits)
        stats = torch.empty(N.NUM_STATS, dtype=torch.float32, device=device)
        logp = torch.empty_like(logp_old)
        nbytes = lib.cm_token_workspace_bytes(rows.rows, rows.vocab)
        ws = _workspace(nbytes, device)
        N.check(lib.cm_token_policy_fwd_bwd(C.byref(rows), old, ad, ref, w, clip_low, clip_high, kl_coef, entropy_coef, d.data_ptr(), ld, logp.data_ptr(),
                                            stats.data_ptr(), ws.data_ptr(), nbytes, N.raw_stream(index)), "cm_token_policy_fwd_bwd")
    return PolicyLoss(stats, _wrote(d, out), logp)


def preference_loss_fwd_bwd(logits, token, seq_start, logp_ref, beta=0.1, label_smoothing=0.0, kind="sigmoid", scale=None, avail=None,
                            temperature=1.0, out=None):
    """Preference loss on paired log ratios, forward and backward in one call.

    ``logits`` [rows, vocab]: the packed rows of 2P sequences, the P chosen answers first, then the P rejected ones; sequence q has the rows
    ``seq_start[q]:seq_start[q + 1]`` (int32, on the device).  Tokens that are not part of an answer are negative.  ``logp_ref`` [2P]: the
    reference policy's sums.  ``kind``: "sigmoid", or "squared" (without label_smoothing).  ``scale``: factor of the gradient, 1/P (the mean
    over the pairs) by default.  Rows outside all sequences of ``out`` are not written (zeros in a tensor that is made here)."""
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
    lib, device, index = N.load(), logits.device, logits.get_device()
    with N.on_device(index):
        d, ld = _grad(torch.zeros_like(logits, memory_format=torch.contiguous_format) if out is None else out, logits)
        stats = torch.empty(N.NUM_STATS, dtype=torch.float32, device=device)
        margin = torch.empty(pairs, dtype=torch.float32, device=device)
        seq_logp = torch.empty(2 * pairs, dtype=torch.float32, device=device)
        nbytes = lib.cm_preference_workspace_bytes(rows.rows, rows.vocab, pairs)
        ws = _workspace(nbytes, device)
        N.check(lib.cm_preference_fwd_bwd(C.byref(rows), seq_start.data_ptr(), pairs, logp_ref.data_ptr(), beta, label_smoothing, _KINDS[kind],
                                          1.0 / pairs if scale is None else scale, d.data_ptr(), ld, margin.data_ptr(), seq_logp.data_ptr(),
                                          stats.data_ptr(), ws.data_ptr(), nbytes, N.raw_stream(index)), "cm_preference_fwd_bwd")
    return PreferenceLoss(stats, _wrote(d, out), margin, seq_logp)
