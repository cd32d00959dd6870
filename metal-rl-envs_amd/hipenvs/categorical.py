"""Log probabilities of given tokens under logits, with entropies, the most likely tokens and the
gradient of the logits: what a policy over actions is trained by and answers with. The reference has
no counterpart.

    log_prob = x[token] - log sum exp x        entropy = -sum p log p, p = softmax x

A logit of -inf is a token that is not allowed: it adds nothing to any sum, and its gradient is zero
(that of the given token apart). A row of nothing else has log probabilities of -inf, entropy 0 and a
gradient of zeros. A negative token is none: log probability 0, and only the entropy has a gradient. A
token past the row is a mistake that the host does not wait to see: its log probability is no number.
Logits are float32 or bfloat16, everything else float32.
"""

import torch

from . import _checks, _lib

MAX_TOP = 64


def _forward(logits, tokens, top, train):
    """(log_prob, entropy, top_log_prob, top_index, stats) for logits (rows, v)."""
    rows, v = logits.shape
    device, ptr = logits.device, _lib.ptr
    log_prob, entropy = (torch.empty(rows, dtype=torch.float32, device=device) for _ in range(2))
    stats = torch.empty((rows, 2), dtype=torch.float32, device=device) if train else None
    top_log_prob = torch.empty((rows, top), dtype=torch.float32, device=device) if top else None
    top_index = torch.empty((rows, top), dtype=torch.int64, device=device) if top else None
    with _lib.on(device):
        nbytes = _lib.lib().hipenvs_log_probs_workspace_bytes(rows, v, top)
        if nbytes < 0:
            raise _lib.HipEnvsError(f"hipenvs_log_probs: unsupported sizes ({rows}, {v}, {top})")
        held = torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None
        _lib.call("hipenvs_log_probs", _checks.DTYPES[logits.dtype], logits.data_ptr(), logits.stride(0),
                  tokens.data_ptr(), log_prob.data_ptr(), entropy.data_ptr(), ptr(stats), top, ptr(top_log_prob),
                  ptr(top_index), rows, v, ptr(held), nbytes, _lib.stream_of(device))
    return log_prob, entropy, top_log_prob, top_index, stats


def _backward(ctx, dlog_prob, dentropy, *_):
    logits, tokens, stats, entropy = ctx.saved_tensors
    dtype, (rows, v), index = ctx.ready
    if logits.dtype is not dtype or logits.shape != (rows, v) or logits.stride(1) != 1 or logits.get_device() != index:
        logits = _checks.saved(logits, dtype, (rows, v), index)
    tokens = _checks.saved(tokens, torch.int64, (rows,), index)
    stats = _checks.saved(stats, torch.float32, (rows, 2), index)
    entropy = _checks.saved(entropy, torch.float32, (rows,), index)
    _checks.refuse_tangents("the gradient of log_probs", dlog_prob, dentropy)
    dlog_prob = _checks.saved(dlog_prob, torch.float32, (rows,), index)
    dentropy = _checks.saved(dentropy, torch.float32, (rows,), index)
    ptr = _lib.ptr
    dlogits = torch.empty((rows, v), dtype=dtype, device=logits.device)
    with _lib.on(logits.device):
        _lib.call("hipenvs_log_probs_backward", _checks.DTYPES[dtype], logits.data_ptr(), logits.stride(0),
                  tokens.data_ptr(), ptr(stats), entropy.data_ptr(), ptr(dlog_prob), ptr(dentropy), dlogits.data_ptr(),
                  rows, v, _lib.stream_of(logits.device))
    return dlogits, None, None


class _LogProbs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, tokens, top):
        ctx.set_materialize_grads(False)
        log_prob, entropy, top_log_prob, top_index, stats = _forward(logits, tokens, top, True)
        ctx.save_for_backward(logits, tokens, stats, entropy)
        ctx.ready = (logits.dtype, tuple(logits.shape), logits.get_device())
        if not top:
            return log_prob, entropy
        ctx.mark_non_differentiable(top_log_prob, top_index)
        return log_prob, entropy, top_log_prob, top_index

    backward = _checks.once(_backward)


def log_probs(logits, tokens, top=0):
    """logits (*lead, v) float32 or bfloat16, tokens (*lead) integers. Returns (log_prob (*lead),
    entropy (*lead)) in float32, differentiable once in logits, in reverse mode; with ``top`` k of 1 to
    64 also (top_log_prob (*lead, k) float32, top_index (*lead, k) int64), the most likely tokens in
    order, of equals the lowest first, without gradients. Asynchronous on the current stream."""
    device = _checks.first(logits, "logits", None)
    lead, v, top = tuple(logits.shape[:-1]), logits.shape[-1], int(top)
    if not 1 <= v <= 0x7FFFFFFF:
        raise ValueError(f"logits must have rows of 1 to 2^31 - 1 values, got shape {tuple(logits.shape)}")
    if not 0 <= top <= min(MAX_TOP, v):
        raise ValueError(f"top must be 0 to {min(MAX_TOP, v)}, got {top}")
    if _checks.tensor(tokens, "tokens").dtype not in (torch.int32, torch.int64):
        raise TypeError(f"tokens must be int32 or int64, got {tokens.dtype}")
    if tuple(tokens.shape) != lead:
        raise ValueError(f"tokens must have shape {lead}, got {tuple(tokens.shape)}")
    if tokens.get_device() != device:
        raise ValueError(f"tokens are on {tokens.device}, logits is on GPU {device}")
    if tokens.numel() > 0x7FFFFFFF:
        raise ValueError(f"there must be fewer than 2^31 rows, got {tokens.numel()}")
    _checks.refuse_tangents("log_probs", logits)
    flat = logits
    if len(lead) != 1:
        flat = logits.reshape(-1, v) if tokens.numel() else logits.reshape(0, v)
        tokens = tokens.reshape(-1)
    if flat.stride(-1) != 1:
        flat = flat.contiguous()
    if tokens.dtype is not torch.int64 or not tokens.is_contiguous():
        tokens = tokens.to(torch.int64).contiguous()
    if _checks.wants_grad(flat):
        found = _LogProbs.apply(flat, tokens, top)
    else:
        found = _forward(flat, tokens, top, False)[:4 if top else 2]
    if len(lead) == 1:
        return tuple(found)
    return tuple(x.view(lead + x.shape[1:]) for x in found)
