"""Loss functions with the reference's names (transvae/loss.py), computed by the fused HIP kernel."""
import torch
from torch.autograd import forward_ad

from . import ops


def trans_vae_loss(x, x_out, mu, logvar, true_len, pred_len, true_prop, pred_prop, weights, beta=1, pad_idx=None):
    """Weighted token cross-entropy + length cross-entropy + beta * KL (+ property MSE).

    Same signature and return order as the reference (transvae/loss.py:23-38):
    ``(total, BCEmol, BCEmask, KLD, MSE)``.  ``x`` are the (B, 127) source token ids (float or
    long); ``true_len`` (B,) or (B,1) are the length classes (the reference passes
    src_mask.sum(-1), trans_models.py:219); None lets the kernel count the non-pad tokens itself
    (``pad_idx``, default len(weights) - 1 = the '_' id of the shipped vocabularies).
    All five values stay on the device; gradients for x_out, mu, logvar, pred_len and pred_prop
    are produced in the same pass and handed to autograd.
    """
    tokens = x.long()
    if pad_idx is None:
        pad_idx = weights.shape[0] - 1
    return ops.LossFn.apply(tokens, x_out, mu, logvar, pred_len, true_prop, pred_prop,
                            weights.to(torch.float32), float(beta), pad_idx, true_len)


def vae_loss(x, x_out, mu, logvar, true_prop, pred_prop, weights, beta=1):
    """Weighted token cross-entropy + beta * KL (+ property MSE): the loss of the RNN models, same signature and return
    order as the reference (transvae/loss.py:8-21): ``(total, BCE, KLD, MSE)``.  The same fused kernel as trans_vae_loss,
    launched without a length head."""
    total, bce, _, kld, mse = ops.LossFn.apply(x.long(), x_out, mu, logvar, None, true_prop, pred_prop,
                                               weights.to(torch.float32), float(beta), weights.shape[0] - 1, None)
    return total, bce, kld, mse


MAX_TOP = 64


def token_logprobs(logits, tokens=None, top=0):
    """Log probabilities of given tokens under logits (..., V), with the entropy of every row and its `top` (0 .. 64) most likely
    alternatives: ``(logp, entropy, top_logp, top_ids)`` of shapes (...), (...), (..., top), (..., top).

    logits: float32, bfloat16 or float16; tokens: integer class ids (...), or None (logp is then 0).  A token outside [0, V) is
    padding: its logp is 0 and passes no gradient, entropy and alternatives are the row's all the same.  Alternatives come in
    descending order, equal logits in ascending order of their ids.  A class at -inf has probability 0 (and gradient 0); a
    row of nothing else has logp -inf, entropy 0 and gradient 0; a NaN or +inf makes its row NaN.  Results are float32 (ids
    int64).  logp, entropy and top_logp are differentiable in the logits, once and backward (forward-mode tangents
    are refused); a captured backward pass is to be captured while no eager autograd graph of the same leaves is alive, as with
    any other op.  No counterpart in the reference, whose losses (transvae/loss.py:8-38) only give weighted means."""
    if logits.dim() < 1 or logits.shape[-1] < 1 or logits.dtype not in ops.LOGIT_TYPES:
        raise ops._lib.TvaeError("token_logprobs: logits must be float32, bfloat16 or float16 (..., V), got %s %s" % (tuple(logits.shape), logits.dtype))
    V, lead = logits.shape[-1], logits.shape[:-1]
    if not 0 <= top <= min(V, MAX_TOP):
        raise ops._lib.TvaeError("token_logprobs: top must be in [0, min(V, %d)] (got %s for V = %d)" % (MAX_TOP, top, V))
    if tokens is not None:
        if tokens.shape != lead or tokens.is_floating_point() or tokens.dtype == torch.bool or tokens.device != logits.device:
            raise ops._lib.TvaeError("token_logprobs: tokens must be integers of shape %s on %s, got %s %s on %s"
                                     % (tuple(lead), logits.device, tuple(tokens.shape), tokens.dtype, tokens.device))
        if tokens.dim() != 1 or tokens.dtype != torch.int64:
            tokens = tokens.reshape(-1).long()
    if forward_ad._current_level >= 0 and forward_ad.unpack_dual(logits).tangent is not None:    # the level first: 0.6 us less a call
        raise ops._lib.TvaeError("token_logprobs: no forward-mode derivatives (its gradient is a backward pass)")
    if logits.requires_grad and torch.is_grad_enabled():
        logp, entropy, top_logp, top_ids = ops.TokenLogpFn.apply(logits, tokens, int(top))
    else:
        logp, entropy, _, top_logp, top_ids = ops.token_logp(logits, tokens, int(top))
    if logits.dim() == 2:
        return logp, entropy, top_logp, top_ids
    return logp.view(lead), entropy.view(lead), top_logp.view(*lead, top), top_ids.view(*lead, top)
