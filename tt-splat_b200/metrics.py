"""Image metrics and the photometric loss (mirrors spike/metrics.py:1-28).

``loss_fn`` runs the fused L1 + SSIM kernel, which returns the loss and its gradient in one
pass; the autograd backward scales the stored gradient.  Images are [H,W,3] (or [V,H,W,3]).
``label_log_probs`` scores rows of label logits (a render's [H,W,C], a batch's [N,C]).
"""
from typing import NamedTuple

import torch

from ._lib import on_device, torch_ops
from . import ops


class _LossFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, pred, gt, lam):
        p = pred.detach().float().contiguous()
        g = gt.detach().float().contiguous().to(p.device)
        out = ops.loss_l1_ssim(p, g, lam, 1.0)
        ctx.save_for_backward(out["gimg"].reshape(pred.shape))
        return out["loss"].sum()

    @staticmethod
    def backward(ctx, gout):
        (gimg,) = ctx.saved_tensors
        return gimg * gout, None, None


def loss_fn(pred, gt, lambda_ssim=0.2):
    """(1-l)*L1 + l*(1-SSIM) (spike/metrics.py:26-28); SSIM on [0,1]-clamped inputs, window 11
    shrunk for small images (:15-19).  For a [V,H,W,3] batch, the sum of the per-view losses."""
    with on_device(pred):
        return _LossFn.apply(pred, gt, float(lambda_ssim))


def psnr(pred, gt):
    """spike/metrics.py:10-12."""
    mse = (pred.clamp(0.0, 1.0) - gt.clamp(0.0, 1.0)).pow(2).mean()
    return -10.0 * torch.log10(mse.clamp(min=1e-12))


def l1(pred, gt):
    """spike/metrics.py:22-23."""
    return (pred - gt).abs().mean()


def ssim(pred, gt, win_size=11):
    """SSIM of [H,W,3] images (spike/metrics.py:15-19) from the fused kernel (lambda = 1 makes
    the loss 1 - SSIM)."""
    return 1.0 - ops.loss_l1_ssim(pred.detach().float().contiguous(), gt.float().contiguous().to(pred.device),
                                  1.0, 1.0)["loss"].sum()


class LabelLogProbs(NamedTuple):
    logp: torch.Tensor        # [...] log probability of the given label
    entropy: torch.Tensor     # [...] entropy of the row's distribution
    top_logp: torch.Tensor    # [..., top] log probabilities of the best labels, best first
    top_ids: torch.Tensor     # [..., top] their ids (int64)


def label_log_probs(logits, labels, top=0):
    """Log probabilities of ``labels`` [...] under the softmax of ``logits`` [..., C], with the
    entropy of each row and its ``top`` (0 to 16) best labels -> ``LabelLogProbs`` in fp32.

    Logits are float32, bfloat16 or float16 with any row stride; labels int32 or int64.  A negative
    label is unlabelled (log probability 0, no gradient), one past the last gives NaN.  Logits of
    -inf are masked labels: never among the best (id -1, log probability -inf where fewer are
    left), and a row of nothing else has log probability -inf, entropy 0 and no gradient.  Ties go
    to the lowest id.  A row with NaN or +inf has NaN results.

    Differentiable once in the logits through all three, in reverse mode only (a forward-mode tangent
    raises); a row whose incoming gradients are zero
    gets zeros whatever it holds, one with NaN or +inf that any gradient reaches gets NaN.  To capture a training step in a CUDA graph, take its gradients
    with ``torch.autograd.grad`` and drop the outputs of eager calls on the same leaves first: torch
    ties a leaf's gradient to the stream of the graph that is still alive, and the capture fails."""
    return LabelLogProbs(*torch_ops().label_log_probs(logits, labels, top))
