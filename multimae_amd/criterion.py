"""Masked losses with the reference's constructor / forward contract (multimae/criterion.py)."""
from typing import NamedTuple, Optional

import torch
from torch import nn

from . import functional as Fn


class _MaskedPixelLoss(nn.Module):
    kind = 0

    def __init__(self, patch_size: int = 16, stride: int = 1, norm_pix=False):
        super().__init__()
        self.patch_size = patch_size
        self.stride = stride
        self.scale_factor = patch_size // stride
        self.norm_pix = norm_pix

    def forward(self, input, target, mask=None):
        """input [B,C,H,W] (fp32 or bf16), target fp32, mask [B, nh*nw] (1 = masked = contributes) or None.

        Mean over channels, masked mean over pixels per sample, mean over the samples that have masked tokens.
        One difference from the reference: when no token is masked at all it returns an fp32 zero (the reference
        returns an int64 zero) because the count stays on the device."""
        if mask is not None and mask.dtype != torch.int64:
            mask = mask.to(torch.int64)
        return Fn.MaskedLossFn.apply(input, target.float(), None if mask is None else mask.contiguous(), self.kind,
                                     bool(self.norm_pix), self.scale_factor)


class MaskedMSELoss(_MaskedPixelLoss):
    """Reference: multimae/criterion.py:68-130."""
    kind = 0


class MaskedL1Loss(_MaskedPixelLoss):
    """Reference: multimae/criterion.py:133-195."""
    kind = 1


class MaskedCrossEntropyLoss(nn.Module):
    """Reference: multimae/criterion.py:23-65.  input [B,C,H,W] logits (fp32 or bf16), target int64 [B,H,W],
    mask [B, (H/scale)*(W/scale)] with scale = patch_size // stride.  As with the pixel losses, an all-zero mask
    yields an fp32 zero (the reference returns an int64 zero)."""

    def __init__(self, patch_size: int = 16, stride: int = 1, label_smoothing: float = 0.0):
        super().__init__()
        self.patch_size = patch_size
        self.stride = stride
        self.scale_factor = patch_size // stride
        self.label_smoothing = label_smoothing

    def forward(self, input, target, mask=None):
        if mask is not None and mask.dtype != torch.int64:
            mask = mask.to(torch.int64)
        return Fn.MaskedCEFn.apply(input, target.to(torch.int64), None if mask is None else mask.contiguous(),
                                   self.scale_factor, float(self.label_smoothing))


class ClassLogProbs(NamedTuple):
    """What class_log_probs returns: the alternatives have the shape [B, top_k, ...], None for top_k = 0."""
    log_prob: torch.Tensor
    entropy: torch.Tensor
    top_log_prob: Optional[torch.Tensor]
    top_class: Optional[torch.Tensor]


def class_log_probs(input, target, top_k: int = 0, temperature: float = 1.0) -> ClassLogProbs:
    """Log probability of a given class, entropy, and the most probable classes at every position, from one pass over the
    logits (no counterpart in the reference).

    input [B, C, ...] logits (fp32, bf16 or fp16; rows [N, C] or class maps [B, C, H, W]), target integer classes [B, ...];
    the distribution is softmax(input / temperature) over dimension 1.  A target outside [0, C) (-100: an ignored pixel) has
    log probability 0 and no gradient.  Up to 64 alternatives in descending order, equal logits by the lower class; these
    carry no gradient (they are what MaskedDistillationLoss takes from a teacher).  log_prob and entropy are fp32 and
    differentiable once, in reverse mode; forward mode and tracing are refused.  A position whose logits are all -inf has log probability -inf, entropy 0 and no gradient."""
    if target.dtype != torch.int64:
        target = target.to(torch.int64)
    return ClassLogProbs(*Fn.class_log_probs(input, target, int(top_k), float(temperature)))


class MaskedDistillationLoss(nn.Module):
    """Distillation from a teacher's most probable classes, beside MaskedCrossEntropyLoss and averaged like it (no
    counterpart in the reference): temperature^2 * KL(teacher || student) per position, masked mean over the positions of a
    sample, then mean over the samples that have any.

    teacher="logits": the target's values are the teacher's logits of the kept classes, and its distribution is
    softmax(values / temperature) over these.  teacher="log_probs": they are its log probabilities at this temperature (the
    top_log_prob of class_log_probs), and what the kept classes leave of 1 is compared with the student's probability of
    all other classes together.  Differentiable once, in the student's logits, in reverse mode; forward mode and tracing are refused."""

    def __init__(self, patch_size: int = 16, stride: int = 1, temperature: float = 1.0, teacher: str = "logits"):
        super().__init__()
        if teacher not in ("logits", "log_probs"):
            raise ValueError(f"MaskedDistillationLoss: teacher {teacher!r} is neither 'logits' nor 'log_probs'")
        self.patch_size = patch_size
        self.stride = stride
        self.scale_factor = patch_size // stride
        self.temperature = temperature
        self.teacher = teacher

    def forward(self, input, target, mask=None):
        """input [B, C, H, W] logits (fp32, bf16 or fp16; also rows [N, C] or sequences [B, C, L]); target = (classes int32 or
        int64 [B, k, H, W], values [B, k, H, W]) with k <= 64; a class outside [0, C) (-1) is padding.  mask
        [B, (H/scale)*(W/scale)] with scale = patch_size // stride (rows: [N], sequences: [B, L]), nonzero = in the loss.
        A mask that is zero everywhere gives a loss and a gradient of zero.  A position in the loss whose logits are all -inf makes
        the loss +inf and has no gradient."""
        top_class, top_value = target
        if mask is not None:
            if mask.dtype != torch.int64:
                mask = mask.to(torch.int64)
            mask = mask.reshape(input.shape[0], -1).contiguous()
        patch = self.scale_factor if input.dim() == 4 else 1
        return Fn.distill(input, top_class, top_value, mask, patch, float(self.temperature), self.teacher == "log_probs")
