"""Alternative classification losses and GroupDRO re-weighting with the reference's names and
call signatures (src/losses.py:9-202).  Off by default in the reference (task.py:133-134,
config.py:80) and tiny (B x n_classes): plain torch, no kernels.

``linear_cross_entropy`` / ``LinearCrossEntropyLoss``: the cross entropy of the discrete cell-property heads
(task.py:129-137) for heads with many classes, on the HIP kernels and without keeping the logits."""
from __future__ import annotations

from typing import List, Optional

import numpy as np
import torch
import torch.nn as nn
import torch.nn.functional as F


def _smoothed_targets(target: torch.Tensor, num_classes: int) -> torch.Tensor:
    """Label smoothing used by both focal losses: binary 0.95/0.05; otherwise 0.9 on the class
    and 0.05 on each neighbour (clipped at the ends, so an end class keeps 0.95)."""
    target = target.clamp(0, num_classes - 1)
    if num_classes == 2:
        hot = F.one_hot(target, num_classes)
        return 0.95 * hot + 0.05 * (1 - hot)
    out = 0.9 * F.one_hot(target, num_classes)
    for step in (-1, 1):
        out = out + 0.05 * F.one_hot((target + step).clamp(0, num_classes - 1), num_classes)
    return out


class Poly1FocalLoss(nn.Module):
    def __init__(self, num_classes: int, epsilon: float = 1.0, alpha: float = 0.25, gamma: float = 2.0,
                 reduction: str = "none", weight: torch.Tensor = None, pos_weight: torch.Tensor = None,
                 label_is_onehot: bool = False):
        super().__init__()
        self.num_classes, self.epsilon, self.alpha, self.gamma = num_classes, epsilon, alpha, gamma
        self.reduction, self.weight, self.pos_weight, self.label_is_onehot = reduction, weight, pos_weight, label_is_onehot

    def _convert_target(self, target):
        return _smoothed_targets(target, self.num_classes)

    def forward(self, logits, labels):
        if not self.label_is_onehot:
            if labels.ndim == 1:
                labels = self._convert_target(labels)
            else:
                labels = F.one_hot(labels.unsqueeze(1), self.num_classes).transpose(1, -1).squeeze_(-1)
        labels = labels.to(device=logits.device, dtype=logits.dtype)
        p = torch.sigmoid(logits)
        bce = F.binary_cross_entropy_with_logits(logits, labels, reduction="none", weight=self.weight,
                                                 pos_weight=self.pos_weight)
        one_minus_pt = 1 - (labels * p + (1 - labels) * (1 - p))
        focal = bce * one_minus_pt ** self.gamma
        if self.alpha >= 0:
            focal = (self.alpha * labels + (1 - self.alpha) * (1 - labels)) * focal
        poly1 = (focal + self.epsilon * one_minus_pt ** (self.gamma + 1)).sum(dim=-1)
        if self.reduction == "mean":
            return poly1.mean()
        if self.reduction == "sum":
            return poly1.sum()
        return poly1


class FocalLoss(nn.Module):
    def __init__(self, num_classes: int, gamma: float = 2.0, alpha: float = 1.0):
        super().__init__()
        self.gamma, self.num_classes, self.alpha = gamma, num_classes, alpha

    def _convert_target(self, target):
        return _smoothed_targets(target, self.num_classes)

    def forward(self, input, target):
        logp = F.log_softmax(input, dim=-1)
        loss = -self._convert_target(target) * logp * (1 - logp.exp()) ** self.gamma
        return self.alpha * loss.sum(dim=-1)


class GroupDRO:
    """Running per-group loss -> per-sample weights, balanced within each list of groups."""

    DEFAULT_GROUPS = [0, 1, 10, 11, 20, 21, 30, 31, 40, 41, 50, 51, 60, 61, 998, 999]
    DEFAULT_BALANCES = [[0, 1, 60, 61], [10, 11, 50, 51], [20, 21, 40, 41], [30, 31]]

    def __init__(self, groups: Optional[List] = None, balances: Optional[List] = None, alpha: float = 0.99):
        self.groups = list(self.DEFAULT_GROUPS) if groups is None else groups
        self.alpha = alpha
        self.batch_loss = dict.fromkeys(self.groups, 0.0)
        self.batch_count = dict.fromkeys(self.groups, 0)
        self.running_loss = dict.fromkeys(self.groups, 0.0)
        self.weights = dict.fromkeys(self.groups, 1.0)
        self.balances = [list(b) for b in self.DEFAULT_BALANCES] if balances is None else balances

    def update_batch(self, loss, mask, group_idx):
        for l, m, g in zip(loss.tolist(), mask.tolist(), group_idx):
            self.batch_loss[g] += l * m
            self.batch_count[g] += m

    def update_weights(self):
        for g in self.groups:
            if self.batch_count[g] > 1:
                batch_mean = self.batch_loss[g] / self.batch_count[g]
                self.running_loss[g] = self.alpha * self.running_loss[g] + (1 - self.alpha) * batch_mean
            self.batch_loss[g], self.batch_count[g] = 0.0, 0
        for members in self.balances:
            mean_w = np.mean(np.array([self.running_loss[g] for g in members]))
            for g in members:
                self.weights[g] = self.running_loss[g] / mean_w

    def get_weights(self, group_idx):
        return torch.from_numpy(np.array([self.weights[g] for g in group_idx]))


def linear_cross_entropy(x: torch.Tensor, w: torch.Tensor, target: torch.Tensor, *, bias: Optional[torch.Tensor] = None,
                         weight: Optional[torch.Tensor] = None, ignore_index: int = -100, reduction: str = "mean") -> torch.Tensor:
    """``F.cross_entropy(x @ w.T + bias, target, weight, ignore_index=..., reduction=...)`` as float32, differentiable once in
    ``x`` (..., D), ``w`` (V, D) and ``bias`` (V), without the (..., V) logits being kept.

    ``x``, ``w`` and ``bias`` are float32, bfloat16 or float16, all of one type; sums, the softmax statistics and the loss are
    held in 32 bits.  The gradients of the logits are rounded to that type (float32: to 24 bits) ahead of the products that
    give those of ``x`` and ``w``, as the backward pass of a linear layer in 16 bits does.  ``target`` (...) int64; ``weight`` (V)
    float32 class weights.  Rows whose target is ``ignore_index`` take no part: their loss and gradient are 0, and they cost
    next to nothing.  Any other target outside [0, V) makes its row's loss and gradient in ``x`` NaN, and what sums over rows:
    the reduced loss and the gradients in ``w`` and ``bias`` (torch stops with a device assertion).  "mean" divides by the sum of
    the class weights that took part (NaN when none did; the gradients are 0 then).  A class is ruled out by a bias of -inf or
    of the type's lowest value; what an infinity in ``w`` or in a row of ``x`` that takes part reaches is infinite or NaN.

    The backward pass holds the logits' gradients of all rows and as many classes as 512 MiB take, 256 at least: a batch of
    millions of rows is better given in parts (include/vae_amd.h lists the workspaces)."""
    from .autograd import LinearCrossEntropyFn
    if x.dim() < 1 or tuple(target.shape) != tuple(x.shape[:-1]):
        raise ValueError(f"vae_amd.linear_cross_entropy: target must be {tuple(x.shape[:-1])}, got {tuple(target.shape)}")
    if weight is not None and weight.requires_grad:
        raise ValueError("vae_amd.linear_cross_entropy: weight is not differentiable (as in torch); detach it")
    rows = x if x.dim() == 2 else x.reshape(-1, x.shape[-1])
    if rows.numel() and rows.stride(1) != 1 and rows.shape[1] > 1:
        rows = rows.contiguous()
    if w.dim() == 2 and ((w.shape[1] > 1 and w.stride(1) != 1) or (w.shape[0] > 1 and w.stride(0) < w.shape[1])):
        w = w.contiguous()
    bias, weight = (t if t is None else t.contiguous() for t in (bias, weight))
    if rows.shape[0] == 0 and w.dim() == 2 and w.shape[1] == rows.shape[1]:   # as torch: nothing, 0 or 0 / 0, with zero gradients
        if reduction not in ("none", "sum", "mean"):
            raise ValueError(f"vae_amd.linear_cross_entropy: reduction must be 'none', 'sum' or 'mean', got {reduction!r}")
        if not x.is_cuda:
            raise RuntimeError("vae_amd.linear_cross_entropy: all tensors must live on one GPU (no CPU fallback)")
        zero = (rows.float().sum() + 0.0 * sum(t.float().flatten()[:1].sum() for t in (w, bias) if t is not None))
        return rows.float().sum(1).view(target.shape) if reduction == "none" else zero if reduction == "sum" else zero + float("nan")
    loss = LinearCrossEntropyFn.apply(rows, w, bias, target.reshape(-1).contiguous(), weight, ignore_index, reduction)
    return loss.view(target.shape) if reduction == "none" else loss


class LinearCrossEntropyLoss(nn.Module):
    """A class head and its loss in one: ``forward(x, target)`` is the cross entropy of ``nn.Linear(in_features, num_classes)``
    on ``x`` (``linear_cross_entropy``); ``weight`` as ``task.class_balance_weights`` makes it."""

    def __init__(self, in_features: int, num_classes: int, bias: bool = True, weight: Optional[torch.Tensor] = None,
                 ignore_index: int = -100, reduction: str = "mean"):
        super().__init__()
        self.linear = nn.Linear(in_features, num_classes, bias=bias)
        self.register_buffer("weight", weight, persistent=False)
        self.ignore_index, self.reduction = ignore_index, reduction

    def _apply(self, fn, recurse=True):
        """The class weights follow the head to its device and not to its type (``.bfloat16()`` would round them)."""
        weight = self.weight
        super()._apply(fn, recurse)
        if weight is not None and self.weight.dtype != weight.dtype:
            self.weight = weight.to(self.weight.device)
        return self

    def forward(self, x: torch.Tensor, target: torch.Tensor) -> torch.Tensor:
        weight = None if self.weight is None else self.weight.float()
        return linear_cross_entropy(x, self.linear.weight, target, bias=self.linear.bias, weight=weight,
                                    ignore_index=self.ignore_index, reduction=self.reduction)
