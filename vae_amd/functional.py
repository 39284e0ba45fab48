"""Gradient reversal for the adversarial cell heads (role of the reference's src/functional.py:8-30):
the forward pass is the identity, the backward pass multiplies the incoming gradient by -lambd.
Host-side plumbing of the module API; the fused step applies the same sign flip through dz_extra.

``gated_residual_norm``: the norms, gate and residual scale between two residual blocks, on the HIP kernels."""
import functools
from typing import Callable, Optional, Tuple

import torch
from torch import nn


class GradReverse(torch.autograd.Function):
    """``GradReverse.apply(x, lambd)`` -> a tensor equal to ``x`` whose gradient is ``-lambd * dL/dy``."""

    @staticmethod
    def forward(ctx, x: torch.Tensor, lambd: float) -> torch.Tensor:  # noqa: D102
        ctx.neg_scale = -float(lambd)
        return x.view(x.shape)

    @staticmethod
    def backward(ctx, grad_output: torch.Tensor) -> Tuple[Optional[torch.Tensor], None]:  # noqa: D102
        return (grad_output * ctx.neg_scale if ctx.needs_input_grad[0] else None), None


def grad_reverse(x: torch.Tensor, lambd: float = 1.0) -> torch.Tensor:
    """Functional form; ``lambd`` is the reversal strength (grad_reverse_dict of the model config)."""
    return GradReverse.apply(x, lambd)


class GradReverseLayer(nn.Module):
    """Module form, placed in front of an adversarial head (networks.py: CellDecoder)."""

    def __init__(self, lambd: float = 1.0) -> None:
        super().__init__()
        self.lambd = lambd

    def extra_repr(self) -> str:
        return f"lambd={self.lambd}"

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return GradReverse.apply(x, self.lambd)


def gated_residual_norm(r: torch.Tensor, b: torch.Tensor, gate: Optional[torch.Tensor] = None, *,
                        post_weight: Optional[torch.Tensor] = None, post_bias: Optional[torch.Tensor] = None,
                        scale: Optional[torch.Tensor] = None, norm_weight: Optional[torch.Tensor] = None,
                        norm_bias: Optional[torch.Tensor] = None, kind: str = "rms", gate_act: str = "sigmoid",
                        eps: float = 1e-5) -> Tuple[torch.Tensor, torch.Tensor]:
    """Residual stream ``r`` and a block's output ``b`` (..., D), 1 <= D <= 16384, -> (y, h):

        ``y = r + scale * act(gate) * (norm(b) * post_weight + post_bias)``   the new residual stream
        ``h = norm(y) * norm_weight + norm_bias``                            what the next block reads

    in one pass over the rows, forward and backward.  ``norm``: ``kind`` "rms" or "layer", over the last dimension.  Without
    ``post_weight`` the block's output is taken as it is.  ``gate``: (..., D) or (..., 1), through ``gate_act`` "sigmoid",
    "tanh" or "identity".  Absent vectors are 1 or 0.  Rows are float32, bfloat16 or float16; the vectors are all of that type
    or all float32.  ``y`` is rounded to its type before ``h`` is formed.  Gradients reach every tensor given (once: there
    is no second derivative)."""
    if b.dim() < 1 or r.shape != b.shape:
        raise ValueError(f"vae_amd.gated_residual_norm: r is {tuple(r.shape)}, b is {tuple(b.shape)}")
    if gate is not None and tuple(gate.shape[:-1]) != tuple(b.shape[:-1]):
        raise ValueError(f"vae_amd.gated_residual_norm: gate is {tuple(gate.shape)}, b is {tuple(b.shape)}")
    vectors = (t if t is None else t.contiguous() for t in (post_weight, post_bias, scale, norm_weight, norm_bias))
    y, h = _gated_residual_norm()(_rows(r), _rows(b), None if gate is None else _rows(gate), *vectors, kind, gate_act, eps)
    return (y, h) if b.dim() == 2 else (y.view(b.shape), h.view(b.shape))


def _rows(t: torch.Tensor) -> torch.Tensor:
    """(..., D) as (rows, D) with a contiguous last dim."""
    if t.dim() != 2:
        t = t.reshape(-1, t.shape[-1]) if t.shape[-1] else t.reshape(0, 0)
    return t if t.stride(1) == 1 or t.shape[1] <= 1 else t.contiguous()


@functools.lru_cache(maxsize=None)
def _gated_residual_norm() -> Callable:
    from .autograd import GatedResidualNormFn          # (modules that need no kernels import this one)
    return GatedResidualNormFn.apply
