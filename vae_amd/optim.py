"""Fused optimiser step on the flat arenas: gradient clipping by global norm
(``Trainer(gradient_clip_val=0.5)``, train.py:54) + AdamW with the reference's groups
(``betas=(0.9, 0.998)``, ``eps=1e-7``, weight decay on ``z_encoder`` / ``cell_decoder`` only,
task.py:534-553) in two HIP launches (``vae_adamw_step``), replacing ``clip_grad_norm_`` +
``torch.optim.AdamW.step`` (dozens of multi-tensor launches, seven passes over 18 M parameters).

The learning-rate schedule stays on the host: pass ``lr_lambda`` (e.g.
``WarmupConstantAndDecaySchedule.lr_lambda``, task.py:662-676); ``step()`` evaluates it at the number
of steps already taken, exactly like ``LambdaLR`` stepped once per optimiser step.
"""
from __future__ import annotations

import ctypes as C
import struct
from typing import Callable, Dict, Iterable, List, Optional, Sequence, Tuple, Union

import torch

from . import _lib
from .arena import ParamArena
from .ops import _on, _raw_stream


def reference_weight_decay(name: str, weight_decay: float) -> float:
    """The reference's two groups (task.py:534-553): decay only on z_encoder.* and cell_decoder.*."""
    return weight_decay if ("z_encoder" in name or "cell_decoder" in name) else 0.0


class FusedAdamW:
    def __init__(self, arena: ParamArena, lr: float = 5e-4, betas: Tuple[float, float] = (0.9, 0.998), eps: float = 1e-7,
                 weight_decay: float = 0.0, max_grad_norm: float = 0.5,
                 decay_of: Callable[[str, float], float] = reference_weight_decay,
                 lr_lambda: Optional[Callable[[int], float]] = None, skip: Iterable[str] = (),
                 track_weight_maxima: bool = False, track_bf16_images: bool = False):
        """``skip``: parameter names that receive no gradient in this run (e.g. the cell heads when no
        cell loss is used) in addition to ``arena.no_grad``: torch leaves grad=None parameters alone.

        ``track_weight_maxima``: every step also leaves the partial maxima of the two gene-sized weight matrices
        (first-layer encoder weights, decoder-head weights) in ``self.weight_maxima`` (2, P) while it stores the updated
        weights; ``ElboStep.use_weight_maxima(opt)`` then skips the step's own 72 MB scan for the two-f16-term GEMM
        scales.  Anything else that changes those weights must call ``arena.touch()`` (``broadcast_parameters`` and
        ``LitVAE``'s state-dict load hook do) or ``refresh_weight_maxima()``.

        ``track_bf16_images``: the bf16-mode counterpart -- every step also leaves bf16 images (nearest even) of the same
        two matrices in ``self.weight_images`` while it stores the updated weights; ``ElboStep.use_weight_images(opt)``
        then skips the step's own cast launch (6 bytes per weight per step).  Same rule: ``refresh_weight_images()`` after
        anything else changed the weights.  One of the two options at a time (they belong to different precision modes)."""
        if not arena.flat.is_cuda:
            raise RuntimeError("vae_amd: FusedAdamW needs the arena on a GPU (there is no CPU fallback)")
        self.lib = _lib.load()
        self.arena = arena
        self.base_lr, self.betas, self.eps = float(lr), (float(betas[0]), float(betas[1])), float(eps)
        self.max_grad_norm = float(max_grad_norm) if max_grad_norm else 0.0
        self.lr_lambda = lr_lambda
        self.steps = 0
        self.exp_avg = torch.zeros_like(arena.flat)
        self.exp_avg_sq = torch.zeros_like(arena.flat)
        self.grad_norm = torch.zeros(1, dtype=torch.float32, device=arena.device)
        self._ws = torch.empty(self.lib.vae_adamw_workspace_bytes() // 4, dtype=torch.float32, device=arena.device)
        # contiguous ranges with one weight decay each, in arena order
        skipped = set(skip) | set(arena.no_grad)
        ranges: List[Tuple[int, int, float]] = []
        for name, (off, shape) in arena.offsets.items():
            if name in skipped:
                continue
            n = arena.extent(name)
            wd = float(decay_of(name, weight_decay))
            if ranges and ranges[-1][1] == off and ranges[-1][2] == wd:
                ranges[-1] = (ranges[-1][0], off + n, wd)
            else:
                ranges.append((off, off + n, wd))
        # alignment padding between groups (<= 3 floats, zero in every arena) is bridged between equal-decay neighbours --
        # but only when the gap really is padding: a skipped / gradient-less parameter of <= 3 elements sitting there
        # must stay untouched, as torch leaves grad=None parameters alone
        def is_padding(lo: int, hi: int) -> bool:
            for name, (off, shape) in arena.offsets.items():
                n = arena.extent(name)
                if off < hi and off + n > lo:
                    return False
            return True

        merged: List[Tuple[int, int, float]] = []
        for r in ranges:
            if merged and r[0] - merged[-1][1] <= 3 and merged[-1][2] == r[2] and is_padding(merged[-1][1], r[0]):
                merged[-1] = (merged[-1][0], r[1], r[2])
            else:
                merged.append(r)
        if len(merged) > 16:
            raise RuntimeError(f"vae_amd: FusedAdamW supports up to 16 ranges, this arena needs {len(merged)}")
        self.ranges = merged
        self._segs = (_lib.AdamWSegment * len(merged))(*[_lib.AdamWSegment(b, e, wd) for b, e, wd in merged])
        self.weight_maxima = None
        self.weight_images = None
        if track_weight_maxima and track_bf16_images:
            raise ValueError("vae_amd: FusedAdamW: track_weight_maxima (two-f16-term mode) or track_bf16_images (bf16 mode), not both")
        if track_weight_maxima or track_bf16_images:
            from .arena import _enc
            def span(first, last):
                b = arena.offsets[first][0]
                e = arena.offsets[last][0] + arena.extent(last)
                return b, e
            enc = span(_enc("z_encoder", 0, "w"), _enc("l_encoder", 0, "w"))
            heads = span("decoder.px_scale_decoder.0.weight",
                         "decoder.px_dropout_decoder.weight" if arena.likelihood == "zinb" else "decoder.px_scale_decoder.0.weight")
            if any(v % 4 for v in enc + heads):
                raise RuntimeError("vae_amd: FusedAdamW(track_weight_maxima / track_bf16_images): the weight matrices are "
                                   "not 16-byte multiples")
            self._max_ranges = (C.c_int64 * 4)(enc[0], enc[1], heads[0], heads[1])
            self._max_spans = (enc, heads)
        if track_weight_maxima:
            self.weight_maxima = torch.zeros(2, int(self.lib.vae_adamw_wmax_partials()), dtype=torch.float32, device=arena.device)
            self.refresh_weight_maxima()
        if track_bf16_images:
            self.weight_images = tuple(torch.empty(e - b, dtype=torch.bfloat16, device=arena.device) for b, e in self._max_spans)
            self.refresh_weight_images()
        self._seen_version = arena.version

    def sync(self) -> None:
        """Refresh the tracked side products when the arena was written by anything but ``step()`` since they were made
        (``ParamArena.touch()``: ``broadcast_parameters`` and ``LitVAE``'s load hook call it; ``ElboStep`` calls this before
        every step that consumes them -- an integer compare)."""
        if self._seen_version != self.arena.version:
            self.refresh_weight_maxima()
            self.refresh_weight_images()
            self._seen_version = self.arena.version

    def refresh_weight_images(self) -> None:
        """Recompute the bf16 images from the weights as they are now (after anything but ``step()`` changed them)."""
        if self.weight_images is None:
            return
        for img, (b, e) in zip(self.weight_images, self._max_spans):
            img.copy_(self.arena.flat[b:e])          # torch rounds to nearest even, as the kernels do

    def refresh_weight_maxima(self) -> None:
        """Recompute the tracked maxima from the weights as they are now (after anything but ``step()`` changed them)."""
        if self.weight_maxima is None:
            return
        self.weight_maxima.zero_()
        for r, (b, e) in enumerate(self._max_spans):
            self.weight_maxima[r, 0] = self.arena.flat[b:e].abs().max()

    @property
    def lr(self) -> float:
        """Learning rate of the NEXT step."""
        return self.base_lr * (float(self.lr_lambda(self.steps)) if self.lr_lambda is not None else 1.0)

    def step(self, grad_scale: float = 1.0) -> None:
        lr = self.lr
        self.steps += 1
        a = self.arena
        if self.weight_maxima is not None:
            rc = self.lib.vae_adamw_step_wmax(a.flat.data_ptr(), a.flat_grad.data_ptr(), self.exp_avg.data_ptr(),
                                              self.exp_avg_sq.data_ptr(), a.total, self._segs, len(self.ranges), lr, self.betas[0],
                                              self.betas[1], self.eps, self.steps, self.max_grad_norm, float(grad_scale),
                                              self._ws.data_ptr(), self._ws.numel() * 4, self.grad_norm.data_ptr(),
                                              self._max_ranges, self.weight_maxima.data_ptr(),
                                              C.c_void_p(torch.cuda.current_stream().cuda_stream))
            _lib.check(rc, "adamw_step_wmax")
            return
        if self.weight_images is not None:
            rc = self.lib.vae_adamw_step_bf16(a.flat.data_ptr(), a.flat_grad.data_ptr(), self.exp_avg.data_ptr(),
                                              self.exp_avg_sq.data_ptr(), a.total, self._segs, len(self.ranges), lr, self.betas[0],
                                              self.betas[1], self.eps, self.steps, self.max_grad_norm, float(grad_scale),
                                              self._ws.data_ptr(), self._ws.numel() * 4, self.grad_norm.data_ptr(),
                                              self._max_ranges, self.weight_images[0].data_ptr(), self.weight_images[1].data_ptr(),
                                              C.c_void_p(torch.cuda.current_stream().cuda_stream))
            _lib.check(rc, "adamw_step_bf16")
            return
        rc = self.lib.vae_adamw_step(a.flat.data_ptr(), a.flat_grad.data_ptr(), self.exp_avg.data_ptr(),
                                     self.exp_avg_sq.data_ptr(), a.total, self._segs, len(self.ranges), lr, self.betas[0],
                                     self.betas[1], self.eps, self.steps, self.max_grad_norm, float(grad_scale),
                                     self._ws.data_ptr(), self._ws.numel() * 4, self.grad_norm.data_ptr(),
                                     C.c_void_p(torch.cuda.current_stream().cuda_stream))
        _lib.check(rc, "adamw_step")

    def state_dict(self) -> Dict[str, object]:
        return {"steps": self.steps, "exp_avg": self.exp_avg, "exp_avg_sq": self.exp_avg_sq}

    def load_state_dict(self, sd: Dict[str, object]) -> None:
        self.steps = int(sd["steps"])
        self.exp_avg.copy_(sd["exp_avg"])
        self.exp_avg_sq.copy_(sd["exp_avg_sq"])


class L1Penalty:
    """``l1_lambda * sum(|p|)`` over the parameters the reference regularises (task.py:491-496: every
    ``z_encoder`` parameter whose name has no "bias" -- the Linear weights AND the LayerNorm scales), on the
    flat arena: one launch adds ``coeff * sign(p)`` to the gradients and sums ``|p|`` (``vae_l1_penalty``)."""

    def __init__(self, arena: ParamArena, selects: Callable[[str], bool] = lambda n: "z_encoder" in n and "bias" not in n):
        if not arena.flat.is_cuda:
            raise RuntimeError("vae_amd: L1Penalty needs the arena on a GPU (there is no CPU fallback)")
        self.lib = _lib.load()
        self.arena = arena
        ranges: List[Tuple[int, int]] = []
        for name, (off, shape) in arena.offsets.items():
            if name in arena.no_grad or not selects(name):
                continue
            n = arena.extent(name)
            if ranges and ranges[-1][1] == off:
                ranges[-1] = (ranges[-1][0], off + n)
            else:
                ranges.append((off, off + n))
        ranges.sort()
        if not 0 < len(ranges) <= 16:
            raise RuntimeError(f"vae_amd: L1Penalty supports 1..16 ranges, got {len(ranges)}")
        self.ranges = ranges
        self._segs = (_lib.AdamWSegment * len(ranges))(*[_lib.AdamWSegment(b, e, 0.0) for b, e in ranges])
        self._ws = torch.empty(self.lib.vae_adamw_workspace_bytes() // 4, dtype=torch.float32, device=arena.device)
        self.total = torch.zeros(1, dtype=torch.float32, device=arena.device)

    def apply(self, grad_coeff: float, backward: bool = True) -> torch.Tensor:
        """-> sum(|p|) as a 0-dim GPU tensor; gradients += grad_coeff * sign(p) when ``backward``."""
        a = self.arena
        rc = self.lib.vae_l1_penalty(a.flat.data_ptr(), a.flat_grad.data_ptr() if backward else None, a.total, self._segs,
                                     len(self.ranges), float(grad_coeff), self._ws.data_ptr(), self._ws.numel() * 4,
                                     self.total.data_ptr(), C.c_void_p(torch.cuda.current_stream().cuda_stream))
        _lib.check(rc, "l1_penalty")
        return self.total[0]


ADAMW_BLOCK = 256                      # VAE_ADAMW_BLOCK: elements of a block of the flat state
_ADAMW_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def adamw_blocks(n: int) -> int:
    """Blocks of the flat state that a tensor of ``n`` elements owns."""
    return -(-n // ADAMW_BLOCK)


def multi_tensor_adamw_(params: Sequence[torch.Tensor], grads: Sequence[Optional[torch.Tensor]], exp_avg: torch.Tensor,
                        exp_avg_sq: torch.Tensor, *, step: Union[int, Sequence[int]], lr: float, betas: Tuple[float, float] = (0.9, 0.998),
                        eps: float = 1e-7, weight_decay: Union[float, Sequence[float]] = 0.0, scales: Optional[torch.Tensor] = None,
                        master: Optional[torch.Tensor] = None, max_grad_norm: float = 0.0, grad_scale: float = 1.0, seed: int = 0,
                        return_norm: bool = False) -> Optional[torch.Tensor]:
    """One AdamW step in place over ``params`` (contiguous fp32 / bf16 / fp16 tensors on one GPU) in one launch for every 96 of
    them, or for every 8 counts of steps among them (include/vae_amd.h, ``vae_adamw_multi``).  A parameter whose gradient is
    None is left alone, with its state.

    The state is flat, in the order of ``params``: every tensor starts a new block of ``ADAMW_BLOCK`` elements.  fp32
    ``exp_avg`` / ``exp_avg_sq``: 32-bit moments.  float8_e4m3fn ones: 8-bit moments, where ``exp_avg_sq`` holds the ROOT of
    the second moment and a code times ``scales[0 | 1, block]`` is the value; the root is rounded at random by
    ``(seed, the tensor's step, element)``, so equal calls give equal bits.  ``master``: fp32 weights in the same layout, which
    are updated in the parameters' place; the parameters then receive their rounding.  Start all of them at zero (``master``: at
    the parameters).

    ``step`` counts from 1: one value, or a list with one for each tensor, by which its bias is corrected (``torch.optim.AdamW``
    counts a parameter's own steps, and one without a gradient takes none).  ``weight_decay``: one value, or one for each
    tensor.  ``max_grad_norm`` > 0 clips by the norm over all gradients; ``return_norm`` returns that norm (of ``grad_scale``
    times the gradients, before clipping) as a 1-element tensor.  The learning rate and the step count are host values: a captured graph would repeat them, so capturing raises."""
    lib = _lib.load()
    n = len(params)
    if len(grads) != n:
        raise ValueError(f"vae_amd.optim.multi_tensor_adamw_: {n} params and {len(grads)} grads")
    dev = exp_avg.device
    if dev.type != "cuda":
        raise RuntimeError("vae_amd.optim.multi_tensor_adamw_: the state must live on the GPU (no CPU fallback)")
    bits = 8 if exp_avg.dtype == torch.float8_e4m3fn else 32
    if exp_avg.dtype not in (torch.float8_e4m3fn, torch.float32) or exp_avg_sq.dtype != exp_avg.dtype:
        raise TypeError("vae_amd.optim.multi_tensor_adamw_: exp_avg and exp_avg_sq must both be float32 or both float8_e4m3fn")
    if isinstance(weight_decay, (int, float)):
        decay: Sequence[float] = [float(weight_decay)] * n
    else:
        decay = weight_decay
        if len(decay) != n:
            raise ValueError(f"vae_amd.optim.multi_tensor_adamw_: {n} params and {len(decay)} weight decays")
    if isinstance(step, (list, tuple)):
        counts, step = step, 1
        if len(counts) != n:
            raise ValueError(f"vae_amd.optim.multi_tensor_adamw_: {n} params and {len(counts)} counts of steps")
        if n and min(counts) < 1:
            raise ValueError("vae_amd.optim.multi_tensor_adamw_: step counts from 1")
    else:
        counts = [0] * n                                                # (the call's)
    table: List[Union[int, float]] = []
    at, live, index = 0, [], dev.index
    for p, g, wd, count_of in zip(params, grads, decay, counts):
        count = p.numel()
        if g is not None and count:
            dtype = p.dtype
            kind = _ADAMW_DTYPES.get(dtype)
            if kind is None or g.dtype is not dtype:
                raise TypeError(f"vae_amd.optim.multi_tensor_adamw_: a parameter of {p.dtype} with a gradient of {g.dtype}; "
                                "float32, bfloat16 and float16 are supported, both of the same type")
            if p.get_device() != index or g.get_device() != index:      # (-1: on the CPU)
                raise RuntimeError(f"vae_amd.optim.multi_tensor_adamw_: parameters, gradients and state must be on {dev}")
            if g.shape != p.shape or not p.is_contiguous() or not g.is_contiguous():
                raise ValueError("vae_amd.optim.multi_tensor_adamw_: parameters and gradients must be contiguous and of one shape")
            table += (p.data_ptr(), g.data_ptr(), count, at, wd, kind, count_of)
            live.append(p)
        at += -(-count // ADAMW_BLOCK)
    for t, name in ((exp_avg, "exp_avg"), (exp_avg_sq, "exp_avg_sq"), (master, "master")):
        if t is None:
            continue
        if t.numel() != at * ADAMW_BLOCK or t.device != dev or not t.is_contiguous():
            raise ValueError(f"vae_amd.optim.multi_tensor_adamw_: {name} must hold {at * ADAMW_BLOCK} contiguous elements on {dev}")
    if master is not None and master.dtype != torch.float32:
        raise TypeError("vae_amd.optim.multi_tensor_adamw_: master must be float32")
    if bits == 8:
        if scales is None or scales.dtype != torch.float32 or scales.numel() != 2 * at or scales.device != dev or not scales.is_contiguous():
            raise ValueError(f"vae_amd.optim.multi_tensor_adamw_: 8-bit moments need contiguous float32 scales (2, {at}) on {dev}")
    clip = max_grad_norm > 0 or return_norm
    norm = None
    with _on(dev):
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("vae_amd.optim.multi_tensor_adamw_: step and learning rate are host values; a captured step would repeat them")
        if return_norm:
            norm = torch.zeros(1, dtype=torch.float32, device=dev)
        if not live:
            return norm
        nbytes = lib.vae_adamw_multi_workspace_bytes(len(live)) if clip else 0
        ws = torch.empty(nbytes // 8, dtype=torch.float64, device=dev) if clip else None
        rc = lib.vae_adamw_multi(struct.pack("=" + "QQqqfiq" * len(live), *table), len(live), bits, exp_avg.data_ptr(), exp_avg_sq.data_ptr(),
                                 scales.data_ptr() if bits == 8 else None, at, None if master is None else master.data_ptr(), float(lr),
                                 float(betas[0]), float(betas[1]), float(eps), int(step), float(max_grad_norm), float(grad_scale),
                                 int(seed) & (2 ** 64 - 1), None if ws is None else ws.data_ptr(), nbytes,
                                 None if norm is None else norm.data_ptr(), _raw_stream(dev.index))
    _lib.check(rc, "multi_tensor_adamw_")
    torch.autograd.graph.increment_version(live)       # a backward pass that saved the old values then says so
    return norm


class MultiTensorAdamW:
    """AdamW over separate tensors of any of the three float types, beside ``FusedAdamW`` (which owns ONE fp32 arena): moments
    in 32 or (asked for) 8 bits, optional fp32 master weights, the reference's betas / eps by default (task.py:534-553).

    ``params``: an iterable of tensors, or of dicts ``{"params": [...], "weight_decay": ...}``.  ``state_bits`` 8 keeps two bytes
    and 1/32 of a byte per parameter in place of eight (see ``multi_tensor_adamw_``)."""

    def __init__(self, params: Iterable, lr: float = 5e-4, betas: Tuple[float, float] = (0.9, 0.998), eps: float = 1e-7,
                 weight_decay: float = 0.0, max_grad_norm: float = 0.0, state_bits: int = 32, master_weights: bool = False,
                 lr_lambda: Optional[Callable[[int], float]] = None, seed: int = 0):
        self.params: List[torch.Tensor] = []
        self.decay: List[float] = []
        for group in params:
            members, wd = (list(group["params"]), group.get("weight_decay", weight_decay)) if isinstance(group, dict) else ([group], weight_decay)
            self.params += members
            self.decay += [float(wd)] * len(members)
        if not self.params:
            raise ValueError("vae_amd: MultiTensorAdamW got no parameters")
        if len({id(p) for p in self.params}) != len(self.params):
            raise ValueError("vae_amd: MultiTensorAdamW got a parameter twice")
        if state_bits not in (8, 32):
            raise ValueError(f"vae_amd: MultiTensorAdamW: state_bits must be 8 or 32, got {state_bits}")
        dev = self.params[0].device
        for p in self.params:
            if p.dtype not in _ADAMW_DTYPES:
                raise TypeError(f"vae_amd: MultiTensorAdamW: parameters of {p.dtype} are not supported")
            if not p.is_contiguous():
                raise ValueError("vae_amd: MultiTensorAdamW needs contiguous parameters")
            if not p.is_cuda or p.device != dev:
                raise RuntimeError("vae_amd: MultiTensorAdamW needs all parameters on one GPU (there is no CPU fallback)")
        self.base_lr, self.betas, self.eps = float(lr), (float(betas[0]), float(betas[1])), float(eps)
        self.max_grad_norm = float(max_grad_norm) if max_grad_norm else 0.0
        self.lr_lambda, self.seed, self.state_bits = lr_lambda, int(seed), state_bits
        self.steps = 0                                     # calls of step(), by which the learning rate goes
        self.param_steps = [0] * len(self.params)          # and in how many of them each parameter had a gradient
        self.starts, blocks = [], 0
        for p in self.params:
            self.starts.append(blocks * ADAMW_BLOCK)
            blocks += adamw_blocks(p.numel())
        kind = torch.float32 if state_bits == 32 else torch.float8_e4m3fn
        self.exp_avg = torch.zeros(blocks * ADAMW_BLOCK, dtype=torch.uint8 if state_bits == 8 else kind, device=dev).view(kind)
        self.exp_avg_sq = torch.zeros_like(self.exp_avg.view(torch.uint8)).view(kind)
        self.scales = torch.zeros(2, blocks, dtype=torch.float32, device=dev) if state_bits == 8 else None
        self.master = None
        if master_weights:
            self.master = torch.zeros(blocks * ADAMW_BLOCK, dtype=torch.float32, device=dev)
            self.refresh_master()
        self.grad_norm: Optional[torch.Tensor] = None

    def refresh_master(self) -> None:
        """Take the master weights from the parameters as they are now (after anything but ``step()`` changed them)."""
        if self.master is not None:
            for p, b in zip(self.params, self.starts):
                self.master[b:b + p.numel()].copy_(p.detach().reshape(-1))

    @property
    def lr(self) -> float:
        """Learning rate of the NEXT step."""
        return self.base_lr * (float(self.lr_lambda(self.steps)) if self.lr_lambda is not None else 1.0)

    def zero_grad(self) -> None:
        for p in self.params:
            p.grad = None

    def step(self, grad_scale: float = 1.0) -> None:
        """Update from ``p.grad``; ``grad_norm`` holds the unclipped norm afterwards when clipping is on."""
        grads = [p.grad for p in self.params]
        counts = [k + 1 for k in self.param_steps]
        self.grad_norm = multi_tensor_adamw_(self.params, grads, self.exp_avg, self.exp_avg_sq, step=counts, lr=self.lr, betas=self.betas,
                                             eps=self.eps, weight_decay=self.decay, scales=self.scales, master=self.master,
                                             max_grad_norm=self.max_grad_norm, grad_scale=grad_scale, seed=self.seed,
                                             return_norm=self.max_grad_norm > 0)
        self.param_steps = [old if g is None else new for old, new, g in zip(self.param_steps, counts, grads)]
        self.steps += 1

    def moments(self, index: int) -> Tuple[torch.Tensor, torch.Tensor]:
        """-> (exp_avg, exp_avg_sq) of parameter ``index`` in fp32 and in its shape, whatever they are held in."""
        p, b = self.params[index], self.starts[index]
        n = p.numel()
        m, v = (t[b:b + adamw_blocks(n) * ADAMW_BLOCK].float() for t in (self.exp_avg, self.exp_avg_sq))
        if self.state_bits == 8:
            k = b // ADAMW_BLOCK
            m, v = ((t.view(-1, ADAMW_BLOCK) * s[k:k + adamw_blocks(n), None]).view(-1) for t, s in zip((m, v), self.scales))
            v = v * v
        return m[:n].view(p.shape), v[:n].view(p.shape)

    def state_dict(self) -> Dict[str, object]:
        return {"steps": self.steps, "param_steps": list(self.param_steps), "seed": self.seed, "exp_avg": self.exp_avg,
                "exp_avg_sq": self.exp_avg_sq, "scales": self.scales, "master": self.master}

    def load_state_dict(self, sd: Dict[str, object]) -> None:
        """State of an optimiser over the same parameters with the same ``state_bits``.  One that was saved without the parameters'
        own counts of steps: all of them took every step."""
        mine = {k: getattr(self, k) for k in ("exp_avg", "exp_avg_sq", "scales", "master")}
        for k, t in mine.items():
            s = sd[k]
            if (t is None) != (s is None) or (t is not None and (t.shape != s.shape or t.dtype != s.dtype)):
                raise ValueError(f"vae_amd: MultiTensorAdamW.load_state_dict: {k} does not fit (other parameters, state_bits or master_weights)")
        counts = [int(k) for k in sd.get("param_steps", [sd["steps"]] * len(self.params))]
        if len(counts) != len(self.params):
            raise ValueError(f"vae_amd: MultiTensorAdamW.load_state_dict: {len(counts)} counts of steps, {len(self.params)} parameters")
        for k, t in mine.items():
            if t is not None:
                t.copy_(sd[k])
        self.steps, self.param_steps, self.seed = int(sd["steps"]), counts, int(sd["seed"])
