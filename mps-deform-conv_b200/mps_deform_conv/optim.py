"""The optimizer step of a network of these layers: AdamW over all parameters
in one launch, and the gradient norm whose clipping factor it reads on the
device.

    opt = AdamW(model.parameters(), lr=1e-3, state_bits=8)
    loss.backward()                              # allreduce_param_grads(...) across ranks
    norm, factor = grad_norm([p.grad for p in model.parameters()], max_norm=1.0)
    opt.step(grad_scale=factor)

Nothing waits for the host: the norm, the factor, the step counters and a
learning rate given as a tensor stay on the device, so a whole training step
can be captured into a CUDA graph.  A norm that is not finite gives the factor
NaN, and a step with a factor that is not finite writes nothing (the usual
skip of fp16 training with a scaled loss).

The reference has no optimizer of its own; its users train with torch's.
"""
from __future__ import annotations

from typing import List, Optional, Sequence, Tuple, Union

import torch
from torch import Tensor

_SCALE_BLOCK = 256               # elements of one scale of an 8-bit state
_ZERO_SCALE = 2.0 ** -107        # scale of a block of zeros (the smallest one)


def _require_cuda(tensors: Sequence[Tensor], name: str) -> None:
    if tensors and tensors[0].device.type != "cuda":
        raise ValueError(f"{name} must be on CUDA device, got {tensors[0].device}")


def _same_order(a: Tensor, b: Tensor) -> bool:
    """The two tensors' elements lie in the same order in memory."""
    return a.shape == b.shape and ((a.is_contiguous() and b.is_contiguous()) or a.stride() == b.stride())


def new_step(device, taken: int = 0) -> Tensor:
    """A step counter of ``adamw_step``: two int32, the steps taken and a ticket
    that the kernel uses and leaves at 0."""
    return torch.tensor([taken, 0], dtype=torch.int32, device=device)


def new_state(param: Tensor, bits: int = 32) -> Tuple[Tensor, Optional[Tensor]]:
    """One zero state of `param` and its scales: float32 and None, or with 8
    bits float8 e4m3 codes and one float32 scale per 256 elements (in memory
    order)."""
    if bits == 32:
        return torch.zeros_like(param, dtype=torch.float32, memory_format=torch.preserve_format), None
    if bits != 8:
        raise ValueError(f"state_bits must be 32 or 8, got {bits}")
    codes = torch.zeros_like(param, dtype=torch.uint8, memory_format=torch.preserve_format).view(torch.float8_e4m3fn)
    blocks = -(-param.numel() // _SCALE_BLOCK)
    return codes, torch.full((blocks,), _ZERO_SCALE, dtype=torch.float32, device=param.device)


def adamw_step(
    params: Sequence[Tensor],
    grads: Sequence[Tensor],
    exp_avgs: Sequence[Tensor],
    exp_avg_sqs: Sequence[Tensor],
    steps: Sequence[Tensor],
    *,
    lr: Union[float, Tensor],
    betas: Tuple[float, float] = (0.9, 0.999),
    eps: float = 1e-8,
    weight_decay: float = 1e-2,
    masters: Optional[Sequence[Tensor]] = None,
    exp_avg_scales: Optional[Sequence[Tensor]] = None,
    exp_avg_sq_scales: Optional[Sequence[Tensor]] = None,
    grad_scale: Optional[Tensor] = None,
    seed: int = 0,
) -> None:
    """One AdamW step, in place, over many tensors at once.

    Args:
        params: float32, float16 or bfloat16 tensors, dense in memory, on one device
        grads: Gradients of the same shapes and dtypes; not written
        exp_avgs, exp_avg_sqs: States in the parameters' memory formats: float32, or
            with scales given float8_e4m3fn codes of the first moment and of the
            square root of the second (``new_state``)
        steps: One counter per tensor (``new_step``); several may be the same tensor.
            Each is advanced by one
        lr: Learning rate, or one float32 element on the device
        eps: 0, or at least 2^-126
        masters: float32 copies that hold the parameters' values between steps
        exp_avg_scales, exp_avg_sq_scales: Scales of 8-bit states
        grad_scale: One float32 element on the device that multiplies the gradients
            (``grad_norm``'s factor). Not finite: the step is skipped
        seed: Of the stochastic rounding of 8-bit states

    Raises:
        ValueError: If a tensor is not on a CUDA device.
        RuntimeError: If shapes, dtypes, layouts or hyperparameters do not fit, or a
            written tensor overlaps another one of the call (counters may be shared,
            gradients the same).
    """
    from mps_deform_conv import _get_lib
    _require_cuda(params, "params")
    on_device = isinstance(lr, Tensor)
    _get_lib().adamw_step(params, grads, exp_avgs, exp_avg_sqs, steps, masters, exp_avg_scales, exp_avg_sq_scales,
                          0.0 if on_device else lr, lr if on_device else None, betas[0], betas[1], eps, weight_decay,
                          grad_scale, seed & 0xFFFFFFFF)


def grad_norm(grads: Sequence[Tensor], max_norm: Optional[float] = None,
              loss_scale: float = 1.0) -> Tuple[Tensor, Tensor]:
    """The norm of all gradients together, and the factor that clips it.

    Returns ``norm = sqrt(sum of squares) / loss_scale`` and ``factor =
    min(1, max_norm / (norm + 1e-6)) / loss_scale`` as 0-d float32 tensors on
    the device.  Without `max_norm` nothing is clipped.  A norm that is not
    finite gives the factor NaN: ``adamw_step`` then skips its step.  Sums are
    fp64 in a fixed order.

    Raises:
        ValueError: If the gradients are not on a CUDA device or max_norm is negative.
    """
    from mps_deform_conv import _get_lib
    grads = [g for g in grads if g is not None]
    if not grads:
        raise ValueError("grads holds no gradient")
    _require_cuda(grads, "grads")
    if max_norm is not None and not max_norm >= 0:
        raise ValueError(f"max_norm must be non-negative, got {max_norm}")
    return _get_lib().grad_norm(grads, -1.0 if max_norm is None else float(max_norm), float(loss_scale))


class AdamW(torch.optim.Optimizer):
    """AdamW with decoupled weight decay on ``adamw_step``.

    Args:
        params: Parameters or parameter groups (CUDA; float32, float16 or bfloat16)
        lr: Learning rate, or one float32 element on the device that a schedule writes
            (a captured step then follows it)
        betas, eps, weight_decay: As in torch.optim.AdamW
        state_bits: 32, or 8 for float8 states with a scale per 256 elements
        master_weights: Keep float32 copies of 16-bit parameters
        seed: Of the stochastic rounding of 8-bit states

    A parameter without a gradient is left alone and its step not counted.
    """

    def __init__(self, params, lr: Union[float, Tensor] = 1e-3, betas: Tuple[float, float] = (0.9, 0.999),
                 eps: float = 1e-8, weight_decay: float = 1e-2, state_bits: int = 32, master_weights: bool = False,
                 seed: int = 0):
        if not isinstance(lr, Tensor) and not lr >= 0:
            raise ValueError(f"lr must be non-negative, got {lr}")
        if not (0 <= betas[0] < 1 and 0 <= betas[1] < 1):
            raise ValueError(f"betas must be in [0, 1), got {betas}")
        if not eps >= 0:
            raise ValueError(f"eps must be non-negative, got {eps}")
        if not weight_decay >= 0:
            raise ValueError(f"weight_decay must be non-negative, got {weight_decay}")
        if state_bits not in (32, 8):
            raise ValueError(f"state_bits must be 32 or 8, got {state_bits}")
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, state_bits=state_bits,
                                      master_weights=master_weights, seed=seed))

    def _init_state(self, p: Tensor, group) -> dict:
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("AdamW: a parameter has no state yet; take one step before capturing a graph "
                               "(a captured initialisation would reset the state at every replay)")
        state = self.state[p]
        state["step"] = new_step(p.device)
        state["exp_avg"], scale = new_state(p, group["state_bits"])
        state["exp_avg_sq"], scale_sq = new_state(p, group["state_bits"])
        if scale is not None:
            state["exp_avg_scale"], state["exp_avg_sq_scale"] = scale, scale_sq
        if group["master_weights"] and p.dtype != torch.float32:
            state["master"] = p.detach().to(torch.float32, memory_format=torch.preserve_format)
        return state

    @torch.no_grad()
    def step(self, closure=None, grad_scale: Optional[Tensor] = None):
        """One step over every parameter that has a gradient.  `grad_scale`: see
        ``adamw_step``."""
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            # one call per (device, master copy or not); most groups are one
            calls = {}
            for p in group["params"]:
                if p.grad is None:
                    continue
                _require_cuda([p], "parameters")
                state = self.state[p] or self._init_state(p, group)
                calls.setdefault((p.device, "master" in state), []).append((p, state))
            for (device, master), items in calls.items():
                states = [s for _, s in items]

                def column(key: str) -> List[Tensor]:
                    return [s[key] for s in states]

                bits8 = group["state_bits"] == 8
                # one tensor serves parameters on several devices
                lr, scale = (t.to(device) if isinstance(t, Tensor) and t.is_cuda else t for t in (group["lr"], grad_scale))
                adamw_step([p for p, _ in items], [p.grad for p, _ in items], column("exp_avg"),
                           column("exp_avg_sq"), column("step"), lr=lr, betas=group["betas"], eps=group["eps"],
                           weight_decay=group["weight_decay"], masters=column("master") if master else None,
                           exp_avg_scales=column("exp_avg_scale") if bits8 else None,
                           exp_avg_sq_scales=column("exp_avg_sq_scale") if bits8 else None,
                           grad_scale=scale, seed=group["seed"])
        return loss

    def load_state_dict(self, state_dict) -> None:
        """As torch's, but the states keep their own dtypes (torch casts floating
        point states to the parameter's), and a learning rate held as a tensor
        stays that tensor and takes the loaded value, since a schedule writes it.
        The states are new tensors: a step captured before is captured again.
        32-bit states saved from a parameter in another memory format are brought
        to this one's.

        Raises:
            ValueError: If 8-bit states are of another memory format; their scales
                belong to 256 elements in memory order.
        """
        saved = [i for g in state_dict["param_groups"] for i in g["params"]]
        params = [p for g in self.param_groups for p in g["params"]]
        for i, p in zip(saved, params):
            for key, value in state_dict["state"].get(i, {}).items():
                if isinstance(value, Tensor) and value.dtype == torch.float8_e4m3fn and not _same_order(value, p):
                    raise ValueError(f"{key} of parameter {i} holds 8-bit codes in another memory format than the parameter")
        held = [g["lr"] for g in self.param_groups]
        super().load_state_dict(state_dict)
        taken = {}
        for group, lr in zip(self.param_groups, held):
            value = float(group["lr"])
            if isinstance(lr, Tensor):
                if taken.setdefault(id(lr), value) != value:  # groups that shared it and are loaded with different ones
                    lr = lr.detach().clone()
                group["lr"] = lr.fill_(value)
            elif isinstance(group["lr"], Tensor) and group["params"]:
                group["lr"] = group["lr"].detach().to(group["params"][0].device)
        for i, p in zip(saved, params):
            for key, value in state_dict["state"].get(i, {}).items():
                if isinstance(value, Tensor):
                    if value.dtype == torch.float32 and value.shape == p.shape and not _same_order(value, p):
                        value = torch.empty_like(p, dtype=torch.float32, memory_format=torch.preserve_format).copy_(value)
                    self.state[p][key] = value.detach().to(p.device, copy=True)
