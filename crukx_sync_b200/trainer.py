"""The trainer's side of a sync step: the policy loss that the update comes from, the global norm of
the gradients and clipping, and the AdamW step on fp32 masters whose bf16 weights are the `new` of
encode_update.  No counterpart in the reference, which starts at the two weight dicts.

    out = policy_loss(logits, tokens, advantages, old_logp=old, ref_logp=ref, mask=mask, kl_coef=0.04)
    out.loss.backward()
    norm = grad_norm(grads)
    adamw_step(masters, grads, exp_avg, exp_avg_sq, cur, lr=1e-6, step=t, norm=norm, max_norm=1.0)
    update = encode_update(prev, cur, send_chk)

Gradients, masters, moments and weights are dicts of name -> contiguous CUDA tensor on one device,
as encode_update takes its weights.  Every call runs on the tensors' device and the current stream,
waits for nothing, and takes its scratch from torch's allocator, so calls on different streams do
not meet and a call can be captured into a CUDA graph.  In a captured graph the Python numbers
among the arguments are fixed; adamw_step's `lr` and `step` may be tensors that it reads when it
runs.  Numbers are taken in fp32, and refused where they would be 0 or infinite there.  Caller mistakes are ValueErrors, raised before anything is launched.
"""

from __future__ import annotations

import math
import operator
from collections.abc import Mapping
from dataclasses import dataclass

import torch

from . import _ext
from .codec import _cuda_device

_LEAST, _MOST = 2.0 ** -149, torch.finfo(torch.float32).max   # of fp32: beyond them a number would be 0 or infinite there
_GRADS, _F32, _BF16 = (torch.bfloat16, torch.float16, torch.float32), (torch.float32,), (torch.bfloat16,)


def _names(dtypes) -> str:
    return " or ".join(str(t).replace("torch.", "") for t in dtypes)


def _dict(what: str, d) -> dict:
    if type(d) is dict:
        return d
    if not isinstance(d, Mapping):
        raise ValueError(f"{what} must be a dict of name -> tensor, got {type(d)}")
    return dict(d)


def _real(what: str, x) -> float:
    if type(x) is float:
        return x
    try:
        if not isinstance(x, (str, bytes, bytearray)):
            return float(x)
    except (TypeError, ValueError, OverflowError, RuntimeError):
        pass
    raise ValueError(f"{what}: expected a number, got {type(x)}")


def _reals(what: str, x) -> tuple[float, float]:
    try:
        a, b = x
    except (TypeError, ValueError):
        raise ValueError(f"{what}: expected two numbers, got {x!r}") from None
    return _real(what, a), _real(what, b)


def _count(what: str, x) -> int:
    try:
        n = x if type(x) is int else operator.index(x)
    except TypeError:
        raise ValueError(f"{what}: expected an int, got {type(x)}") from None
    if not 1 <= n < 1 << 63:
        raise ValueError(f"{what} counts from 1, got {n}")
    return n


def _empty_device(grads) -> int:
    """The device of a result that no tensor determines."""
    return -1 if grads else _cuda_device(torch.device("cuda")).index


# ------------------------------------------------------------------ what is wrong with refused arguments

def _check_set(what: str, tensors: dict, dtypes, device=None):
    """Raises for the first tensor that does not fit; returns their one device."""
    for name, t in tensors.items():
        if not isinstance(t, torch.Tensor) or t.dtype not in dtypes:
            raise ValueError(f"{name}: expected a {_names(dtypes)} torch tensor, got {getattr(t, 'dtype', type(t))}")
        if t.layout != torch.strided or not t.is_contiguous():
            raise ValueError(f"{name}: tensor must be contiguous")
        if not t.is_cuda:
            raise ValueError(f"{name}: expected a CUDA tensor")
        if t.is_inference() and what != "gradients":
            raise ValueError(f"{name}: an inference tensor cannot be written")
        if device is None:
            device = t.device
        elif t.device != device:
            raise ValueError("all tensors must be on one device")
    return device


def _check_match(what: str, tensors: dict, grads: dict, dtypes, device) -> None:
    if tensors.keys() != grads.keys():
        raise ValueError(f"{what} and the gradients differ in tensor names: {sorted(tensors.keys() ^ grads.keys())[:5]}")
    _check_set(what, tensors, dtypes, device)
    for name, t in tensors.items():
        if t.numel() != grads[name].numel():
            raise ValueError(f"{name}: {what} and the gradient differ in shape")


def _check_scalar(what: str, t, dtype, device) -> None:
    if t is not None and (not isinstance(t, torch.Tensor) or t.dtype != dtype or t.numel() != 1 or t.device != device):
        raise ValueError(f"{what}: expected one {_names([dtype])} on the gradients' device")


def _refused(what: str):
    raise ValueError(f"{what}: these tensors cannot be taken")


def _tensor(what: str, t):
    if t is not None and not isinstance(t, torch.Tensor):
        raise ValueError(f"{what}: expected a torch tensor, got {type(t)}")
    return t


# ------------------------------------------------------------------ gradients and the step

def grad_norm(grads: Mapping[str, torch.Tensor]) -> torch.Tensor:
    """sqrt(sum of g^2) over every element of every gradient, as a 0-d fp32 CUDA tensor.

    bf16, fp16 and fp32 gradients may be mixed.  The sum is held in 64 bits and squares that would
    overflow or vanish in fp32 count in full; its order is fixed, so equal gradients give equal bits."""
    grads = _dict("gradients", grads)
    norm = _ext.glue().grad_norm(grads, _empty_device(grads))
    if norm is None:
        _check_set("gradients", grads, _GRADS)
        _refused("gradients")
    return norm


def clip_grads(grads: Mapping[str, torch.Tensor], max_norm: float, *, out: Mapping[str, torch.Tensor] | None = None,
               norm: torch.Tensor | None = None) -> torch.Tensor:
    """Scale the gradients so that their global norm is at most `max_norm`; returns the norm before.

    Every gradient is multiplied by min(1, max_norm / (norm + 1e-6)) and rounded to its type: in
    place, or into the tensors of `out` (same names, sizes and types).  `norm` (0-d fp32, on the
    device) takes the place of the gradients' own, for gradients spread over ranks
    (dist.grad_norm_global).  A norm that is not finite is not clipped away: NaN leaves NaN, and an
    infinite one 0, or NaN where the gradient is infinite, as the products say.  Tensors that share
    memory (a tied weight under two names) are refused."""
    max_norm = _real("max_norm", max_norm)
    if not max_norm >= _LEAST:   # (NaN too)
        raise ValueError(f"max_norm must be positive (in fp32), got {max_norm}")
    grads = _dict("gradients", grads)
    if out is not None:
        out = _dict("out", out)
    result = _ext.glue().clip_grads(grads, max_norm, out, _tensor("norm", norm), _empty_device(grads))
    if result is None:
        device = _check_set("gradients" if out is not None else "gradients that are clipped in place", grads, _GRADS)
        if out is not None:
            _check_match("out", out, grads, _GRADS, device)
            for name, g in grads.items():
                if g.dtype != out[name].dtype:
                    raise ValueError(f"{name}: out and the gradient differ in type")
        _check_scalar("norm", norm, torch.float32, device)
        _refused("gradients")
    return result


def adamw_step(masters: Mapping[str, torch.Tensor], grads: Mapping[str, torch.Tensor],
               exp_avg: Mapping[str, torch.Tensor], exp_avg_sq: Mapping[str, torch.Tensor],
               weights: Mapping[str, torch.Tensor] | None = None, *, lr, step, betas=(0.9, 0.999), eps: float = 1e-8,
               weight_decay: float = 0.0, norm: torch.Tensor | None = None, max_norm: float | None = None) -> None:
    """One AdamW step (decoupled weight decay) on fp32 masters and moments, in place.

    `weights` receives the bf16 rounding of the new masters: the `new` of encode_update, while the
    dict of the step before stays its `old`.  `step` counts from 1.  `norm` is the gradients' global
    norm (grad_norm, dist.grad_norm_global): with `max_norm` the gradients are scaled by
    min(1, max_norm / (norm + 1e-6)) on the way, without another pass over them; and where the norm
    is not finite, masters and moments stay as they are (weights get the masters' rounding all the
    same).  `lr` (fp32) and `step` (int64) may be one-element tensors on the device, read when the
    step runs: a captured graph then follows them.  Memory that the step writes may not be shared."""
    b1, b2 = _reals("betas", betas)
    eps, weight_decay = _real("eps", eps), _real("weight_decay", weight_decay)
    if not (0 <= b1 < 1 and 0 <= b2 < 1):
        raise ValueError(f"betas must be in [0, 1), got {betas}")
    if not eps >= _LEAST:
        raise ValueError(f"eps must be positive (in fp32), got {eps}")
    if not abs(weight_decay) <= _MOST:
        raise ValueError(f"weight_decay must be finite (in fp32), got {weight_decay}")
    if max_norm is not None:
        max_norm = _real("max_norm", max_norm)
        if norm is None or not max_norm >= _LEAST:
            raise ValueError(f"max_norm must be positive (in fp32) and comes with norm, got {max_norm}")
    lr, lr_t = (0.0, lr) if isinstance(lr, torch.Tensor) else (_real("lr", lr), None)
    step, step_t = (1, step) if isinstance(step, torch.Tensor) else (_count("step", step), None)
    if not abs(lr) <= _MOST:
        raise ValueError(f"lr must be finite (in fp32), got {lr}")
    grads, masters = _dict("gradients", grads), _dict("masters", masters)
    exp_avg, exp_avg_sq = _dict("exp_avg", exp_avg), _dict("exp_avg_sq", exp_avg_sq)
    if weights is not None:
        weights = _dict("weights", weights)
    if not _ext.glue().adamw_step(masters, grads, exp_avg, exp_avg_sq, weights, lr, lr_t, step, step_t, b1, b2, eps, weight_decay,
                                  _tensor("norm", norm), max_norm or 0.0):
        device = _check_set("gradients", grads, _GRADS)
        for what, d in (("masters", masters), ("exp_avg", exp_avg), ("exp_avg_sq", exp_avg_sq)):
            _check_match(what, d, grads, _F32, device)
        if weights is not None:
            _check_match("weights", weights, grads, _BF16, device)
        for what, t, dtype in (("norm", norm, torch.float32), ("lr", lr_t, torch.float32), ("step", step_t, torch.int64)):
            _check_scalar(what, t, dtype, device)
        _refused("gradients")


# ------------------------------------------------------------------ policy loss

@dataclass(slots=True)
class PolicyLoss:
    loss: torch.Tensor        # 0-d fp32, differentiable to the logits
    logp: torch.Tensor        # fp32, the tokens' shape: log-probability of each token (0 where it does not count)
    kl: torch.Tensor          # 0-d fp32: mean KL estimate to the reference policy
    clip_frac: torch.Tensor   # 0-d fp32: share of the tokens whose ratio was clipped


def policy_loss(logits: torch.Tensor, tokens: torch.Tensor, advantages: torch.Tensor, *,
                old_logp: torch.Tensor | None = None, ref_logp: torch.Tensor | None = None,
                mask: torch.Tensor | None = None, clip=(0.2, 0.2), kl_coef: float = 0.0, temperature: float = 1.0,
                denom: float | None = None) -> PolicyLoss:
    """Clipped policy loss with a KL term, from the logits; differentiable to them.

    logits [tokens' shape, V] (bf16, fp16 or fp32; rows at any strides, the vocabulary contiguous);
    tokens [T] or [B, T] (int64 or int32), the sampled ones; advantages (fp32), the tokens' shape or
    1 along a dimension.  Per token, with logp = log softmax(logits / temperature)[token]:

        ratio = exp(logp - old_logp)                    (1 where old_logp is None)
        l = -min(ratio A, clip(ratio, 1 - clip[0], 1 + clip[1]) A) + kl_coef (e^x - x - 1),  x = ref_logp - logp
        loss = sum(mask l) / denom

    mask: bool, or fp32 weights, shaped as advantages may be; tokens where it is 0 are left out whatever
    stands there (their logits are not read).  denom: None for the sum of the mask; a batch's total
    when it is split, or the number of sequences when the weights are 1 / length.  A mask of zeros
    gives 0.  advantages, old_logp, ref_logp and mask are constants: nothing is propagated to them.
    A token outside the vocabulary that counts makes the loss NaN.

    Where the logits require a gradient it is computed in this same call (they are read once), for
    loss.backward() as it stands; a loss that is scaled first is right too, and costs a second pass.
    Forward-mode gradients are refused."""
    lo, hi = _reals("clip", clip)
    temperature, kl_coef = _real("temperature", temperature), _real("kl_coef", kl_coef)
    if not (lo >= 0 and hi >= 0):
        raise ValueError(f"clip bounds must not be negative, got {clip}")
    if not 1e-30 < temperature < math.inf:   # (1 / temperature is a number fp32 holds)
        raise ValueError(f"temperature must be more than 1e-30 and finite, got {temperature}")
    if not abs(kl_coef) < 1e30:
        raise ValueError(f"kl_coef must be less than 1e30, got {kl_coef}")
    if kl_coef and ref_logp is None:
        raise ValueError("kl_coef needs ref_logp")
    if denom is not None:
        denom = _real("denom", denom)
        if not denom > 0:
            raise ValueError(f"denom must be positive, got {denom}")
    given = dict(tokens=tokens, advantages=advantages, old_logp=old_logp, ref_logp=ref_logp, mask=mask)
    for what, t in (("logits", logits), *given.items()):
        if t is None and what in ("logits", "tokens", "advantages"):
            raise ValueError(f"{what}: expected a torch tensor, got None")
        _tensor(what, t)
    out = _ext.glue().policy_loss(logits, tokens, advantages, old_logp, ref_logp, mask, lo, hi, kl_coef, temperature, denom or 0.0)
    if out is None:
        _check_policy(logits, **given)
    return PolicyLoss(*out)


def _check_policy(logits, tokens, **given) -> None:
    if logits.dtype not in _GRADS or logits.layout != torch.strided:
        raise ValueError(f"logits: expected a {_names(_GRADS)} torch tensor, got {logits.dtype}")
    if tokens.dtype not in (torch.int64, torch.int32):
        raise ValueError(f"tokens: expected an int64 or int32 torch tensor, got {tokens.dtype}")
    if tokens.dim() not in (1, 2) or logits.shape[:-1] != tokens.shape or logits.dim() < 2 or logits.shape[-1] < 1:
        raise ValueError(f"logits {tuple(logits.shape)} do not go with tokens {tuple(tokens.shape)}: "
                         "expected [T, V] and [T], or [B, T, V] and [B, T]")
    if logits.shape[-1] > 1 and logits.stride(-1) != 1:
        raise ValueError("logits: the vocabulary must be contiguous")
    if not logits.is_cuda:
        raise ValueError("logits: expected a CUDA tensor")
    if torch.autograd.forward_ad.unpack_dual(logits).tangent is not None:
        raise ValueError("logits: forward-mode gradients are not supported")
    for what, t in (("tokens", tokens), *given.items()):
        if t is None:
            continue
        if what != "tokens" and t.dtype != torch.float32 and not (what == "mask" and t.dtype == torch.bool):
            raise ValueError(f"{what}: expected a {'bool or ' if what == 'mask' else ''}float32 torch tensor, got {t.dtype}")
        if t.dim() != tokens.dim() or any(a != b and (a != 1 or what not in ("advantages", "mask")) for a, b in zip(t.shape, tokens.shape)):
            raise ValueError(f"{what}: shape {tuple(t.shape)} does not go with tokens {tuple(tokens.shape)}")
        if t.device != logits.device:
            raise ValueError(f"{what}: all tensors must be on one device")
    _refused("logits")
