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
runs.  Caller mistakes are ValueErrors, raised before anything is launched.
"""

from __future__ import annotations

import ctypes
import math
import operator
import struct
from collections.abc import Mapping
from contextlib import nullcontext
from dataclasses import dataclass

import torch

from . import _ext
from .codec import _cuda_device, _raise

_CODES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}   # CRX_BF16, CRX_FP16, CRX_FP32
_GRADS, _F32, _BF16 = frozenset(_CODES), frozenset([torch.float32]), frozenset([torch.bfloat16])
_GRAD_TYPES = "bfloat16, float16 or float32"


def _on(index: int):
    """The device current for a call (its launches, its scratch)."""
    return nullcontext() if torch.cuda.current_device() == index else torch.cuda.device(index)


def _stream(index: int):
    return torch.cuda.current_stream(index).cuda_stream


def _check(name: str, t, dtypes, what: str) -> None:
    if not isinstance(t, torch.Tensor) or t.dtype not in dtypes:
        raise ValueError(f"{name}: expected a {what} torch tensor, got {getattr(t, 'dtype', type(t))}")
    if t.layout != torch.strided or not t.is_contiguous():
        raise ValueError(f"{name}: tensor must be contiguous")
    if not t.is_cuda:
        raise ValueError(f"{name}: expected a CUDA tensor")


_T = torch.Tensor
_dtype_of = operator.attrgetter("dtype")


def _gather(what: str, tensors: Mapping, dtypes, types: str, index: int | None):
    """The dict's tensors, checked, their addresses, element counts and types, and the index of
    their one device.  Whole-list calls: a model has hundreds of tensors and the step waits for this."""
    if not isinstance(tensors, Mapping):
        raise ValueError(f"{what} must be a dict of name -> tensor, got {type(tensors)}")
    out = list(tensors.values())
    try:
        types_of = list(map(_dtype_of, out))
        kinds = set(types_of)
        devices = set(map(_T.get_device, out))
        fine = kinds <= dtypes and -1 not in devices and all(map(_T.is_contiguous, out))
        if fine:
            ptrs, numels = list(map(_T.data_ptr, out)), list(map(_T.numel, out))
    except (TypeError, AttributeError, RuntimeError, NotImplementedError):   # not tensors, or not strided ones
        fine = False
    if not fine:
        for name, t in tensors.items():
            _check(name, t, dtypes, types)
        raise ValueError(f"{what}: expected contiguous {types} CUDA tensors")
    if index is not None:
        devices.add(index)
    if len(devices) > 1:
        raise ValueError("all tensors must be on one device")
    codes = [_CODES[kinds.pop()]] * len(out) if len(kinds) == 1 else list(map(_CODES.__getitem__, types_of))
    return out, ptrs, numels, codes, next(iter(devices), None)


def _match(what: str, tensors: Mapping, names, numels, dtypes, types: str, index: int):
    """`tensors` under the same names and sizes, in the order of `names`: (tensors, addresses, types)."""
    if not isinstance(tensors, Mapping) or tensors.keys() != names:
        odd = sorted(set(tensors) ^ set(names))[:5] if isinstance(tensors, Mapping) else type(tensors)
        raise ValueError(f"{what} and the gradients differ in tensor names: {odd}")
    if list(tensors) != list(names):
        tensors = {n: tensors[n] for n in names}
    out, ptrs, n, codes, _ = _gather(what, tensors, dtypes, types, index)
    if n != numels:
        name = next(name for name, a, b in zip(names, n, numels) if a != b)
        raise ValueError(f"{name}: {what} and the gradient differ in shape")
    return out, ptrs, codes


def _scalar(what: str, t, dtype, index: int) -> None:
    if not isinstance(t, torch.Tensor) or t.dtype != dtype or t.numel() != 1 or t.get_device() != index:
        raise ValueError(f"{what}: expected one {str(dtype).replace('torch.', '')} on the gradients' device")


def _no_tensors() -> int:
    return _cuda_device(torch.device("cuda")).index


def grad_norm(grads: Mapping[str, torch.Tensor]) -> torch.Tensor:
    """sqrt(sum of g^2) over every element of every gradient, as a 0-d fp32 CUDA tensor.

    bf16, fp16 and fp32 gradients may be mixed.  The sum is held in 64 bits and squares that would
    overflow or vanish in fp32 count in full; its order is fixed, so equal gradients give equal bits."""
    tensors, ptrs, numels, codes, index = _gather("gradients", grads, _GRADS, _GRAD_TYPES, None)
    if index is None:
        index = _no_tensors()
    L = _ext.load()
    n = len(tensors)
    err = ctypes.create_string_buffer(512)
    with _on(index):
        norm = torch.empty((), dtype=torch.float32, device=index)
        size = L.crx_grads_workspace(n)
        ws = torch.empty(size, dtype=torch.uint8, device=index)
        st = L.crx_grad_norm(n, _ext.ptr_array(ptrs), _ext.CBuf("i", codes), _ext.CBuf("q", numels), ws.data_ptr(), size,
                             norm.data_ptr(), _stream(index), err, 512)
    if st != _ext.CRX_OK:
        _raise(st, err)
    return norm


def clip_grads(grads: Mapping[str, torch.Tensor], max_norm: float, *, out: Mapping[str, torch.Tensor] | None = None,
               norm: torch.Tensor | None = None) -> torch.Tensor:
    """Scale the gradients so that their global norm is at most `max_norm`; returns the norm before.

    Every gradient is multiplied by min(1, max_norm / (norm + 1e-6)) and rounded to its type: in
    place, or into the tensors of `out` (same names, sizes and types).  `norm` (0-d fp32, on the
    device) takes the place of the gradients' own, for gradients spread over ranks
    (dist.grad_norm_global).  A norm that is not finite is not clipped away: it leaves NaN, as its
    product says.  Tensors that share memory (a tied weight under two names) are refused."""
    if not max_norm > 0:   # (NaN too)
        raise ValueError(f"max_norm must be positive, got {max_norm}")
    tensors, ptrs, numels, codes, index = _gather("gradients", grads, _GRADS, _GRAD_TYPES, None)
    if index is None:
        index = _no_tensors()
    outs, out_ptrs = tensors, ptrs
    if out is not None:
        outs, out_ptrs, out_codes = _match("out", out, grads.keys(), numels, _GRADS, _GRAD_TYPES, index)
        if out_codes != codes:
            name = next(name for name, a, b in zip(grads, codes, out_codes) if a != b)
            raise ValueError(f"{name}: out and the gradient differ in type")
    if norm is not None:
        _scalar("norm", norm, torch.float32, index)
    L = _ext.load()
    n = len(tensors)
    err = ctypes.create_string_buffer(512)
    with _on(index):
        size = 0 if norm is not None else L.crx_grads_workspace(n)
        ws = torch.empty(size, dtype=torch.uint8, device=index) if size else None
        result = norm if norm is not None else torch.empty((), dtype=torch.float32, device=index)
        st = L.crx_clip_grads(n, _ext.ptr_array(ptrs), _ext.ptr_array(out_ptrs), _ext.CBuf("i", codes), _ext.CBuf("q", numels),
                              max_norm, None if norm is None else norm.data_ptr(),
                              ws.data_ptr() if size else None, size, result.data_ptr() if norm is None else None,
                              _stream(index), err, 512)
    if st != _ext.CRX_OK:
        _raise(st, err)
    torch.autograd.graph.increment_version(outs)   # written through raw pointers
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
    tensors, ptrs, numels, codes, index = _gather("gradients", grads, _GRADS, _GRAD_TYPES, None)
    names = grads.keys()
    b1, b2 = betas
    if not (0 <= b1 < 1 and 0 <= b2 < 1):
        raise ValueError(f"betas must be in [0, 1), got {betas}")
    if not eps > 0:
        raise ValueError(f"eps must be positive, got {eps}")
    if not math.isfinite(weight_decay):
        raise ValueError(f"weight_decay must be finite, got {weight_decay}")
    if max_norm is not None and (norm is None or not max_norm > 0):
        raise ValueError("max_norm must be positive and comes with norm")
    if not isinstance(step, torch.Tensor) and step < 1:
        raise ValueError(f"step counts from 1, got {step}")
    if not isinstance(lr, torch.Tensor) and not math.isfinite(lr):
        raise ValueError(f"lr must be finite, got {lr}")
    (p, p_ptrs, _), (m, m_ptrs, _), (v, v_ptrs, _) = (
        _match(what, d, names, numels, _F32, "float32", index)
        for what, d in (("masters", masters), ("exp_avg", exp_avg), ("exp_avg_sq", exp_avg_sq)))
    w, w_ptrs, _ = ([], None, None) if weights is None else _match("weights", weights, names, numels, _BF16, "bfloat16", index)
    if not tensors:
        return
    for what, t, dtype in (("norm", norm, torch.float32), ("lr", lr, torch.float32), ("step", step, torch.int64)):
        if isinstance(t, torch.Tensor) or what == "norm" and t is not None:
            _scalar(what, t, dtype, index)
    lr_p = lr.data_ptr() if isinstance(lr, torch.Tensor) else 0
    step_p = step.data_ptr() if isinstance(step, torch.Tensor) else 0
    args = _ADAMW.pack(0.0 if lr_p else lr, b1, b2, eps, weight_decay, 1 if step_p else int(step), lr_p, step_p,
                       0 if norm is None else norm.data_ptr(), max_norm or 0.0)
    L = _ext.load()
    err = ctypes.create_string_buffer(512)
    with _on(index):
        st = L.crx_adamw_step(len(tensors), _ext.ptr_array(p_ptrs), _ext.ptr_array(ptrs), _ext.CBuf("i", codes),
                              _ext.ptr_array(m_ptrs), _ext.ptr_array(v_ptrs), None if w_ptrs is None else _ext.ptr_array(w_ptrs),
                              _ext.CBuf("q", numels), args, _stream(index), err, 512)
    if st != _ext.CRX_OK:
        _raise(st, err)
    torch.autograd.graph.increment_version(p + m + v + w)


_INTS, _MASKS, _NONE = frozenset([torch.int64, torch.int32]), frozenset([torch.bool, torch.float32]), (0, 0, 0)
_POLICY = struct.Struct("28qd4f4i")    # crx_policy_args
_ADAMW = struct.Struct("5d4qf4x")      # crx_adamw_args


@dataclass(slots=True)
class PolicyLoss:
    loss: torch.Tensor        # 0-d fp32, differentiable to the logits
    logp: torch.Tensor        # fp32, the tokens' shape: log-probability of each token (0 where it does not count)
    kl: torch.Tensor          # 0-d fp32: mean KL estimate to the reference policy
    clip_frac: torch.Tensor   # 0-d fp32: share of the tokens whose ratio was clipped


def _rows(what: str, t, shape, index: int, dtypes, types: str, broadcast: bool):
    """(address, stride over sequences, stride over tokens) of per-token values."""
    if not isinstance(t, _T) or t.dtype not in dtypes or t.layout is not torch.strided:
        raise ValueError(f"{what}: expected a {types} torch tensor, got {getattr(t, 'dtype', type(t))}")
    if t.get_device() != index:
        raise ValueError(f"{what}: all tensors must be on one device")
    strides = t.stride()
    if t.shape != shape:
        if not broadcast or t.dim() != len(shape) or any(a != b and a != 1 for a, b in zip(t.shape, shape)):
            raise ValueError(f"{what}: shape {tuple(t.shape)} does not go with tokens {tuple(shape)}")
        strides = [0 if n == 1 else s for n, s in zip(t.shape, strides)]
    return (t.data_ptr(), *strides) if len(strides) == 2 else (t.data_ptr(), 0, strides[0])


def _grad_like(logits: torch.Tensor) -> torch.Tensor:
    """Memory for the gradient: laid out as the logits are, with rows starting at the same places
    between 16-byte boundaries (a row is then written in the vectors it was read in), unless that
    would waste or share memory; then rows padded to 16 bytes."""
    size, stride, V = logits.shape, logits.stride(), logits.shape[-1]
    es = logits.element_size()
    phase = logits.data_ptr() % 16 // es
    if phase == 0 and logits.is_contiguous():
        return torch.empty(size, dtype=logits.dtype, device=logits.device)
    end, fits = V, True   # elements up to the end of what the dims so far span
    for s, n in sorted((s, n) for s, n in zip(stride[:-1], size[:-1]) if n > 1):
        fits = fits and s >= end
        end += s * (n - 1)
    if fits and end <= 2 * logits.numel() + 64:
        flat = torch.empty(end + phase, dtype=logits.dtype, device=logits.device)
        return flat.as_strided(size, stride, phase)
    pad = -V % (16 // es)
    return torch.empty((*size[:-1], V + pad), dtype=logits.dtype, device=logits.device)[..., :V]


class _Call:
    """The arguments of one policy loss, as the library takes them."""

    __slots__ = ("index", "shape", "vocab", "small", "numbers", "keep")

    def pack(self, logits, grad, logp, loss, stats, rows) -> bytes:
        ls, g, gs = logits.stride(), 0, (0, 0, 0)
        if grad is not None:
            g, gs = grad.data_ptr(), grad.stride()
        if len(ls) == 2:
            ls, gs = (0, *ls), (0, *gs)
        return _POLICY.pack(*self.shape, self.vocab, logits.data_ptr(), ls[0], ls[1], g, gs[0], gs[1], *self.small, logp, loss,
                            stats, rows, *self.numbers)

    def run(self, logits, want_grad: bool):
        index, (b, t) = self.index, self.shape
        err = ctypes.create_string_buffer(512)
        with _on(index):
            grad = _grad_like(logits) if want_grad else None
            loss = torch.empty((), dtype=torch.float32, device=logits.device)
            logp = torch.empty(self.keep[0].shape, dtype=torch.float32, device=logits.device)
            stats = torch.empty(2, dtype=torch.float32, device=logits.device)
            rows = torch.empty(_ext.load().crx_policy_workspace(b, t), dtype=torch.uint8, device=logits.device)
            st = _ext.load().crx_policy_loss(
                self.pack(logits, grad, logp.data_ptr(), loss.data_ptr(), stats.data_ptr(), rows.data_ptr()), _stream(index), err, 512)
        if st != _ext.CRX_OK:
            _raise(st, err)
        return loss, stats, logp, rows, grad


class _PolicyLossFn(torch.autograd.Function):
    """The forward pass leaves the gradient for an incoming gradient of 1.  backward() hands it out;
    for another one (and the second time) it is computed again from the logits, so that it is
    rounded once whatever its scale."""

    @staticmethod
    def forward(ctx, logits, call):
        loss, stats, logp, rows, grad = call.run(logits, True)
        kl, clip_frac = stats.unbind(0)
        ctx.call, ctx.rows, ctx.grad = call, rows, grad
        ctx.save_for_backward(logits, call.keep[0])
        ctx.mark_non_differentiable(logp, kl, clip_frac)
        ctx.set_materialize_grads(False)
        return loss, logp, kl, clip_frac

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, scale, *_):
        if scale is None:
            return None, None
        logits, _ = ctx.saved_tensors   # (refuses tensors modified since)
        call = ctx.call
        grad, ctx.grad = ctx.grad, None
        err = ctypes.create_string_buffer(512)
        with _on(call.index):
            unless_one = grad is not None
            if grad is None:
                grad = _grad_like(logits)
            rows = ctx.rows.data_ptr()   # (in the places of results that the backward pass does not touch, too)
            st = _ext.load().crx_policy_backward(call.pack(logits, grad, rows, rows, rows, rows), scale.data_ptr(), unless_one,
                                                 _stream(call.index), err, 512)
        if st != _ext.CRX_OK:
            _raise(st, err)
        return grad, None


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
    loss.backward() as it stands; a loss that is scaled first is right too, and costs a second pass."""
    if not isinstance(logits, _T) or logits.dtype not in _CODES or logits.layout is not torch.strided:
        raise ValueError(f"logits: expected a {_GRAD_TYPES} torch tensor, got {getattr(logits, 'dtype', type(logits))}")
    if not isinstance(tokens, _T):
        raise ValueError(f"tokens: expected an int64 or int32 torch tensor, got {type(tokens)}")
    size, shape = logits.shape, tokens.shape
    if len(shape) not in (1, 2) or size[:-1] != shape or len(size) < 2 or size[-1] < 1:
        raise ValueError(f"logits {tuple(size)} do not go with tokens {tuple(shape)}: "
                         "expected [T, V] and [T], or [B, T, V] and [B, T]")
    if size[-1] > 1 and logits.stride(-1) != 1:
        raise ValueError("logits: the vocabulary must be contiguous")
    if not logits.is_cuda:
        raise ValueError("logits: expected a CUDA tensor")
    call = _Call()
    index = call.index = logits.get_device()
    call.shape = shape if len(shape) == 2 else (1, shape[0])
    call.vocab = size[-1]
    call.small = (
        *_rows("tokens", tokens, shape, index, _INTS, "int64 or int32", False),
        *_rows("advantages", advantages, shape, index, _F32, "float32", True),
        *(_NONE if old_logp is None else _rows("old_logp", old_logp, shape, index, _F32, "float32", False)),
        *(_NONE if ref_logp is None else _rows("ref_logp", ref_logp, shape, index, _F32, "float32", False)),
        *(_NONE if mask is None else _rows("mask", mask, shape, index, _MASKS, "bool or float32", True)))
    lo, hi = clip
    if not (lo >= 0 and hi >= 0):
        raise ValueError(f"clip bounds must not be negative, got {clip}")
    if not 0 < temperature < math.inf:
        raise ValueError(f"temperature must be positive and finite, got {temperature}")
    if not math.isfinite(kl_coef):
        raise ValueError(f"kl_coef must be finite, got {kl_coef}")
    if kl_coef and ref_logp is None:
        raise ValueError("kl_coef needs ref_logp")
    if denom is not None and not denom > 0:
        raise ValueError(f"denom must be positive, got {denom}")
    call.numbers = (denom or 0.0, lo, hi, kl_coef, temperature, _CODES[logits.dtype], tokens.dtype == torch.int64,
                    mask is not None and mask.dtype == torch.float32, 0)
    call.keep = (tokens, advantages, old_logp, ref_logp, mask)
    if logits.requires_grad and torch.is_grad_enabled():
        return PolicyLoss(*_PolicyLossFn.apply(logits, call))
    loss, stats, logp, _, _ = call.run(logits, False)
    kl, clip_frac = stats.unbind(0)
    return PolicyLoss(loss, logp, kl, clip_frac)
