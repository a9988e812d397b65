"""The trainer-side operators from their definitions, in 64 bits on the CPU, with how far each of the
library's results may be from them.

Roundings are counted as half a step: H = 2^-24 of the value for fp32, torch.finfo(t).eps / 2 for
the type t a result is rounded to, and half of t's smallest subnormal where it is that small."""

import math

import torch

H = 2.0 ** -24
NORM = 10 * H   # 16 squares added in fp32 (16 H of the sum, 8 H of its root), sqrt and its rounding to fp32


def half_step(x, dtype):
    f = torch.finfo(dtype)
    return x.abs() * f.eps / 2 + f.smallest_normal * f.eps / 2


def norm(grads):
    big = max([float(g.double().abs().max()) for g in grads if g.numel()], default=0.0)
    if not 0 < big < math.inf:
        return big if big == big else math.nan
    n = big * math.sqrt(sum(float((g.double() / big).square().sum()) for g in grads))
    return n if n <= torch.finfo(torch.float32).max else math.inf   # the result's type holds no more than 3.4e38


def coef(n, max_norm):
    return min(1.0, max_norm / (n + 1e-6))


def clip(g, c):
    """(c g, tolerance): c has the norm's error and three roundings, the product one more."""
    want = g.double() * c
    return want, half_step(want, g.dtype) + want.abs() * (NORM + 4 * H) * 1.01


def adamw(p, g, m, v, *, lr, step, b1, b2, eps, wd, c=1.0):
    """New (p, m, v) and their tolerances."""
    p, g, m, v = (t.double() for t in (p, g, m, v))
    g = g * c
    m2 = b1 * m + (1 - b1) * g
    v2 = b2 * v + (1 - b2) * g * g
    den = (v2 / (1 - b2 ** step)).sqrt() + eps
    up = lr / (1 - b1 ** step) * m2 / den
    p2 = p * (1 - lr * wd) - up
    tiny = 2.0 ** -149
    # g: c's error (above) and a rounding; each coefficient, product and sum one rounding
    tol_m = 3 * H * (b1 * m).abs() + (NORM + 10 * H) * ((1 - b1) * g).abs() + tiny
    tol_v = 3 * H * b2 * v + (2 * NORM + 20 * H) * (1 - b2) * g * g + 4 * tiny
    # den: half of v's relative error, and the bias, product, root, sum; then rate, product, division
    rel_v = (tol_v / v2.clamp(min=tiny)).clamp(max=1)
    tol_up = lr / (1 - b1 ** step) * tol_m / den + up.abs() * (0.5 * rel_v + 10 * H)
    tol_p = H * p2.abs() + tol_up + 4 * H * (lr * wd * p).abs() + H * up.abs() + tiny
    return (p2, m2, v2), (1.01 * tol_p, 1.01 * tol_m, 1.01 * tol_v)


def policy(logits, tokens, adv, *, old=None, ref=None, mask=None, clip=(0.2, 0.2), kl_coef=0.0, tau=1.0, denom=None):
    """dict of loss, logp, kl, clip_frac, grad, and the same with "tol_" before it.  Two-dimensional or
    one-dimensional tokens; a token outside the vocabulary is not handled here."""
    z = logits.double() / tau
    w = torch.ones(tokens.shape, dtype=torch.float64) if mask is None else mask.double().expand(tokens.shape)
    on = w != 0
    D = float(w.sum()) if denom is None else float(denom)
    inv = 1 / D if D else 0.0
    A = adv.double().expand(tokens.shape)
    at = tokens.long().clamp(0, logits.shape[-1] - 1)[..., None]
    logq = torch.log_softmax(z, -1)
    logp = logq.gather(-1, at)[..., 0]
    r = torch.ones_like(logp) if old is None else (logp - old.double()).exp()
    cut = ((A > 0) & (r > 1 + clip[1])) | ((A < 0) & (r < 1 - clip[0]))
    bound = torch.where(A > 0, torch.tensor(1.0 + clip[1], dtype=torch.float64), 1.0 - clip[0])
    gain = torch.where(A == 0, 0.0, torch.where(cut, bound, r) * A)
    x = torch.zeros_like(logp) if ref is None else ref.double() - logp
    k = torch.expm1(x) - x
    wi = w * inv

    def mean(t):
        return torch.where(on, wi * t, 0.0).sum()

    dl = torch.where(cut | (A == 0), 0.0, -r * A) - kl_coef * torch.expm1(x)
    u = torch.where(on, wi * dl / tau, 0.0)
    p = logq.exp()
    hot = torch.zeros_like(p).scatter_(-1, at, 1.0)
    grad = torch.where(on[..., None], u[..., None] * (hot - p), 0.0)
    # logp: s is a sum of at most V / 512 + 16 + 32 fp32 additions deep, of terms each off by the
    # exponent's rounding (X 2^-X < 0.54 of H), 4 H of 2^x and the rescalings; log2, the exponent of
    # the token (H of its size), two products; and c = log2(e) / tau is half a step off, which tilts
    # the softmax by H |z_a - mean z|.
    V = logits.shape[-1]
    fin = torch.where(torch.isfinite(z), z, 0.0)
    spread = torch.where(on, (fin.gather(-1, at)[..., 0] - (p * fin).sum(-1)).abs(), 0.0)
    depth = V / 512 + 16 + 32
    tol_lp = H * (depth + 12 + 4 * logp.abs() + 2 * spread + math.log(V + 1))
    wa = torch.where(on, wi.abs(), 0.0)
    tol_r = torch.where(A == 0, 0.0, r * A.abs()) * (tol_lp + 8 * H) * 1.1
    tol_x = tol_lp + 2 * H * (x.abs() + logp.abs())
    tol_k = torch.expm1(x).abs() * tol_x + tol_x ** 2 + 4 * H * (torch.expm1(x).abs() + x.abs())
    tol_u = wa / tau * (tol_r + abs(kl_coef) * (x.exp() * tol_x + 6 * H * torch.expm1(x).abs())) + 6 * H * u.abs()
    big = torch.where(on, u.abs(), 0.0)[..., None]
    # p: s, the exponent (H of it and the tilt), 2^x, the products
    expo = torch.where(torch.isfinite(logq), logq, 0.0).abs() * 1.45
    tol_p = p * H * (depth + 20 + 2 * expo + 2 * spread[..., None] + math.log(V + 1))
    tol_g = tol_u[..., None] * (hot + p) * 1.1 + big * (tol_p + 2 * H * (hot + p)) + half_step(grad, logits.dtype)
    return {"loss": mean(-gain + kl_coef * k), "logp": torch.where(on, logp, 0.0), "kl": mean(k),
            "clip_frac": mean(cut.double()), "grad": grad,
            "tol_loss": ((wa * (tol_r + abs(kl_coef) * tol_k)).nansum() + 4 * H * (wa * (gain.abs() + abs(kl_coef) * k)).nansum()) * 1.01 + H * 1e-6,
            "tol_logp": torch.where(on, tol_lp, 0.0), "tol_kl": (wa * tol_k).nansum() * 1.01 + 4 * H * (wa * k).nansum() + H * 1e-6,
            "tol_clip_frac": 4 * H, "tol_grad": tol_g}
