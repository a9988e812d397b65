"""Cases of the trainer-side operators: the clipped policy loss, the gradient norm and clipping, and the
AdamW step on fp32 masters.  `run` computes them in elementary torch operations, or (own = True) through
the package's public entry points."""

import math
import random

import torch

own = False

# A decoder's parameter shapes, as this repository's workloads use them: (layers, d, kv, ffn, vocab);
# vocab 0 leaves the embedding to another rank.
TOY = (4, 1024, 1024, 2816, 32768)
SHAPE_1P5B = (28, 1536, 256, 8960, 151936)
RANK_OF_7B = (4, 3584, 512, 18944, 0)     # about an eighth of 28 such layers


def listed():
    loss = {"op": "loss", "grad": True, "lo": 0.2, "hi": 0.2, "beta": 0.0, "tau": 1.0, "old": True, "shift": False,
            "weights": "none", "pad": 0}
    return [
        # a few tokens of the toy decoder: what a call costs before any data moves
        {**loss, "name": "loss_16x32k", "B": 1, "T": 16, "V": 32768, "dtype": "bf16"},
        # a micro-batch of ragged answers; the logits are a model's [:, :-1]
        {**loss, "name": "loss_255x152k_shifted", "B": 3, "T": 85, "V": 151936, "dtype": "bf16", "shift": True,
         "weights": "mask", "beta": 0.04},
        # a training batch of the 7B shape's vocabulary with a reference model, asymmetric clipping
        {**loss, "name": "loss_4096x152k", "B": 8, "T": 512, "V": 152064, "dtype": "bf16", "weights": "mask",
         "hi": 0.28, "beta": 0.001},
        # fp32 logits with an odd vocabulary in padded rows, sequence-mean weights, sampling temperature 0.7
        {**loss, "name": "loss_1015x32771_fp32", "B": 5, "T": 203, "V": 32771, "dtype": "fp32", "weights": "mean",
         "beta": 0.04, "tau": 0.7, "pad": 5},
        # log-probabilities and loss without gradients: a scoring pass over a batch
        {**loss, "name": "score_4096x152k", "B": 8, "T": 512, "V": 151936, "dtype": "bf16", "grad": False,
         "weights": "mask", "beta": 0.04},
        # adapters packed one behind the other in one buffer: small, many and unaligned
        {**_ragged("clip", 112, 1100000, 1, "bf16"), "name": "clip_adapters"},
        # the toy decoder's fp32 gradients
        {**_decoder("clip", TOY, "fp32"), "name": "clip_toy_fp32"},
        # one rank's share of the 7B shape
        {**_decoder("clip", RANK_OF_7B, "bf16"), "name": "clip_rank_of_7b"},
        # the norm alone over the whole 1.5B shape (logged, or passed on to the step)
        {**_decoder("norm", SHAPE_1P5B, "bf16"), "name": "norm_1p5b"},
        {**_ragged("norm", 30, 50000, 8, "fp16"), "name": "norm_small"},
        # the toy decoder's step with fp32 gradients, clipped
        {**_decoder("step", TOY, "fp32"), "name": "step_toy_fp32"},
        # one rank's share of the 7B shape, clipped: norm, then the step
        {**_decoder("step", RANK_OF_7B, "bf16"), "name": "step_rank_of_7b"},
    ]


def _decoder(op, shape, dtype):
    return {"op": op, "layers": shape[0], "d": shape[1], "kv": shape[2], "ffn": shape[3], "vocab": shape[4],
            "dtype": dtype, "align": 8, "max_norm": 0.5}


def _ragged(op, tensors, elements, align, dtype):
    return {"op": op, "tensors": tensors, "elements": elements, "align": align, "dtype": dtype, "max_norm": 0.5}


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["loss", "loss", "loss", "clip", "norm", "step"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if op != "loss":
        return _ragged(op, _log(rng, 1, 500), _log(rng, 1000, 400000000), rng.choice([1, 8]), dtype)
    V = _log(rng, 256, 152064)
    n = _log(rng, 1, min(16384, 200000000 // V))
    B = min(n, _log(rng, 1, 16))
    return {"op": "loss", "B": B, "T": max(1, n // B), "V": V, "dtype": dtype, "grad": rng.random() < 0.75,
            "shift": rng.random() < 0.3, "pad": rng.choice([0, 0, 3, 8]), "weights": rng.choice(["none", "mask", "mean"]),
            "old": rng.random() < 0.8, "lo": 0.2, "hi": rng.choice([0.2, 0.28]), "beta": rng.choice([0.0, 0.001, 0.04]),
            "tau": rng.choice([1.0, 1.0, 0.6])}


_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}


def _sizes(case):
    """Element counts of the case's tensors."""
    if "layers" in case:
        d, kv, ffn = case["d"], case["kv"], case["ffn"]
        layer = [d * d, d, kv * d, kv, kv * d, kv, d * d, ffn * d, ffn * d, d * ffn, d, d]
        return ([case["vocab"] * d] if case["vocab"] else []) + layer * case["layers"] + [d]
    r = random.Random(case["tensors"] * 1000003 + case["elements"])
    cut = [math.exp(r.uniform(0, 5)) for _ in range(case["tensors"])]
    return [max(1, int(c / sum(cut) * case["elements"])) for c in cut]


def _places(case):
    """(offset, elements) of each tensor in the flat buffer, and the buffer's size."""
    a, at, places = case["align"], 0, []
    for n in _sizes(case):
        places.append((at, n))
        at += -(-n // a) * a
    return places, at


def _views(flat, places):
    return {"t%d" % i: flat[o:o + n] for i, (o, n) in enumerate(places)}


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (_prepare_loss if case["op"] == "loss" else _prepare_set)(case, g)


def _lengths(case):
    """Tokens of each sequence that count: half of T to T, and none in one of three or more."""
    if case["weights"] == "none":
        return [case["T"]] * case["B"]
    r = random.Random(case["V"])
    n = [r.randint((case["T"] + 1) // 2, case["T"]) for _ in range(case["B"])]
    if case["B"] > 2:
        n[case["B"] // 2] = 0
    return n


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _prepare_set(case, g):
    """Gradients as views of one buffer (and, for the step, masters and moments beside them); the space
    between tensors holds zeros, which stay zeros in every formula here."""
    places, total = _places(case)
    hole = torch.zeros(total, dtype=torch.bool, device="cuda")
    for (o, n), (q, _) in zip(places, places[1:] + [(total, 0)]):
        if o + n < q:
            hole[o + n:q] = True

    def flat(scale, dtype):
        return (_randn(g, total) * scale).masked_fill_(hole, 0).to(dtype)

    grad = flat(1e-3, _TYPES[case["dtype"]])
    s = {"case": case, "grad": grad, "grads": _views(grad, places)}
    if case["op"] == "clip":
        s["out"] = torch.zeros_like(grad)
        s["outs"] = _views(s["out"], places)
    if case["op"] == "step":
        s["master"], s["m"] = flat(0.02, torch.float32), flat(1e-4, torch.float32)
        s["v"] = flat(1e-3, torch.float32).square_()
        s["weight"] = s["master"].to(torch.bfloat16)
        for k in ("master", "m", "v", "weight"):
            s[k + "s"] = _views(s[k], places)
    return s


def _prepare_loss(case, g):
    """Logits in which the sampled token stands out by a varying amount, log-probabilities of a slightly
    older policy and of a reference beside the present ones, normalised advantages per sequence."""
    B, T, V, tau = case["B"], case["T"], case["V"], case["tau"]
    rows = T + 1 if case["shift"] else T
    whole = (_randn(g, B, rows, V + case["pad"]) * 2.5).to(_TYPES[case["dtype"]])
    tokens = torch.randint(0, V, (B, T), generator=g, device="cuda")
    z = whole[:, :T, :V]
    bump = torch.rand(B, T, 1, generator=g, device="cuda") * 14 + 2
    z.scatter_add_(2, tokens[:, :, None], bump.to(z.dtype))
    logp = torch.empty(B, T, device="cuda")
    for b in range(B):
        x = z[b].float() / tau
        logp[b] = x.gather(1, tokens[b, :, None])[:, 0] - torch.logsumexp(x, -1)
    drift = _randn(g, B, T) * 0.15
    ratio = drift.neg().exp()   # a token whose ratio stands at a border has no gradient to agree on
    edge = ((ratio - 1 + case["lo"]).abs() < 2e-3) | ((ratio - 1 - case["hi"]).abs() < 2e-3)
    drift = torch.where(edge, torch.zeros_like(drift), drift)
    s = {"case": case, "tokens": tokens, "old": logp + drift if case["old"] else None,
         "ref": logp + _randn(g, B, T) * 0.2 if case["beta"] else None, "advantages": _randn(g, B, 1), "mask": None}
    if case["weights"] != "none":
        length = torch.tensor(_lengths(case), device="cuda")[:, None]
        mask = torch.arange(T, device="cuda") < length
        s["mask"] = mask if case["weights"] == "mask" else mask.float() / length.clamp(min=1)
    s["logits"] = z.detach().requires_grad_(case["grad"])
    return s


def run(state):
    return {"loss": _run_loss, "norm": _run_norm, "clip": _run_clip, "step": _run_step}[state["case"]["op"]](state)


def _denom(case):
    return float(case["B"]) if case["weights"] == "mean" else None


def _run_loss(s):
    c = s["case"]
    if own:
        import crukx_sync_b200 as crx
        out = crx.policy_loss(s["logits"], s["tokens"], s["advantages"], old_logp=s["old"], ref_logp=s["ref"],
                              mask=s["mask"], clip=(c["lo"], c["hi"]), kl_coef=c["beta"], temperature=c["tau"],
                              denom=_denom(c))
        got = {"loss": out.loss.detach(), "logp": out.logp, "kl": out.kl, "clip_frac": out.clip_frac}
        if c["grad"]:
            got["grad"], = torch.autograd.grad(out.loss, s["logits"])
        return got
    with torch.no_grad():
        return _plain_loss(s, c)


def _plain_loss(s, c):
    logits, tokens, A = s["logits"], s["tokens"], s["advantages"]
    z = logits.float() / c["tau"]
    top = z.amax(-1, keepdim=True)
    at = (z.gather(2, tokens[:, :, None]) - top)[:, :, 0]
    e = z.sub_(top).exp_()
    total = e.sum(-1, keepdim=True)
    logp = at - total[:, :, 0].log()
    r = (logp - s["old"]).exp() if c["old"] else torch.ones_like(logp)
    surrogate = torch.minimum(r * A, r.clamp(1 - c["lo"], 1 + c["hi"]) * A)
    cut = ((A > 0) & (r > 1 + c["hi"])) | ((A < 0) & (r < 1 - c["lo"]))
    w = s["mask"].float() if s["mask"] is not None else torch.ones_like(logp)
    D = w.double().sum() if _denom(c) is None else _denom(c)
    x = s["ref"] - logp if c["beta"] else torch.zeros_like(logp)
    kl = x.exp() - x - 1

    def mean(t):
        return (torch.where(w != 0, w.double() * t.double(), 0.0).sum() / D).float()

    got = {"loss": mean(-surrogate.double() + c["beta"] * kl.double()), "logp": torch.where(w != 0, logp, 0.0),
           "kl": mean(kl), "clip_frac": mean(cut.float())}
    if c["grad"]:
        up = torch.where(cut, 0.0, -A * r) + c["beta"] * (1 - x.exp())
        up = torch.where(w != 0, w / D * up / c["tau"], 0.0).float()[:, :, None]
        p = e.div_(total).mul_(-up)
        p.scatter_add_(2, tokens[:, :, None], up)
        got["grad"] = p.to(logits.dtype)
    return got


def _plain_norm(grad):
    return grad.float().square().sum().sqrt()


def _run_norm(s):
    if own:
        import crukx_sync_b200 as crx
        return crx.grad_norm(s["grads"])
    return _plain_norm(s["grad"])


def _run_clip(s):
    if own:
        import crukx_sync_b200 as crx
        return crx.clip_grads(s["grads"], s["case"]["max_norm"], out=s["outs"]), s["out"]
    norm = _plain_norm(s["grad"])
    coef = (s["case"]["max_norm"] / (norm + 1e-6)).clamp(max=1.0)
    s["out"].copy_(s["grad"].float() * coef)
    return norm, s["out"]


_LR, _STEP, _BETAS, _EPS, _DECAY = 2e-6, 7, (0.9, 0.95), 1e-8, 0.1


def _run_step(s):
    max_norm = s["case"]["max_norm"]
    if own:
        import crukx_sync_b200 as crx
        norm = crx.grad_norm(s["grads"])
        crx.adamw_step(s["masters"], s["grads"], s["ms"], s["vs"], s["weights"], lr=_LR, step=_STEP, betas=_BETAS,
                       eps=_EPS, weight_decay=_DECAY, norm=norm, max_norm=max_norm)
    else:
        norm = _plain_norm(s["grad"])
        g = s["grad"].float() * (max_norm / (norm + 1e-6)).clamp(max=1.0)
        m, v, p = s["m"], s["v"], s["master"]
        m.mul_(_BETAS[0]).add_(g * (1 - _BETAS[0]))
        v.mul_(_BETAS[1]).add_(g.square_().mul_(1 - _BETAS[1]))
        den = (v / (1 - _BETAS[1] ** _STEP)).sqrt_().add_(_EPS)
        p.mul_(1 - _LR * _DECAY).sub_((m / den).mul_(_LR / (1 - _BETAS[0] ** _STEP)))
        s["weight"].copy_(p)
    return {"norm": norm, "master": s["master"], "m": s["m"], "v": s["v"], "weight": s["weight"]}


def work(case):
    e = _BYTES[case["dtype"]]
    if case["op"] == "loss":
        n, counted = case["B"] * case["T"], sum(_lengths(case))
        b = 1 if case["weights"] == "mask" else 4 if case["weights"] == "mean" else 0
        small = n * (8 + b + (4 if case["old"] else 0) + (4 if case["beta"] else 0) + 4) + 4 * case["B"]
        return {"bytes": (counted + (n if case["grad"] else 0)) * case["V"] * e + small,
                "flops": counted * case["V"] * (8 if case["grad"] else 4)}
    n = sum(_sizes(case))
    if case["op"] == "norm":
        return {"bytes": n * e, "flops": 2 * n}
    if case["op"] == "clip":
        return {"bytes": 2 * n * e, "flops": 3 * n}
    return {"bytes": n * (e + 12 + 14), "flops": 18 * n}


def exact(case, seed):
    """The definitions in 64 bits, sequence by sequence and piece by piece."""
    s = prepare(case, seed)
    if case["op"] == "loss":
        with torch.no_grad():
            return _exact_loss(s, case)
    g = s["grad"].double()
    norm = torch.linalg.vector_norm(g)
    if case["op"] == "norm":
        return norm
    g *= min(1.0, case["max_norm"] / (float(norm) + 1e-6))
    if case["op"] == "clip":
        return norm, g
    (b1, b2), t = _BETAS, _STEP
    m = b1 * s["m"].double() + (1 - b1) * g
    v = b2 * s["v"].double() + (1 - b2) * g * g
    del g
    step = torch.sqrt(v / (1 - b2 ** t))
    step += _EPS
    step = _LR * m / (1 - b1 ** t) / step
    p = s["master"].double() * (1 - _LR * _DECAY) - step
    return {"norm": norm, "master": p, "m": m, "v": v, "weight": p}


def _exact_loss(s, c):
    B, T = c["B"], c["T"]
    w = torch.ones(B, T, dtype=torch.float64, device="cuda") if s["mask"] is None else s["mask"].double()
    D = float(B) if c["weights"] == "mean" else float(w.sum())
    grads, logps, kls, losses, cuts = [], [], [], [], []
    for b in range(B):
        logq = torch.log_softmax(s["logits"][b].double() / c["tau"], -1)
        lp = logq[torch.arange(T, device="cuda"), s["tokens"][b]]
        a = float(s["advantages"][b, 0])
        r = torch.exp(lp - s["old"][b].double()) if c["old"] else torch.ones_like(lp)
        out = r > 1 + c["hi"] if a > 0 else r < 1 - c["lo"]
        inside = torch.clamp(r, 1 - c["lo"], 1 + c["hi"])
        x = s["ref"][b].double() - lp if c["beta"] else torch.zeros_like(lp)
        kl = torch.expm1(x) - x
        losses.append(-torch.where(out, inside, r) * a + c["beta"] * kl)
        kls.append(kl)
        cuts.append(out.double())
        logps.append(torch.where(w[b] != 0, lp, 0.0))
        if c["grad"]:
            up = torch.where(out, 0.0, -a * r) - c["beta"] * torch.expm1(x)
            up = w[b] * up / ((D or 1.0) * c["tau"])
            dz = torch.exp(logq) * -up[:, None]
            dz[torch.arange(T, device="cuda"), s["tokens"][b]] += up
            grads.append(dz)
    mean = [(w * torch.stack(v)).sum() / (D or 1.0) for v in (losses, kls, cuts)]
    got = {"loss": mean[0], "logp": torch.stack(logps), "kl": mean[1], "clip_frac": mean[2]}
    if c["grad"]:
        got["grad"] = torch.stack(grads)
    return got
