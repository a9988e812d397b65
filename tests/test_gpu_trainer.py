"""policy_loss, grad_norm, clip_grads and adamw_step against their definitions in 64 bits, at the
sizes, layouts, masks and values where they can go wrong, and run together as a trainer does."""

import contextlib
import gc
import math

import pytest
import torch

import trainer_ref as ref

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16, torch.float32]
SIZES = [1, 2, 7, 8, 9, 63, 4095, 8191, 8192, 8193, 8200, 16384, 3 * 8192 + 77, 100003]


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA GPU")
    from crukx_sync_b200 import _ext
    _ext.load()


@pytest.fixture(scope="module", autouse=True)
def _collected():
    """No tensors stay behind in reference cycles (a graphed callable is one): a later test counts memory."""
    yield
    gc.collect()


@pytest.fixture(scope="module")
def crx():
    import crukx_sync_b200
    return crukx_sync_b200


def gen(seed):
    return torch.Generator().manual_seed(seed)


def gradients(sizes, dtype, seed=0, shift=0, scale=1.0):
    """CPU gradients and CUDA copies that start `shift` elements after a 16-byte boundary."""
    g = gen(seed)
    cpu = {f"t{i}": (torch.randn(n, generator=g) * scale).to(dtype) for i, n in enumerate(sizes)}
    return cpu, {k: shifted(v, shift) for k, v in cpu.items()}


def shifted(t, shift):
    flat = torch.zeros(t.numel() + shift + 8, dtype=t.dtype, device="cuda")
    out = flat[shift:shift + t.numel()]
    out.copy_(t)
    return out


def near(got, want, tol, what=""):
    got, want = got.detach().double().cpu(), torch.as_tensor(want, dtype=torch.float64)
    assert got.shape == want.shape, what
    fine = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    same = (got == want) | torch.isnan(want)
    assert bool((fine | same).all()), what
    off = ((got - want).abs() - tol)[fine] if torch.is_tensor(tol) and tol.dim() else (got - want).abs()[fine] - tol
    assert off.numel() == 0 or float(off.max()) <= 0, f"{what}: {float(off.max())} beyond the tolerance"


# ---------------------------------------------------------------------------------- norm and clipping

@pytest.mark.parametrize("shift", [0, 1, 3])
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_norm(crx, dtype, shift):
    cpu, gpu = gradients(SIZES, dtype, 1, shift)
    want = ref.norm(cpu.values())
    got = crx.grad_norm(gpu)
    assert got.shape == () and got.dtype == torch.float32
    near(got, want, want * ref.NORM)
    assert torch.equal(got, crx.grad_norm(gpu))


@pytest.mark.parametrize("n", [1, 5, 8192, 300001])
def test_norm_one_tensor(crx, n):
    cpu, gpu = gradients([n], torch.bfloat16, n)
    want = ref.norm(cpu.values())
    near(crx.grad_norm(gpu), want, want * ref.NORM)


@pytest.mark.parametrize("scale", [1e-36, 1e-22, 1e-12, 1e15, 1e25, 1e36])
def test_norm_of_values_whose_squares_leave_fp32(crx, scale):
    cpu, gpu = gradients([5, 100003], torch.bfloat16, 2, 0, scale)
    want = ref.norm(cpu.values())
    near(crx.grad_norm(gpu), want, want * ref.NORM)


@pytest.mark.parametrize("most", [1e38, 1e36, 1e3])   # 1e38: the norm is 7.7e38, more than fp32 holds
def test_norm_of_mixed_magnitudes_and_zeros(crx, most):
    g = gen(3)
    t = torch.randn(50000, generator=g) * torch.exp(torch.randn(50000, generator=g) * 30)
    t[:20000] = 0
    t = t.clamp(-most, most)
    want = ref.norm([t])
    near(crx.grad_norm({"a": t.cuda(), "z": torch.zeros(9999, device="cuda")}), want,
         want * ref.NORM if want < math.inf else 0.0)


def test_norm_of_nothing_and_of_many(crx):
    assert float(crx.grad_norm({})) == 0
    assert float(crx.grad_norm({"e": torch.empty(0, device="cuda")})) == 0
    sizes = [(i * 37) % 61 for i in range(2100)]   # more tensors than one launch takes, empty ones among them
    cpu, gpu = gradients(sizes, torch.float16, 4)
    want = ref.norm(cpu.values())
    near(crx.grad_norm(gpu), want, want * ref.NORM)
    crx.clip_grads(gpu, want / 3)
    for k in cpu:
        near(gpu[k], *ref.clip(cpu[k], ref.coef(want, want / 3)), k)


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("place", [0, 8191, 9000])
def test_norm_that_is_not_finite(crx, bad, place):
    t = torch.ones(9001, dtype=torch.bfloat16)
    t[place] = bad
    got = float(crx.grad_norm({"a": t.cuda()}))
    assert math.isnan(got) if math.isnan(bad) else got == math.inf


def test_norm_of_mixed_types(crx):
    cpu, gpu = {}, {}
    for i, dt in enumerate(TYPES * 3):
        c, d = gradients([1000 * i + 3], dt, i, i % 4)
        cpu[f"x{i}"], gpu[f"x{i}"] = c["t0"], d["t0"]
    want = ref.norm(cpu.values())
    near(crx.grad_norm(gpu), want, want * ref.NORM)
    got = crx.clip_grads(gpu, want / 7)
    near(got, want, want * ref.NORM)
    for k in cpu:
        near(gpu[k], *ref.clip(cpu[k], ref.coef(want, want / 7)), k)


@pytest.mark.parametrize("into", ["in place", "aligned", "unaligned"])
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_clip(crx, dtype, into):
    cpu, gpu = gradients(SIZES, dtype, 5, 1 if into == "unaligned" else 0)
    before = {k: v.clone() for k, v in gpu.items()}
    out = None if into == "in place" else {k: shifted(torch.full_like(v, 7.0), 2 if into == "unaligned" else 0) for k, v in cpu.items()}
    n = ref.norm(cpu.values())
    versions = {k: v._version for k, v in (out or gpu).items()}
    got = crx.clip_grads(gpu, n / 3, out=out)
    near(got, n, n * ref.NORM)
    for k in cpu:
        near((out or gpu)[k], *ref.clip(cpu[k], ref.coef(n, n / 3)), k)
        assert (out or gpu)[k]._version > versions[k]
        if out:
            assert torch.equal(gpu[k], before[k])


def test_clip_that_has_nothing_to_do(crx):
    cpu, gpu = gradients([1000, 9], torch.float32, 6)
    out = {k: torch.empty_like(v) for k, v in gpu.items()}
    crx.clip_grads(gpu, 1e9)
    crx.clip_grads(gpu, 1e9, out=out)
    crx.clip_grads(gpu, math.inf)
    for k in cpu:
        assert torch.equal(gpu[k].cpu(), cpu[k]) and torch.equal(out[k].cpu(), cpu[k])


def test_clip_by_a_given_norm(crx):
    cpu, gpu = gradients([70000], torch.float32, 7)
    norm = torch.tensor(12.5, device="cuda")
    assert crx.clip_grads(gpu, 2.0, norm=norm) is norm
    near(gpu["t0"], *ref.clip(cpu["t0"], ref.coef(12.5, 2.0)))


@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_clip_by_a_norm_that_is_not_finite(crx, bad):
    g = {"a": torch.tensor([1.0, bad, 2.0], device="cuda")}
    crx.clip_grads(g, 1.0)
    got = g["a"].cpu()
    assert math.isnan(got[1]) and (math.isnan(got[0]) if math.isnan(bad) else got[0] == 0)


def test_tensors_that_share_memory_are_refused(crx):
    base = torch.ones(100, device="cuda")
    a, b, c = base[:50], base[49:80], base[80:]
    with pytest.raises(ValueError, match="share memory"):
        crx.clip_grads({"a": a, "b": b}, 1.0)
    with pytest.raises(ValueError, match="share memory"):
        crx.clip_grads({"a": a, "tied": a}, 1.0)
    with pytest.raises(ValueError, match="share memory"):
        crx.clip_grads({"c": c}, 1.0, out={"c": base[79:99]})
    near(crx.grad_norm({"a": a, "tied": a}), 10.0, 10 * ref.NORM)   # reading the same memory twice is fine
    assert torch.equal(base, torch.ones_like(base))
    m, v, g = (torch.ones(20, device="cuda") for _ in range(3))
    w = torch.ones(40, device="cuda", dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="share memory"):
        crx.adamw_step({"a": a[:20], "b": a[10:30]}, {"a": g, "b": g}, {"a": m, "b": m.clone()}, {"a": v, "b": v.clone()}, lr=1e-3, step=1)
    with pytest.raises(ValueError, match="share memory"):
        crx.adamw_step({"a": a[:20]}, {"a": a[10:30]}, {"a": m}, {"a": v}, lr=1e-3, step=1)
    with pytest.raises(ValueError, match="share memory"):
        crx.adamw_step({"a": w.view(torch.float32)}, {"a": g}, {"a": m}, {"a": v}, {"a": w[:20]}, lr=1e-3, step=1)


# ---------------------------------------------------------------------------------- AdamW

HYPER = dict(lr=2e-4, b1=0.9, b2=0.95, eps=1e-8, wd=0.1)


def state_of(cpu, shift=0, seed=11):
    g = gen(seed)
    p = {k: torch.randn(t.numel(), generator=g) * 0.02 for k, t in cpu.items()}
    m = {k: torch.randn(t.numel(), generator=g) * 0.1 for k, t in cpu.items()}
    v = {k: torch.randn(t.numel(), generator=g).square() for k, t in cpu.items()}
    host = (p, m, v)
    return host, [{k: shifted(t, shift) for k, t in d.items()} for d in host]


def check_step(cpu, host, dev, weights, step, c=1.0):
    for k, g in cpu.items():
        want, tol = ref.adamw(host[0][k], g, host[1][k], host[2][k], step=step, c=c, **HYPER)
        for d, x, t, what in zip(dev, want, tol, "pmv"):
            near(d[k], x, t, f"{k} {what}")
        if weights is not None:
            assert torch.equal(weights[k], dev[0][k].to(torch.bfloat16)), k


def step_args(n):
    return dict(lr=HYPER["lr"], step=n, betas=(HYPER["b1"], HYPER["b2"]), eps=HYPER["eps"], weight_decay=HYPER["wd"])


@pytest.mark.parametrize("shift,state_shift", [(0, 0), (3, 3), (1, 2)])
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_adamw(crx, dtype, shift, state_shift):
    cpu, gpu = gradients(SIZES, dtype, 8, shift)
    host, dev = state_of(cpu, state_shift)
    w = {k: shifted(torch.zeros(t.numel(), dtype=torch.bfloat16), state_shift) for k, t in cpu.items()}
    crx.adamw_step(dev[0], gpu, dev[1], dev[2], w, **step_args(3))
    check_step(cpu, host, dev, w, 3)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=str)
def test_adamw_clipped_and_chained(crx, dtype):
    cpu, gpu = gradients([7, 4096, 20001], dtype, 9)
    host, dev = state_of(cpu)
    for step in (1, 2, 1000):
        before = [{k: t.cpu() for k, t in d.items()} for d in dev]
        norm = crx.grad_norm(gpu)
        crx.adamw_step(dev[0], gpu, dev[1], dev[2], norm=norm, max_norm=0.25, **step_args(step))
        check_step(cpu, before, dev, None, step, ref.coef(ref.norm(cpu.values()), 0.25))


def test_adamw_of_many_tensors(crx):
    sizes = [(i * 53) % 97 for i in range(1100)]
    cpu, gpu = gradients(sizes, torch.bfloat16, 10)
    host, dev = state_of(cpu)
    w = {k: torch.zeros(t.numel(), dtype=torch.bfloat16, device="cuda") for k, t in cpu.items()}
    crx.adamw_step(dev[0], gpu, dev[1], dev[2], w, **step_args(2))
    check_step(cpu, host, dev, w, 2)


@pytest.mark.parametrize("b1,b2", [(0.0, 0.0), (0.9, 0.999)])
def test_adamw_first_step_from_zero_moments(crx, b1, b2):
    p, g = torch.randn(1000, generator=gen(1)), torch.randn(1000, generator=gen(2))
    g[:10] = 0
    dev = [{"a": t.cuda()} for t in (p, torch.zeros(1000), torch.zeros(1000))]
    crx.adamw_step(dev[0], {"a": g.cuda()}, dev[1], dev[2], lr=1e-3, step=1, betas=(b1, b2))
    z = torch.zeros(1000)
    want, tol = ref.adamw(p, g, z, z, lr=1e-3, step=1, b1=b1, b2=b2, eps=1e-8, wd=0.0)
    for d, x, t in zip(dev, want, tol):
        near(d["a"], x, t)


@pytest.mark.parametrize("eps", [1e-30, 1e-15, 9e-13, 1e-12, 1e-6])
def test_adamw_of_tiny_gradients(crx, eps):
    """Second moments near and below the smallest normal number, next to an eps of any size."""
    g = torch.randn(20000, generator=gen(3)) * torch.logspace(-23, -15, 20000)
    p, z = torch.zeros(20000), torch.zeros(20000)
    dev = [{"a": t.cuda()} for t in (p, z, z)]
    crx.adamw_step(dev[0], {"a": g.cuda()}, dev[1], dev[2], lr=1e-3, step=1, eps=eps)
    want, tol = ref.adamw(p, g, z, z, lr=1e-3, step=1, b1=0.9, b2=0.999, eps=eps, wd=0.0)
    # below 2^-126 the root may count as 0: at most 2^-63 / eps of the update, where eps is 1e-12 or more;
    # and v is a multiple of 2^-149, so its root is known to half of that over the root
    v = want[2]
    loose = want[0].abs() * (2.0 ** -63 / eps if eps >= 1e-12 else 0.0)
    den = (v / (1 - 0.999)).sqrt()
    steps = want[0].abs() * 2.0 * (2.0 ** -149 / (1 - 0.999)) / (den * (den + eps)).clamp(min=1e-60)
    fine = steps < 0.1 * want[0].abs()   # (elsewhere v is a few of its steps and says nothing)
    near(dev[0]["a"].cpu()[fine], want[0][fine], (tol[0] + loose + steps)[fine])
    near(dev[2]["a"], v, tol[2])


@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_adamw_leaves_the_state_when_the_norm_is_not_finite(crx, bad):
    cpu, gpu = gradients([4001], torch.float32, 12)
    gpu["t0"][17] = bad
    host, dev = state_of(cpu)
    w = {"t0": torch.zeros(4001, dtype=torch.bfloat16, device="cuda")}
    crx.adamw_step(dev[0], gpu, dev[1], dev[2], w, norm=crx.grad_norm(gpu), max_norm=1.0, **step_args(2))
    for d, h in zip(dev, host):
        assert torch.equal(d["t0"].cpu(), h["t0"])
    assert torch.equal(w["t0"].cpu(), host[0]["t0"].to(torch.bfloat16))


def test_adamw_moves_versions(crx):
    cpu, gpu = gradients([64], torch.bfloat16, 13)
    host, dev = state_of(cpu)
    w = {"t0": torch.zeros(64, dtype=torch.bfloat16, device="cuda")}
    was = [d["t0"]._version for d in dev] + [w["t0"]._version]
    crx.adamw_step(dev[0], gpu, dev[1], dev[2], w, **step_args(1))
    assert all(d["t0"]._version > v for d, v in zip(dev + [w], was))


def test_a_captured_step_follows_its_tensors(crx):
    cpu, gpu = gradients([5000], torch.bfloat16, 14)
    host, dev = state_of(cpu)
    w = {"t0": torch.zeros(5000, dtype=torch.bfloat16, device="cuda")}
    lr = torch.tensor(HYPER["lr"], device="cuda")
    step = torch.ones(1, dtype=torch.int64, device="cuda")

    def body():
        n = crx.grad_norm(gpu)
        crx.adamw_step(dev[0], gpu, dev[1], dev[2], w, norm=n, max_norm=0.5, **{**step_args(1), "lr": lr, "step": step})
        return n

    body()
    for d, h in zip(dev, host):
        d["t0"].copy_(h["t0"])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        n = body()
    for s in (1, 2, 30):
        before = [{k: t.cpu() for k, t in d.items()} for d in dev]
        new, _ = gradients([5000], torch.bfloat16, 100 + s)
        gpu["t0"].copy_(new["t0"])
        step.fill_(s)
        graph.replay()
        torch.cuda.synchronize()
        want = ref.norm(new.values())
        near(n, want, want * ref.NORM)
        check_step(new, before, dev, w, s, ref.coef(want, 0.5))


# ---------------------------------------------------------------------------------- policy loss

def batch(B, T, V, dtype, seed=0, scale=2.5, old=True, with_ref=True, mask=None, pad=0):
    g = gen(seed)
    wide = (torch.randn(B, T, V + pad, generator=g) * scale).to(dtype)
    z = wide[..., :V]
    tokens = torch.randint(0, V, (B, T), generator=g)
    z.scatter_add_(2, tokens[..., None], (torch.rand(B, T, 1, generator=g) * 9).to(dtype))
    logp = torch.log_softmax(z.double(), -1).gather(2, tokens[..., None])[..., 0]
    d = torch.randn(B, T, generator=g) * 0.2
    r = (-d).exp()
    d = torch.where(((r - 0.8).abs() < 1e-3) | ((r - 1.2).abs() < 1e-3) | ((r - 1.28).abs() < 1e-3), 0.0, d)   # a border has no one gradient
    return {"logits": wide, "V": V, "tokens": tokens, "adv": torch.randn(B, 1, generator=g),
            "old": (logp + d).float() if old else None,
            "ref": (logp + torch.randn(B, T, generator=g) * 0.2).float() if with_ref else None, "mask": mask}


def dev(t):
    return None if t is None else t.cuda()


def run(crx, d, view=None, **kw):
    z = d["logits"].cuda()[..., :d["V"]]
    z = view(z) if view else z
    z = z.detach().requires_grad_()
    out = crx.policy_loss(z, dev(d["tokens"]), dev(d["adv"]), old_logp=dev(d["old"]), ref_logp=dev(d["ref"]), mask=dev(d["mask"]), **kw)
    grad, = torch.autograd.grad(out.loss, z)
    return out, grad


def verify(crx, d, **kw):
    out, grad = run(crx, d, **kw)
    rkw = {k: v for k, v in kw.items() if k in ("clip", "kl_coef", "denom")}
    want = ref.policy(d["logits"][..., :d["V"]], d["tokens"], d["adv"], old=d["old"], ref=d["ref"], mask=d["mask"],
                      tau=kw.get("temperature", 1.0), **rkw)
    for k in ("loss", "kl", "clip_frac", "logp"):
        near(getattr(out, k), want[k], want["tol_" + k], k)
    near(grad, want["grad"], want["tol_grad"], "grad")
    with torch.no_grad():   # the same values without the gradient
        kw.pop("view", None)
        again = crx.policy_loss(d["logits"].cuda()[..., :d["V"]], dev(d["tokens"]), dev(d["adv"]), old_logp=dev(d["old"]),
                                ref_logp=dev(d["ref"]), mask=dev(d["mask"]), **kw)
    assert not again.loss.requires_grad
    near(again.loss, want["loss"], want["tol_loss"])
    near(again.logp, want["logp"], want["tol_logp"])
    return out, grad


@pytest.mark.parametrize("V", [1, 2, 3, 7, 8, 9, 31, 255, 1000, 4096, 4099, 16387, 33000])
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_policy_loss(crx, dtype, V):
    verify(crx, batch(2, 5, V, dtype, V), kl_coef=0.04)


@pytest.mark.parametrize("B,T,V", [(1, 1, 152064), (1, 3, 151936), (2, 40, 50001), (3, 333, 1031), (1, 700, 257), (7, 150, 300)])
def test_policy_loss_sizes(crx, B, T, V):
    verify(crx, batch(B, T, V, torch.bfloat16, T), kl_coef=0.001, clip=(0.2, 0.28))


@pytest.mark.parametrize("pad", [1, 4, 8, 5000])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=str)
def test_policy_loss_of_padded_rows(crx, dtype, pad):
    verify(crx, batch(3, 17, 1003, dtype, pad, pad=pad), kl_coef=0.04)


def test_policy_loss_layouts(crx):
    d = batch(4, 6, 515, torch.bfloat16, 3)
    # the rows of a longer batch (logits[:, :-1]), sequences behind tokens, rows apart, rows shared
    def longer(z):
        return torch.cat([z, z[:, :1]], 1)[:, :-1]

    def swapped(z):
        return z.transpose(0, 1).contiguous().transpose(0, 1)

    def apart(z):
        return z.repeat_interleave(3, 0)[::3]

    def odd(z):
        flat = torch.zeros(z.numel() + 1, dtype=z.dtype, device="cuda")[1:].view(z.shape)
        return flat.copy_(z)

    for view in (longer, swapped, apart, odd):
        verify(crx, d, view=view, kl_coef=0.04)
    shared = {**d, "logits": d["logits"][:1, :1].clone().expand(4, 6, 515), "old": None}
    z = shared["logits"][:1, :1].cuda().expand(4, 6, 515).requires_grad_()
    out = crx.policy_loss(z, dev(d["tokens"]), dev(d["adv"]), ref_logp=dev(d["ref"]), kl_coef=0.04)
    g, = torch.autograd.grad(out.loss, z)
    want = ref.policy(shared["logits"], d["tokens"], d["adv"], ref=d["ref"], kl_coef=0.04)
    near(out.loss, want["loss"], want["tol_loss"])
    near(g, want["grad"], want["tol_grad"])


def test_policy_loss_of_a_broadcast_leaf(crx):
    row = torch.randn(1, 1, 130, generator=gen(5))
    d = batch(3, 4, 130, torch.float32, 5)
    leaf = row.cuda().requires_grad_()
    out = crx.policy_loss(leaf.expand(3, 4, 130), dev(d["tokens"]), dev(d["adv"]))
    out.loss.backward()
    want = ref.policy(row.expand(3, 4, 130), d["tokens"], d["adv"])
    near(leaf.grad, want["grad"].sum((0, 1), keepdim=True), want["tol_grad"].sum((0, 1), keepdim=True) + 12 * ref.H * want["grad"].abs().sum((0, 1), keepdim=True))


@pytest.mark.parametrize("tau,roundings", [(1.0, 1), (0.75, 2)])
def test_log_probabilities_of_unlikely_tokens(crx, tau, roundings):
    """Next to one large logit: the difference of two logits, which bf16 ones have exactly, over the temperature."""
    z = torch.zeros(4000, 2, dtype=torch.bfloat16)
    z[:, 0] = torch.rand(4000, generator=gen(44)) * 100 - 40
    z[:, 1] = z[:, 0].float() - 18 - torch.rand(4000, generator=gen(45)) * 40
    tokens = torch.ones(4000, dtype=torch.int64)
    out = crx.policy_loss(z.cuda(), dev(tokens), torch.ones(4000, device="cuda"), temperature=tau)
    want = torch.log_softmax(z.double() / tau, -1)[:, 1]
    # the quotient (exact where it is by 1) and the sum with log s are rounded; s is 1 to e^-18 + H, twice that in 2^x
    near(out.logp, want, roundings * ref.H * want.abs() + 2 * (math.exp(-17) + ref.H))


def test_policy_loss_of_one_sequence(crx):
    d = batch(1, 23, 999, torch.float16, 6)
    one = {k: v[0] if torch.is_tensor(v) else v for k, v in d.items()}
    verify(crx, one, kl_coef=0.1)
    i32 = {**one, "tokens": one["tokens"].int(), "adv": torch.randn(23, generator=gen(1))}
    verify(crx, i32)


def test_operands_at_any_stride(crx):
    d = batch(3, 8, 300, torch.float32, 7, mask=torch.rand(3, 8, generator=gen(9)) < 0.7)
    base, grad = run(crx, d, kl_coef=0.04)

    def wide(t):
        out = torch.full((t.shape[0], 2 * t.shape[1] + 1), 1, dtype=t.dtype, device="cuda")[:, 1::2]
        return out.copy_(t)

    z = d["logits"].cuda().requires_grad_()
    out = crx.policy_loss(z, wide(d["tokens"]), wide(d["adv"].expand(3, 8)), old_logp=wide(d["old"].cuda().t().contiguous().t()),
                          ref_logp=wide(d["ref"]), mask=wide(d["mask"]), kl_coef=0.04)
    g, = torch.autograd.grad(out.loss, z)
    assert torch.equal(out.loss, base.loss) and torch.equal(g, grad) and torch.equal(out.logp, base.logp)


@pytest.mark.parametrize("kind", ["bool", "weights", "one", "per sequence"])
def test_masks(crx, kind):
    g = gen(8)
    mask = {"bool": torch.rand(5, 9, generator=g) < 0.6, "weights": torch.rand(5, 9, generator=g).float(),
            "one": torch.zeros(5, 9, dtype=torch.bool), "per sequence": torch.tensor([[1.], [0.], [2.], [0.5], [0.]])}[kind]
    if kind == "one":
        mask[3, 4] = True
    if kind == "bool":
        mask[2] = False
    verify(crx, batch(5, 9, 777, torch.bfloat16, 8, mask=mask), kl_coef=0.04)
    verify(crx, batch(5, 9, 777, torch.bfloat16, 8, mask=mask), kl_coef=0.04, denom=5.0)


@pytest.mark.parametrize("size", [1e-41, 1e-30, 1e30, 1e38])
def test_weights_of_any_size(crx, size):
    """Weights and their sum far from 1: only their proportions count."""
    d = batch(2, 8, 500, torch.float32, 38)
    steps = torch.randint(1, 4, (2, 8), generator=gen(39)).float()
    mask = steps * torch.tensor(size)
    verify(crx, {**d, "mask": mask}, kl_coef=0.04)
    verify(crx, {**d, "mask": mask}, kl_coef=0.04, denom=float(mask.double().sum()) / 2)


@pytest.mark.parametrize("n", [1, 31, 32, 33, 255, 1023, 1024, 1025, 8191, 30001, 262147])
def test_masks_over_many_rows(crx, n):
    """The order in which rows are taken covers each once, wherever its runs end."""
    mask = torch.rand(n, generator=gen(n)) < 0.5
    d = batch(1, n, 5, torch.float32, 24, with_ref=False)
    one = {k: v[0] if torch.is_tensor(v) else v for k, v in d.items()}
    verify(crx, {**one, "mask": mask})
    out, grad = run(crx, {**one, "mask": mask})
    assert bool((grad.abs().sum(-1) != 0).cpu()[~mask].sum() == 0)


@pytest.mark.parametrize("B,T,V,dtype", [
    (1, 1300, 152064, torch.bfloat16),   # clusters whose rows do not fit the rings, about nine rows each
    (2, 350, 33000, torch.float32),      # clusters of two
    (1, 1300, 33001, torch.bfloat16),    # CTAs whose rows do not fit
    (1, 1900, 12001, torch.bfloat16),    # CTAs whose rows do
    (1, 1400, 12001, torch.float32),
    (3, 2000, 4099, torch.float16),      # warps
    (1, 5000, 9001, torch.bfloat16),     # warps whose rows do not fit
], ids=str)
@pytest.mark.parametrize("masked", [False, True], ids=["all", "masked"])
def test_many_rows_that_count_for_every_unit(crx, B, T, V, dtype, masked):
    """Rings, barriers and the parts of a cluster over many rows, row by row; equal bits when it runs again."""
    g = torch.Generator(device="cuda").manual_seed(41)
    z = (torch.randn(B, T, V, generator=g, device="cuda") * 2.5).to(dtype)
    tokens = torch.randint(0, V, (B, T), generator=g, device="cuda")
    z.scatter_add_(2, tokens[..., None], (torch.rand(B, T, 1, generator=g, device="cuda") * 9).to(dtype))
    adv = torch.randn(B, T, generator=g, device="cuda")
    mask = torch.rand(B, T, generator=g, device="cuda") < 0.8 if masked else torch.ones(B, T, dtype=torch.bool, device="cuda")
    leaf = z.detach().requires_grad_()

    def once():
        out = crx.policy_loss(leaf, tokens, adv, mask=mask if masked else None)
        return out, torch.autograd.grad(out.loss, leaf)[0]

    out, grad = once()
    u = (-adv.double() / mask.sum()) * mask
    depth = V / 512 + 48
    for b in range(B):
        for lo in range(0, T, 50):
            part = slice(lo, min(T, lo + 50))
            q = torch.log_softmax(z[b, part].double(), -1)
            a = tokens[b, part, None]
            logp = q.gather(1, a)[:, 0]
            on = mask[b, part]
            tilt = (z[b, part].double().gather(1, a)[:, 0] - (q.exp() * z[b, part].double()).sum(-1)).abs()
            tol = ref.H * (depth + 12 + 4 * logp.abs() + 2 * tilt + math.log(V))   # as in trainer_ref
            assert bool(((out.logp[b, part].double() - torch.where(on, logp, 0.0)).abs() <= tol).all()), (b, lo)
            p = q.exp()
            hot = torch.zeros_like(p).scatter_(1, a, 1.0)
            ub = u[b, part, None]
            want = ub * (hot - p)
            bound = ub.abs() * (8 * ref.H * (hot + p) + p * ref.H * (depth + 20 + 3 * q.abs() + 2 * math.log(V))) + ref.half_step(want, dtype)
            assert bool(((grad[b, part].double() - want).abs() <= bound).all()), (b, lo)
    loss = float((adv.double() * mask).sum() / -mask.sum())   # (every ratio is 1)
    assert abs(float(out.loss.detach()) - loss) <= 4 * ref.H * float((adv.double().abs() * mask).sum() / mask.sum())
    with torch.no_grad():
        alone = crx.policy_loss(z, tokens, adv, mask=mask if masked else None)
    # another split of the row, each within the tolerance (the tilt is at most |logp| + log V)
    assert bool(((alone.logp - out.logp).abs().double() <= 2 * ref.H * (depth + 12 + 6 * out.logp.abs().double() + 3 * math.log(V))).all())
    for _ in range(3):
        out2, grad2 = once()
        assert torch.equal(out2.logp, out.logp) and torch.equal(out2.loss, out.loss) and torch.equal(grad2, grad)


def test_a_mask_that_leaves_nothing(crx):
    d = batch(2, 3, 100, torch.float32, 9, mask=torch.zeros(2, 3, dtype=torch.bool))
    out, grad = run(crx, d, kl_coef=0.04)
    assert float(out.loss.detach()) == float(out.kl) == float(out.clip_frac) == 0 and not out.logp.any() and not grad.any()


def test_what_stands_in_masked_places_does_not_count(crx):
    mask = torch.ones(3, 6, dtype=torch.bool)
    mask[0, 2:] = False
    mask[2] = False
    d = batch(3, 6, 1000, torch.bfloat16, 10, mask=mask)
    out, grad = run(crx, d, kl_coef=0.04)
    bad = {k: v.clone() if torch.is_tensor(v) else v for k, v in d.items()}
    for name, value in (("logits", math.nan), ("old", math.inf), ("ref", -math.inf), ("tokens", -100)):
        bad[name][~mask] = value
    bad["adv"] = d["adv"].expand(3, 6).clone()
    bad["adv"][~mask] = math.nan
    out2, grad2 = run(crx, bad, kl_coef=0.04)
    assert torch.equal(out.loss, out2.loss) and torch.equal(grad, grad2) and torch.equal(out.logp, out2.logp)
    assert not grad[2].any() and not out.logp[2].any()


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_vocabulary_masks(crx, dtype):
    """Tokens ruled out by -inf or the type's lowest value, up to all but one."""
    d = batch(2, 4, 5000, dtype, 11, old=False, with_ref=False)
    low = torch.finfo(dtype).min
    keep = torch.rand(2, 4, 5000, generator=gen(1)) < 0.1
    keep.scatter_(2, d["tokens"][..., None], True)
    keep[0, 0] = False
    keep[0, 0, d["tokens"][0, 0]] = True
    for value in (-math.inf, low):
        z = torch.where(keep, d["logits"], torch.tensor(value, dtype=dtype))
        verify(crx, {**d, "logits": z})


@pytest.mark.parametrize("value", ["low", "high", "mixed"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=str)
def test_rows_of_extreme_logits(crx, dtype, value):
    """Logits that fp32 cannot hold once scaled: a row of the type's lowest (or highest) value is uniform."""
    f = torch.finfo(dtype)
    d = batch(1, 3, 5001, dtype, 12, old=False, with_ref=False)
    z = torch.full((1, 3, 5001), f.min if value == "low" else f.max, dtype=dtype)
    if value == "mixed":
        z[..., 100:] = f.min
        z[..., 4000:] = -math.inf
        d["tokens"] = torch.tensor([[5, 99, 50]])
    verify(crx, {**d, "logits": z})
    verify(crx, {**d, "logits": z}, temperature=0.5)


# What a row's small probabilities may lose beside the tolerances of trainer_ref: 2^x is 0 below 2^-126, of
# a sum that a maximum of up to 2^30 (in units of log2; its rounding is 2^5 at most) may have lowered to 2^-32.
FLUSH = 2.0 ** -94


def verify_rows(crx, d, tau=1.0):
    """Loss, log-probabilities and gradient of rows without an older policy (so each ratio is 1, whatever
    the log-probability), with the gradient's own error where a probability is as good as 0."""
    out, grad = run(crx, d, temperature=tau)
    want = ref.policy(d["logits"][..., :d["V"]], d["tokens"], d["adv"], tau=tau)
    near(out.logp, want["logp"], want["tol_logp"], "logp")
    near(out.loss, want["loss"], 4 * ref.H * float(d["adv"].abs().double().mean()) + 1e-12, "loss")
    u = (d["adv"].double().expand(d["tokens"].shape) / d["tokens"].numel() / tau).abs()[..., None]
    z = d["logits"][..., :d["V"]].double() / tau
    p = torch.log_softmax(z, -1).exp()
    hot = torch.zeros_like(p).scatter_(-1, d["tokens"][..., None], 1.0)
    # u: advantage, 1 / number, 1 / temperature and their products; p: as in trainer_ref
    depth = d["V"] / 512 + 48
    expo = torch.where(p > 0, p.clamp(min=1e-300).log(), 0.0).abs() * 1.45
    tol = u * (8 * ref.H * (hot + p) + p * ref.H * (depth + 20 + 4 * expo + 3 * math.log(d["V"])) + FLUSH) + ref.half_step(want["grad"], grad.dtype)
    near(grad, want["grad"], tol, "grad")
    return out, grad


@pytest.mark.parametrize("fill", [1e7, 5e8, 1e9, 1e10, 1e12, 1e20, 1e30])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=str)
def test_vocabulary_masks_of_any_fill(crx, dtype, fill):
    """Tokens ruled out by a large negative number: scattered ones, runs longer than a CTA's chunks, a row's first
    and last elements; and rows of nothing but that number, or of the opposite one."""
    V = 33333
    d = batch(1, 8, V, dtype, 25, old=False, with_ref=False)
    d["tokens"][:] = 20001
    d["adv"] = torch.randn(1, 8, generator=gen(26))
    z = d["logits"][0]
    z[0, ::2] = -fill
    z[1, :20000] = -fill
    z[2, 20002:] = -fill
    z[3, :9] = -fill
    z[3, -9:] = -fill
    z[4] = -fill
    z[4, 20001] = 3.0
    z[5] = -fill
    z[6] = fill
    z[7, 20001] = fill
    verify_rows(crx, d)
    warps = {**d, "logits": z[:7].repeat_interleave(100, 0)[None], "tokens": d["tokens"][:, :7].repeat_interleave(100, 1),
             "adv": d["adv"][:, :7].repeat_interleave(100, 1)}
    warps["logits"] = warps["logits"][..., 19000:20000 + 2048 + 3]   # as many short rows as take a warp each
    verify_rows(crx, {**warps, "V": 3051, "tokens": warps["tokens"] - 19000})


@pytest.mark.parametrize("tau", [1e-1, 1e-3, 1e-6, 1e-7, 1e-8, 1e-9, 1e-12, 1e-20, 2e-30, 1e4, 1e30])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=str)
def test_temperatures_down_to_the_limit(crx, dtype, tau):
    """Ordinary logits; the largest was sampled, and in the last rows another."""
    d = batch(1, 12, 1003, dtype, 27, old=False, with_ref=False)
    d["tokens"] = d["logits"].argmax(-1)
    d["tokens"][0, 8:] = 17
    d["adv"] = torch.randn(1, 12, generator=gen(28))
    verify_rows(crx, d, tau)


@pytest.mark.parametrize("far", [1e-9, 1.0])
def test_a_scaled_loss_of_large_logits(crx, far):
    """The second pass over the logits takes the same exponents as the first."""
    d = batch(1, 6, 1003, torch.float32, 43, old=False, with_ref=False)
    if far == 1.0:
        d["logits"][0, :3] *= 1e12
        d["logits"][0, 4] = -1e10
    z = d["logits"].cuda().requires_grad_()
    out = crx.policy_loss(z, dev(d["tokens"]), dev(d["adv"]), temperature=far)
    once, = torch.autograd.grad(out.loss, z, retain_graph=True)
    twice, = torch.autograd.grad(out.loss * 2, z)
    assert torch.isfinite(once).all() and torch.equal(twice, once * 2)


def test_values_that_are_not_numbers(crx):
    d = batch(1, 4, 600, torch.float32, 13, old=False, with_ref=False)
    d["logits"][0, 1, 5] = math.nan
    d["logits"][0, 2] = -math.inf
    d["logits"][0, 3, 7] = math.inf
    out, grad = run(crx, d)
    assert math.isnan(out.loss) and torch.isnan(out.logp[0, 1:]).all() and torch.isfinite(out.logp[0, 0])
    assert torch.isnan(grad[0, 1:]).all() and torch.isfinite(grad[0, 0]).all()


@pytest.mark.parametrize("token", [-1, -100, 600, 1 << 40])
def test_a_token_outside_the_vocabulary(crx, token):
    d = batch(1, 3, 600, torch.float32, 14)
    d["tokens"][0, 1] = token
    out, grad = run(crx, d)
    assert math.isnan(out.loss) and math.isnan(out.logp[0, 1]) and torch.isfinite(out.logp[0, ::2]).all()
    assert torch.isfinite(grad[0, ::2]).all()


@pytest.mark.parametrize("what", ["token", "logits", "old"])
def test_an_advantage_of_zero_hides_nothing(crx, what):
    d = batch(1, 3, 600, torch.float32, 32, with_ref=False)
    d["adv"] = torch.tensor([[1.0, 0.0, -1.0]])
    if what == "token":
        d["tokens"][0, 1] = 600
    elif what == "logits":
        d["logits"][0, 1, 7] = math.nan
    else:
        d["old"][0, 1] = math.nan
    out, grad = run(crx, d)
    assert torch.isnan(out.loss) and torch.isnan(grad[0, 1]).all() and torch.isfinite(grad[0, ::2]).all()


def test_a_token_that_was_ruled_out(crx):
    """A sampled token of probability 0: logp -inf, ratio 0; without a KL term its gradient is finite."""
    d = batch(1, 2, 300, torch.float32, 15, with_ref=False)
    d["logits"][0, 1, d["tokens"][0, 1]] = -math.inf
    d["adv"] = torch.tensor([[0.5]])
    out, grad = run(crx, d)
    assert out.logp[0, 1] == -math.inf and torch.isfinite(out.loss) and not grad[0, 1].any()


def test_zero_advantage_and_far_ratios(crx):
    d = batch(1, 6, 400, torch.float32, 16, with_ref=False)
    d["adv"] = torch.tensor([[0.0, 0.0, 1.0, -1.0, 1.0, -1.0]])
    d["old"] += torch.tensor([[-200.0, 200.0, -200.0, 200.0, 90.0, 90.0]])
    out, grad = verify(crx, d)
    assert torch.isfinite(out.loss) and not grad[0, :4].any()


def test_a_reference_that_is_only_reported(crx):
    """Without a coefficient the KL term may be anything: loss and gradient do not see it."""
    d = batch(1, 4, 200, torch.float32, 16)
    base, grad = run(crx, {**d, "ref": None})
    d["ref"][0, 1] = 200.0
    out, grad2 = run(crx, d)
    assert torch.equal(out.loss, base.loss) and torch.equal(grad, grad2) and out.kl == math.inf


@pytest.mark.parametrize("clip", [(0.0, 0.0), (5.0, math.inf), (0.2, 1e300)])
def test_clip_bounds_of_any_size(crx, clip):
    d = batch(2, 20, 300, torch.float32, 22, with_ref=False)
    d["old"] += 0.01   # no ratio of exactly 1
    verify(crx, d, clip=clip)


def test_dicts_in_different_orders(crx):
    cpu, gpu = gradients([100, 33, 7000], torch.bfloat16, 15)
    host, dev = state_of(cpu)
    turned = [dict(reversed(list(x.items()))) for x in dev]
    w = {k: torch.zeros(t.numel(), dtype=torch.bfloat16, device="cuda") for k, t in sorted(cpu.items(), reverse=True)}
    crx.adamw_step(turned[0], gpu, dev[1], turned[2], w, **step_args(3))
    check_step(cpu, host, dev, w, 3)
    out = {k: torch.zeros_like(t) for k, t in reversed(list(gpu.items()))}
    crx.clip_grads(gpu, 1.0, out=out)
    n = ref.norm(cpu.values())
    for k in cpu:
        near(out[k], *ref.clip(cpu[k], ref.coef(n, 1.0)), k)


def test_empty_batches(crx):
    for shape in [(0,), (0, 4), (3, 0)]:
        z = torch.zeros(*shape, 10, device="cuda", requires_grad=True)
        out = crx.policy_loss(z, torch.zeros(shape, dtype=torch.int64, device="cuda"), torch.zeros(shape, device="cuda"))
        out.loss.backward()
        assert float(out.loss) == 0 and out.logp.shape == shape and z.grad.shape == z.shape


@pytest.mark.parametrize("scale", [0.5, -3.0, 0.0, 65536.0])
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32], ids=str)
def test_a_scaled_loss(crx, dtype, scale):
    d = batch(3, 30, 2000, dtype, 17, mask=torch.rand(3, 30, generator=gen(2)) < 0.5)
    z = d["logits"].cuda().requires_grad_()
    out = crx.policy_loss(z, dev(d["tokens"]), dev(d["adv"]), old_logp=dev(d["old"]), mask=dev(d["mask"]))
    g, = torch.autograd.grad(out.loss * scale, z)
    want = ref.policy(d["logits"], d["tokens"], d["adv"], old=d["old"], mask=d["mask"])
    exact = want["grad"] * scale
    # the scaled gradient is rounded once, so small ones that fp16 cannot hold come through a large scale
    tol = (want["tol_grad"] - ref.half_step(want["grad"], dtype)) * abs(scale) + 2 * ref.H * exact.abs() + ref.half_step(exact, dtype)
    near(g, exact, tol)


def test_backward_twice(crx):
    d = batch(2, 9, 700, torch.bfloat16, 18)
    z = d["logits"].cuda().requires_grad_()
    out = crx.policy_loss(z, dev(d["tokens"]), dev(d["adv"]), old_logp=dev(d["old"]))
    a, = torch.autograd.grad(out.loss, z, retain_graph=True)
    keep = a.clone()
    a.zero_()   # the caller's own now
    b, = torch.autograd.grad(out.loss, z, retain_graph=True)
    c, = torch.autograd.grad(out.loss, z, grad_outputs=torch.tensor(2.0, device="cuda"))
    assert torch.equal(b, keep)
    near(c, 2 * keep.double().cpu(), 1e-30)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(out.loss, z)


def test_a_gradient_of_the_gradient_is_refused(crx):
    d = batch(1, 2, 50, torch.float32, 19)
    z = d["logits"].cuda().requires_grad_()
    out = crx.policy_loss(z, dev(d["tokens"]), dev(d["adv"]))
    with pytest.raises(RuntimeError, match="not differentiable"):
        torch.autograd.grad(out.loss, z, create_graph=True)


@pytest.mark.parametrize("needs_grad", [False, True])
def test_forward_gradients_are_refused(crx, needs_grad):
    from torch.autograd import forward_ad
    d = batch(1, 2, 50, torch.float32, 40)
    z = d["logits"].cuda().requires_grad_(needs_grad)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(z, torch.ones_like(z))
        with pytest.raises(ValueError, match="forward"):
            crx.policy_loss(dual, dev(d["tokens"]), dev(d["adv"]))
        with pytest.raises(ValueError, match="forward"), torch.no_grad():
            crx.policy_loss(dual, dev(d["tokens"]), dev(d["adv"]))
    crx.policy_loss(z, dev(d["tokens"]), dev(d["adv"]))


def test_inference_tensors_are_not_written(crx):
    with torch.inference_mode():
        t = torch.ones(8, device="cuda")
        near(crx.grad_norm({"t": t}), math.sqrt(8), math.sqrt(8) * ref.NORM)
        crx.clip_grads({"t": t}, 1.0)
    near(t.clone(), torch.full((8,), 1 / math.sqrt(8)), 1e-6)
    before = t.clone()
    near(crx.grad_norm({"t": t}), 1.0, 1e-6)
    with pytest.raises(ValueError, match="inference"):
        crx.clip_grads({"t": t}, 0.5)
    assert torch.equal(t.clone(), before)


def test_logits_changed_before_backward_are_noticed(crx):
    d = batch(1, 2, 50, torch.float32, 19)
    z = d["logits"].cuda().requires_grad_()
    y = z * 1.0
    out = crx.policy_loss(y, dev(d["tokens"]), dev(d["adv"]))
    with torch.no_grad():
        y.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.loss.backward()


class Offloaded:
    """Hooks that hand saved tensors to the backward pass as contiguous copies, as offloading them does."""

    def __init__(self, there=lambda t: t.to("cpu", copy=True), back=lambda t: t.cuda()):
        self.hooks = torch.autograd.graph.saved_tensors_hooks(lambda t: there(t.contiguous()), back)


@pytest.mark.parametrize("scale", [1.0, 0.5])
def test_saved_tensors_that_come_back_laid_out_otherwise(crx, scale):
    """Shifted tokens and logits, saved by hooks that return contiguous ones."""
    d = batch(4, 10, 301, torch.bfloat16, 29, mask=torch.rand(4, 10, generator=gen(30)) < 0.8)
    z = d["logits"].cuda()
    tokens, rest = dev(d["tokens"])[:, 1:], {k: dev(d[k])[:, 1:] for k in ("old", "ref", "mask")}

    def grads(hooks):
        x = z.clone().requires_grad_()
        with hooks:
            out = crx.policy_loss(x[:, :-1], tokens, dev(d["adv"]), old_logp=rest["old"], ref_logp=rest["ref"], mask=rest["mask"], kl_coef=0.04)
        first, = torch.autograd.grad(out.loss * scale, x, retain_graph=True)
        second, = torch.autograd.grad(out.loss * scale, x)
        return first, second

    want = grads(contextlib.nullcontext())
    assert torch.equal(*want)
    for hooks in (Offloaded().hooks, torch.autograd.graph.save_on_cpu(), torch.autograd.graph.save_on_cpu(pin_memory=True)):
        for g, w in zip(grads(hooks), want):
            assert torch.equal(g, w)


@pytest.mark.parametrize("back", [lambda t: t, lambda t: t.cuda()[..., :1], lambda t: t.cuda().to(torch.int32 if t.dtype == torch.int64 else t.dtype),
                                  lambda t: t.cuda().to(torch.float16 if t.dtype == torch.bfloat16 else t.dtype)],
                         ids=["host", "shape", "tokens' type", "logits' type"])
def test_saved_tensors_that_come_back_as_others_are_refused(crx, back):
    d = batch(2, 5, 64, torch.bfloat16, 31)
    z = d["logits"].cuda().requires_grad_()
    with Offloaded(back=back).hooks:
        out = crx.policy_loss(z, dev(d["tokens"]), dev(d["adv"]))
    with pytest.raises(RuntimeError, match="saved"):
        torch.autograd.grad(out.loss * 0.5, z)


def test_gradient_against_differences(crx):
    d = batch(1, 2, 9, torch.float32, 20, scale=1.0)
    kw = dict(old=d["old"], ref=d["ref"], kl_coef=0.3, tau=0.8)
    out, grad = run(crx, d, kl_coef=0.3, temperature=0.8)
    h = 1e-5
    for t in range(2):
        for j in range(9):
            up, down = d["logits"].double().clone(), d["logits"].double().clone()
            up[0, t, j] += h
            down[0, t, j] -= h

            def loss(z):
                logp = torch.log_softmax(z / 0.8, -1).gather(2, d["tokens"][..., None])[..., 0]
                r = (logp - d["old"].double()).exp()
                s = torch.minimum(r * d["adv"].double(), r.clamp(0.8, 1.2) * d["adv"].double())
                x = d["ref"].double() - logp
                return float((-s + 0.3 * (x.exp() - x - 1)).mean())
            assert kw["tau"] == 0.8
            slope = (loss(up) - loss(down)) / (2 * h)
            # the difference quotient: h^2 of a third derivative of order 10, and 64-bit roundings over h
            assert abs(float(grad[0, t, j]) - slope) < 1e-8 + 1e-5 * abs(slope) + 40 * ref.H


def test_elements_past_2_31(crx):
    """More logits than 32 bits count: rows at the far end."""
    T, V = 16500, 131072
    z = torch.zeros(T, V, dtype=torch.bfloat16, device="cuda")
    d = batch(1, 4, V, torch.bfloat16, 21, with_ref=False)
    z[-4:] = d["logits"][0].cuda()
    tokens = torch.zeros(T, dtype=torch.int64, device="cuda")
    tokens[-4:] = d["tokens"][0].cuda()
    mask = torch.zeros(T, dtype=torch.bool, device="cuda")
    mask[-4:] = True
    out = crx.policy_loss(z.requires_grad_(), tokens, torch.ones(T, device="cuda"), mask=mask)
    g, = torch.autograd.grad(out.loss, z)
    want = ref.policy(d["logits"], d["tokens"], torch.ones(1, 4))
    near(out.logp[-4:], want["logp"][0], want["tol_logp"][0])
    near(g[-4:], want["grad"][0], want["tol_grad"][0])
    assert not g[:100].any() and not g[T // 2:T // 2 + 100].any() and not g[-104:-4].any()


def test_gradients_past_2_31(crx):
    n = (1 << 31) + 4099
    g = torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    g[-5000:] = 3.0
    g[:7] = 4.0
    want = math.sqrt(5000 * 9 + 7 * 16)
    near(crx.grad_norm({"g": g}), want, want * ref.NORM)
    p, m, v = (torch.zeros(n, device="cuda") for _ in range(3))
    crx.adamw_step({"g": p}, {"g": g}, {"g": m}, {"g": v}, lr=1e-3, step=1)
    for part in (slice(0, 5000), slice(n - 6000, n)):
        x, z = g[part].cpu(), torch.zeros(p[part].numel())
        new, tol = ref.adamw(z, x, z, z, lr=1e-3, step=1, b1=0.9, b2=0.999, eps=1e-8, wd=0.0)
        for t, w, e in zip((p, m, v), new, tol):
            near(t[part], w, e)
    assert not p[n // 2:n // 2 + 100000].any()
    crx.clip_grads({"g": g}, want / 2)
    near(g[-5000:], *ref.clip(torch.full((5000,), 3.0, dtype=torch.bfloat16), ref.coef(want, want / 2)))
    assert not g[n // 2:n // 2 + 100000].any()


def test_calls_on_two_streams_and_equal_bits(crx):
    ds = [batch(4, 50, 9001, torch.bfloat16, 30 + i) for i in range(2)]
    ins = [(d["logits"].cuda().requires_grad_(), dev(d["tokens"]), dev(d["adv"]), dev(d["old"])) for d in ds]
    alone = [run(crx, {**d, "ref": None}) for d in ds]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in ds]
    for _ in range(5):
        got = []
        for s, (z, tok, adv, old) in zip(streams, ins):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                out = crx.policy_loss(z, tok, adv, old_logp=old)
                got.append((out, torch.autograd.grad(out.loss, z)[0], crx.grad_norm({"z": z.detach()})))
        torch.cuda.synchronize()
        for (o, g, n), (o1, g1), (z, *_), d in zip(got, alone, ins, ds):
            assert torch.equal(o.loss, o1.loss) and torch.equal(g, g1) and torch.equal(o.logp, o1.logp)
            want = ref.norm([d["logits"]])
            near(n, want, want * ref.NORM)


def test_two_captured_losses(crx):
    """Two graphs captured side by side, replayed in either order on new inputs."""
    graphs = []
    for i in range(2):
        d = batch(2, 20, 3001 + i, torch.bfloat16, 40 + i, mask=torch.ones(2, 20, dtype=torch.bool))
        z = d["logits"].cuda()
        args = {k: dev(d[k]) for k in ("tokens", "adv", "old", "ref", "mask")}

        def body(z=z, a=args):
            x = z.detach().requires_grad_()
            out = crx.policy_loss(x, a["tokens"], a["adv"], old_logp=a["old"], ref_logp=a["ref"], mask=a["mask"], kl_coef=0.04)
            return out, torch.autograd.grad(out.loss, x)[0]

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            body()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out, g = body()
        graphs.append((graph, z, args, out, g, 3001 + i))
    for order in ((0, 1), (1, 0)):
        fresh = {}
        for i in order:
            graph, z, args, out, g, V = graphs[i]
            d = batch(2, 20, V, torch.bfloat16, 50 + 2 * i + order[0], mask=torch.rand(2, 20, generator=gen(i)) < 0.5)
            z.copy_(d["logits"])
            for k, v in args.items():
                v.copy_(d[k])
            fresh[i] = d
            graph.replay()
        torch.cuda.synchronize()
        for i in order:
            _, _, _, out, g, V = graphs[i]
            d = fresh[i]
            want = ref.policy(d["logits"], d["tokens"], d["adv"], old=d["old"], ref=d["ref"], mask=d["mask"], kl_coef=0.04)
            near(out.loss, want["loss"], want["tol_loss"])
            near(g, want["grad"], want["tol_grad"])


def test_a_backward_pass_captured_without_its_loss(crx):
    """Each replay gives the gradient for the incoming gradient of that time, whatever was done with the one before."""
    d = batch(2, 12, 900, torch.bfloat16, 33)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for captured in (False, True):
        with torch.cuda.stream(side):
            z = d["logits"].cuda().requires_grad_()
            args = [dev(d["tokens"]), dev(d["adv"])]
            old, scale = dev(d["old"]), torch.ones((), device="cuda")
            want = {}
            for f in (1.0, 2.0, -0.5):
                out = crx.policy_loss(z, *args, old_logp=old)
                want[f], = torch.autograd.grad(out.loss, z, grad_outputs=torch.tensor(f, device="cuda"))
            first = torch.cuda.CUDAGraph()
            if captured:
                with torch.cuda.graph(first, stream=side):
                    out = crx.policy_loss(z, *args, old_logp=old)
                first.replay()
            else:
                out = crx.policy_loss(z, *args, old_logp=old)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                g, = torch.autograd.grad(out.loss, z, grad_outputs=scale, retain_graph=True)
            for f in (2.0, 1.0, 1.0, -0.5, 1.0):
                scale.fill_(f)
                graph.replay()
                assert torch.equal(g, want[f]), (captured, f)
                g.zero_()   # the caller's own
            if captured:   # a gradient taken outside stays as it is when the loss is replayed on other logits
                kept, = torch.autograd.grad(out.loss, z, retain_graph=True)
                assert torch.equal(kept, want[1.0])
                with torch.no_grad():
                    z.zero_()
                first.replay()
                assert torch.equal(kept, want[1.0])
        torch.cuda.synchronize()


def test_a_graphed_callable(crx):
    """Loss and backward pass captured one after the other, replayed on new inputs."""
    shape = (2, 9, 701)
    d = batch(*shape, torch.bfloat16, 34, with_ref=False)
    tokens, adv, old = dev(d["tokens"]), dev(d["adv"]), dev(d["old"])
    z = d["logits"].cuda().requires_grad_()
    graphed = torch.cuda.make_graphed_callables(lambda x: crx.policy_loss(x, tokens, adv, old_logp=old).loss, (z,))
    for seed, f in ((35, 1.0), (36, 3.0), (37, 1.0)):
        x = batch(*shape, torch.bfloat16, seed)["logits"].cuda().requires_grad_()
        loss = graphed(x)
        g, = torch.autograd.grad(loss * f, x)
        y = x.detach().clone().requires_grad_()
        out = crx.policy_loss(y, tokens, adv, old_logp=old)
        w, = torch.autograd.grad(out.loss * f, y)
        assert torch.equal(loss, out.loss) and torch.equal(g, w)


# ---------------------------------------------------------------------------------- together

def test_a_trainers_step_through_to_the_worker(crx):
    """Loss, backward, norm, clipped step and sync, three steps: the worker's weights are the
    trainer's bits, and the parameters are those of the same steps in plain torch."""
    g = gen(60)
    V, D, B, T = 997, 64, 4, 12
    p0 = {"embed": torch.randn(V, D, generator=g) * 0.1, "head": torch.randn(V, D, generator=g) * 0.1,
          "norm": torch.ones(D)}
    masters = {k: v.cuda() for k, v in p0.items()}
    m, v = ({k: torch.zeros_like(t) for k, t in masters.items()} for _ in range(2))
    prev = {k: t.bfloat16() for k, t in masters.items()}
    cur = {k: t.clone() for k, t in prev.items()}
    worker = {k: t.clone() for k, t in prev.items()}
    plain = {k: t.double() for k, t in p0.items()}
    pm, pv = ({k: torch.zeros_like(t) for k, t in plain.items()} for _ in range(2))
    send, recv = {}, {}
    for step in range(1, 4):
        tokens = torch.randint(0, V, (B, T + 1), generator=g)
        adv = torch.randn(B, 1, generator=g)
        mask = torch.arange(T) < torch.tensor([T, 5, 0, 9])[:, None]
        w = {k: t.clone().requires_grad_() for k, t in prev.items()}

        def forward(w, tokens):
            return (w["embed"][tokens[:, :-1]] * w["norm"]) @ w["head"].t()

        dt = tokens.cuda()
        logits = forward(w, dt)
        out = crx.policy_loss(logits, dt[:, 1:], adv.cuda(), mask=mask.cuda(), denom=float(mask.sum()))
        out.loss.backward()
        grads = {k: t.grad for k, t in w.items()}
        norm = crx.grad_norm(grads)
        crx.adamw_step(masters, grads, m, v, cur, lr=1e-3, step=step, norm=norm, max_norm=0.1)
        update = crx.encode_update(prev, cur, send)
        crx.apply_update(worker, update, recv)
        for k in cur:
            assert torch.equal(worker[k].view(torch.int16), cur[k].view(torch.int16)), k
            assert torch.equal(cur[k], masters[k].bfloat16()), k
        # the same step from these gradients in 64 bits
        host = {k: t.cpu() for k, t in grads.items()}
        n = ref.norm(host.values())
        near(norm, n, n * ref.NORM)
        for k in plain:
            (plain[k], pm[k], pv[k]), tol = ref.adamw(plain[k], host[k], pm[k], pv[k], lr=1e-3, step=step, b1=0.9, b2=0.999,
                                                      eps=1e-8, wd=0.0, c=ref.coef(n, 0.1))
            near(masters[k], plain[k], step * (tol[0] + 2e-6 * 1e-3))
            plain[k], pm[k], pv[k] = masters[k].double().cpu(), m[k].double().cpu(), v[k].double().cpu()
        prev, cur = cur, prev
    assert send == {k: c for k, (c, _) in recv.items()}
