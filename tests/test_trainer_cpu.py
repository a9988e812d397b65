"""The trainer-side operators without a GPU: caller mistakes are refused before anything runs, in
Python and at the C entry points, the gradient's memory is laid out as documented, and the global
norm over two ranks."""

import ctypes
import math
import struct

import pytest
import torch
import torch.multiprocessing as mp

import crukx_sync_b200 as crx
from crukx_sync_b200 import _ext, trainer


@pytest.fixture(scope="module", autouse=True)
def lib():
    from crukx_sync_b200 import build
    build.build()
    return _ext.load()


class OnCuda(torch.Tensor):
    """A CPU tensor that says it is on cuda:0, for the checks that come after that one."""

    is_cuda = True
    device = torch.device("cuda", 0)


def fake(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype).as_subclass(OnCuda)


def test_gradients_that_are_refused():
    ok = fake(4)
    for bad, match in [({"a": torch.zeros(4)}, "CUDA"), ({"a": fake(4, dtype=torch.float64)}, "float32"), ({"a": None}, "NoneType"),
                       ({"a": fake(4, 4).t()[1:]}, "contiguous"), ({"a": torch.zeros(4, 4).to_sparse()}, "contiguous"), ([ok], "dict")]:
        with pytest.raises(ValueError, match=match):
            crx.grad_norm(bad)
        with pytest.raises(ValueError, match=match):
            crx.clip_grads(bad, 1.0)
        with pytest.raises(ValueError, match=match):
            crx.adamw_step(bad, bad, bad, bad, lr=1e-3, step=1)


def test_clip_arguments_that_are_refused():
    g = {"a": fake(4), "b": fake(3)}
    for bad in (0.0, -1.0, math.nan):
        with pytest.raises(ValueError, match="max_norm"):
            crx.clip_grads(g, bad)
    with pytest.raises(ValueError, match="names"):
        crx.clip_grads(g, 1.0, out={"a": fake(4)})
    with pytest.raises(ValueError, match="shape"):
        crx.clip_grads(g, 1.0, out={"a": fake(4), "b": fake(4)})
    with pytest.raises(ValueError, match="type"):
        crx.clip_grads(g, 1.0, out={"a": fake(4), "b": fake(3, dtype=torch.bfloat16)})
    with pytest.raises(ValueError, match="norm"):
        crx.clip_grads(g, 1.0, norm=torch.zeros(()))
    with pytest.raises(ValueError, match="norm"):
        crx.clip_grads(g, 1.0, norm=2.0)


def test_step_arguments_that_are_refused():
    def call(g=None, p=None, m=None, v=None, w=None, **kw):
        d = {"a": fake(4)}
        crx.adamw_step(p or d, g or {"a": fake(4, dtype=torch.bfloat16)}, m or d, v or d, w, **{"lr": 1e-3, "step": 1, **kw})

    for kw, match in [(dict(step=0), "step"), (dict(lr=math.nan), "lr"), (dict(betas=(1.0, 0.9)), "betas"), (dict(betas=(0.9, -0.1)), "betas"),
                      (dict(eps=0.0), "eps"), (dict(weight_decay=math.inf), "weight_decay"), (dict(max_norm=1.0), "max_norm"),
                      (dict(norm=fake(()), max_norm=0.0), "max_norm"), (dict(norm=fake(2)), "norm"), (dict(norm=1.0), "norm"),
                      (dict(step=fake(1)), "step"), (dict(lr=fake((), dtype=torch.float64)), "lr"),
                      (dict(p={"b": fake(4)}), "names"), (dict(m={"a": fake(5)}), "shape"), (dict(v={"a": fake(4, dtype=torch.bfloat16)}), "float32"),
                      (dict(w={"a": fake(4)}), "bfloat16"), (dict(w={"a": fake(4, dtype=torch.float16)}), "bfloat16")]:
        with pytest.raises(ValueError, match=match):
            call(**kw)


def test_loss_arguments_that_are_refused():
    def call(z=None, tok=None, adv=None, **kw):
        crx.policy_loss(fake(2, 3, 8) if z is None else z, fake(2, 3, dtype=torch.int64) if tok is None else tok,
                        fake(2, 1) if adv is None else adv, **kw)

    for kw, match in [(dict(z=torch.zeros(2, 3, 8)), "CUDA"), (dict(z=fake(2, 3, 8, dtype=torch.float64)), "logits"),
                      (dict(z=fake(2, 4, 8)), "tokens"), (dict(z=fake(2, 3, 0)), "tokens"), (dict(z=fake(2, 8, 3).transpose(1, 2)), "contiguous"),
                      (dict(z=fake(1, 2, 3, 8), tok=fake(1, 2, 3, dtype=torch.int64)), "tokens"), (dict(tok=fake(2, 3)), "tokens"),
                      (dict(adv=fake(2)), "advantages"), (dict(adv=fake(3, 3)), "advantages"), (dict(adv=fake(2, 1, dtype=torch.float64)), "advantages"),
                      (dict(old_logp=fake(2, 1)), "old_logp"), (dict(old_logp=fake(2, 3, dtype=torch.bfloat16)), "old_logp"),
                      (dict(ref_logp=fake(3, 2)), "ref_logp"), (dict(mask=fake(2, 3, dtype=torch.int64)), "mask"), (dict(mask=fake(3)), "mask"),
                      (dict(adv=torch.zeros(2, 1)), "one device"), (dict(tok=torch.zeros(2, 3, dtype=torch.int64)), "one device"),
                      (dict(clip=(-0.1, 0.2)), "clip"), (dict(clip=(0.1, math.nan)), "clip"), (dict(temperature=0.0), "temperature"),
                      (dict(temperature=math.inf), "temperature"), (dict(temperature=1e-38), "temperature"), (dict(kl_coef=0.1), "ref_logp"), (dict(kl_coef=math.nan), "kl_coef"), (dict(kl_coef=math.inf, ref_logp=fake(2, 3)), "kl_coef"),
                      (dict(denom=0.0), "denom"), (dict(denom=-1.0), "denom")]:
        with pytest.raises(ValueError, match=match):
            call(**kw)


@pytest.mark.parametrize("max_norm", [1e-46, 1e-300])
def test_limits_that_fp32_does_not_hold(max_norm):
    """Not taken as 0, which would mean that nothing is clipped."""
    d = {"a": fake(4)}
    with pytest.raises(ValueError, match="max_norm"):
        crx.clip_grads(d, max_norm)
    with pytest.raises(ValueError, match="max_norm"):
        crx.adamw_step(d, {"a": fake(4)}, d, d, lr=1e-3, step=1, norm=fake(()), max_norm=max_norm)


def test_values_that_are_no_numbers_are_value_errors():
    d, z = {"a": fake(4)}, fake(2, 3, 8)
    words = ["1e-3", None, object(), 1j, [1.0], 10 ** 400]
    for bad in words:
        with pytest.raises(ValueError, match="max_norm"):
            crx.clip_grads(d, bad)
        for name in ("lr", "step", "eps", "weight_decay", "betas", "max_norm"):
            if (name, bad) == ("max_norm", None):
                continue   # (no clipping)
            kw = {"lr": 1e-3, "step": 1, "norm": fake(()), name: (0.9, bad) if name == "betas" else bad}
            with pytest.raises(ValueError, match=name):
                crx.adamw_step(d, {"a": fake(4)}, d, d, **kw)
        for name in ("clip", "kl_coef", "temperature", "denom"):
            if (name, bad) == ("denom", None):
                continue   # (the sum of the mask)
            kw = {"ref_logp": fake(2, 3), name: (bad, 0.2) if name == "clip" else bad}
            with pytest.raises(ValueError, match=name):
                crx.policy_loss(z, fake(2, 3, dtype=torch.int64), fake(2, 1), **kw)
    for bad in (2.5, 1 << 63, -(1 << 63)):
        with pytest.raises(ValueError, match="step"):
            crx.adamw_step(d, {"a": fake(4)}, d, d, lr=1e-3, step=bad)
    for bad in (0.9, None, (0.9,), (0.9, 0.99, 0.999)):
        with pytest.raises(ValueError, match="betas"):
            crx.adamw_step(d, {"a": fake(4)}, d, d, lr=1e-3, step=1, betas=bad)
        with pytest.raises(ValueError, match="clip"):
            crx.policy_loss(z, fake(2, 3, dtype=torch.int64), fake(2, 1), clip=bad)


def test_numbers_of_other_types_are_taken():
    """Integers, numpy's and torch's numbers get as far as the tensors."""
    import numpy as np
    d = {"a": fake(4)}
    for one, half in ((np.int64(1), np.float32(0.5)), (True, np.float64(0.5)), (1, torch.tensor(0.5))):
        with pytest.raises(ValueError, match="these tensors"):
            crx.adamw_step(d, {"a": fake(4)}, d, d, lr=half if not isinstance(half, torch.Tensor) else 1, step=one, betas=(half, half), eps=half,
                           weight_decay=half, norm=fake(()), max_norm=half)
        with pytest.raises(ValueError, match="these tensors"):
            crx.policy_loss(fake(2, 3, 8), fake(2, 3, dtype=torch.int64), fake(2, 1), ref_logp=fake(2, 3), clip=(half, one), kl_coef=half,
                            temperature=half, denom=one)


@pytest.mark.parametrize("quiet", [False, True])
def test_forward_gradients_are_refused(quiet):
    """Without gradients of the backward kind too: no_grad does not stop the forward kind."""
    from torch.autograd import forward_ad
    with forward_ad.dual_level():
        z = forward_ad.make_dual(fake(2, 3, 8), torch.ones(2, 3, 8))
        with pytest.raises(ValueError, match="forward"), torch.set_grad_enabled(not quiet):
            crx.policy_loss(z, fake(2, 3, dtype=torch.int64), fake(2, 1))


def test_gradient_memory_follows_the_logits(lib):
    glue = _ext.glue()
    base = torch.zeros(3, 5, 20, dtype=torch.bfloat16)
    same = [base, base[:, :-1], base[..., :13], base.transpose(0, 1), torch.zeros(301, dtype=torch.bfloat16)[1:].view(3, 5, 20)]
    for z in same:
        g = glue.grad_like(z)
        assert g.shape == z.shape and g.stride() == z.stride() and g.data_ptr() % 16 == z.data_ptr() % 16
    for z in (base[:1, :1].expand(3, 5, 20), torch.zeros(3, 5, 100, dtype=torch.bfloat16)[..., :20], base.as_strided((3, 5, 20), (40, 10, 1))):
        g = glue.grad_like(z)
        assert g.shape == z.shape and g.stride() == (5 * 24, 24, 1)   # rows padded to 16 bytes


def pointers(*values):
    return _ext.CBuf("Q", values)


def test_c_entry_points_refuse(lib):
    err = ctypes.create_string_buffer(512)
    one, n4 = _ext.CBuf("i", [2]), _ext.CBuf("q", [4])
    ws = 1 << 20
    size = lib.crx_grads_workspace(1)
    assert size > 0 and lib.crx_grads_workspace(5000) > size and lib.crx_grads_workspace(-1) == 0
    bad = [(-1, pointers(4096), one, n4, ws, size, 4096), (1, None, one, n4, ws, size, 4096), (1, pointers(0), one, n4, ws, size, 4096),
           (1, pointers(4097), one, n4, ws, size, 4096), (1, pointers(4096), _ext.CBuf("i", [7]), n4, ws, size, 4096),
           (1, pointers(4096), one, _ext.CBuf("q", [-4]), ws, size, 4096), (1, pointers(4096), one, n4, None, size, 4096),
           (1, pointers(4096), one, n4, ws, size - 1, 4096), (1, pointers(4096), one, n4, ws + 4, size, 4096),
           (1, pointers(4096), one, n4, ws, size, None)]
    for a in bad:
        assert lib.crx_grad_norm(*a, None, err, 512) == _ext.CRX_BAD_ARGUMENT and err.value, a

    def clip(g, o, numel, max_norm=1.0):
        k = len(g)
        return lib.crx_clip_grads(k, pointers(*g), pointers(*o), _ext.CBuf("i", [2] * k), _ext.CBuf("q", numel), max_norm, None, ws,
                                  lib.crx_grads_workspace(k), 4096, None, err, 512)

    assert clip([4096], [4096], [4], 0.0) == _ext.CRX_VALUE_ERROR
    assert clip([4096], [0], [4]) == _ext.CRX_BAD_ARGUMENT
    for g, o, numel in [([4096, 4096], [4096, 4096], [4, 4]), ([4096, 4108], [4096, 4108], [4, 4]), ([4096], [4104], [4]),
                        ([4096, 8192], [16384, 4100], [4, 4]), ([4096, 8192], [8192, 4096], [4, 4]),
                        ([4096, 65536, 4200], [4096, 65536, 4200], [1000, 4, 1])]:
        assert clip(g, o, numel) == _ext.CRX_VALUE_ERROR and b"share memory" in err.value, (g, o)

    def step(p=4096, g=8192, m=12288, v=16384, w=20480, beta1=0.9, eps=1e-8, t=1):
        args = struct.pack("5d4qf4x", 1e-3, beta1, 0.99, eps, 0.0, t, 0, 0, 0, 0.0)
        return lib.crx_adamw_step(1, pointers(p), pointers(g), one, pointers(m), pointers(v), pointers(w), n4, args, None, err, 512)

    for kw, status in [(dict(beta1=1.0), 1), (dict(eps=0.0), 1), (dict(t=0), 1), (dict(p=0), 5), (dict(m=12290), 5), (dict(w=20481), 5),
                       (dict(m=4100), 1), (dict(v=8200), 1), (dict(w=4096), 1), (dict(g=16380), 1)]:
        assert step(**kw) == status and err.value, kw

    def loss(batch=1, steps=1, vocab=8, logits=4096, tokens=4096, adv=4096, logp=4096, out=4096, stats=4096, rows=4096, denom=0.0, lo=0.2,
             tau=1.0, dtype=0):
        a = struct.pack("28qd4f4i", batch, steps, vocab, logits, 8, 8, 0, 0, 0, tokens, 1, 1, adv, 1, 1, *[0] * 9, logp, out, stats, rows,
                        denom, lo, 0.2, 0.0, tau, dtype, 1, 0, 0)
        return lib.crx_policy_loss(a, None, err, 512)

    for kw, status in [(dict(batch=-1), 5), (dict(steps=-1), 5), (dict(vocab=0), 5), (dict(batch=1 << 30, steps=1 << 30), 5), (dict(logits=0), 5),
                       (dict(logits=4097), 5), (dict(tokens=0), 5), (dict(adv=0), 5), (dict(logp=0), 5), (dict(out=0), 5), (dict(stats=0), 5),
                       (dict(rows=0), 5), (dict(rows=4104), 5), (dict(dtype=3), 5), (dict(denom=-1.0), 1), (dict(lo=-0.5), 1), (dict(lo=math.nan), 1),
                       (dict(tau=0.0), 1), (dict(tau=math.inf), 1), (dict(tau=1e-38), 1), (dict(vocab=1 << 31), 5)]:
        assert loss(**kw) == status and err.value, kw
    assert lib.crx_policy_loss(None, None, err, 512) == 5 and lib.crx_policy_backward(None, None, 0, None, err, 512) == 5


@pytest.mark.parametrize("kw", [dict(eps=1e-46), dict(lr=1e39), dict(lr=-1e39), dict(weight_decay=1e39)], ids=str)
def test_step_numbers_that_fp32_does_not_hold(lib, kw):
    """An eps that would be 0 and rates that would be infinite, in Python and at the C entry."""
    d = {"a": fake(4)}
    with pytest.raises(ValueError, match=next(iter(kw))):
        crx.adamw_step(d, {"a": fake(4)}, d, d, **{"lr": 1e-3, "step": 1, **kw})
    err = ctypes.create_string_buffer(512)
    args = struct.pack("5d4qf4x", kw.get("lr", 1e-3), 0.9, 0.99, kw.get("eps", 1e-8), kw.get("weight_decay", 0.0), 1, 0, 0, 0, 0.0)
    assert lib.crx_adamw_step(1, pointers(4096), pointers(8192), _ext.CBuf("i", [2]), pointers(12288), pointers(16384), pointers(20480),
                              _ext.CBuf("q", [4]), args, None, err, 512) == _ext.CRX_VALUE_ERROR and err.value


@pytest.fixture
def glue_files(tmp_path, monkeypatch):
    """A build whose torch side is one made-up source and whose compiler copies it."""
    from crukx_sync_b200 import build
    build.build()
    for name in ("GLUE", "GLUE_SRC", "GLUE_BUILT"):
        monkeypatch.setattr(build, name, str(tmp_path / name))
    (tmp_path / "GLUE_SRC").write_text("one")
    monkeypatch.setattr(build, "glue_command", lambda out: ["cp", build.GLUE_SRC, out])
    return build, tmp_path


def test_the_torch_side_is_built_again_for_another_torch(glue_files, monkeypatch):
    build, tmp = glue_files
    build.build()
    assert (tmp / "GLUE").read_text() == "one"
    (tmp / "GLUE").write_text("kept")
    build.build()
    assert (tmp / "GLUE").read_text() == "kept"   # nothing changed
    monkeypatch.setattr(build.importlib.metadata, "version", lambda name: "0.0")
    build.build()
    assert (tmp / "GLUE").read_text() == "one"


@pytest.mark.parametrize("how", ["fails", "no compiler", "no torch"])
def test_a_torch_side_that_cannot_be_built_leaves_the_library(glue_files, monkeypatch, capsys, how):
    """The codec does without it; what was built of an older source is gone."""
    build, tmp = glue_files
    (tmp / "GLUE").write_text("old")

    def no_torch(out):
        raise RuntimeError("torch not found")

    monkeypatch.setattr(build, "glue_command", {"fails": lambda out: ["false"], "no compiler": lambda out: [str(tmp / "none")], "no torch": no_torch}[how])
    assert build.build() == build.LIB
    assert not (tmp / "GLUE").exists() and "_glue.so" in capsys.readouterr().err


def _rank(rank, world, port, queue):
    import os

    import torch.distributed as td
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    td.init_process_group("gloo", rank=rank, world_size=world)
    from crukx_sync_b200 import dist
    trainer.grad_norm = lambda grads: torch.tensor(math.sqrt(sum(float(g.double().square().sum()) for g in grads.values())))
    queue.put((rank, float(dist.grad_norm_global({"a": torch.full((4,), 1.0 + rank)})),
               float(dist.grad_norm_global({"a": torch.full((1,), 3e30 if rank else 4e30)}))))
    td.destroy_process_group()


def test_global_norm_over_two_ranks():
    import socket
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    ctx = mp.get_context("spawn")
    queue = ctx.Queue()
    procs = [ctx.Process(target=_rank, args=(r, 2, port, queue)) for r in range(2)]
    for p in procs:
        p.start()
    got = sorted(queue.get(timeout=120) for _ in procs)
    for p in procs:
        p.join(60)
    for _, small, large in got:
        assert small == pytest.approx(math.sqrt(4 + 16), rel=1e-6) and large == pytest.approx(5e30, rel=1e-6)
