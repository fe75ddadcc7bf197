"""nn.optimizer.FusedMuon: the orthogonalised update on engine and foreign parameters, beside layer normalisation, through the plugin
API, against the formulas in 64 bits (bounds: test_muon.py); functional.adam_update against torch.optim.Adam."""
import argparse
import copy
import os
import sys

import pytest
import torch
import torch.nn as nn
import torch.nn.functional as F

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
for _p in (os.path.join(ROOT, "oracle"), os.path.dirname(os.path.abspath(__file__))):
    if _p not in sys.path:
        sys.path.insert(0, _p)
from test_muon import muon_close, muon_exact  # noqa: E402

DEV = "cuda"


def adam_exact(p, g, m, v, lr, betas, eps, step):
    p, g, m, v = (t.double().cpu() for t in (p, g, m, v))
    m = betas[0] * m + (1 - betas[0]) * g
    v = betas[1] * v + (1 - betas[1]) * g * g
    return p - lr / (1 - betas[0] ** step) * m / ((v / (1 - betas[1] ** step)).sqrt() + eps), m, v


def adam_close(p, want, before, lr, half=2.0 ** -24):
    """a dozen fp32 roundings of the step, which is at most a few lr, and one of the parameter"""
    lim = 16 * 2.0 ** -24 * (want[0] - before.double().cpu()).abs() + 2 * (half + 2.0 ** -24) * want[0].abs() + 1e-37
    assert ((p.double().cpu() - want[0]).abs() <= lim).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_adam_update(dtype):
    """more tensors than one launch takes, from one element up, over three steps"""
    from pixelssl_amd import functional as PF
    g = torch.Generator().manual_seed(1)
    shapes = [(1 + 37 * k % 700,) for k in range(90)] + [(12000,), (5, 7), (4, 3, 2, 2), (0,)]
    ps = [torch.randn(s, generator=g).to(dtype).cuda() for s in shapes]
    ms, vs = [torch.zeros(s, device="cuda") for s in shapes], [torch.zeros(s, device="cuda") for s in shapes]
    for step in range(1, 4):
        gs = [torch.randn(s, generator=g).to(dtype).cuda() for s in shapes]
        before = [p.clone() for p in ps]
        want = [adam_exact(p, gr, m, v, 1e-3, (0.9, 0.99), 1e-8, step) for p, gr, m, v in zip(ps, gs, ms, vs)]
        PF.adam_update(ps, gs, ms, vs, lr=1e-3, betas=(0.9, 0.99), eps=1e-8, step=step)
        for p, m, v, w, b in zip(ps, ms, vs, want, before):
            adam_close(p, w, b, 1e-3, 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -24)
            assert ((m.double().cpu() - w[1]).abs() <= 4 * 2.0 ** -24 * (w[1].abs() + 1)).all()
            assert ((v.double().cpu() - w[2]).abs() <= 4 * 2.0 ** -24 * (w[2].abs() + 1e-3)).all()


def snapshot(opt):
    """(parameter, its state tensors) before a step, by parameter"""
    out = {"lr": [g["lr"] for g in opt.param_groups]}           # (a scheduler moves on right after the step)
    for p in opt._param_list():
        ref = getattr(p, "_pxl_flat", None)
        if ref is None:
            st = [opt.state[p].get(k) if p in opt.state else None for k, _ in opt._keys_of(p)]
            st = [torch.zeros_like(p, dtype=torch.float32) if t is None else t.clone() for t in st]
        else:
            from pixelssl_amd.nn.optimizer import _flat_view
            st = [_flat_view(ref[0], getattr(ref[0], a), p).clone() for _, a in opt._keys_of(p)]
        out[id(p)] = (p.detach().clone(), st)
    return out


def verify_step(opt, before, grads):
    for lr, group in zip(before["lr"], opt.param_groups):
        for p in group["params"]:
            old, st = before[id(p)]
            g = grads.get(id(p))
            if g is None:
                assert torch.equal(p.detach(), old)
                continue
            ref = getattr(p, "_pxl_flat", None)
            if len(st) == 1:
                want = muon_exact(old.contiguous(), g.contiguous(), st[0].contiguous(), lr, group["momentum"], group["nesterov"],
                                  group["weight_decay"])
                if ref is None:
                    new = opt.state[p]["momentum_buffer"]
                else:
                    from pixelssl_amd.nn.optimizer import _flat_view
                    new = _flat_view(ref[0], ref[0].momentum, p)
                # gradients of any scale here: the momentum's own relative bound, its parts at least as large as 2^-20 of the largest
                lim = 4 * 2.0 ** -24 * torch.linalg.vector_norm(st[0].double().cpu().abs() + g.double().cpu().abs()).item()
                assert torch.linalg.vector_norm(new.double().cpu() - want[1]).item() <= lim, tuple(p.shape)
                off = torch.linalg.vector_norm(p.detach().double().cpu() - want[0]).item()
                lim = (want[2] + 8 * 2.0 ** -24 * torch.linalg.vector_norm(want[0]) + 2.0 ** -22 * want[3]).item()
                assert off <= lim, tuple(p.shape)
            else:
                want = adam_exact(old, g, st[0], st[1], lr * group["vector_scale"], group["betas"], group["eps"], opt._step)
                adam_close(p.detach(), want, old, lr)


@pytest.mark.gpu
def test_on_an_engine_model():
    """every convolution (21-class head and 7 x 7 stem in padded slots among them) and every vector of a small DeepLab, two steps; the
    padding of the slots stays zero; the networks' packed weights follow"""
    from pixelssl_amd.engine import DeepLabV2Core
    from pixelssl_amd.nn.optimizer import FusedMuon
    core = DeepLabV2Core(backbone=(1, 1, 1, 1), device=DEV, engine_dtype=torch.float32)
    params = list(core.parameters())
    opt = FusedMuon([{"params": params[:20]}, {"params": params[20:], "lr": 0.05, "nesterov": False, "weight_decay": 0.1}], lr=0.02)
    store = core.flat
    mask = torch.ones_like(store.params, dtype=torch.bool)
    for p in params:
        from pixelssl_amd.nn.optimizer import _flat_view
        _flat_view(store, mask, p).fill_(False)
    g = torch.Generator().manual_seed(3)
    version = store.version()
    for _ in range(2):
        grads = {}
        for p in params:
            gr = (torch.randn(p.shape, generator=g) * 0.01).to(DEV)
            p.grad.copy_(gr)
            grads[id(p)] = gr
        before = snapshot(opt)
        opt.step()
        verify_step(opt, before, grads)
    assert store.version() != version
    assert not store.params[mask].any() and not store.momentum[mask].any()
    opt.zero_grad()
    assert not store.grads.any()


class _NormedSegModel(nn.Module):
    """a plugin's torch task model: convolutions and linear layers between layer norms, both layouts"""

    def __init__(self, args=None):
        super().__init__()
        import pixelssl_amd as P
        g = torch.Generator().manual_seed(17)
        self.stem = nn.Conv2d(3, 24, 3, padding=1)
        self.norm1 = P.nn.LayerNorm(24, channels_first=True)
        self.mix = nn.Conv2d(24, 40, 1)
        self.norm2 = P.nn.LayerNorm(40)
        self.proj = nn.Linear(40, 21)
        with torch.no_grad():
            for p in self.parameters():
                p.copy_(torch.randn(p.shape, generator=g) * 0.2)
        self.param_groups = [{"params": [p for n, p in self.named_parameters() if not n.startswith("proj")], "lr": args.lr},
                             {"params": list(self.proj.parameters()), "lr": args.lr * 10, "muon": False}]

    def logits(self, x, norm_channels, norm_rows):
        h = F.gelu(norm_channels(self.stem(x), self.norm1))
        h = norm_rows(self.mix(h).movedim(1, -1), self.norm2)
        return self.proj(h).movedim(-1, 1).contiguous()

    def forward(self, inp):
        pred = self.logits(inp[0], lambda t, m: m(t), lambda t, m: m(t))
        return {"pred": (pred,), "activated_pred": (F.softmax(pred, dim=1),)}, {}


def _plain_norm(axis):
    def norm(t, m):
        shape = [1] * t.dim()
        shape[axis] = -1
        c = t - t.mean(axis, keepdim=True)
        return c / (c.square().mean(axis, keepdim=True) + m.eps).sqrt() * m.weight.view(shape) + m.bias.view(shape)
    return norm


@pytest.mark.gpu
def test_layer_norm_and_muon_train_a_plugin_model_through_mean_teacher():
    """ssl_mt iterations on a torch task model of layer norms and matrices with the `muon` factory: its gradients against the same
    network in 64 bits with plain norms, its updates against the formulas on those gradients, the checkpoint round trip"""
    import torch_oracle as TO
    import pixelssl_amd as P
    from pixelssl_amd.nn import optimizer as popt, lrer as plr
    a = argparse.Namespace(lr=0.01, momentum=-1, weight_decay=1e-3, dampening=-1, nesterov=True, beta1=-1, beta2=-1, eps=-1, power=-1,
                           last_epoch=-1, epochs=1, iters_per_epoch=8, ignore_index=255, labeled_batch_size=2, unlabeled_batch_size=2,
                           batch_size=4, ignore_unlabeled=False, is_epoch_lrer=False, log_freq=1000, task="sseg", gpus=1,
                           gaussian_noise_std=None, cons_for_labeled=False, cons_scale=1.0, cons_rampup_epochs=3, ema_decay=0.99, num_classes=21)
    algo = P.ssl_algorithm.ssl_mt.ssl_mt(a, {"model": lambda args: _NormedSegModel(args).to(DEV)}, {"model": popt.muon(a)},
                                         {"model": plr.polynomiallr(a)}, {"model": P.sseg.criterion.sseg_criterion()}, None)
    assert type(algo.s_optimizer) is popt.FusedMuon and a.momentum == 0.95 and a.beta2 == 0.999
    algo.s_model.train(), algo.t_model.train()
    model, opt = algo.s_model.module, algo.s_optimizer
    for it in range(3):
        x, gt = TO.synthetic_batch(4, 33, 2, seed=70 + it, block=16)
        x, gt = x.to(DEV), gt.to(DEV)
        before = snapshot(opt)
        ref = copy.deepcopy(model).double().cpu()
        teacher = copy.deepcopy(algo.t_model.module).double().cpu()
        out, _, _ = algo.train_step((x,), (gt,), it, 6)
        grads = {id(p): p.grad.clone() for p in model.parameters()}
        verify_step(opt, before, grads)
        xd, lab = x.double().cpu(), gt[:2, 0].long().cpu()
        pred = ref.logits(xd, _plain_norm(1), _plain_norm(-1))
        with torch.no_grad():
            t_pred = teacher.logits(xd, _plain_norm(1), _plain_norm(-1))
        task = (F.cross_entropy(pred[:2], lab, ignore_index=255, reduction="none").sum((1, 2)) / (33 * 33)).mean()
        cons = P.nn.func.sigmoid_rampup(it, 6) * F.mse_loss(pred[2:], t_pred[2:])
        (task + cons).backward()
        assert abs(out["s_task_loss"].item() - task.item()) < 2e-5 * abs(task.item())
        for (n, p), r in zip(model.named_parameters(), ref.parameters()):
            err = (grads[id(p)].double().cpu() - r.grad).norm() / r.grad.norm()
            assert err < 1e-4, (it, n, err.item())           # fp32 convolutions and sums over 4 x 33 x 33 positions
    # a checkpoint into a new optimizer: the next step has the same bits
    twin = _NormedSegModel(a).to(DEV)
    twin.load_state_dict(model.state_dict())
    opt2 = popt.FusedMuon(twin.param_groups, lr=0.01)
    opt2.load_state_dict(copy.deepcopy(opt.state_dict()))
    g = torch.Generator().manual_seed(5)
    for p, q in zip(model.parameters(), twin.parameters()):
        p.grad = torch.randn(p.shape, generator=g).to(DEV)
        q.grad = p.grad.clone()
    opt.step(), opt2.step()
    assert all(torch.equal(p, q) for p, q in zip(model.parameters(), twin.parameters()))


@pytest.mark.gpu
def test_ssl_null_trains_an_engine_model_with_muon():
    """SupOnly on a small DeepLab (bf16 engine, the default path: no fused SGD update applies) with the `muon` factory: the update of
    every parameter from the gradients of its own backward"""
    import torch_oracle as TO
    from pixelssl_amd.engine import DeepLabV2Core
    from pixelssl_amd import functional as PF
    from pixelssl_amd.nn.optimizer import FusedMuon
    core = DeepLabV2Core(backbone=(1, 1, 1, 1), device=DEV, engine_dtype=torch.bfloat16)
    core.load_state_dict({k: v for k, v in core.state_dict().items()})
    core.train()
    opt = FusedMuon(core.parameters(), lr=0.005)
    x, gt = TO.synthetic_batch(2, 65, 2, seed=4, block=16)
    for _ in range(2):
        opt.zero_grad()
        logits, _, _ = core(x.to(DEV))
        PF.cross_entropy_per_sample(logits, gt.to(DEV), 255).mean().backward()
        grads = {id(p): p.grad.clone() for p in core.parameters()}
        before = snapshot(opt)
        opt.step()
        verify_step(opt, before, grads)
    assert all(torch.isfinite(p).all() for p in core.parameters())


@pytest.mark.gpu
def test_parameters_without_a_gradient_and_other_layouts():
    from pixelssl_amd.nn.optimizer import FusedMuon
    g = torch.Generator().manual_seed(6)
    ps = [nn.Parameter(t.to(DEV)) for t in (torch.randn(12, 8, 3, 3, generator=g).contiguous(memory_format=torch.channels_last),
                                            torch.randn(30, 20, generator=g), torch.randn(20, generator=g), torch.randn(9, 5, generator=g))]
    opt = FusedMuon([{"params": ps[:3]}, {"params": ps[3:], "muon": False}], lr=0.02)
    for it in range(3):
        for k, p in enumerate(ps):
            p.grad = torch.randn(p.shape, generator=g).to(DEV) if k != 1 or it == 2 else None
        before = snapshot(opt)
        opt.step()
        verify_step(opt, before, {id(p): p.grad for p in ps if p.grad is not None})
    sd = copy.deepcopy(opt.state_dict())
    assert set(sd["state"][0]) == {"momentum_buffer", "step"} and set(sd["state"][3]) == {"exp_avg", "exp_avg_sq", "step"}
    sd["state"][0]["momentum_buffer"] = sd["state"][0]["momentum_buffer"].contiguous()      # saved by something with another layout
    opt.load_state_dict(sd)
    before = snapshot(opt)
    opt.step()
    verify_step(opt, before, {id(p): p.grad for p in ps})


@pytest.mark.gpu
def test_a_captured_step_is_refused():
    from pixelssl_amd import _lib
    from pixelssl_amd.nn.optimizer import FusedMuon
    p = nn.Parameter(torch.randn(8, 8, device=DEV))
    opt = FusedMuon([p], lr=0.02)
    p.grad = torch.randn(8, 8, device=DEV)
    opt.step()
    before = p.detach().clone()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s):
        g.capture_begin()
        with pytest.raises(_lib.PixelHipError, match="captured"):
            opt.step()
        torch.zeros(1, device=DEV)
        g.capture_end()
    torch.cuda.synchronize()
    assert torch.equal(before, p.detach()) and opt._step == 1


def test_refusals():
    from pixelssl_amd import _lib, functional as PF
    from pixelssl_amd.nn import optimizer as popt
    p = nn.Parameter(torch.randn(4, 6))
    for kw in (dict(momentum=1.0), dict(betas=(0.9, 1.0)), dict(eps=0.0), dict(ns_eps=-1.0), dict(adjust_lr="rms"), dict(ns_steps=0),
               dict(ns_coefficients=(1.0, 2.0))):
        with pytest.raises(ValueError):
            popt.FusedMuon([p], **kw)
    with pytest.raises(ValueError, match="dense"):
        popt.FusedMuon([nn.Parameter(torch.randn(4, 6).t())])
    with pytest.raises(ValueError, match="float32 or bfloat16"):
        popt.FusedMuon([nn.Parameter(torch.randn(4, 6).double())])
    opt = popt.FusedMuon([p])
    p.grad = torch.randn(4, 6)
    with pytest.raises(_lib.PixelHipError, match="GPU only"):
        opt.step()
    v = torch.zeros(3)
    with pytest.raises(_lib.PixelHipError, match="GPU only"):
        PF.adam_update([v], [v], [v], [v], lr=0.1)
    with pytest.raises(ValueError, match="step"):
        PF.adam_update([v], [v], [v], [v], lr=0.1, step=0)
    with pytest.raises(ValueError, match="shapes"):
        PF.adam_update([v], [v[:2]], [v], [v], lr=0.1)
    with pytest.raises(ValueError, match="moments"):
        PF.adam_update([v, v], [v, v], [v], [v, v], lr=0.1)
    with pytest.raises(ValueError, match="moments float32"):
        PF.adam_update([v], [v], [v.double()], [v], lr=0.1)
    assert "muon" not in popt.VALID_OPTIMIZER
    h = _lib.lib()
    it = (_lib.AdamItem * 1)((1, 1, None, 1, 4))
    assert h.pxl_adam_list(0, it, 1, 0.1, 0.9, 0.99, 1e-8, 1, None) == -1 and b"item 0" in h.pxl_last_error()
    assert h.pxl_adam_list(5, it, 1, 0.1, 0.9, 0.99, 1e-8, 1, None) == -1 and h.pxl_adam_list(0, None, 0, 0.1, 0.9, 0.99, 1e-8, 1, None) == 0


def test_factory_defaults_and_formulas():
    from pixelssl_amd.nn import optimizer as popt
    a = argparse.Namespace(lr=-1, momentum=-1, weight_decay=-1, nesterov=True, beta1=-1, beta2=-1, eps=-1)
    opt = popt.muon(a)([{"params": [nn.Parameter(torch.zeros(3, 2))], "lr": 0.3}, {"params": [nn.Parameter(torch.zeros(3))]}])
    assert (a.lr, a.momentum, a.weight_decay, a.beta1, a.beta2, a.eps) == (0.02, 0.95, 0.0, 0.9, 0.999, 1e-8)
    assert opt.param_groups[0]["lr"] == 0.3 and opt.param_groups[1]["lr"] == 0.02 and opt.param_groups[0]["nesterov"] is True
    # the formula of the oracle against torch's own Adam
    g = torch.Generator().manual_seed(1)
    p = nn.Parameter(torch.randn(7, generator=g, dtype=torch.float64))
    ref = torch.optim.Adam([p], lr=0.1, betas=(0.8, 0.9))
    q, m, v = p.detach().clone(), torch.zeros(7, dtype=torch.float64), torch.zeros(7, dtype=torch.float64)
    for step in range(1, 4):
        p.grad = torch.randn(7, generator=g, dtype=torch.float64)
        ref.step()
        q, m, v = adam_exact(q, p.grad, m, v, 0.1, (0.8, 0.9), 1e-8, step)
        assert torch.allclose(q, p.detach(), rtol=1e-12)


@pytest.mark.gpu
def test_adam_update_refuses_memory_that_appears_twice():
    """the same vector, or a piece of it, twice in a call: two of its workgroups would race"""
    from pixelssl_amd import _lib, functional as PF
    new = lambda: torch.ones(40, device="cuda")
    p, q = new(), new()
    a, b = p[:24], p[20:]
    for lists in (([p, p], [new(), new()], [new(), new()], [new(), new()]), ([p], [p], [new()], [new()]), ([a, b], [new()[:24], new()[:20]], [new()[:24], new()[:20]],
                  [new()[:24], new()[:20]]), ([p, new()], [q, new()], [new(), q], [new(), new()])):
        with pytest.raises(_lib.PixelHipError, match="twice"):
            PF.adam_update(*lists, lr=0.1)
    m = new()
    with pytest.raises(_lib.PixelHipError, match="twice"):
        PF.adam_update([p], [q], [m], [m], lr=0.1)
    assert torch.equal(p, new()) and torch.equal(q, new()) and torch.equal(m, new())
    PF.adam_update([p, new()], [q, q], [new(), new()], [new(), new()], lr=0.1)          # (one gradient of two parameters is only read)
