"""FusedMuon on two ranks (gloo, CPU): the gradients it steps with are the mean over the ranks, each in its parameter's own type, and the
replicas stay equal.  The kernels are replaced by the formulas in torch; the exchange is what is tested."""
import os
import sys

import torch
import torch.multiprocessing as mp

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
from test_dist_gloo import _free_port  # noqa: E402
from test_muon import exact  # noqa: E402

HERE = os.path.dirname(os.path.abspath(__file__))


def _plain_muon(params, grads, momenta, lr, momentum, nesterov, weight_decay, steps, coefficients, eps, adjust):
    for p, g, m, s in zip(params, grads, momenta, adjust):
        m.mul_(momentum).add_(g.float() * (1 - momentum))
        u = g.float() * (1 - momentum) + m * momentum if nesterov else m
        p.copy_(p * (1 - lr * weight_decay) - lr * s * exact(u.flatten(1), steps, coefficients, eps).view(p.shape).float())


def _plain_adam(params, grads, ms, vs, lr, betas, eps, step):
    for p, g, m, v in zip(params, grads, ms, vs):
        m.lerp_(g.float(), 1 - betas[0])
        v.mul_(betas[1]).addcmul_(g.float(), g.float(), value=1 - betas[1])
        p.sub_(lr / (1 - betas[0] ** step) * m / ((v / (1 - betas[1] ** step)).sqrt() + eps))


def _value(rank, k, n, dtype):
    """gradients with more bits than bf16 holds, another one on each rank"""
    return (1 + 2.0 ** -12 * (k + 1 + 2 * rank) + torch.arange(n) * 2.0 ** -16).to(dtype)


def _worker(rank, world, port, q):
    import torch.distributed as dist
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port), RANK=str(rank), WORLD_SIZE=str(world), LOCAL_RANK=str(rank), PXL_FORCE_DEVICE="cpu")
    from pixelssl_amd import dist as pdist, functional as PF
    from pixelssl_amd.nn.optimizer import FusedMuon, FusedSGD
    pdist.init_from_env(backend="gloo")
    PF.muon_update, PF.adam_update = _plain_muon, _plain_adam
    torch.manual_seed(0)
    shapes = [((6, 4), torch.bfloat16), ((5,), torch.float32), ((3, 4), torch.float32), ((4,), torch.float32), ((2, 3), torch.bfloat16)]
    same = []
    for make in (lambda ps: FusedMuon([dict(params=ps[:3]), dict(params=ps[3:])], lr=0.02), lambda ps: FusedSGD([dict(params=ps)], lr=0.5)):
        ps = [torch.nn.Parameter(torch.randn(s).to(t)) for s, t in shapes]
        opt = make(ps)
        for k, p in enumerate(ps):
            if k < 3 or (k == 3 and rank == 0):              # the fourth only on one rank, the last one on none
                p.grad = _value(rank, k, p.numel(), p.dtype).view_as(p)
        opt.step()
        ok = ps[4].grad is None
        for k, p in enumerate(ps[:4]):
            each = [_value(r, k, p.numel(), p.dtype) if k < 3 or r == 0 else torch.zeros(p.numel(), dtype=p.dtype) for r in range(world)]
            ok = ok and p.grad.dtype == p.dtype and torch.equal(p.grad.reshape(-1), ((each[0] + each[1]) * 0.5))
        flat = torch.cat([p.detach().reshape(-1).float() for p in ps])
        both = [torch.zeros_like(flat) for _ in range(world)]
        dist.all_gather(both, flat)
        same.append((bool(ok), bool(torch.equal(*both)), bool(torch.isfinite(flat).all())))
    q.put((rank, same))
    dist.barrier()
    dist.destroy_process_group()


def test_two_ranks_average_each_gradient_in_its_own_type():
    ctx = mp.get_context("spawn")
    q = ctx.Queue()
    port = _free_port()
    procs = [ctx.Process(target=_worker, args=(r, 2, port, q)) for r in range(2)]
    for p in procs:
        p.start()
    res = [q.get(timeout=120) for _ in procs]
    for p in procs:
        p.join(timeout=60)
        assert p.exitcode == 0
    assert all(all(x) for _, s in res for x in s), res
