"""Layer normalisation and the matrix updates under what records or transforms a program: a recorder sees the allocations of a call and not
its kernels, so a traced module would return whatever its memory held; a forward-mode tangent would be dropped.  All are refused."""
import pytest
import torch
from torch.autograd import forward_ad

DEVICES = [pytest.param("cpu"), pytest.param("cuda", marks=pytest.mark.gpu)]


def calls(dev):
    from pixelssl_amd import functional as PF
    w, b = torch.ones(8, device=dev), torch.zeros(8, device=dev)
    z = lambda: torch.zeros(4, 8, device=dev)
    return {"layer_norm": lambda x: PF.layer_norm(x, w, b), "layer_norm_channels": lambda x: PF.layer_norm_channels(x, w, b),
            "orthogonalize": lambda x: PF.orthogonalize(x), "muon_update": lambda x: (PF.muon_update([x], [z()], [z()], lr=0.1), x)[1],
            "adam_update": lambda x: (PF.adam_update([x], [z()], [z()], [z()], lr=0.1), x)[1]}


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("name", ["layer_norm", "layer_norm_channels", "orthogonalize", "muon_update", "adam_update"])
def test_recorders_and_forward_mode_are_refused(name, dev):
    from pixelssl_amd import _lib
    f, x = calls(dev)[name], torch.randn(4, 8, device=dev)
    with pytest.raises(_lib.PixelHipError, match="traced"):
        torch.jit.trace(f, (x,), check_trace=False)
    from torch.fx.experimental.proxy_tensor import make_fx
    with pytest.raises(_lib.PixelHipError, match="traced"):
        make_fx(f)(x)
    with forward_ad.dual_level():
        with pytest.raises(_lib.PixelHipError, match="forward-mode"):
            f(forward_ad.make_dual(x, torch.ones_like(x)))
    with pytest.raises(_lib.PixelHipError, match="torch.func"):
        torch.func.vmap(f)(x[None])
    with pytest.raises(_lib.PixelHipError, match="torch.func|traced"):
        torch.func.jvp(f, (x,), (torch.ones_like(x),))


@pytest.mark.gpu
def test_tangents_of_parameters_and_what_still_runs():
    from pixelssl_amd import _lib, functional as PF
    x, w = torch.randn(4, 8, device="cuda"), torch.ones(8, device="cuda")
    with forward_ad.dual_level():
        with pytest.raises(_lib.PixelHipError, match="forward-mode"):
            PF.layer_norm(x, forward_ad.make_dual(w, torch.ones_like(w)))
        with pytest.raises(_lib.PixelHipError, match="forward-mode"):
            PF.layer_norm(x, w, forward_ad.make_dual(w, torch.ones_like(w)))
        inside = PF.layer_norm(x, w)                      # no tangent: nothing is lost
    assert torch.equal(inside, PF.layer_norm(x, w))
    with pytest.raises(_lib.PixelHipError, match="traced"):          # with gradients, as a module in training is traced
        torch.jit.trace(lambda t: PF.layer_norm(t, w), (x.requires_grad_(True),), check_trace=False)
