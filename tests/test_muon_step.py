"""FusedMuon.step and the list updates as one action: settings as users and checkpoints give them, and refusals that come before anything moved."""
import pytest
import torch
import torch.nn as nn


def settings_of(monkeypatch, **kw):
    """the keyword arguments that one step hands to muon_update (stubbed: no GPU here)"""
    from pixelssl_amd import functional as PF
    from pixelssl_amd.nn.optimizer import FusedMuon
    seen = []
    monkeypatch.setattr(PF, "muon_update", lambda p, g, m, **k: seen.append(k))
    monkeypatch.setattr(PF, "adam_update", lambda *a, **k: None)
    ps = [nn.Parameter(torch.randn(4, 6)), nn.Parameter(torch.randn(3, 5)), nn.Parameter(torch.randn(5))]
    opt = FusedMuon([{"params": ps[:1]}, {"params": ps[1:]}], **kw)
    for p in ps:
        p.grad = torch.randn(p.shape)
    opt.step()
    return opt, seen


@pytest.mark.parametrize("coefs", [[1.5, -0.5, 0.0], (1.5, -0.5, 0.0), [[1.5, -0.5, 0.0]] * 5, ([1.5, -0.5, 0.0],) * 5])
def test_coefficients_in_lists(monkeypatch, coefs):
    opt, seen = settings_of(monkeypatch, ns_coefficients=coefs)
    assert len(seen) == 1 and len(seen[0]["adjust"]) == 2             # both groups' matrices in one call
    flat = torch.tensor(seen[0]["coefficients"]).reshape(-1, 3)
    assert torch.equal(flat, torch.tensor([[1.5, -0.5, 0.0]] * len(flat)))
    opt.param_groups[1]["ns_coefficients"] = [[1.5, -0.5, 0.0]] * 5   # (as an edited or loaded group may hold them)
    opt.step()
    assert opt._step == 2
