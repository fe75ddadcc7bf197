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


@pytest.fixture
def launches(monkeypatch):
    """checks on the host as on a GPU, launches counted and not made"""
    from pixelssl_amd import functional as PF
    seen = []
    monkeypatch.setattr(PF, "_gpu", lambda *a: None)
    monkeypatch.setattr(PF, "_launch", lambda index, fn, *args: seen.append(fn.__name__))
    return seen


def parameters(n_vectors=2, overlap=False):
    flat = torch.zeros(64)
    mats = [nn.Parameter(flat[:24].view(4, 6)), nn.Parameter(flat[20:44].view(4, 6) if overlap else torch.randn(4, 6))]
    vecs = [nn.Parameter(torch.randn(7)) for _ in range(n_vectors)]
    for p in mats + vecs:
        p.grad = torch.randn(p.shape)
    return mats, vecs


@pytest.mark.parametrize("fault", ["overlap", "grow", "steps", "layout", "lr"])
def test_a_refused_step_launches_nothing_and_counts_nothing(launches, fault):
    """groups whose vectors come first, and a matrix group that is refused"""
    from pixelssl_amd.nn.optimizer import FusedMuon
    mats, vecs = parameters(overlap=fault == "overlap")
    opt = FusedMuon([{"params": vecs}, {"params": mats[:1]}, {"params": mats[1:]}], lr=0.02)
    if fault == "grow":
        opt.param_groups[2]["ns_coefficients"] = (30.0, 0.0, 0.0)
    elif fault == "steps":
        opt.param_groups[2]["ns_steps"] = 17
    elif fault == "layout":
        mats[1].data = torch.randn(6, 4).t()
    elif fault == "lr":
        opt.param_groups[2]["lr"] = float("nan")
    for _ in range(2):
        with pytest.raises(Exception, match="twice|grow|steps|lie alike|lr nan"):
            opt.step()
        assert launches == [] and opt._step == 0 and opt._steps_taken == 0 and all("step" not in opt.state[p] for p in vecs)


def test_a_step_launches_everything_once(launches):
    from pixelssl_amd.nn.optimizer import FusedMuon
    mats, vecs = parameters()
    opt = FusedMuon([{"params": vecs[:1] + mats[:1]}, {"params": vecs[1:] + mats[1:], "lr": 0.1}], lr=0.02)
    opt.step()
    assert sorted(launches) == ["pxl_adam_list"] * 2 + ["pxl_muon_step"] * 2 and opt._step == 1
    assert all(opt.state[p]["step"].item() == 1 for p in mats + vecs)


def test_a_refused_update_of_two_types_launches_nothing(launches):
    """the parameters of the first type are fine, those of the second share memory"""
    from pixelssl_amd import _lib, functional as PF
    z = lambda t: torch.zeros(4, 6, dtype=t)
    p16 = [z(torch.bfloat16), None]
    p16[1] = p16[0]
    with pytest.raises(_lib.PixelHipError, match="twice"):
        PF.muon_update([z(torch.float32)] + p16, [z(torch.float32)] + [z(torch.bfloat16) for _ in p16], [z(torch.float32) for _ in range(3)], lr=0.1)
    with pytest.raises(_lib.PixelHipError, match="twice"):
        PF.adam_update([z(torch.float32)] + p16, [z(torch.float32)] + [z(torch.bfloat16) for _ in p16], *[[z(torch.float32) for _ in range(3)] for _ in range(2)], lr=0.1)
    assert launches == []


def test_checks_of_the_c_interface():
    import ctypes
    from pixelssl_amd import _lib
    h = _lib.lib()
    coef = (ctypes.c_float * 15)(*((3.4445, -4.7750, 2.0315) * 5))
    apart = (_lib.NsItem * 2)((1 << 20, 1 << 21, 1 << 22, 8, 16, 1.0, 0), (1 << 23, 1 << 24, 1 << 25, 8, 16, 1.0, 0))
    same = (_lib.NsItem * 2)((1 << 20, 1 << 21, 1 << 22, 8, 16, 1.0, 0), ((1 << 20) + 508, 1 << 24, 1 << 25, 8, 16, 1.0, 0))
    ok = (1e-7, 0.1, 0.9, 0.0)
    assert h.pxl_muon_check(0, apart, 2, 5, coef, *ok) == 0 and h.pxl_muon_check(0, None, 0, 5, coef, *ok) == 0
    assert h.pxl_muon_check(0, same, 2, 5, coef, *ok) == -1 and b"twice" in h.pxl_last_error()
    assert h.pxl_muon_check(0, apart, 2, 17, coef, *ok) == -1 and h.pxl_muon_check(2, apart, 2, 5, coef, *ok) == -1 and h.pxl_muon_check(0, None, 2, 5, coef, *ok) == -1
    assert h.pxl_muon_check(0, apart, 2, 5, None, *ok) == -1 and h.pxl_muon_check(0, apart, 2, 5, coef, 0.0, 0.1, 0.9, 0.0) == -1
    for bad in ((1e-7, float("nan"), 0.9, 0.0), (1e-7, 0.1, 1.0, 0.0), (1e-7, 0.1, 0.9, float("inf"))):
        assert h.pxl_muon_check(0, apart, 2, 5, coef, *bad) == -1
    it = (_lib.AdamItem * 2)((1 << 20, 1 << 21, 1 << 22, 1 << 23, 4), (1 << 24, 1 << 21, 1 << 25, (1 << 23) + 8, 4))
    assert h.pxl_adam_check(0, it, 1, 0.9, 0.99, 1e-8, 1) == 0 and h.pxl_adam_check(0, it, 2, 0.9, 0.99, 1e-8, 1) == -1 and b"twice" in h.pxl_last_error()
    assert h.pxl_adam_check(0, it, 1, 1.0, 0.99, 1e-8, 1) == -1 and h.pxl_adam_check(0, it, 1, 0.9, 0.99, 1e-8, 0) == -1


@pytest.mark.gpu
def test_a_refused_step_moves_no_parameter():
    from pixelssl_amd import _lib
    from pixelssl_amd.nn.optimizer import FusedMuon
    flat = torch.randn(64, device="cuda")
    a, b, v = nn.Parameter(flat[:24].view(4, 6)), nn.Parameter(flat[20:44].view(4, 6)), nn.Parameter(torch.randn(7, device="cuda"))
    c = nn.Parameter(torch.randn(4, 6, device="cuda"))
    for p in (a, b, v, c):
        p.grad = torch.randn(p.shape, device="cuda")
    opt = FusedMuon([{"params": [v]}, {"params": [c], "lr": 0.1}, {"params": [a, b]}], lr=0.02)
    before = [t.detach().clone() for t in (flat, v, c)]
    with pytest.raises(_lib.PixelHipError, match="twice"):
        opt.step()
    assert all(torch.equal(t, o) for t, o in zip((flat, v.detach(), c.detach()), before)) and opt._step == 0
    b.grad = None
    opt.step()
    assert opt._step == 1 and not any(torch.equal(t, o) for t, o in zip((flat, v.detach(), c.detach()), before))


def test_parameters_without_elements(launches):
    """an axis of length 0 is left alone, beside parameters that step"""
    from pixelssl_amd import functional as PF
    from pixelssl_amd.nn.optimizer import FusedMuon
    ps = [nn.Parameter(torch.randn(s)) for s in ((5, 0), (0, 5), (4, 6), (0,), (3,))]
    for p in ps:
        p.grad = torch.randn(p.shape)
    opt = FusedMuon(ps)
    opt.step()
    assert launches == ["pxl_adam_list", "pxl_muon_step"] and opt._step == 1
    assert PF.muon_scale((5, 0)) == PF.muon_scale((0, 5)) == 1.0


def test_a_group_added_later(launches):
    from pixelssl_amd.nn.optimizer import FusedMuon
    mats, vecs = parameters()
    opt = FusedMuon(mats[:1])
    opt.step()
    with pytest.raises(ValueError, match="dense"):
        opt.add_param_group({"params": [nn.Parameter(torch.randn(4, 6).t())]})
    assert len(opt.param_groups) == 1
    opt.add_param_group({"params": mats[1:] + vecs, "lr": 0.1})
    launches.clear()
    opt.step()
    assert launches == ["pxl_adam_list", "pxl_muon_step", "pxl_muon_step"] and opt._foreign[1] == mats[1:] + vecs
    assert set(opt.state_dict()["state"][2]) == {"exp_avg", "exp_avg_sq", "step"}


def test_as_many_workgroups_as_no_grid_holds_are_refused():
    """2^22 matrices of 1 x 449 are 2^25 tiles: with 256 threads each past the 2^32 of a grid"""
    import ctypes
    import numpy as np
    from pixelssl_amd import _lib
    h = _lib.lib()
    n = 1 << 22
    items = np.zeros(n, dtype=np.dtype([("p", "u8"), ("g", "u8"), ("mom", "u8"), ("rows", "i4"), ("cols", "i4"), ("scale", "f4"), ("reserved", "i4")]))
    assert items.itemsize == ctypes.sizeof(_lib.NsItem)
    items["p"], items["g"], items["mom"], items["rows"], items["cols"] = 1, 1, 1, 1, 449
    at = items.ctypes.data_as(ctypes.c_void_p)
    for dtype in (0, 1):
        assert h.pxl_ns_workspace(dtype, at, n) == 0 and b"too many" in h.pxl_last_error()
        assert h.pxl_ns_workspace(dtype, at, n // 4) > 0
    items["cols"] = 300                                  # on one CU each: a workgroup a matrix
    assert h.pxl_ns_workspace(1, at, n) > 0
    items["rows"], items["cols"] = 4096, 4096             # 2^15 tiles are fine, 2^24 are not
    assert h.pxl_ns_workspace(0, at, 8) > 0 and h.pxl_ns_workspace(0, at, 1 << 12) == 0 and b"too many" in h.pxl_last_error()
