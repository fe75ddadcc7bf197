"""bf16 parameters under the orthogonalised updates: what is computed for them in 32 bits is rounded once, at the end."""
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
from test_muon import muon_exact  # noqa: E402


def strong(shape, seed, strength):
    """six directions of `strength` times the noise"""
    g = torch.Generator().manual_seed(seed)
    rows, cols = shape
    return torch.randn(rows, cols, generator=g) + strength * torch.randn(rows, 6, generator=g) @ torch.randn(6, cols, generator=g)


SHAPES = [(16, 27), (64, 147), (147, 64), (64, 400), (64, 448), (64, 449), (21, 4608), (33, 1000), (100, 300), (256, 1024), (1024, 256), (129, 2305)]


@pytest.mark.gpu
@pytest.mark.parametrize("strength", [0.5, 50.0])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_muon_step_is_the_32_bit_step_rounded_once(shape, strength):
    """the update is formed from an fp32 momentum: a bf16 gradient does not make it a bf16 matrix.  Equal bits with the fp32 step of the same
    values, rounded; and that step against the definition"""
    from pixelssl_amd import functional as PF
    g = (strong(shape, 1, strength) * 1e-3).bfloat16()
    m = strong(shape, 2, strength) * 1e-3
    for p in (torch.zeros(shape), torch.randn(shape, generator=torch.Generator().manual_seed(3)).bfloat16().float() * 0.125):
        want = muon_exact(p, g, m, 0.02, wd=0.1)
        p16, p32, m16, m32 = p.bfloat16().cuda(), p.cuda(), m.cuda(), m.cuda()
        PF.muon_update([p16], [g.cuda()], [m16], lr=0.02, weight_decay=0.1)
        PF.muon_update([p32], [g.float().cuda()], [m32], lr=0.02, weight_decay=0.1)
        off = torch.linalg.vector_norm(p32.double().cpu() - want[0])
        assert off <= want[2] + 8 * 2.0 ** -24 * torch.linalg.vector_norm(want[0]) + 2.0 ** -22 * want[3]
        assert torch.equal(m16, m32) and torch.equal(p16, p32.bfloat16())


def test_the_workspace_serves_both_forms():
    """a bf16 step needs what the fp32 step of the same matrices needs"""
    from pixelssl_amd import _lib
    h = _lib.lib()
    for rows, cols in SHAPES + [(2048, 4608)]:
        items = (_lib.NsItem * 3)(*[(1, 1, 1, rows, cols, 1.0, 0)] * 3)
        assert h.pxl_ns_workspace(1, items, 3) >= h.pxl_ns_workspace(0, items, 3)


@pytest.mark.gpu
@pytest.mark.parametrize("steps", [6, 7, 10])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_steps_past_one_segment_are_the_32_bit_steps_rounded_once(shape, steps):
    """between two segments the iterate is no bf16 matrix any more"""
    from pixelssl_amd import functional as PF
    x = strong(shape, steps, 0.5).bfloat16().cuda()
    assert torch.equal(PF.orthogonalize(x, steps=steps), PF.orthogonalize(x.float(), steps=steps).bfloat16())


def test_workspace_of_the_form_that_runs():
    """bf16 matrices in five steps are one plane: their workspace is that of one, and enough for the call; refusals are 0"""
    import ctypes
    from pixelssl_amd import _lib
    h = _lib.lib()
    coef = (ctypes.c_float * 21)(*((3.4445, -4.7750, 2.0315) * 7))
    items = (_lib.NsItem * 2)((1 << 20, 1 << 26, 0, 512, 4608, 1.0, 0), (1 << 30, 1 << 31, 0, 512, 4608, 1.0, 0))
    five, seven, both = h.pxl_orthogonalize_workspace(1, items, 2, 5, coef), h.pxl_orthogonalize_workspace(1, items, 2, 7, coef), h.pxl_ns_workspace(1, items, 2)
    assert 0 < five < 0.6 * seven and seven <= both
    assert h.pxl_orthogonalize_workspace(0, items, 2, 5, coef) == h.pxl_ns_workspace(0, items, 2)
    assert h.pxl_orthogonalize(1, items, 2, 5, coef, 1e-7, 1, five - 1, None) == -4
    assert h.pxl_orthogonalize_workspace(1, items, 2, 17, coef) == 0 and h.pxl_orthogonalize_workspace(2, items, 2, 5, coef) == 0
    assert h.pxl_orthogonalize_workspace(1, None, 2, 5, coef) == 0 and h.pxl_orthogonalize_workspace(1, items, 2, 5, None) == 0
