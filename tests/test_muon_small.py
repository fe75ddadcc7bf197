"""orthogonalize of small fp32 matrices is as exact as the formula in 32 bits as written.

Both make the same roundings of the same quantities (A = X X', its square, the product with X, one each a step, sums of at most 128 terms),
independent and of random sign: the Frobenius norm of 256 and more of them differs by a few per cent from run to run, the order of a sum (one after
the other or in blocks) changes its share by less than 1.5.  So over six matrices the error is at most 1.5 times the plain form's, both against the
definition in 64 bits; single rows and columns, of few errors, 4 times that.  (Planes of 22 bits were at 1.4 to 1.9 times here.)"""
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
from test_muon import COEF, exact, gradient  # noqa: E402


def plain(x, steps=5, coef=COEF):
    tall = x.shape[-2] > x.shape[-1]
    x = x.float().mT.contiguous() if tall else x.float()
    x = x / x.square().sum((-2, -1), keepdim=True).sqrt()
    a, b, c = coef
    for _ in range(steps):
        s = x @ x.mT.contiguous()
        x = a * x + (b * s + c * (s @ s)) @ x
    return x.mT if tall else x


def off(got, want):
    return (torch.linalg.vector_norm(got.double().cpu() - want) / torch.linalg.vector_norm(want)).item()


SHAPES = [(16, 16), (20, 24), (24, 20), (30, 30), (32, 32), (33, 33), (40, 40), (48, 48), (64, 64), (50, 60), (64, 33), (94, 22), (22, 94), (32, 128), (128, 32),
          (1, 100), (17, 1)]


@pytest.mark.gpu
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_as_exact_as_32_bits(shape):
    from pixelssl_amd import functional as PF
    x = gradient((6,) + shape, sum(shape), rank=6)
    want = exact(x)
    mine, theirs = off(PF.orthogonalize(x.cuda()), want), off(plain(x), want)
    assert mine <= (1.5 if min(shape) > 1 else 4) * max(theirs, 2.0 ** -24), "%.2g, the plain form %.2g" % (mine, theirs)


EDGES = [(1, 1), (1, 2), (3, 1), (31, 64), (33, 64), (64, 33), (1, 128), (128, 1), (1, 129), (129, 1), (32, 129), (1, 448), (447, 3), (5, 449), (33, 65), (65, 33), (64, 65)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("shape", EDGES, ids=lambda s: "x".join(map(str, s)))
def test_edges_of_the_forms(shape, dtype):
    """sizes on both sides of where one form ends, alone and three of them, nothing around the result touched; a Muon step of the same"""
    from pixelssl_amd import functional as PF
    from test_muon import close, make, muon_close, muon_exact
    x = gradient((3,) + shape, sum(shape), dtype)
    got = PF.orthogonalize(x.cuda())
    close(got, exact(x), dtype, what=str(shape))
    assert torch.equal(got[1], PF.orthogonalize(x[1].cuda()))
    p, g, m = make(shape, 5)
    want = muon_exact(p, g, m, 0.02, wd=0.1)
    n = p.numel()
    flat = torch.full((n + 256,), 7.0, device="cuda")
    view = flat[128:128 + n].view(shape)
    view.copy_(p)
    PF.muon_update([view], [g], [m], lr=0.02, weight_decay=0.1)
    muon_close(view, m, want, torch.float32, str(shape))
    assert (flat[:128] == 7).all() and (flat[128 + n:] == 7).all()


@pytest.mark.gpu
def test_many_small_matrices_of_every_form():
    """one call over all the forms, more matrices than travel in the arguments of a launch; steps other than five"""
    from pixelssl_amd import functional as PF
    from test_muon import make, muon_close, muon_exact
    shapes = [(64, 64), (32, 128), (20, 300), (64, 147), (40, 30), (21, 1000), (100, 90)] * 8
    trip = [make(s, k) for k, s in enumerate(shapes)]
    for steps in (1, 3, 7):
        now = [[t.clone() for t in tr] for tr in trip]
        want = [muon_exact(*tr, 0.02, steps=steps) for tr in now]
        PF.muon_update(*zip(*now), lr=0.02, steps=steps)
        for (p, _, m), w, s in zip(now, want, shapes):
            muon_close(p, m, w, torch.float32, "%s, %d steps" % (s, steps))
