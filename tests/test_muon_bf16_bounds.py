"""The bf16 form of orthogonalize under bounds that a lost row, column or factor does not pass.

All steps of a bf16 matrix run as one segment: A = X X', then per step Q = a + b A + c A^2, P <- Q P, A <- Q (Q A); X is one exact plane, every other
matrix a pair of planes, off by h = 2^-22 of an entry, and every product is summed in fp32.  An error E of A at the start of step k reaches
the result as (the divided differences of l -> P_k(l), the product of the q from step k on) * E * (X at step k): in the Frobenius norm
at most  max_ij |P_k[l_i, l_j]| sigma_j(k) |E|_F  (eigenvectors of A on both sides).  With the exact singular values that is a number:
  E_0 = h (2 + sqrt(n / 16) / 4) |A|_F               (A's planes, its sums over n in steps of 16: rounding of random sign)
  E_k = 2 h (|Q|_F max|l q| + max|q| |Q A|_F + |A|_F)  (planes of Q, Q A and A, sums)
and Q's and P's own rounding reaches it as 2 h |Q|_F max(later q) max(earlier q sigma) and 2 h |P|_F max(later q).  The result is rounded once: what an
entry is off beyond half a step of bf16, 2^-8 of it, is the error before that rounding.  1.1: terms of second order, the factor 1 + 2^-8."""
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
from test_muon import COEF, exact, gradient, spectrum  # noqa: E402

H = 2.0 ** -22


def bound(x, steps=5, coef=COEF, eps=1e-7):
    """the error before the last rounding of one matrix x, Frobenius norm"""
    x = x.double()
    n = max(x.shape)
    s = torch.linalg.svdvals(x) / torch.linalg.vector_norm(x).clamp(min=eps)
    m, (a, b, c) = len(s), coef
    norm = lambda v: torch.linalg.vector_norm(v).item()
    S, L, Q = [s], [s * s], []
    for k in range(steps):
        Q.append(a + L[k] * (b + c * L[k]))
        S.append(S[k] * Q[k])
        L.append(S[k + 1] ** 2)
    total = 0.0
    for k in range(steps):
        dA, dP, P = torch.ones(m, m).double(), torch.zeros(m, m).double(), torch.ones(m).double()
        for j in range(k, steps):                  # divided differences of A -> q(A), of the product and of A -> q(A)^2 A
            dQ = (b + c * (L[j][:, None] + L[j][None, :])) * dA
            dP = dQ * P[None, :] + Q[j][:, None] * dP
            P = P * Q[j]
            dA = (Q[j][:, None] + Q[j][None, :]) * dQ * L[j][None, :] + (Q[j] ** 2)[:, None] * dA
        if k == 0:
            E = (2 + (n / 16) ** 0.5 / 4) * norm(L[0])
        else:
            q, l = Q[k - 1], L[k - 1]
            E = 2 * (norm(q) * (l * q).abs().max().item() + q.abs().max().item() * norm(l * q) + norm(L[k]))
        total += H * E * (dP.abs() * S[k][None, :]).max().item()
        before, after = torch.ones(m).double(), torch.ones(m).double()
        for j in range(k):
            before = before * Q[j]
        for j in range(k + 1, steps):
            after = after * Q[j]
        total += 2 * H * after.abs().max().item() * (norm(Q[k]) * (before * s).abs().max().item() + norm(before * Q[k]) * s.max().item())
    return 1.1 * total


def beyond_rounding(got, want):
    return ((got.double().cpu() - want).abs() - 2.0 ** -8 * want.abs()).clamp(min=0)


def check(got, x, steps=5, what=""):
    rows = lambda t: t.reshape(-1, *t.shape[-2:])
    for g, m in zip(rows(got), rows(x)):
        want, lim = exact(m, steps), bound(m, steps)
        off = torch.linalg.vector_norm(beyond_rounding(g, want)).item()
        assert off <= lim, "%s: %.3g at a bound of %.3g" % (what, off, lim)
        least = min(torch.linalg.vector_norm(want, dim=d).min().item() for d in (0, 1))
        assert 2 * lim < least, "%s: the bound %.3g would let a line of %.3g go" % (what, lim, least)


SHAPES = [(1, 1), (1, 64), (70, 1), (3, 5), (31, 33), (2, 32, 32), (64, 147), (147, 64), (129, 257), (3, 200, 640), (300, 128), (21, 4608), (2304, 96), (65, 65),
          (64, 384), (384, 63), (64, 385), (33, 256), (257, 64), (449, 64), (2, 32, 417), (48, 40007), (40007, 21), (1024, 256), (2, 513, 768)]


@pytest.mark.gpu
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_shapes(shape):
    from pixelssl_amd import functional as PF
    x = gradient(shape, sum(shape), torch.bfloat16)
    check(PF.orthogonalize(x.cuda()), x, what=str(shape))


@pytest.mark.gpu
@pytest.mark.parametrize("steps", [1, 2, 3, 4, 5])
def test_steps(steps):
    from pixelssl_amd import functional as PF
    x = gradient((96, 224), steps, torch.bfloat16)
    check(PF.orthogonalize(x.cuda(), steps=steps), x, steps, "%d steps" % steps)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["equal", "harmonic", "square", "six_decades", "one_strong", "half_rank"])
def test_spectra(kind):
    from pixelssl_amd import functional as PF
    for m, n in ((60, 130), (96, 160), (160, 160)):
        x = spectrum(m, n, kind, 3).to(torch.bfloat16)
        for y in (x, x.t().contiguous()):
            check(PF.orthogonalize(y.cuda()), y, what="%s %s" % (kind, tuple(y.shape)))


def test_the_bound_refuses_what_is_wrong():
    """an exact result rounded to bf16 passes; one without its last row or column, 2 % too large, or with a small block turned does not"""
    for shape in [(64, 147), (257, 64), (64, 385), (33, 256), (48, 4000), (300, 128)]:
        x = gradient(shape, sum(shape), torch.bfloat16)
        right = exact(x).bfloat16()
        check(right, x, what=str(shape))
        row, col, block = right.clone(), right.clone(), right.clone()
        row[-1], col[:, -1] = 0, 0
        block[-16:, -16:] = right[-16:, -16:].t() if shape[0] > 16 else 0
        for wrong in (row, col, block, right * 1.02):
            with pytest.raises(AssertionError, match="at a bound of"):
                check(wrong, x, what=str(shape))
