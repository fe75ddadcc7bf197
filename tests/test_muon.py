"""Orthogonalised updates (csrc/muon.hip; functional.orthogonalize, functional.muon_update) against the definitions in 64 bits.

Tolerances (Frobenius norms, h = 2^-22 a plane pair's rounding): a run of `steps` steps makes at most 3 products a step plus two a segment,
each relatively exact to h (planes) and 2^-24 sqrt(K) < h for every K here (fp32 sums of random sign); within a segment an error of A grows at
most by `grow` (the limit that ends segments: 16 with 32-bit results, 2^15 with bf16 results; the default coefficients reach 11.9 and
19800), and the entry error of X0 (h |X0| = h) at most by prod q(0) = a^steps on directions with singular values near zero:
    |error| <= h (a^steps + grow (5 steps) |O|)  +  e |O|,      e: half a step of bf16 for bf16 results (2^-8), else 2^-24."""
import math

import pytest
import torch

COEF = (3.4445, -4.7750, 2.0315)
H = 2.0 ** -22


def exact(x, steps=5, coef=COEF, eps=1e-7):
    """the iteration as written, in 64 bits"""
    x = x.double()
    tall = x.shape[-2] > x.shape[-1]
    if tall:
        x = x.mT
    x = x / torch.linalg.vector_norm(x, dim=(-2, -1), keepdim=True).clamp(min=eps)
    for s in range(steps):
        a, b, c = coef[s] if isinstance(coef[0], tuple) else coef
        lam = x @ x.mT
        x = a * x + (b * lam + c * (lam @ lam)) @ x
    return x.mT if tall else x


def bound(want, dtype, steps=5, coef=COEF):
    norm = torch.linalg.vector_norm(want, dim=(-2, -1))
    a = 1.0
    for s in range(steps):
        a *= max(1.0, abs(coef[s][0] if isinstance(coef[0], tuple) else coef[0]))
    grow = 16.0 if dtype == torch.float32 else max(16.0, min(32768.0, 19800.0))
    return H * (a + grow * 5 * steps * norm) + (2.0 ** -24 if dtype == torch.float32 else 2.0 ** -8) * norm


def close(got, want, dtype, steps=5, coef=COEF, what=""):
    off = torch.linalg.vector_norm(got.double().cpu() - want, dim=(-2, -1))
    lim = bound(want, dtype, steps, coef)
    assert (off <= lim).all(), "%s: %.3g at a bound of %.3g" % (what, (off / lim).max().item() * lim.max().item(), lim.max().item())


def gradient(shape, seed, dtype=torch.float32, rank=4):
    """a few strong directions over noise, a small scale"""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g)
    x = x + 0.5 * torch.randn(shape[:-1] + (rank,), generator=g) @ torch.randn(shape[:-2] + (rank, shape[-1]), generator=g)
    return (x * 1e-3).to(dtype)


SHAPES = [(1, 1), (1, 64), (70, 1), (3, 5), (31, 33), (2, 32, 32), (64, 147), (147, 64), (5, 40, 70), (129, 257), (256, 256), (3, 200, 640), (300, 128),
          (21, 4608), (2304, 96), (513, 640), (2, 3, 16, 24), (65, 65), (64, 384), (384, 63), (64, 385), (33, 256), (257, 64), (2, 64, 448), (448, 61), (449, 64), (2, 32, 417), (300, 1, 5),
          (48, 40007), (40007, 21), (2, 64, 1025)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("shape", SHAPES, ids=["x".join(map(str, s)) for s in SHAPES])
def test_orthogonalize(shape, dtype):
    from pixelssl_amd import functional as PF
    x = gradient(shape, sum(shape), dtype)
    before = x.clone()
    xd = x.cuda()
    got = PF.orthogonalize(xd)
    assert got.shape == x.shape and got.dtype == dtype and torch.equal(xd.cpu(), before)
    close(got, exact(x), dtype, what=str(shape))


@pytest.mark.gpu
@pytest.mark.parametrize("shape,dtype", [((8, 1000, 1056), torch.float32), ((8, 2100, 1024), torch.float32), ((8, 1024, 1024), torch.bfloat16),
                                         ((5, 2, 900, 1700), torch.float32), ((1, 2930, 2940), torch.bfloat16)],
                         ids=lambda v: "x".join(map(str, v)) if isinstance(v, tuple) else str(v)[6:])
def test_more_tiles_than_compute_units(shape, dtype):
    """the tiles of the last round run in shares (the 64-bit products on the GPU: the plain formula all the same)"""
    from pixelssl_amd import functional as PF
    x = gradient(shape, 7, dtype).cuda()
    got = PF.orthogonalize(x)
    close(got, exact(x).cpu(), dtype, what=str(shape))
    assert torch.equal(got, PF.orthogonalize(x))


def spectrum(m, n, kind, seed):
    g = torch.Generator().manual_seed(seed)
    u, _, vh = torch.linalg.svd(torch.randn(m, n, generator=g, dtype=torch.float64), full_matrices=False)
    i = torch.arange(m, dtype=torch.float64)
    s = {"equal": torch.ones(m).double(), "harmonic": 1 / (1 + i), "square": 1 / (1 + i) ** 2, "six_decades": 10 ** (-6 * i / m),
         "one_strong": torch.where(i == 0, 1.0, 1e-3).double(), "rank_1": (i == 0).double(), "half_rank": (i < m // 2).double()}[kind]
    return (u * s) @ vh


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("kind", ["equal", "harmonic", "square", "six_decades", "one_strong", "rank_1", "half_rank"])
def test_spectra(kind, dtype):
    """from one strong direction to singular values over six decades: where rounding of A next to zero would grow"""
    from pixelssl_amd import functional as PF
    for m, n in ((60, 130), (96, 160), (160, 160)):
        x = spectrum(m, n, kind, 3).to(dtype)
        for y in (x, x.t().contiguous()):
            close(PF.orthogonalize(y.cuda()), exact(y), dtype, what="%s %s" % (kind, tuple(y.shape)))


@pytest.mark.gpu
def test_singular_values_come_out_near_one():
    from pixelssl_amd import functional as PF
    s = torch.linalg.svdvals(PF.orthogonalize(torch.randn(96, 400, generator=torch.Generator().manual_seed(1)).cuda()).double().cpu())
    assert s.min() > 0.65 and s.max() < 1.25


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("steps", [1, 2, 3, 4, 6, 7, 10])
def test_steps(steps, dtype):
    from pixelssl_amd import functional as PF
    x = gradient((96, 224), steps, dtype)
    close(PF.orthogonalize(x.cuda(), steps=steps), exact(x, steps), dtype, steps, what="%d steps" % steps)


@pytest.mark.gpu
def test_other_coefficients_one_per_step():
    from pixelssl_amd import functional as PF
    x = gradient((64, 160), 5)
    cubic = (1.5, -0.5, 0.0)
    close(PF.orthogonalize(x.cuda(), coefficients=cubic, steps=12), exact(x, 12, cubic), torch.float32, 12, cubic, "cubic")
    mixed = ((3.4445, -4.7750, 2.0315), (2.0, -1.5, 0.5), (1.5, -0.5, 0.0))
    close(PF.orthogonalize(x.cuda(), coefficients=mixed, steps=3), exact(x, 3, mixed), torch.float32, 3, mixed, "mixed")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_scales_zeros_and_what_is_not_finite(dtype):
    """norms from far below eps to near the type's end; a matrix of zeros, with zero rows and columns; a NaN or an infinity makes its own
    matrix NaN and no other"""
    from pixelssl_amd import functional as PF
    base = gradient((40, 72), 2).double() * 1e3
    x = torch.stack([base, base * 1e-30, base * 2.0 ** 100, base * 1e-9, base * 0, base, base, base, base]).to(dtype)
    x[5, 7], x[5, :, 9] = 0, 0
    x[6, 3, 3], x[7, 39, 71] = float("nan"), -float("inf")
    x[8, 0, 0] = 1e38
    got = PF.orthogonalize(x.cuda()).cpu()
    ok = [0, 1, 2, 3, 4, 5, 8]
    close(got[ok], exact(x[ok]), dtype, what="scales")
    assert not got[4].any() and not got[5, 7].any() and not got[5, :, 9].any()
    assert torch.isnan(got[[6, 7]]).all()


@pytest.mark.gpu
def test_layouts_streams_and_same_bits():
    from pixelssl_amd import functional as PF
    x = gradient((3, 70, 90), 6).cuda()
    want = PF.orthogonalize(x)
    close(want, exact(x.cpu()), torch.float32)
    for view in (x.mT.contiguous().mT, torch.cat([x, x], -1)[..., :90], x[None], x.flip(0)):
        got = PF.orthogonalize(view)
        assert torch.equal(got, want.flip(0) if view.shape == x.shape and not torch.equal(view, x) else want.view(view.shape))
    close(PF.orthogonalize(x[1]), exact(x[1].cpu()), torch.float32, what="alone")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = PF.orthogonalize(x)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    assert PF.orthogonalize(torch.zeros(0, 4, 5, device="cuda")).shape == (0, 4, 5)
    assert PF.orthogonalize(torch.zeros(2, 0, 5, device="cuda")).shape == (2, 0, 5)


def muon_exact(p, g, m, lr, mu=0.95, nesterov=True, wd=0.0, steps=5, coef=COEF, eps=1e-7, scale=None):
    p, g, m = p.double().cpu(), g.double().cpu(), m.double().cpu()
    m = mu * m + (1 - mu) * g
    u = (1 - mu) * g + mu * m if nesterov else m
    o = exact(u.reshape(u.shape[0], -1), steps, coef, eps)
    rows, cols = o.shape
    s = math.sqrt(max(1.0, rows / cols)) if scale is None else scale
    return p * (1 - lr * wd) - lr * s * o.view(p.shape), m, lr * s * bound(o, torch.float32, steps, coef), lr * s * torch.linalg.vector_norm(o)


def make(shape, seed, dtype=torch.float32, fmt=torch.contiguous_format):
    cols = 1
    for n in shape[1:]:
        cols *= n
    gen = torch.Generator().manual_seed(seed)
    out = []
    for k in range(3):
        t = (torch.randn(shape, generator=gen) * 0.1) if k == 0 else gradient((shape[0], cols), seed * 3 + k).view(shape)
        out.append(t.to(dtype if k < 2 else torch.float32).cuda().contiguous(memory_format=fmt if len(shape) == 4 else torch.contiguous_format))
    return out


def muon_close(p, m, want, dtype, what=""):
    """the momentum is off by three roundings, the parameter by the orthogonalised update's bound, four roundings and its type's half
    step; a bf16 gradient's update is formed and orthogonalised like a bf16 matrix' (its bound from bound())"""
    wp, wm, tol, unorm = want
    assert ((m.double().cpu() - wm).abs() <= 4 * 2.0 ** -24 * (wm.abs() + 1e-4)).all(), what
    off = torch.linalg.vector_norm(p.double().cpu() - wp)
    half = 2.0 ** -24 if dtype == torch.float32 else 2.0 ** -8
    lim = tol + (4 * 2.0 ** -24 + half) * torch.linalg.vector_norm(wp) + 2.0 ** -22 * unorm
    assert off <= lim, "%s: %.3g at a bound of %.3g" % (what, off, lim)


MIX = [(64, 3, 7, 7), (64, 64, 1, 1), (64, 64, 3, 3), (256, 64, 1, 1), (21, 128, 3, 3), (128, 300), (300, 128), (10, 7, 5), (1, 40), (40, 1), (33, 65),
       (65, 33), (96, 96), (64, 64, 3, 3), (2, 2), (128, 300)]


@pytest.mark.gpu
@pytest.mark.parametrize("nesterov,wd", [(True, 0.0), (False, 0.1)], ids=["nesterov", "plain_decay"])
def test_muon_update_of_mixed_shapes(nesterov, wd):
    """more shapes than one set of launches takes, in one call; the same again in one call per matrix"""
    from pixelssl_amd import functional as PF
    trip = [make(s, 10 + k) for k, s in enumerate(MIX)]
    want = [muon_exact(p, g, m, 0.02, nesterov=nesterov, wd=wd) for p, g, m in trip]
    alone = [[t.clone() for t in tr] for tr in trip]
    grads = [g.clone() for _, g, _ in trip]
    versions = [t[0]._version for t in trip]
    PF.muon_update(*zip(*trip), lr=0.02, nesterov=nesterov, weight_decay=wd)
    for k, (p, g, m) in enumerate(trip):
        muon_close(p, m, want[k], torch.float32, str(MIX[k]))
        assert torch.equal(g, grads[k]) and p._version > versions[k]
        a = alone[k]
        PF.muon_update([a[0]], [a[1]], [a[2]], lr=0.02, nesterov=nesterov, weight_decay=wd)
        muon_close(a[0], a[2], want[k], torch.float32, "alone, %s" % (MIX[k],))
        assert torch.equal(a[2], m)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,first,step", [(20, 24, 3), (40, 24, 30), (100, 24, 11), (0, 460, 41)])
def test_muon_update_of_many_shapes(rows, first, step):
    """15 shapes that run alike, more than the arguments of one launch hold, tall and wide; the last of 9 to 64 rows (columns)"""
    from pixelssl_amd import functional as PF
    small = [rows or 9 + 55 * k // 14 for k in range(15)]
    trip = [make((small[k], first + step * k) if k % 2 else (first + step * k, small[k]), k) for k in range(15)]
    want = [muon_exact(p, g, m, 0.01) for p, g, m in trip]
    PF.muon_update(*zip(*trip), lr=0.01)
    for (p, g, m), w in zip(trip, want):
        muon_close(p, m, w, torch.float32, str(tuple(p.shape)))


@pytest.mark.gpu
def test_muon_update_of_large_matrices_of_two_shapes():
    """more tiles than compute units, of two shapes, the last round's of the second one"""
    from pixelssl_amd import functional as PF
    trip = [make((1000, 1024) if k < 4 else (900, 1300), k) for k in range(9)]
    want = [muon_exact(p, g, m, 0.01) for p, g, m in trip]
    PF.muon_update(*zip(*trip), lr=0.01)
    for (p, g, m), w in zip(trip, want):
        muon_close(p, m, w, torch.float32, str(tuple(p.shape)))


@pytest.mark.gpu
def test_muon_update_of_many_matrices():
    """more matrices than one table launch carries, some hundred of them"""
    from pixelssl_amd import functional as PF
    trip = [make((8 + 8 * (k % 3), 24), k) for k in range(150)]
    want = [muon_exact(p, g, m, 0.01) for p, g, m in trip]
    PF.muon_update(*zip(*trip), lr=0.01)
    for (p, g, m), w in zip(trip, want):
        muon_close(p, m, w, torch.float32)


@pytest.mark.gpu
def test_muon_update_types_layouts_and_adjustments():
    from pixelssl_amd import functional as PF
    for fmt in (torch.contiguous_format, torch.channels_last):
        p, g, m = make((48, 20, 3, 3), 3, fmt=fmt)
        w = muon_exact(p, g, m, 0.02)
        g2 = g.contiguous() if fmt == torch.channels_last else g.contiguous(memory_format=torch.channels_last)
        p2, m2 = p.clone(), m.clone()
        PF.muon_update([p], [g], [m], lr=0.02)
        muon_close(p, m, w, torch.float32, str(fmt))
        PF.muon_update([p2], [g2], [m2], lr=0.02)               # a gradient laid out otherwise
        assert torch.equal(p2, p) and torch.equal(m2, m)
    p, g, m = make((48, 90), 4, torch.bfloat16)
    f = make((64, 90), 5)
    w, wf = muon_exact(p, g, m, 0.02, wd=0.1), muon_exact(*f, 0.02, wd=0.1)
    PF.muon_update([p, f[0]], [g, f[1]], [m, f[2]], lr=0.02, weight_decay=0.1)
    muon_close(p, m, w, torch.bfloat16, "bf16 parameter")
    muon_close(f[0], f[2], wf, torch.float32, "fp32 parameter beside it")
    p, g, m = make((30, 200), 6)
    w = muon_exact(p, g, m, 0.02, scale=0.2 * math.sqrt(200))
    PF.muon_update([p], [g], [m], lr=0.02, adjust="match_rms_adamw")
    muon_close(p, m, w, torch.float32, "match_rms_adamw")
    PF.muon_update([], [], [], lr=0.02)


@pytest.mark.gpu
def test_captured_updates_replay():
    """two captured updates over their own state, replayed in turn with eager work between, against eager runs of the same steps"""
    from pixelssl_amd import functional as PF
    shapes = [(64, 96), (96, 64, 1, 1), (21, 300)]
    runs = []
    for r in range(2):
        trip = [make(s, 40 + 10 * r + k) for k, s in enumerate(shapes)]
        mirror = [[t.clone() for t in tr] for tr in trip]
        x = gradient((2, 40, 50), 70 + r).cuda()
        g = torch.cuda.CUDAGraph()
        warm = [[t.clone() for t in tr] for tr in trip]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            PF.muon_update(*zip(*warm), lr=0.02)
            PF.orthogonalize(x)
        torch.cuda.current_stream().wait_stream(side)
        with torch.cuda.graph(g):
            PF.muon_update(*zip(*trip), lr=0.02)
            o = PF.orthogonalize(x)
        runs.append((g, trip, mirror, x, o))
    gen = torch.Generator().manual_seed(9)
    for rep in range(3):
        for g, trip, mirror, x, o in runs:
            x.copy_(gradient((2, 40, 50), 100 + rep))
            for (_, gd, _), (_, gm, _) in zip(trip, mirror):
                gd.copy_(torch.randn(gd.shape, generator=gen))
                gm.copy_(gd)
            g.replay()
            PF.muon_update(*zip(*mirror), lr=0.02)
            assert torch.equal(o, PF.orthogonalize(x))
            for a, b in zip(trip, mirror):
                assert torch.equal(a[0], b[0]) and torch.equal(a[2], b[2])
            torch.cuda.synchronize()


@pytest.mark.gpu
def test_nothing_around_the_matrices_is_touched():
    from pixelssl_amd import functional as PF
    for rows, cols in ((33, 70), (70, 33), (64, 64)):
        n, pad = rows * cols, 128
        flat = [torch.full((n + 2 * pad,), 5.0, device="cuda") for _ in range(3)]
        views = [f[pad:pad + n].view(rows, cols) for f in flat]
        for v, s in zip(views, make((rows, cols), 8)):
            v.copy_(s)
        PF.muon_update([views[0]], [views[1]], [views[2]], lr=0.02)
        for f in flat:
            assert (f[:pad] == 5).all() and (f[pad + n:] == 5).all()


# ---- refusals: no kernel is reached --------------------------------------------------------------------------------------------
def test_orthogonalize_refusals():
    from pixelssl_amd import _lib, functional as PF
    x = torch.randn(4, 8)
    with pytest.raises(_lib.PixelHipError, match="GPU only"):
        PF.orthogonalize(x)
    with pytest.raises(ValueError, match="no matrix"):
        PF.orthogonalize(x[0])
    with pytest.raises(ValueError, match="float32 or bfloat16"):
        PF.orthogonalize(x.double())
    with pytest.raises(ValueError, match="eps"):
        PF.orthogonalize(x, eps=0.0)
    with pytest.raises(ValueError, match="Newton-Schulz"):
        PF.orthogonalize(x, steps=0)
    with pytest.raises(ValueError, match="Newton-Schulz"):
        PF.orthogonalize(x, steps=3, coefficients=((1.5, -0.5, 0.0),) * 2)
    with pytest.raises(ValueError, match="Newton-Schulz"):
        PF.orthogonalize(x, coefficients=(1.5, -0.5))
    with pytest.raises(_lib.PixelHipError, match="no gradient"):
        PF.orthogonalize(x.requires_grad_(True))


def test_muon_update_refusals():
    from pixelssl_amd import _lib, functional as PF
    p, g, m = torch.randn(6, 4), torch.randn(6, 4), torch.zeros(6, 4)
    with pytest.raises(_lib.PixelHipError, match="GPU only"):
        PF.muon_update([p], [g], [m], lr=0.1)
    with pytest.raises(ValueError, match="1 gradients"):
        PF.muon_update([p, p], [g], [m], lr=0.1)
    with pytest.raises(ValueError, match="entry 0"):
        PF.muon_update([p[0]], [g[0]], [m[0]], lr=0.1)
    with pytest.raises(ValueError, match="entry 0"):
        PF.muon_update([p], [g[:3]], [m], lr=0.1)
    with pytest.raises(ValueError, match="momentum float32"):
        PF.muon_update([p], [g], [m.bfloat16()], lr=0.1)
    with pytest.raises(ValueError, match="both"):
        PF.muon_update([p], [g.bfloat16()], [m], lr=0.1)
    with pytest.raises(ValueError, match="dense"):
        PF.muon_update([torch.randn(4, 6).t()], [g], [m], lr=0.1)
    with pytest.raises(ValueError, match="lie alike"):
        PF.muon_update([torch.randn(6, 4, 3, 3)], [torch.randn(6, 4, 3, 3)], [torch.zeros(6, 4, 3, 3).contiguous(memory_format=torch.channels_last)], lr=0.1)
    for kw in (dict(momentum=1.0), dict(momentum=-0.1), dict(lr=float("nan")), dict(weight_decay=float("inf")), dict(eps=0.0)):
        with pytest.raises(ValueError):
            PF.muon_update([p], [g], [m], **{"lr": 0.1, **kw})
    with pytest.raises(ValueError, match="adjust"):
        PF.muon_scale((4, 4), "rms")


@pytest.mark.gpu
def test_refusals_that_need_device_tensors():
    from pixelssl_amd import _lib, functional as PF
    p, g, m = make((6, 4), 1)
    q = make((6, 4), 2)
    flat = torch.zeros(60, device="cuda")
    a, b = flat[:24].view(6, 4), flat[20:44].view(6, 4)
    for lists in (([p, p], [g, q[1]], [m, q[2]]), ([p, q[0]], [g, q[1]], [m, m]), ([p, g], [g, q[1]], [m, q[2]]), ([p], [p], [m]),
                  ([a], [b], [m]), ([p], [a], [b]), ([a, b], [g, q[1]], [m, q[2]])):
        with pytest.raises(_lib.PixelHipError, match="twice"):
            PF.muon_update(*lists, lr=0.1)
    with pytest.raises(_lib.PixelHipError, match="grow"):
        PF.orthogonalize(p, coefficients=(30.0, 0.0, 0.0))
    with pytest.raises(_lib.PixelHipError, match="finite"):
        PF.orthogonalize(p, coefficients=(float("nan"), 0.0, 0.0))
    with pytest.raises(_lib.PixelHipError, match="steps"):
        PF.orthogonalize(p, steps=17)
    with pytest.raises(ValueError, match="lies on"):
        PF.muon_update([p], [g.cpu()], [m], lr=0.1)


def test_c_entry_points_refuse_bad_arguments():
    import ctypes
    from pixelssl_amd import _lib
    h = _lib.lib()
    coef = (ctypes.c_float * 15)(*(COEF * 5))
    one = (_lib.NsItem * 1)((1, 1, 1, 8, 16, 1.0, 0))
    need = h.pxl_ns_workspace(0, one, 1)
    assert need > 0 and h.pxl_ns_workspace(0, one, 0) == 0 and h.pxl_ns_workspace(2, one, 1) == 0 and b"dtype" in h.pxl_last_error()
    assert h.pxl_orthogonalize(0, one, 1, 5, coef, 1e-7, 1, need - 1, None) == -4 and b"workspace" in h.pxl_last_error()
    assert h.pxl_orthogonalize(0, one, 1, 5, coef, 1e-7, None, need, None) == -4
    assert h.pxl_orthogonalize(3, one, 1, 5, coef, 1e-7, 1, need, None) == -1
    assert h.pxl_orthogonalize(0, one, 1, 0, coef, 1e-7, 1, need, None) == -1 and h.pxl_orthogonalize(0, one, 1, 17, coef, 1e-7, 1, need, None) == -1
    assert h.pxl_orthogonalize(0, one, 1, 5, None, 1e-7, 1, need, None) == -1
    assert h.pxl_orthogonalize(0, one, 1, 5, coef, 0.0, 1, need, None) == -1
    assert h.pxl_orthogonalize(0, None, 1, 5, coef, 1e-7, 1, need, None) == -1
    big = (ctypes.c_float * 15)(*((8.0, 0.0, 0.0) * 5))
    assert h.pxl_orthogonalize(0, one, 1, 5, big, 1e-7, 1, need, None) == -1 and b"grow" in h.pxl_last_error()
    for bad in ((1, 1, 1, 0, 16, 1.0, 0), (1, 1, 1, 8, -1, 1.0, 0), (1, 1, 1, 40000, 40000, 1.0, 0), (1, 1, 1, 1 << 25, 4, 1.0, 0)):
        it = (_lib.NsItem * 1)(bad)
        assert h.pxl_orthogonalize(0, it, 1, 5, coef, 1e-7, 1, 1 << 40, None) == -1 and b"item 0" in h.pxl_last_error()
    for bad in ((None, 1, 1, 8, 16, 1.0, 0), (1, None, 1, 8, 16, 1.0, 0)):
        it = (_lib.NsItem * 1)(bad)
        assert h.pxl_orthogonalize(0, it, 1, 5, coef, 1e-7, 1, need, None) == -1 and b"null" in h.pxl_last_error()
    it = (_lib.NsItem * 1)((1, 1, None, 8, 16, 1.0, 0))
    assert h.pxl_muon_step(0, it, 1, 5, coef, 1e-7, 0.1, 0.9, 1, 0.0, 1, need, None) == -1 and b"null" in h.pxl_last_error()
    assert h.pxl_muon_step(0, one, 1, 5, coef, 1e-7, 0.1, 1.0, 1, 0.0, 1, need, None) == -1 and b"momentum" in h.pxl_last_error()
    assert h.pxl_muon_step(0, one, 1, 5, coef, 1e-7, float("nan"), 0.9, 1, 0.0, 1, need, None) == -1
    assert h.pxl_orthogonalize(0, one, 0, 5, coef, 1e-7, None, 0, None) == 0
    two = (_lib.NsItem * 2)((1 << 20, 1 << 21, 1 << 22, 8, 16, 1.0, 0), ((1 << 20) + 508, 1 << 23, 1 << 24, 8, 16, 1.0, 0))
    room = h.pxl_ns_workspace(0, two, 2)
    assert h.pxl_muon_step(0, two, 2, 5, coef, 1e-7, 0.1, 0.9, 1, 0.0, 1 << 30, room, None) == -1 and b"twice" in h.pxl_last_error()
    assert h.pxl_orthogonalize(0, two, 2, 5, coef, 1e-7, 1 << 30, room, None) == -1 and b"twice" in h.pxl_last_error()


def test_scale_of_the_learning_rate():
    from pixelssl_amd.functional import muon_scale
    assert muon_scale((64, 64, 3, 3)) == 1.0 and muon_scale((256, 64)) == 2.0 and muon_scale((4, 100), "none") == 1.0
    assert abs(muon_scale((64, 64, 3, 3), "match_rms_adamw") - 0.2 * 24) < 1e-12
