"""Layer normalisation over very many features, rows and positions, and over maps of few positions: what the register kernels do not hold.

There sums are taken in 64 bits, so that their length is in no bound.  With h = 2^-24: the mean is off by its own rounding and that of its quotient,
d_m = 2 h |mean| at most, the variance relatively by 6 h and by d_m^2 / var (rounding of the differences, their squares, the quotient, eps), rstd
relatively by e_r = 8 h + d_m^2 rstd^2, u by d_u = d_m rstd + |u| (e_r + 4 h), and
  y  by |w| d_u + 4 h (|u w| + |b|) + e |y|          (e: half a step of the type of y, 0 for fp32: counted in the 4 h)
  dx by rstd (8 h (|g| + mean|g| + 2 |u| mean|g u|) + d_u mean|g u| + |u| mean(|g| d_u)) + |dx| (e_r + 4 h + e),   g = dy w
  dw by 8 h sum|dy u| + sum|dy| d_u + e |dw|,    db by 4 h sum|dy| + e |db|      (shares of it are rounded to fp32 once each)."""
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
from test_layer_norm import H, close, rows_of, run  # noqa: E402


def reference(x, w, b, eps, dy):
    x, dy, w, b = (t.double() for t in (x, dy, w, b))
    m = x.mean(1, keepdim=True)
    r = 1 / (((x - m) ** 2).mean(1, keepdim=True) + eps).sqrt()
    u = (x - m) * r
    d_m = 2 * H * m.abs()
    e_r = 8 * H + d_m ** 2 * r ** 2
    d_u = d_m * r + u.abs() * (e_r + 4 * H)
    y = u * w + b
    g = dy * w
    gu = (g * u).abs().mean(1, keepdim=True)
    dx = r * (g - g.mean(1, keepdim=True) - u * (g * u).mean(1, keepdim=True))
    sums = 8 * H * (g.abs() + g.abs().mean(1, keepdim=True) + 2 * u.abs() * gu)
    dw, db = (dy * u).sum(0), dy.sum(0)
    return {"y": (y, lambda e: w.abs() * d_u + 4 * H * ((u * w).abs() + b.abs()) + e * y.abs()),
            "dx": (dx, lambda e: r * (sums + d_u * gu + u.abs() * (g.abs() * d_u).mean(1, keepdim=True)) + dx.abs() * (e_r + 4 * H + e)),
            "dw": (dw, lambda e: 8 * H * (dy * u).abs().sum(0) + (dy.abs() * d_u).sum(0) + e * dw.abs()),
            "db": (db, lambda e: 4 * H * dy.abs().sum(0) + e * db.abs())}


def make(shape, C, dtype, seed):
    """one sign, a mean a hundred times the deviation: where sums one after the other drift"""
    g = torch.Generator().manual_seed(seed)
    x = (0.1 + 1e-3 * torch.randn(shape, generator=g)).to(dtype)
    dy = (0.1 + 1e-2 * torch.randn(shape, generator=g)).to(dtype)
    return x.cuda(), (1 + 0.2 * torch.randn(C, generator=g)).cuda(), (0.2 * torch.randn(C, generator=g)).cuda(), dy.cuda()


LONG = [((2, 300007), False), ((1, 2 ** 21 + 1), False), ((2 ** 20, 3), False), ((2 ** 18, 7), False), ((1, 300007, 1, 3), True), ((2, 200001, 2), True), ((1, 40, 2 ** 22 + 8), True),
        ((2 ** 19 + 3, 2, 1, 2), True), ((50000, 33, 3), True)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("shape,channels", LONG, ids=["x".join(map(str, s)) for s, _ in LONG])
def test_sums_of_many_terms(shape, channels, dtype):
    C = shape[1]
    if not channels and 16 // dtype.itemsize <= C <= 8192:
        pytest.skip("held in registers, sums in 32 bits: the bounds of test_layer_norm.py")
    x, w, b, dy = make(shape, C, dtype, C % 1000)
    got = run(x, w, b, dy, channels, eps=1e-8)
    want = reference(rows_of(x, channels).cpu(), w.cpu(), b.cpu(), 1e-8, rows_of(dy, channels).cpu())
    for name, t in zip(("y", "dx"), got):
        close(rows_of(t, channels), want[name], "%s %s" % (shape, name))
    for name, t in zip(("dw", "db"), got[2:]):
        close(t, want[name], "%s %s" % (shape, name))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_short_rows_that_lie_apart(dtype):
    """read as they lie: the bits of the same rows without gaps"""
    x, w, b, dy = make((1000, 11), 3, dtype, 3)
    apart = run(x[:, 5:8], w, b, dy[:, :3].contiguous(), False, eps=1e-8)
    for a, r in zip(apart, run(x[:, 5:8].contiguous(), w, b, dy[:, :3].contiguous(), False, eps=1e-8)):
        assert torch.equal(a, r)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("shape", [(1, 1, 1, 1), (8, 2048, 1, 1), (3, 5, 1, 1), (5, 9001, 1), (70, 33)], ids=lambda s: "x".join(map(str, s)))
def test_a_map_of_one_position_is_a_row(shape, dtype):
    """the same kernels, so the same bits, forward and backward"""
    g = torch.Generator().manual_seed(shape[1])
    x, dy = (torch.randn(shape, generator=g).to(dtype).cuda() for _ in range(2))
    w, b = torch.randn(shape[1], generator=g).cuda(), torch.randn(shape[1], generator=g).cuda()
    rows = run(x.flatten(1), w, b, dy.flatten(1), False)
    for a, r in zip(run(x, w, b, dy, True), rows):
        assert torch.equal(a.reshape(r.shape), r)


def test_one_position_needs_the_workspace_of_rows():
    from pixelssl_amd import _lib
    h = _lib.lib()
    for n, c in ((1, 1), (70, 33), (100000, 2048), (3, 2 ** 24)):
        assert h.pxl_layer_norm_nchw_bwd_workspace(n, c, 1) == h.pxl_layer_norm_bwd_workspace(n, c)


@pytest.mark.gpu
def test_more_tiles_than_a_grid_holds():
    """2^24 small maps: as many workgroups of 256 threads as no launch takes"""
    from pixelssl_amd import functional as PF
    n = 2 ** 24 + 3
    x = torch.empty(n, 2, 2, 2, device="cuda").normal_(generator=torch.Generator("cuda").manual_seed(1))
    w, b = torch.tensor([0.7, 1.3], device="cuda"), torch.tensor([0.2, -0.1], device="cuda")
    y = PF.layer_norm_channels(x, w, b)
    for part, want in zip(x.split(2 ** 21 - 1), y.split(2 ** 21 - 1)):
        assert torch.equal(PF.layer_norm_channels(part, w, b), want)
    x.requires_grad_(True)
    dy = torch.ones_like(y)
    dx, = torch.autograd.grad(PF.layer_norm_channels(x, w, b), x, dy)
    last = x[-5:].detach().requires_grad_(True)
    assert torch.equal(torch.autograd.grad(PF.layer_norm_channels(last, w, b), last, dy[-5:])[0], dx[-5:])


@pytest.mark.gpu
def test_as_many_channels_as_are_taken():
    """2^24 channels at two positions, the parameters' gradients among what is checked"""
    from pixelssl_amd import functional as PF
    C = 2 ** 24
    g = torch.Generator("cuda").manual_seed(2)
    x, dy = (torch.empty(1, C, 2, device="cuda").normal_(generator=g) for _ in range(2))
    w, b = torch.ones(C, device="cuda"), torch.zeros(C, device="cuda")
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    y = PF.layer_norm_channels(*leaves)
    dx, dw, db = torch.autograd.grad(y, leaves, dy)
    rows = lambda t: t.detach()[0].t().contiguous()
    want = reference(rows(x), w.detach(), b.detach(), 1e-5, rows(dy))
    for name, t in (("y", rows(y)), ("dx", rows(dx)), ("dw", dw), ("db", db)):
        val, bound = want[name]
        assert ((t.double() - val).abs() <= bound(0.0) + 1e-37).all(), name


@pytest.mark.gpu
@pytest.mark.parametrize("shape,channels", [((2 ** 20, 2048), False), ((2 ** 24, 16), False), ((16, 32, 1025, 1025), True)], ids=lambda v: "x".join(map(str, v)) if isinstance(v, tuple) else "")
def test_parameter_gradients_of_a_constant_gradient(shape, channels):
    """one addend over and over is what a running sum in 32 bits drifts with: n of them, each addition off by up to 2^-24 of what there is, by up to
    2^-25 n of the sum.  At most 256 rows, or 512 positions of these maps, are added up so; what adds up those sums is in 64 bits"""
    from pixelssl_amd import functional as PF
    C = shape[1]
    x = torch.empty(shape, device="cuda").normal_(generator=torch.Generator("cuda").manual_seed(1)).bfloat16()
    w, b = torch.ones(C, device="cuda", requires_grad=True), torch.zeros(C, device="cuda", requires_grad=True)
    dy = torch.full(shape, 0.1, device="cuda")
    y = (PF.layer_norm_channels if channels else PF.layer_norm)(x.float(), w, b)
    db, = torch.autograd.grad(y, b, dy)
    want = x.numel() // C * float(dy.flatten()[0])
    assert (db.double() / want - 1).abs().max().item() <= 2.0 ** -25 * 512 * (1 if channels else 0.5)
