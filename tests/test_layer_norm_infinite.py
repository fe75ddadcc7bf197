"""Infinite and NaN gradients through the backward pass of layer normalisation: what the formula gives for them, at their own position or row
and nowhere else."""
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
from test_layer_norm import rows_of, run  # noqa: E402


def formula(x, w, dy, eps=1e-5):
    x, w, dy = x.double(), w.double(), dy.double()
    m = x.mean(1, keepdim=True)
    r = 1 / (((x - m) ** 2).mean(1, keepdim=True) + eps).sqrt()
    u, g = (x - m) * r, dy * w
    return r * (g - g.mean(1, keepdim=True) - u * (g * u).mean(1, keepdim=True)), (dy * u).sum(0), dy.sum(0)


def same_kind(got, want, what):
    got, want = got.double().cpu(), want.cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    assert torch.equal(torch.isinf(got), torch.isinf(want)) and torch.equal(got[torch.isinf(want)], want[torch.isinf(want)]), what


CHANNELS = [(2, 5, 9, 8), (1, 33, 6, 7), (2, 100, 5, 8), (1, 129, 9, 9), (1, 257, 8, 8), (1, 600, 4, 9), (1, 1500, 4, 8), (1, 2050, 3, 3), (2, 40, 1, 3)]
ROWS = [(5, 3), (9, 33), (6, 777), (4, 2051), (3, 9000)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("shape", CHANNELS + ROWS, ids=lambda s: "x".join(map(str, s)))
def test_infinite_gradients(shape, dtype):
    channels, C = len(shape) == 4, shape[1]
    g = torch.Generator().manual_seed(C)
    x, dy = (torch.randn(shape, generator=g).to(dtype) for _ in range(2))
    w = 1 + 0.1 * torch.rand(C, generator=g)
    rows = rows_of(dy, channels).shape[0]
    hit = [(0, C - 1, float("inf")), (rows - 1, C - 1, -float("inf")), (rows // 2, 0, float("inf")), (rows // 2 + 1, C // 2, float("nan"))]
    flat = dy.movedim(1, -1).reshape(-1, C).contiguous() if channels else dy
    for r, c, v in hit:
        flat[r, c] = v
    dy = flat.view(shape[0], *shape[2:], C).movedim(-1, 1).contiguous() if channels else flat
    got = run(x.cuda(), w.cuda(), torch.zeros(C).cuda(), dy.cuda(), channels)
    dx, dw, db = formula(rows_of(x, channels), w, rows_of(dy, channels))
    same_kind(rows_of(got[1], channels), dx, "%s dx" % (shape,))
    same_kind(got[2], dw, "%s dw" % (shape,))
    same_kind(got[3], db, "%s db" % (shape,))
