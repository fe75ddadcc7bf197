"""Timed cases of the training operators next to the convolution engine: the orthogonalised update of the Muon optimizer
and layer normalisation over the last axis and over the channels of a map, each with its gradients.

`run` computes a case in plain torch arithmetic (own = False) or through the framework's entry points (own = True);
`exact` gives the same values from the operators' definitions in 64 bits."""
import math

import torch

own = False

COEFFICIENTS = (3.4445, -4.7750, 2.0315)     # the quintic of the Newton-Schulz step
STEPS = 5
NORM_EPS = 1e-7
LR, MOMENTUM, DECAY = 0.02, 0.95, 0.01       # of the Muon cases
LN_EPS = 1e-5


def listed():
    return [
        # the update of one 7 x 7 stem convolution over three colours: a single small matrix, latency counts
        dict(name="orthogonalize_stem", op="orthogonalize", batch=1, rows=64, cols=147, dtype="float32"),
        # the 23 3 x 3 convolutions of a ResNet-101's third stage
        dict(name="orthogonalize_stage3", op="orthogonalize", batch=23, rows=256, cols=2304, dtype="float32"),
        # the 1 x 1 convolutions that widen the same stage: taller than wide, bf16 updates
        dict(name="orthogonalize_widen_bf16", op="orthogonalize", batch=23, rows=1024, cols=256, dtype="bfloat16"),
        # the largest: two wide matrices, bound by the matrix products
        dict(name="orthogonalize_large", op="orthogonalize", batch=2, rows=2048, cols=4608, dtype="float32"),
        # a whole optimizer step (momentum, orthogonalisation, decay, update) of a ResNet-101's last 3 x 3 convolutions
        dict(name="muon_stage4", op="muon", batch=3, rows=512, channels=512, kernel=3),
        # the same for the multi-rate head: 21 classes, 18432 columns, four branches
        dict(name="muon_head", op="muon", batch=4, rows=21, channels=2048, kernel=3),
        # one feature vector normalised at inference
        dict(name="layer_norm_vector", op="layer_norm", rows=1, cols=2048, dtype="bfloat16", train=False),
        # every position of 8 stride-8 maps of 513 x 513 images, 2048 channels last, forward and backward
        dict(name="layer_norm_map", op="layer_norm", rows=8 * 65 * 65, cols=2048, dtype="bfloat16", train=True),
        # sizes that fit no vector width
        dict(name="layer_norm_odd", op="layer_norm", rows=1003, cols=777, dtype="float32", train=True),
        # a small odd map, channels first
        dict(name="layer_norm_channels_small", op="layer_norm_channels", batch=2, channels=64, height=17, width=19, dtype="float32", train=True),
        # stride-4 maps of 513 x 513 images
        dict(name="layer_norm_channels_stride4", op="layer_norm_channels", batch=8, channels=256, height=129, width=129, dtype="float32", train=True),
        # the deepest stride-8 maps in the throughput type
        dict(name="layer_norm_channels_deep", op="layer_norm_channels", batch=8, channels=2048, height=65, width=65, dtype="bfloat16", train=True),
    ]


def _log_int(rng, lo, hi):
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return max(lo, min(hi, n))


def draw(rng):
    op = rng.choice(["orthogonalize", "muon", "layer_norm", "layer_norm_channels"])
    if op == "orthogonalize":
        rows, cols = _log_int(rng, 16, 2048), _log_int(rng, 16, 4608)
        most = 2 * 2048 * 4608
        return dict(op=op, batch=_log_int(rng, 1, max(1, min(32, most // (rows * cols)))), rows=rows, cols=cols,
                    dtype=rng.choice(["float32", "bfloat16"]))
    if op == "muon":
        kernel = rng.choice([1, 3])
        rows, channels = _log_int(rng, 16, 1024), _log_int(rng, 16, 1024)
        most = 8 * 1024 * 1024
        return dict(op=op, batch=_log_int(rng, 1, max(1, min(24, most // (rows * channels * kernel * kernel)))), rows=rows,
                    channels=channels, kernel=kernel)
    most = 8 * 65 * 65 * 2048
    dtype, train = rng.choice(["float32", "bfloat16"]), rng.random() < 0.75
    if op == "layer_norm":
        cols = _log_int(rng, 8, 8192)
        return dict(op=op, rows=_log_int(rng, 1, most // (cols * 2)), cols=cols, dtype=dtype, train=train)
    channels, height, width = _log_int(rng, 8, 2048), _log_int(rng, 5, 129), _log_int(rng, 5, 129)
    return dict(op=op, batch=_log_int(rng, 1, max(1, min(8, most // (channels * height * width * 2)))), channels=channels, height=height,
                width=width, dtype=dtype, train=train)


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _update(g, batch, rows, cols):
    """what a gradient of a trained layer looks like: a few strong directions over noise, a small scale"""
    noise = torch.randn(batch, rows, cols, generator=g, device="cuda")
    left = torch.randn(batch, rows, 6, generator=g, device="cuda")
    right = torch.randn(batch, 6, cols, generator=g, device="cuda")
    return (noise + 0.5 * (left @ right)) * 1e-3


def prepare(case, seed):
    g = _generator(seed)
    op = case["op"]
    if op == "orthogonalize":
        return dict(op=op, x=_update(g, case["batch"], case["rows"], case["cols"]).to(getattr(torch, case["dtype"])))
    if op == "muon":
        batch, rows, channels, kernel = case["batch"], case["rows"], case["channels"], case["kernel"]
        shape, cols = (batch, rows, channels, kernel, kernel), channels * kernel * kernel
        params = torch.randn(shape, generator=g, device="cuda") * math.sqrt(2.0 / cols)
        grads = _update(g, batch, rows, cols).view(shape)
        momenta = _update(g, batch, rows, cols).view(shape)
        return dict(op=op, params=params, grads=grads, momenta=momenta, lists=[list(t.unbind(0)) for t in (params, grads, momenta)])
    dtype = getattr(torch, case["dtype"])
    if op == "layer_norm":
        shape, features = (case["rows"], case["cols"]), case["cols"]
    else:
        shape, features = (case["batch"], case["channels"], case["height"], case["width"]), case["channels"]
    x = (torch.randn(shape, generator=g, device="cuda") * 1.5 + 0.3).to(dtype)
    weight = 1.0 + 0.1 * torch.randn(features, generator=g, device="cuda")
    bias = 0.1 * torch.randn(features, generator=g, device="cuda")
    state = dict(op=op, train=case["train"], x=x, weight=weight, bias=bias)
    if case["train"]:
        state["dy"] = torch.randn(shape, generator=g, device="cuda").to(dtype)
        for t in (x, weight, bias):
            t.requires_grad_(True)
    return state


def _plain_orthogonalize(x):
    """[batch, rows, cols] in 32 bits -> the orthogonalised matrices in 32 bits"""
    tall = x.shape[-2] > x.shape[-1]
    if tall:
        x = x.transpose(-2, -1).contiguous()
    x = x / x.square().sum((-2, -1), keepdim=True).sqrt().clamp(min=NORM_EPS)
    a, b, c = COEFFICIENTS
    for _ in range(STEPS):
        s = x @ x.transpose(-2, -1)
        x = a * x + (b * s + c * (s @ s)) @ x
    return x.transpose(-2, -1).contiguous() if tall else x


def _plain_layer_norm(s, axis):
    x, w, b = s["x"].detach().float(), s["weight"].detach(), s["bias"].detach()
    shape = [1] * x.dim()
    shape[axis] = -1
    w, b = w.view(shape), b.view(shape)
    centred = x - x.mean(axis, keepdim=True)
    rstd = (centred.square().mean(axis, keepdim=True) + LN_EPS).rsqrt()
    unit = centred * rstd
    y = (unit * w + b).to(s["x"].dtype)
    if not s["train"]:
        return y
    dy = s["dy"].float()
    others = [k for k in range(x.dim()) if k != axis % x.dim()]
    g = dy * w
    dx = rstd * (g - g.mean(axis, keepdim=True) - unit * (g * unit).mean(axis, keepdim=True))
    return y, dx.to(s["x"].dtype), (dy * unit).sum(others), dy.sum(others)


def _run_plain(s):
    if s["op"] == "orthogonalize":
        return _plain_orthogonalize(s["x"].float()).to(s["x"].dtype)
    if s["op"] == "muon":
        p, g, m = s["params"], s["grads"], s["momenta"]
        m.mul_(MOMENTUM).add_(g * (1 - MOMENTUM))
        u = g * (1 - MOMENTUM) + m * MOMENTUM
        rows, cols = p.shape[1], p[0, 0].numel()
        o = _plain_orthogonalize(u.view(p.shape[0], rows, cols)).view(p.shape)
        p.mul_(1 - LR * DECAY).sub_(o * (LR * math.sqrt(max(1.0, rows / cols))))
        return p, m
    return _plain_layer_norm(s, -1 if s["op"] == "layer_norm" else 1)


def _run_own(s):
    from pixelssl_amd import functional as PF
    if s["op"] == "orthogonalize":
        return PF.orthogonalize(s["x"], steps=STEPS, coefficients=COEFFICIENTS, eps=NORM_EPS)
    if s["op"] == "muon":
        PF.muon_update(*s["lists"], lr=LR, momentum=MOMENTUM, nesterov=True, weight_decay=DECAY, steps=STEPS,
                       coefficients=COEFFICIENTS, eps=NORM_EPS)
        return s["params"], s["momenta"]
    norm = PF.layer_norm if s["op"] == "layer_norm" else PF.layer_norm_channels
    if not s["train"]:
        with torch.no_grad():
            return norm(s["x"], s["weight"], s["bias"], eps=LN_EPS)
    y = norm(s["x"], s["weight"], s["bias"], eps=LN_EPS)
    return (y.detach(),) + torch.autograd.grad(y, (s["x"], s["weight"], s["bias"]), s["dy"])


def run(state):
    return _run_own(state) if own else _run_plain(state)


def work(case):
    op = case["op"]
    if op in ("orthogonalize", "muon"):
        rows = case["rows"]
        cols = case["cols"] if op == "orthogonalize" else case["channels"] * case["kernel"] ** 2
        m, n, batch = min(rows, cols), max(rows, cols), case["batch"]
        # multiply-adds as 2 operations, symmetric products at half price.  Step by step: X X', its square and the product with X;
        # or, as all factors are polynomials of X X' and commute, one X X', the recursion on m x m matrices and one product with X
        stepwise = STEPS * (m * m * n + m ** 3 + 2 * m * m * n)
        commuting = m * m * n + (4 * STEPS - 4) * m ** 3 + 2 * m * m * n
        size = batch * rows * cols
        if op == "muon":
            return dict(bytes=5 * 4 * size, flops=batch * min(stepwise, commuting) + 8 * size)
        return dict(bytes=2 * (4 if case["dtype"] == "float32" else 2) * size, flops=batch * min(stepwise, commuting) + 3 * size)
    if op == "layer_norm":
        size, features = case["rows"] * case["cols"], case["cols"]
    else:
        size, features = case["batch"] * case["channels"] * case["height"] * case["width"], case["channels"]
    item = 4 if case["dtype"] == "float32" else 2
    if not case["train"]:
        return dict(bytes=2 * item * size + 8 * features, flops=8 * size)
    # forward and backward as one pass each over what they need: x, y; x, dy, dx (x is needed again after the loss)
    return dict(bytes=5 * item * size + 16 * features, flops=20 * size)


def _exact_orthogonalize(x):
    """the scalar polynomial applied to the singular values: eigenvectors of the smaller Gram matrix, in 64 bits"""
    x = x.double()
    x = x / torch.linalg.vector_norm(x, dim=(-2, -1), keepdim=True).clamp(min=NORM_EPS)
    wide = x.shape[-2] <= x.shape[-1]
    gram = torch.matmul(x, x.mT) if wide else torch.matmul(x.mT, x)
    values, vectors = torch.linalg.eigh(gram.cpu())
    a, b, c = COEFFICIENTS
    lam = values.clamp(min=0.0)
    gain = torch.ones_like(lam)
    for _ in range(STEPS):
        factor = a + lam * (b + c * lam)
        gain, lam = gain * factor, lam * factor * factor
    transform = ((vectors * gain.unsqueeze(-2)) @ vectors.mT).to(x.device)
    return torch.matmul(transform, x) if wide else torch.matmul(x, transform)


def exact(case, seed):
    s = prepare(case, seed)
    if s["op"] == "orthogonalize":
        return _exact_orthogonalize(s["x"])
    if s["op"] == "muon":
        p, g, m = (s[k].double() for k in ("params", "grads", "momenta"))
        m = torch.lerp(m, g, 1 - MOMENTUM)
        u = torch.lerp(g, m, MOMENTUM).flatten(2)
        o = _exact_orthogonalize(u).view(p.shape)
        ratio = u.shape[-2] / u.shape[-1]
        return p * (1 - LR * DECAY) - LR * math.sqrt(ratio if ratio > 1 else 1) * o, m
    axis = -1 if s["op"] == "layer_norm" else 1
    x, w, b = (s[k].detach().double().requires_grad_(s["train"]) for k in ("x", "weight", "bias"))
    lead = (-1,) + (1,) * (0 if axis == -1 else x.dim() - 2)
    var, mean = torch.var_mean(x, dim=axis, correction=0, keepdim=True)
    y = (x - mean) / torch.sqrt(var + LN_EPS) * w.view(lead) + b.view(lead)
    if not s["train"]:
        return y
    return (y.detach(),) + torch.autograd.grad(y, (x, w, b), s["dy"].double())
