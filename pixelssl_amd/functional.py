"""Fused per-pixel losses (NCHW fp32 tensors) and layer normalisation (fp32 / bf16), autograd Functions over libpixelhip kernels;
orthogonalised updates of weight matrices."""
import ctypes
import functools
import threading

import torch
from torch.autograd import forward_ad

from . import _lib
from ._lib import check, dtype_code, lib, ptr, stream_ptr


def _gpu(*ts):
    for t in ts:
        if not t.is_cuda:
            raise _lib.PixelHipError("fused losses run on the GPU only (got %s); there is no CPU path" % t.device)


class _CrossEntropyPerSample(torch.autograd.Function):
    """CommonSSEGCriterion arithmetic (task/sseg/criterion.py:24-38): CE with ignore_index summed over a
    sample and divided by ALL H*W pixels."""

    @staticmethod
    def forward(ctx, logits, gt, ignore_index):
        _gpu(logits, gt)
        logits = logits.contiguous()
        gt = gt.contiguous().float()
        N, C, H, W = logits.shape
        loss = torch.empty(N, device=logits.device, dtype=torch.float32)
        check(lib().pxl_ce_fwd(N, C, H * W, ptr(logits), ptr(gt), int(ignore_index), ptr(loss), stream_ptr()))
        ctx.save_for_backward(logits, gt)
        ctx.ignore_index = int(ignore_index)
        return loss

    @staticmethod
    def backward(ctx, gout):
        logits, gt = ctx.saved_tensors
        N, C, H, W = logits.shape
        gout = gout.contiguous().float()
        dlogits = torch.empty_like(logits)
        check(lib().pxl_ce_bwd(N, C, H * W, ptr(logits), ptr(gt), ctx.ignore_index, ptr(gout), ptr(dlogits), stream_ptr()))
        return dlogits, None, None


def cross_entropy_per_sample(logits, gt, ignore_index=255):
    """logits [N,C,H,W] fp32, gt [N,1,H,W] or [N,H,W] float class ids -> loss [N]."""
    return _CrossEntropyPerSample.apply(logits, gt, ignore_index)


class _MSE(torch.autograd.Function):
    """nn.MSELoss() (mean reduction); the gradient flows to the first operand only (the second is the
    detached teacher / pseudo-label, ssl_mt.py:179-184)."""

    @staticmethod
    def forward(ctx, a, b):
        _gpu(a, b)
        a = a.contiguous()
        b = b.contiguous()
        out = torch.empty(1, device=a.device, dtype=torch.float32)
        check(lib().pxl_mse_fwd(a.numel(), ptr(a), ptr(b), ptr(out), stream_ptr()))
        ctx.save_for_backward(a, b)
        return out.view(())

    @staticmethod
    def backward(ctx, gout):
        a, b = ctx.saved_tensors
        gout = gout.contiguous().float().view(1)
        da = torch.empty_like(a)
        check(lib().pxl_mse_bwd(a.numel(), ptr(a), ptr(b), ptr(gout), ptr(da), stream_ptr()))
        return da, None


def mse_loss(a, b):
    if a.shape != b.shape:
        raise ValueError("mse_loss: shape mismatch %s vs %s" % (tuple(a.shape), tuple(b.shape)))
    return _MSE.apply(a, b.detach())


class _TaskConsistency(torch.autograd.Function):
    """Task loss (per-sample CE on the first `n_ce` samples) + consistency loss (MSE of samples [lo, hi) against a
    detached target) of ONE logits tensor, with ONE backward launch writing d(logits) once: what autograd builds from
    `pred[:lbs]` -> CE, `pred[lo:]` -> MSE, `task + cons` is two zero-filled slice gradients, two copies and a sum over the
    full [N, C, H, W] tensor (ssl_mt.py:166-196 at 8 x 21 x 513 x 513: 0.33 ms of the step).  `ce_values` is the CE forward
    already computed (no-grad) on the same operands -- the caller may have launched it before the target existed."""

    @staticmethod
    def forward(ctx, logits, gt, ce_values, target, lo, hi, ignore_index):
        _gpu(logits, gt, target)
        logits = logits.contiguous()
        target = target.contiguous()
        gt = gt.contiguous().float()
        if target.shape != logits.shape:
            raise ValueError("task_consistency: target %s vs logits %s" % (tuple(target.shape), tuple(logits.shape)))
        N = logits.shape[0]
        n_ce = ce_values.shape[0]
        if not (0 <= lo <= hi <= N and n_ce <= N and gt.shape[0] == n_ce):
            raise ValueError("task_consistency: bad ranges n_ce=%d [%d, %d) of %d" % (n_ce, lo, hi, N))
        out = torch.zeros(1, device=logits.device, dtype=torch.float32)
        if hi > lo:
            a, b = logits[lo:hi], target[lo:hi]
            check(lib().pxl_mse_fwd(a.numel(), ptr(a), ptr(b), ptr(out), stream_ptr()))
        ctx.save_for_backward(logits, gt, target)
        ctx.rng = (int(lo), int(hi), int(n_ce), int(ignore_index))
        ctx.set_materialize_grads(False)
        return ce_values.clone(), out.view(())

    @staticmethod
    def backward(ctx, g_ce, g_mse):
        logits, gt, target = ctx.saved_tensors
        lo, hi, n_ce, ignore = ctx.rng
        if g_ce is None and g_mse is None:
            return (None,) * 7
        N, C, H, W = logits.shape
        g_ce = g_ce.contiguous().float() if g_ce is not None else None
        g_mse = g_mse.contiguous().float().view(1) if g_mse is not None else None
        dlogits = torch.empty_like(logits)
        check(lib().pxl_ce_mse_bwd(N, C, H * W, ptr(logits), ptr(gt), ignore, n_ce, ptr(g_ce), ptr(target), lo, hi, ptr(g_mse),
                                   ptr(dlogits), stream_ptr()))
        return dlogits, None, None, None, None, None, None


def task_consistency(logits, gt, ce_values, target, lo, hi, ignore_index=255):
    """-> (per-sample CE [n_ce] (= ce_values, now differentiable), MSE(logits[lo:hi], target[lo:hi]) scalar)."""
    return _TaskConsistency.apply(logits, gt, ce_values.detach(), target.detach(), int(lo), int(hi), int(ignore_index))


def head_losses(s_head, t_head, gt, n_ce, mse_lo, mse_hi, ce_weight, mse_weight, ignore_index=255, mse_weight_dev=None):
    """The training seam on the low-resolution logits of deferred forward passes (engine.DeferredHead; csrc/head.hip:
    pxl_head_loss): per-sample cross-entropy of the student and of the teacher on the first `n_ce` samples
    (task/sseg/criterion.py:24-38), the MSE between their predictions over samples [mse_lo, mse_hi) (ssl_mt.py:179-184)
    and d(loss)/d(student low-res logits) for loss = ce_weight * sum(CE_student) + mse_weight * MSE, left in the
    student's executor for s_head.backward().  t_head None: student terms only.
    mse_weight_dev: device address of mse_weight (graph.HyperBlock.ptr) -- a captured step reads the ramped weight from there.
    -> (student CE [n_ce], teacher CE [n_ce] or None, MSE mean scalar), detached fp32 device tensors."""
    _gpu(gt)
    gt = gt.contiguous().float()
    B = s_head.batch
    if t_head is not None and (t_head.batch != B or t_head.plan.out_size != s_head.plan.out_size):
        raise ValueError("head_losses: student and teacher passes differ in shape")
    H, W = s_head.plan.out_size
    if n_ce and gt.numel() != n_ce * H * W:
        raise ValueError("head_losses: gt %s does not hold %d maps of %d x %d" % (tuple(gt.shape), n_ce, H, W))
    sums = torch.empty(2 * B + 1, device=gt.device, dtype=torch.float32)
    pl = s_head.plan
    s_head._check_arena("head_losses")
    if t_head is not None:
        t_head._check_arena("head_losses")
    if mse_weight_dev is not None:
        check(lib().pxl_net_head_loss_hp(pl.net, ptr(s_head.arena), t_head.plan.net if t_head is not None else None,
                                         ptr(t_head.arena) if t_head is not None else None, ptr(gt), int(ignore_index), int(n_ce),
                                         int(mse_lo), int(mse_hi), float(ce_weight), mse_weight_dev, ptr(pl.scratch),
                                         pl.scratch.numel(), ptr(sums), stream_ptr()))
    else:
        check(lib().pxl_net_head_loss(pl.net, ptr(s_head.arena), t_head.plan.net if t_head is not None else None,
                                      ptr(t_head.arena) if t_head is not None else None, ptr(gt), int(ignore_index), int(n_ce),
                                      int(mse_lo), int(mse_hi), float(ce_weight), float(mse_weight), ptr(pl.scratch),
                                      pl.scratch.numel(), ptr(sums), stream_ptr()))
    s_head.mark_grad()
    return sums[:n_ce], (sums[B:B + n_ce] if t_head is not None else None), sums[2 * B]


class _DecoderConsistency(torch.autograd.Function):
    """One SSLCCT auxiliary decoder from its (perturbed) latent to its consistency term, without the full-resolution planes:
    the decoder's executor stops at its own-resolution logits, csrc/head.hip: pxl_cons_head_fwd evaluates resize + soft-max + MSE
    and parks the gradient for a unit incoming gradient; the backward scales it by the incoming gradient (a device scalar), runs
    the executor's backward from there and returns the latent's gradient (ssl_cct.py:476-484 + autograd)."""

    @staticmethod
    def forward(ctx, x, anchor, core, target, out_size, holder):
        head = core.forward_deferred(x, out_size=out_size, force_graph=True, seam="cons")
        if head is None:
            raise _lib.PixelHipError("decoder_consistency: the fused seam cannot run on this plan (check decoder_consistency_supported first)")
        pl = head.plan
        loss = torch.empty(1, device=x.device, dtype=torch.float32)
        check(lib().pxl_net_cons_head_fwd(pl.net, ptr(head.arena), ptr(target), ptr(pl.scratch), pl.scratch.numel(), ptr(loss), stream_ptr()))
        pl.grad_gen = getattr(pl, "grad_gen", 0) + 1         # the parked gradient is this plan's seam state from here on
        head._parked_gen = pl.grad_gen
        ctx.head, ctx.x_shape = head, tuple(x.shape)
        holder.append(head)
        return loss.reshape(())

    @staticmethod
    def backward(ctx, gout):
        head = ctx.head
        pl, core = head.plan, head.core
        if getattr(head, "_parked_gen", None) != getattr(pl, "grad_gen", 0):
            raise _lib.PixelHipError("decoder_consistency: the gradient parked by the forward has been overwritten (another pass / seam ran "
                                     "on the same plan before this backward)")
        g = gout.detach().reshape(1).contiguous().float()
        check(lib().pxl_net_cons_head_bwd(pl.net, ptr(pl.scratch), pl.scratch.numel(), ptr(g), stream_ptr()))
        head.mark_grad()
        head.backward()
        dx = None
        if ctx.needs_input_grad[0]:
            dx = torch.empty(ctx.x_shape, device=g.device, dtype=torch.float32)
            check(lib().pxl_net_input_grad(pl.net, ptr(pl.scratch), ptr(dx), stream_ptr()))
        ctx.head = None
        return dx, None, None, None, None, None


def decoder_consistency_supported(core, x, target, out_size):
    """can decoder_consistency run for this decoder / latent / target?  (plans the shape, runs nothing)"""
    if not (x.is_cuda and target.is_cuda and x.dim() == 4 and target.dim() == 4):
        return False
    B, _, H, W = x.shape
    if tuple(target.shape) != (B, core.num_classes) + tuple(out_size) or target.dtype != torch.float32:
        return False
    core._plan(B, H, W, out_size, inference=False)
    return bool(lib().pxl_net_cons_head_supported(core._cur.net))


def decoder_consistency(core, x, target, out_size):
    """MSE(softmax(resize(decoder(x), out_size)), target) of an engine.AuxDecoderCore as ONE differentiable scalar (gradients: the
    decoder's parameters and x).  -> (term, DeferredHead); head.materialize() yields the resized prediction when somebody wants it."""
    _gpu(x, target)
    holder = []
    term = _DecoderConsistency.apply(x.contiguous().float(), core._anchor, core, target.detach().contiguous(), tuple(out_size), holder)
    return term, holder[0]


class MSELoss(torch.nn.Module):
    """Drop-in for the `nn.MSELoss()` the SSL algorithms instantiate."""

    def forward(self, a, b):
        return mse_loss(a, b)


def confusion_matrix(pred, gt, num_classes, out=None):
    """Device confusion matrix of the sseg validation metrics (task/sseg/func.py:41-48): pred [N,C,H,W] fp32 (activated
    or not: only its channel arg-max counts), gt [N,1,H,W] / [N,H,W] float class ids -> int64 [C,C] with
    cm[g][a] = #pixels labeled g (0 <= g < C) predicted a.  Accumulates into `out` when given.  Bit-exact integer counts."""
    _gpu(pred, gt)
    pred = pred.detach().contiguous().float()
    gt = gt.detach().contiguous().float()
    N, C, H, W = pred.shape
    if C != num_classes:
        raise ValueError("confusion_matrix: prediction has %d channels, num_classes = %d" % (C, num_classes))
    if gt.numel() != N * H * W:
        raise ValueError("confusion_matrix: gt %s does not match prediction %s" % (tuple(gt.shape), tuple(pred.shape)))
    cm = out if out is not None else torch.zeros(C, C, device=pred.device, dtype=torch.int64)
    check(lib().pxl_confusion_matrix(N, C, H * W, ptr(pred), ptr(gt), ptr(cm), stream_ptr()))
    return cm


def argmax_u8(pred):
    """[N,C,H,W] fp32 -> uint8 [N,H,W] channel arg-max (np.argmax tie / NaN rules)."""
    _gpu(pred)
    pred = pred.detach().contiguous().float()
    N, C, H, W = pred.shape
    out = torch.empty(N, H, W, device=pred.device, dtype=torch.uint8)
    check(lib().pxl_argmax_u8(N, C, H * W, ptr(pred), ptr(out), stream_ptr()))
    return out


class _SoftmaxChannels(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x):
        _gpu(x)
        x = x.contiguous().float()
        N, C = x.shape[0], x.shape[1]
        p = torch.empty_like(x)
        check(lib().pxl_softmax_nchw_fwd(N, C, x.numel() // (N * C), ptr(x), ptr(p), stream_ptr()))
        ctx.save_for_backward(p)
        return p

    @staticmethod
    def backward(ctx, dp):
        (p,) = ctx.saved_tensors
        N, C = p.shape[0], p.shape[1]
        dx = torch.empty_like(p)
        check(lib().pxl_softmax_nchw_bwd(N, C, p.numel() // (N * C), ptr(p), ptr(dp.contiguous().float()), ptr(dx), stream_ptr()))
        return dx


def softmax_channels(x):
    """F.softmax(x, dim=1) of an NCHW fp32 prediction (the sseg activation), differentiable."""
    return _SoftmaxChannels.apply(x)


# ---- layer normalisation (csrc/layernorm.hip) ---------------------------------------------------------------------------------
def _launch(index, fn, *args):
    """fn(*args, stream) on the current stream of device `index`, which need not be the current device"""
    if index == torch._C._cuda_getDevice():
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    if rc:
        check(rc)


_held = threading.local()


class _AllOrNothing:
    """`with _AllOrNothing():` -- the updates called inside check their arguments there and are launched together at the end; an exception, and
    none of them is."""

    def __enter__(self):
        self.outer, _held.calls = getattr(_held, "calls", None), []

    def __exit__(self, kind, *_):
        calls, _held.calls = _held.calls, self.outer
        if kind is None:
            _submit(calls)


def _submit(calls):
    """calls: (device index, C function, arguments, what has to live until the launch), all checked; launched one after the other"""
    held = getattr(_held, "calls", None)
    if held is not None:
        held += calls
        return
    for index, fn, args, _ in calls:
        _launch(index, fn, *args)


def _refuse_recording(name, *tensors):
    """A recorder (torch.jit.trace, make_fx) sees the allocations of a call but not its kernels: what it made would return what the memory held
    before.  torch.func's wrappers have no memory, and a forward-mode tangent would stop at the outputs without a word."""
    if torch._C._get_tracing_state() is not None or torch._C._get_dispatch_mode(torch._C._TorchDispatchModeKey.PROXY) is not None:
        raise _lib.PixelHipError("%s cannot be traced (torch.jit.trace, make_fx): its kernels would be missing from the result" % name)
    if torch._C._functorch.peek_interpreter_stack() is not None:
        raise _lib.PixelHipError("%s does not run under torch.func / vmap" % name)
    if forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise _lib.PixelHipError("%s has no forward-mode derivative" % name)


_pxlnode = None


def _node():
    """the compiled autograd nodes (pixelssl_amd/node), bound to the loaded libpixelhip.so"""
    global _pxlnode
    if _pxlnode is None:
        try:
            from . import _pxlnode as module
        except ImportError as e:
            raise _lib.PixelHipError("_pxlnode.so is missing or does not load (%s). Build it with `python -m pixelssl_amd.build`; there is "
                                     "no other path." % e)
        raw = ctypes.CDLL(_lib.LIB_PATH)          # (the same loaded library as lib(): its addresses)
        module.bind([ctypes.cast(getattr(raw, name), ctypes.c_void_p).value for name in (
            "pxl_layer_norm_fwd", "pxl_layer_norm_bwd", "pxl_layer_norm_bwd_workspace", "pxl_layer_norm_nchw_fwd", "pxl_layer_norm_nchw_bwd",
            "pxl_layer_norm_nchw_bwd_workspace", "pxl_last_error")])
        _pxlnode = module
    return _pxlnode


def _layer_norm(x, weight, bias, eps, channels):
    y = (_pxlnode or _node()).layer_norm(x, weight, bias, eps, channels)
    if y is None:
        _layer_norm_refuse("layer_norm_channels" if channels else "layer_norm", x, weight, bias, eps, channels)
    return y


def _layer_norm_refuse(name, x, weight, bias, eps, channels):
    """says what the node does not take about the arguments"""
    _refuse_recording(name, x, weight, bias)
    dtype = x.dtype
    if dtype is not torch.float32 and dtype is not torch.bfloat16:
        raise ValueError("%s: float32 or bfloat16, got %s" % (name, dtype))
    if x.dim() < (2 if channels else 1) or x.shape[1 if channels else -1] == 0:
        raise ValueError("%s: no features to normalise over in %s" % (name, tuple(x.shape)))
    C = x.shape[1 if channels else -1]
    if C > 1 << 24:
        raise ValueError("%s: %d features (at most 2^24)" % (name, C))
    for what, t in (("weight", weight), ("bias", bias)):
        if t is None:
            continue
        if t.dim() != 1 or t.shape[0] != C:
            raise ValueError("%s: %s %s for %d features" % (name, what, tuple(t.shape), C))
        if (t.dtype is not torch.float32 and t.dtype is not dtype) or (weight is not None and t.dtype is not weight.dtype):
            raise ValueError("%s: weight and bias are both float32 or both of the type of x (%s), got %s" % (name, dtype, t.dtype))
        if t.device != x.device:
            raise ValueError("%s: %s on %s, x on %s" % (name, what, t.device, x.device))
    if not eps >= 0:
        raise ValueError("%s: eps %r" % (name, eps))
    _gpu(x)
    raise ValueError("%s: a dense tensor, got %s" % (name, x.layout))


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """(x - mean) / sqrt(var + eps) * weight + bias over the LAST axis of x (fp32 or bf16; any leading axes, rows may lie apart in
    memory), statistics in fp32; weight / bias [C]: fp32 or the type of x.  Differentiable once in x, weight and bias; gradients
    are the same bits from call to call."""
    return _layer_norm(x, weight, bias, eps, False)


def layer_norm_channels(x, weight=None, bias=None, eps=1e-5):
    """`layer_norm` over axis 1 of an [N, C, ...] map at each position (a map stored channels last is read as it lies)."""
    return _layer_norm(x, weight, bias, eps, True)


# ---- orthogonalised updates (csrc/muon.hip) -----------------------------------------------------------------------------------
NEWTON_SCHULZ = (3.4445, -4.7750, 2.0315)      # (a, b, c) of x (a + b x^2 + c x^4): singular values to 0.7 .. 1.2 in five steps


@functools.lru_cache(maxsize=64)
def _ns_coefficients(steps, coefficients):
    """(a, b, c) for every step, or one triple per step -> float[steps * 3]"""
    if coefficients and not isinstance(coefficients[0], tuple):
        coefficients = (coefficients,) * steps
    if steps < 1 or len(coefficients) != steps or any(len(t) != 3 for t in coefficients):
        raise ValueError("Newton-Schulz: %d steps need one (a, b, c) or as many, got %r" % (steps, coefficients))
    flat = [float(v) for t in coefficients for v in t]
    return (ctypes.c_float * len(flat))(*flat)


def _coefficient_key(coefficients):
    """one (a, b, c) or one per step, as nested tuples whatever sequences they came in"""
    return tuple(tuple(float(v) for v in t) if isinstance(t, (tuple, list)) else float(t) for t in coefficients)


def _coefficients(steps, coefficients):
    return _ns_coefficients(int(steps), _coefficient_key(coefficients))


def orthogonalize(x, steps=5, coefficients=NEWTON_SCHULZ, eps=1e-7):
    """Every matrix of x [..., rows, cols] (fp32 or bf16) with its singular values driven to about 1 by `steps` of the Newton-Schulz
    iteration X <- (a + b L + c L^2) X, L = X X', from X = x / max(|x|, eps) (Frobenius norm); for rows > cols on the transposed
    matrix.  coefficients: one (a, b, c) or one per step.  A NaN or an infinity makes its own matrix NaN.  Not differentiable."""
    _refuse_recording("orthogonalize", x)
    if x.dim() < 2:
        raise ValueError("orthogonalize: %s is no matrix" % (tuple(x.shape),))
    if x.dtype not in (torch.float32, torch.bfloat16):
        raise ValueError("orthogonalize: float32 or bfloat16, got %s" % x.dtype)
    if not eps > 0:
        raise ValueError("orthogonalize: eps %r" % (eps,))
    coef = _coefficients(steps, coefficients)
    if torch.is_grad_enabled() and x.requires_grad:
        raise _lib.PixelHipError("orthogonalize has no gradient: call it under torch.no_grad() or on a detached tensor")
    _gpu(x)
    x = x.detach().contiguous()
    out = torch.empty_like(x)
    rows, cols = x.shape[-2], x.shape[-1]
    if x.numel():
        size = rows * cols * x.element_size()
        src, dst = x.data_ptr(), out.data_ptr()
        n = x.numel() // (rows * cols)
        items = (_lib.NsItem * n)(*[(dst + k * size, src + k * size, None, rows, cols, 1.0, 0) for k in range(n)])
        nbytes = lib().pxl_orthogonalize_workspace(dtype_code(x.dtype), items, n, int(steps), coef)
        index, fn, args, ws = _ns_call(lib().pxl_orthogonalize, nbytes, x.device, dtype_code(x.dtype), items, n, steps, coef, eps)
        _launch(index, fn, *args)
    return out


def _ns_call(fn, nbytes, dev, code, items, n, steps, coef, eps, *scalars):
    """one call with its workspace of nbytes (0: refused), as _submit takes it"""
    if nbytes == 0:
        raise _lib.PixelHipError("libpixelhip: %s" % lib().pxl_last_error().decode())
    ws = torch.empty(nbytes, device=dev, dtype=torch.uint8)
    return dev.index, fn, (code, items, n, int(steps), coef, float(eps)) + scalars + (ptr(ws), nbytes), ws


def _dense_strides(t):
    """strides of the axes that have any length, when t fills one run of memory with its first axis outermost (contiguous or
    channels last); None otherwise"""
    if not (t.is_contiguous() or (t.dim() == 4 and t.is_contiguous(memory_format=torch.channels_last))):
        return None
    return tuple(s for s, n in zip(t.stride(), t.shape) if n > 1)


def muon_scale(shape, adjust="original"):
    """factor on the learning rate of a [rows, ...] parameter: 'original': sqrt(max(1, rows / cols)); 'match_rms_adamw': 0.2 sqrt(max(rows,
    cols)) (an update of the size AdamW's has); 'none': 1.  cols: the product of the other axes."""
    rows, cols = shape[0], 1
    for n in shape[1:]:
        cols *= n
    if adjust == "original":
        return max(1.0, rows / cols) ** 0.5 if cols else 1.0
    if adjust == "match_rms_adamw":
        return 0.2 * max(rows, cols) ** 0.5
    if adjust == "none":
        return 1.0
    raise ValueError("muon: adjust is 'original', 'match_rms_adamw' or 'none', got %r" % (adjust,))


def muon_update(params, grads, momenta, lr, momentum=0.95, nesterov=True, weight_decay=0.0, steps=5, coefficients=NEWTON_SCHULZ, eps=1e-7,
                adjust="original"):
    """One Muon step on lists of parameters [rows, ...] (two axes or more; a convolution's [out, in, kh, kw] is the matrix of its
    rows), in place, all matrices of all shapes together:
        momentum_k <- momentum * momentum_k + (1 - momentum) * grad_k
        u = (1 - momentum) * grad_k + momentum * momentum_k  (nesterov)  or  momentum_k
        param_k <- param_k * (1 - lr * weight_decay) - lr * muon_scale(...) * orthogonalize(u)
    adjust: the rule of muon_scale, or one factor per parameter in its place.  params / grads fp32 or bf16 (one type per parameter), momenta
    fp32 with the parameter's memory layout (contiguous or channels last).  Parameters and momenta may overlap nothing.  What is refused is
    refused before anything is changed."""
    params, grads, momenta = list(params), list(grads), list(momenta)
    _refuse_recording("muon_update", *params, *grads, *momenta)
    if not len(params) == len(grads) == len(momenta):
        raise ValueError("muon_update: %d parameters, %d gradients, %d momenta" % (len(params), len(grads), len(momenta)))
    lr, momentum, weight_decay = float(lr), float(momentum), float(weight_decay)
    if not 0 <= momentum < 1 or not eps > 0 or not abs(lr) < float("inf") or not abs(weight_decay) < float("inf"):
        raise ValueError("muon_update: lr %r, momentum %r (0 <= momentum < 1), weight decay %r, eps %r" % (lr, momentum, weight_decay, eps))
    coef = _coefficients(steps, coefficients)
    named = isinstance(adjust, str)
    if not named and (len(adjust) != len(params) or not all(abs(float(a)) < float("inf") for a in adjust)):
        raise ValueError("muon_update: adjust is a name or one finite factor per parameter, got %r" % (adjust,))
    work, keep, scales = {}, [], {}
    for k, (p, g, m) in enumerate(zip(params, grads, momenta)):
        shape = p.shape
        if p.dim() < 2 or g.shape != shape or m.shape != shape:
            raise ValueError("muon_update: entry %d: parameter %s, gradient %s, momentum %s" % (k, tuple(shape), tuple(g.shape), tuple(m.shape)))
        if p.dtype not in (torch.float32, torch.bfloat16) or g.dtype != p.dtype or m.dtype != torch.float32:
            raise ValueError("muon_update: entry %d: parameter and gradient both float32 or both bfloat16, momentum float32; got %s, %s, %s" %
                             (k, p.dtype, g.dtype, m.dtype))
        strides = _dense_strides(p)
        if strides is None or _dense_strides(m) != strides:
            raise ValueError("muon_update: entry %d: a parameter and its momentum are dense and lie alike in memory" % k)
        if g.device != p.device or m.device != p.device:
            raise ValueError("muon_update: entry %d lies on %s, %s and %s" % (k, p.device, g.device, m.device))
        _gpu(p)
        if p.numel() == 0:
            continue
        if _dense_strides(g) != strides:
            g = torch.empty_like(p, requires_grad=False).copy_(g.detach())
            keep.append(g)
        if shape not in scales:
            scales[shape] = (shape[0], p.numel() // shape[0], muon_scale(shape, adjust) if named else 0.0, 0)
        geo = scales[shape] if named else scales[shape][:2] + (float(adjust[k]), 0)
        work.setdefault((p.device, p.dtype), []).append((p.data_ptr(), g.data_ptr(), m.data_ptr()) + geo)
    calls = []
    for (dev, dtype), entries in work.items():
        items, n = (_lib.NsItem * len(entries))(*entries), len(entries)
        check(lib().pxl_muon_check(dtype_code(dtype), items, n, int(steps), coef, float(eps), lr, momentum, weight_decay))
        nbytes = lib().pxl_ns_workspace(dtype_code(dtype), items, n)
        index, fn, args, ws = _ns_call(lib().pxl_muon_step, nbytes, dev, dtype_code(dtype), items, n, steps, coef, eps, lr, momentum, int(bool(nesterov)), weight_decay)
        calls.append((index, fn, args, (ws, keep)))
    _submit(calls)
    torch.autograd.graph.increment_version([t for t in params + momenta if t.numel()])


def adam_update(params, grads, exp_avgs, exp_avg_sqs, lr, betas=(0.9, 0.999), eps=1e-8, step=1):
    """torch.optim.Adam's update without weight decay (FusedAdam's arithmetic) on lists of tensors, in place, many in one launch: the
    vectors beside muon_update's matrices.  params / grads fp32 or bf16, exp_avgs / exp_avg_sqs fp32, all four of an entry dense and
    alike in memory (a gradient may lie otherwise).  Parameters and moments may overlap nothing.  step counts from 1.  What is refused is refused
    before anything is changed."""
    params, grads, exp_avgs, exp_avg_sqs = list(params), list(grads), list(exp_avgs), list(exp_avg_sqs)
    _refuse_recording("adam_update", *params, *grads, *exp_avgs, *exp_avg_sqs)
    if not len(params) == len(grads) == len(exp_avgs) == len(exp_avg_sqs):
        raise ValueError("adam_update: %d parameters, %d gradients, %d and %d moments" % (len(params), len(grads), len(exp_avgs), len(exp_avg_sqs)))
    b1, b2 = float(betas[0]), float(betas[1])
    if not (0 <= b1 < 1 and 0 <= b2 < 1 and eps > 0 and int(step) >= 1):
        raise ValueError("adam_update: betas %r, eps %r, step %r" % (betas, eps, step))
    work, keep, touched = {}, [], []
    for k, (p, g, m, v) in enumerate(zip(params, grads, exp_avgs, exp_avg_sqs)):
        if not g.shape == m.shape == v.shape == p.shape:
            raise ValueError("adam_update: entry %d: shapes %s, %s, %s, %s" % (k, tuple(p.shape), tuple(g.shape), tuple(m.shape), tuple(v.shape)))
        if p.dtype not in (torch.float32, torch.bfloat16) or g.dtype != p.dtype or m.dtype != torch.float32 or v.dtype != torch.float32:
            raise ValueError("adam_update: entry %d: parameter and gradient both float32 or both bfloat16, the moments float32" % k)
        strides = _dense_strides(p)
        if strides is None or _dense_strides(m) != strides or _dense_strides(v) != strides:
            raise ValueError("adam_update: entry %d: a parameter and its moments are dense and lie alike in memory" % k)
        if not g.device == m.device == v.device == p.device:
            raise ValueError("adam_update: entry %d lies on several devices" % k)
        _gpu(p)
        if p.numel() == 0:
            continue
        if _dense_strides(g) != strides:
            g = torch.empty_like(p, requires_grad=False).copy_(g.detach())
            keep.append(g)
        work.setdefault((p.device, p.dtype), []).append((p.data_ptr(), g.data_ptr(), m.data_ptr(), v.data_ptr(), p.numel()))
        touched += [p, m, v]
    calls = []
    for (dev, dtype), entries in work.items():
        items, n = (_lib.AdamItem * len(entries))(*entries), len(entries)
        check(lib().pxl_adam_check(dtype_code(dtype), items, n, b1, b2, float(eps), int(step)))
        calls.append((dev.index, lib().pxl_adam_list, (dtype_code(dtype), items, n, float(lr), b1, b2, float(eps), int(step)), keep))
    _submit(calls)
    torch.autograd.graph.increment_version(touched)
