"""Operators of a residual block in 8 bits: quantisation into e4m3 blocks of 128, the block-scaled product, a linear layer on top of
it (forward and backward in 8 bits) and the root-mean-square norm with the residual's addition that feeds it.

The format (``include/monoloco_hip.h``): ``torch.float8_e4m3fn`` codes; 128 values share one ``torch.float8_e8m0fnu`` scale, the
smallest power of two with which their largest magnitude fits into 448.  A block is 1 x 128 of a row -- scales (rows, ceil(n / 128)) --
or 128 x 128 of a weight -- scales (ceil(rows / 128), ceil(n / 128)).  A block that holds a NaN or an infinity becomes NaN.

Plumbing as in ``engine.py``: torch holds the memory and the stream, the arithmetic is ``libmonoloco_hip.so``'s; every call runs on
the current stream of its tensors' device.  Wrong arguments raise ``ValueError``, failures inside the library ``MonolocoHipError``.
The reference has no such layers: its Linear layers are fp32 (monoloco/network/architectures.py:24-43)."""
import ctypes
import functools

import torch

from . import _lib
from ._lib import MonolocoHipError, check_ops
from .engine import _RAW_STREAM, _stream

BLOCK = 128
CODES = torch.float8_e4m3fn
SCALES = torch.float8_e8m0fnu
DTYPES = {torch.float32: _lib.ML_F32, torch.bfloat16: _lib.ML_BF16, torch.float16: _lib.ML_F16}
_current = getattr(torch._C, '_cuda_getDevice', torch.cuda.current_device)


def _blocks(n):
    return -(-n // BLOCK)


def _need(ok, text, *args):
    if not ok:
        raise ValueError(text % args)


def _device_of(name, *tensors):
    """The one device (its index) of the call's tensors.  (Small calls are bound by what Python does: the checks here and below look at
    one thing each and build their texts only when they fail.)"""
    index = None
    for t in tensors:
        if t is None:
            continue
        if not isinstance(t, torch.Tensor):
            raise ValueError("%s: expected tensors, got %s" % (name, type(t).__name__))
        i = t.get_device()
        if i != index:
            if not t.is_cuda:
                raise MonolocoHipError("%s runs on HIP devices only, got a tensor on %s (there is no CPU fallback)" % (name, t.device))
            if index is not None:
                raise ValueError("%s: tensors on cuda:%d and on %s" % (name, index, t.device))
            index = i
    return index


def _run(index, fn, *args):
    """fn(*args, stream) on the current stream of device `index`."""
    if _RAW_STREAM is not None and _current() == index:
        rc = fn(*args, _RAW_STREAM(index))
    else:
        dev = torch.device('cuda', index)
        with torch.cuda.device(dev):
            rc = fn(*args, _stream(dev))
    if rc:
        check_ops(rc)


def _rows(t):
    """A matrix whose rows are contiguous and do not overlap (a copy where they are not)."""
    if not t.is_contiguous() and t.numel() and ((t.shape[1] > 1 and t.stride(1) != 1) or (t.shape[0] > 1 and t.stride(0) < t.shape[1])):
        return t.contiguous()
    return t


def _flat_rows(t, n):
    """(..., n) -> (rows, n) with such rows."""
    if t.dim() != 2:
        t = t.reshape(-1, n)
    return t if t.is_contiguous() else _rows(t)


def _ld(t):
    """Row stride of such a matrix (of a single row: anything that is long enough)."""
    m, n = t.shape
    return t.stride(0) if m > 1 and n else n or 1


def _codes_empty(m, n, dev):
    """(m, n) codes whose rows start on 16 bytes: what the product loads in whole pieces."""
    if n % 16 == 0:
        return torch.empty((m, n), dtype=CODES, device=dev)
    return torch.empty((m, n + -n % 16), dtype=CODES, device=dev)[:, :n]


def _quantize(x, tile, transposed):
    """-> q, scale, qt, scale_t (the last two None where not asked for)."""
    x = _rows(x)
    m, n = x.shape
    dev = x.device
    q = _codes_empty(m, n, dev)
    s = torch.empty((_blocks(m) if tile else m, _blocks(n)), dtype=SCALES, device=dev)
    qt = st = None
    if transposed:
        qt = _codes_empty(n, m, dev)
        st = torch.empty((_blocks(n) if tile else n, _blocks(m)), dtype=SCALES, device=dev)
    if x.numel():
        _run(x.get_device(), _lib.load().ml_fp8_quantize, x.data_ptr(), DTYPES[x.dtype], m, n, _ld(x), int(tile), q.data_ptr(), _ld(q), s.data_ptr(), s.shape[1],
             qt.data_ptr() if transposed else None, _ld(qt) if transposed else 0, st.data_ptr() if transposed else None, st.shape[1] if transposed else 0, None)
    return q, s, qt, st


def quantize(x, block=(1, BLOCK), transposed=False):
    """x (m, n) in fp32, bf16 or fp16 -> (codes (m, n), scales) in blocks of (1, 128) or (128, 128).

    ``transposed=True``: (codes, scales, codes_t, scales_t) from one read of x: the same, and x^T (n, m) in blocks of ITS rows -- what a
    product needs that reduces over the other axis.  With (128, 128) blocks the transposed codes and scales are the straight ones,
    transposed.  Rows of the codes start on 16 bytes (a view of a wider buffer where n is no multiple of 16).  Not differentiable: x's
    values are taken without their history."""
    _device_of('quantize', x)
    _need(x.dim() == 2 and x.dtype in DTYPES, "quantize: needs a matrix in fp32, bf16 or fp16, got %s %s", tuple(x.shape), x.dtype)
    _need(tuple(block) in ((1, BLOCK), (BLOCK, BLOCK)), "quantize: blocks are (1, 128) or (128, 128), got %r", block)
    _lib.load()
    with torch.no_grad():
        q, s, qt, st = _quantize(x.detach(), tuple(block) == (BLOCK, BLOCK), bool(transposed))
    return (q, s, qt, st) if transposed else (q, s)


def _scales_of(name, codes, scale):
    """-> is it a scale per tile (else per row)?"""
    rows, k = codes.shape
    shape, kb = scale.shape, -(-k // BLOCK)
    if scale.dtype == SCALES and len(shape) == 2 and shape[1] == kb:
        if shape[0] == rows:
            return False
        if shape[0] == -(-rows // BLOCK):
            return True
    raise ValueError("matmul: %s_scale is %s %s; %s codes take %s as (%d, %d) (a scale per row and 128 columns) or (%d, %d) (per 128 x 128)"
                     % (name, tuple(shape), scale.dtype, (rows, k), SCALES, rows, kb, -(-rows // BLOCK), kb))


@functools.lru_cache(maxsize=1024)
def _matmul_work(m, n, k, dtype):
    return int(_lib.load().ml_fp8_matmul_work(m, n, k, dtype))


def matmul(a, a_scale, b, b_scale, bias=None, out_dtype=torch.bfloat16, out=None):
    """a (m, k) . b (n, k)^T [+ bias (n)] of e4m3 codes with their block scales -> (m, n) in ``out_dtype`` (fp32, bf16, fp16), accumulated
    in fp32 and rounded once.  16-bit results come from the 8-bit matrix instructions (1.5e-5 of the result's norm beside the rounding: a result
    whose terms cancel to less than that keeps no digits), fp32 results from exact bf16 operands at half the rate (6e-8; the operands' values
    have to lie in fp32's normal range, smaller ones count as 0): ``out_dtype`` is the choice between the two.

    Each scale is (rows, ceil(k / 128)) or (ceil(rows / 128), ceil(k / 128)), as ``quantize`` gives them.  ``out``: an (m, n) tensor of one
    of the three types with contiguous rows to write into (``out_dtype`` is then its type), apart in memory from what is read.  Not
    differentiable: see ``linear``."""
    index = _device_of('matmul', a, a_scale, b, b_scale, bias, out)
    if not (a.dtype == CODES and b.dtype == CODES and a.dim() == 2 and b.dim() == 2):
        raise ValueError("matmul: a and b are matrices of %s, got %s %s and %s %s" % (CODES, tuple(a.shape), a.dtype, tuple(b.shape), b.dtype))
    m, k = a.shape
    n = b.shape[0]
    if b.shape[1] != k:
        raise ValueError("matmul: a has rows of %d, b of %d" % (k, b.shape[1]))
    a_tile, b_tile = _scales_of('a', a, a_scale), _scales_of('b', b, b_scale)
    if bias is not None:
        if bias.dim() != 1 or bias.shape[0] != n or bias.dtype not in DTYPES:
            raise ValueError("matmul: the bias is (%d) in fp32, bf16 or fp16, got %s %s" % (n, tuple(bias.shape), bias.dtype))
        bias = bias.contiguous()
    if torch.is_grad_enabled() and (a.requires_grad or b.requires_grad or a_scale.requires_grad or b_scale.requires_grad or (bias is not None and bias.requires_grad)):
        raise ValueError("matmul is not differentiable: use linear, or detach the operands and the bias")
    given = out is not None
    if not given:
        if out_dtype not in DTYPES:
            raise ValueError("matmul: out_dtype is fp32, bf16 or fp16, got %s" % (out_dtype,))
        out = torch.empty((m, n), dtype=out_dtype, device=a.device)
    else:
        _need(tuple(out.shape) == (m, n) and out.dtype in DTYPES, "matmul: out is %s %s, needed (%d, %d) in fp32, bf16 or fp16", tuple(out.shape), out.dtype, m, n)
        _need(_rows(out) is out, "matmul: the rows of out have to be contiguous and apart")
        _need(not (out.requires_grad and torch.is_grad_enabled()), "matmul is not differentiable: out must not require a gradient")
    if m and n:
        a, b, a_scale, b_scale = _rows(a), _rows(b), _rows(a_scale), _rows(b_scale)
        dt = DTYPES[out.dtype]
        size = _matmul_work(m, n, k, dt)
        work = torch.empty((size,), dtype=torch.uint8, device=a.device) if size else None
        _run(index, _lib.load().ml_fp8_matmul, a.data_ptr(), _ld(a), a_scale.data_ptr(), _ld(a_scale), a_tile, b.data_ptr(), _ld(b), b_scale.data_ptr(), _ld(b_scale),
             b_tile, bias.data_ptr() if bias is not None else None, DTYPES[bias.dtype] if bias is not None else 0, out.data_ptr(), dt, _ld(out), m, n, k,
             work.data_ptr() if size else None, size)
    if given:
        torch.autograd.graph.increment_version(out)
    return out


@functools.lru_cache(maxsize=256)
def _linear_sizes(m, n, k, need_dx, need_dw, need_db):
    """Bytes of the three workspaces of a linear layer of that shape."""
    out = (ctypes.c_int64 * 3)()
    check_ops(_lib.load().ml_fp8_linear_sizes(m, n, k, need_dx, need_dw, need_db, out))
    return tuple(out)


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, grads):
        n, k = weight.shape
        # (needs_input_grad is requires_grad alone, also where gradients are off)
        need_x, need_w, need_b = (grads and need for need in ctx.needs_input_grad[:3])
        x2, w2 = _flat_rows(x, k), _rows(weight)
        m = x2.shape[0]
        dev = x.device
        size, keep, _ = _linear_sizes(m, n, k, need_x, need_w, need_b)
        y = torch.empty(x.shape[:-1] + (n,), dtype=x.dtype, device=dev)
        work = torch.empty((size,), dtype=torch.uint8, device=dev)
        saved = torch.empty((keep,), dtype=torch.uint8, device=dev) if keep else None
        _run(x.get_device(), _lib.load().ml_fp8_linear, x2.data_ptr(), DTYPES[x.dtype], _ld(x2), w2.data_ptr(), DTYPES[weight.dtype], _ld(w2),
             bias.data_ptr() if bias is not None else None, DTYPES[bias.dtype] if bias is not None else 0, y.data_ptr(), n or 1, m, n, k, need_x, need_w, work.data_ptr(),
             saved.data_ptr() if keep else None)
        ctx.save_for_backward(saved)
        ctx.was = (m, n, k, need_x, need_w, x.shape, x.dtype, weight.dtype, bias.dtype if need_b else None)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        want_x, want_w, want_b, _ = ctx.needs_input_grad
        saved, = ctx.saved_tensors
        m, n, k, need_x, need_w, xshape, xdt, wdt, bdt = ctx.was
        dev = dy.device
        dy2 = _flat_rows(dy, n) if n else dy
        dx = torch.empty(xshape, dtype=xdt, device=dev) if want_x else None
        dw = torch.empty((n, k), dtype=wdt, device=dev) if want_w else None
        db = torch.empty((n,), dtype=bdt, device=dev) if want_b else None
        work = torch.empty((_linear_sizes(m, n, k, need_x, need_w, want_b)[2],), dtype=torch.uint8, device=dev)
        if n:
            _run(dy.get_device(), _lib.load().ml_fp8_linear_backward, dy2.data_ptr(), DTYPES[dy.dtype], _ld(dy2), saved.data_ptr() if saved is not None else None,
                 dx.data_ptr() if want_x and m else None, DTYPES[xdt], dw.data_ptr() if want_w else None, DTYPES[wdt], db.data_ptr() if want_b else None,
                 DTYPES[bdt] if want_b else 0, m, n, k, need_x, need_w, work.data_ptr())
        elif want_x:
            dx.zero_()
        return dx, dw, db, None


def linear(x, weight, bias=None):
    """x (..., k) . weight (n, k)^T + bias (n) with both operands rounded to 8 bits, forward and backward; the result has x's type.

    Forward: x in 1 x 128 blocks of its rows, the weight in 128 x 128 tiles.  Backward, from dy rounded the same way: dx from the
    transposed tiles of the weight, dw from dy^T and x^T in 1 x 128 blocks along the batch, the bias gradient from dy itself.  What is kept
    for the backward pass are the 8-bit transposed operands, not x (without gradients nothing is prepared or kept; the weight is still
    quantised in every call: ``quantize`` it once and use ``matmul`` to serve).  x, weight and bias may each be fp32, bf16 or fp16."""
    _device_of('linear', x, weight, bias)
    if not (x.dim() and weight.dim() == 2 and x.shape[-1] == weight.shape[1]):
        raise ValueError("linear: x %s does not fit weight %s" % (tuple(x.shape), tuple(weight.shape)))
    if x.dtype not in DTYPES or weight.dtype not in DTYPES:
        raise ValueError("linear: x and weight are fp32, bf16 or fp16, got %s and %s" % (x.dtype, weight.dtype))
    if not weight.shape[1]:
        raise ValueError("linear: the weight has no columns")
    if bias is not None:
        if bias.dim() != 1 or bias.shape[0] != weight.shape[0] or bias.dtype not in DTYPES:
            raise ValueError("linear: the bias is (%d) in fp32, bf16 or fp16, got %s %s" % (weight.shape[0], tuple(bias.shape), bias.dtype))
        if not bias.is_contiguous():
            bias = bias.contiguous()
    return _Linear.apply(x, weight, bias, torch.is_grad_enabled())


def _norm_args(name, x, weight, residual, eps):
    _device_of(name, x, weight, residual)
    dt = x.dtype
    if dt not in DTYPES or not x.dim():
        raise ValueError("%s: x is fp32, bf16 or fp16 with at least one axis, got %s %s" % (name, tuple(x.shape), dt))
    n = x.shape[-1]
    if not n:
        raise ValueError("%s: the last axis is empty" % name)
    if weight.dim() != 1 or weight.shape[0] != n or (weight.dtype != dt and weight.dtype != torch.float32):
        raise ValueError("%s: the weight is (%d) in x's type or fp32, got %s %s" % (name, n, tuple(weight.shape), weight.dtype))
    if residual is not None and (residual.dtype != dt or residual.shape != x.shape):
        raise ValueError("%s: the residual has to be like x, %s %s" % (name, tuple(x.shape), dt))
    if not eps >= 0:
        raise ValueError("%s: eps is negative" % name)


def _norm(x, weight, residual, eps, eight):
    """-> y or None, h or None (shaped like x), codes, scales."""
    n = x.shape[-1]
    dev = x.device
    x2 = _flat_rows(x, n)
    r2 = _flat_rows(residual, n) if residual is not None else None
    if not weight.is_contiguous():
        weight = weight.contiguous()
    m = x2.shape[0]
    h = torch.empty(x.shape, dtype=x.dtype, device=dev) if r2 is not None else None
    y = q = s = None
    if eight:
        q, s = _codes_empty(m, n, dev), torch.empty((m, -(-n // BLOCK)), dtype=SCALES, device=dev)
    else:
        y = torch.empty(x.shape, dtype=x.dtype, device=dev)
    if m:
        dt = DTYPES[x.dtype]
        _run(x.get_device(), _lib.load().ml_rms_norm, x2.data_ptr(), _ld(x2), r2.data_ptr() if r2 is not None else None, _ld(r2) if r2 is not None else 0, dt,
             weight.data_ptr(), dt if weight.dtype == x.dtype else _lib.ML_F32, m, n, eps, h.data_ptr() if h is not None else None, n,
             y.data_ptr() if y is not None else None, n, q.data_ptr() if eight else None, _ld(q) if eight else 0, s.data_ptr() if eight else None, s.shape[1] if eight else 0)
    return y, h, q, s


@functools.lru_cache(maxsize=256)
def _norm_groups(m, n):
    return int(_lib.load().ml_rms_norm_backward_groups(m, n))


class _RmsNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, residual, eps):
        ctx.set_materialize_grads(False)
        ctx.eps = eps
        y, h, _, _ = _norm(x, weight, residual, eps, False)
        if h is None:
            ctx.save_for_backward(x, weight)
            return y
        ctx.save_for_backward(h, weight)
        return y, h

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, dh=None):
        h, weight = ctx.saved_tensors
        need_x, need_w, need_r, _ = ctx.needs_input_grad
        if dy is None:      # only h is used: it is a sum
            return dh if need_x else None, torch.zeros_like(weight) if need_w else None, dh if need_r else None, None
        n, dev = h.shape[-1], h.device
        dy2, h2 = _flat_rows(dy, n), _flat_rows(h, n)
        d2 = _flat_rows(dh, n) if dh is not None else None
        if not weight.is_contiguous():
            weight = weight.contiguous()
        m = h2.shape[0]
        dt = DTYPES[h.dtype]
        dx, dw = torch.empty(h.shape, dtype=h.dtype, device=dev), torch.empty((n,), dtype=weight.dtype, device=dev)
        work = torch.empty((_norm_groups(m, n) * n,), dtype=torch.float32, device=dev)
        _run(h.get_device(), _lib.load().ml_rms_norm_backward, dy2.data_ptr(), _ld(dy2), h2.data_ptr(), _ld(h2), d2.data_ptr() if d2 is not None else None,
             _ld(d2) if d2 is not None else 0, dt, weight.data_ptr(), dt if weight.dtype == h.dtype else _lib.ML_F32, m, n, ctx.eps, dx.data_ptr(), n, dw.data_ptr(),
             work.data_ptr())
        return dx if need_x else None, dw if need_w else None, dx if need_r else None, None


def rms_norm(x, weight, residual=None, eps=1e-6):
    """h / sqrt(mean(h^2) + eps) * weight over the last axis, h = x (+ residual), in x's type: y, or (y, h) with a residual.

    y comes from h before its rounding to x's type; h is what the next block adds to.  Differentiable in x, weight, residual (the
    gradient that reaches h is added inside the backward kernel).  x in fp32, bf16 or fp16, weight in x's type or fp32."""
    _norm_args('rms_norm', x, weight, residual, eps)
    return _RmsNorm.apply(x, weight, residual, float(eps))


def rms_norm_fp8(x, weight, residual=None, eps=1e-6):
    """The same with y as 8-bit blocks for ``matmul``: (codes, scales), or (codes, scales, h) with a residual; codes and scales are
    matrices of the flattened rows, h has x's shape.  For serving: not differentiable (a call that would need it is refused)."""
    _norm_args('rms_norm_fp8', x, weight, residual, eps)
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or (residual is not None and residual.requires_grad)):
        raise ValueError("rms_norm_fp8 is not differentiable: use rms_norm and linear, or torch.no_grad()")
    _, h, q, s = _norm(x, weight, residual, float(eps), True)
    return (q, s, h) if residual is not None else (q, s)
