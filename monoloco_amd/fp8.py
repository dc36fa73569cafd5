"""Operators of a residual block in 8 bits: quantisation into e4m3 blocks of 128, the block-scaled product, a linear layer on top of
it (forward and backward in 8 bits) and the root-mean-square norm with the residual's addition that feeds it.

The format (``include/monoloco_hip.h``): ``torch.float8_e4m3fn`` codes; 128 values share one ``torch.float8_e8m0fnu`` scale, the
smallest power of two with which their largest magnitude fits into 448.  A block is 1 x 128 of a row -- scales (rows, ceil(n / 128)) --
or 128 x 128 of a weight -- scales (ceil(rows / 128), ceil(n / 128)).  A block that holds a NaN or an infinity becomes NaN.

Plumbing as in ``engine.py``: torch holds the memory and the stream, the arithmetic is ``libmonoloco_hip.so``'s; every call runs on
the current stream of its tensors' device.  Wrong arguments raise ``ValueError``, failures inside the library ``MonolocoHipError``.
The reference has no such layers: its Linear layers are fp32 (monoloco/network/architectures.py:24-43)."""
import torch

from . import _lib
from ._lib import MonolocoHipError, check_ops
from .engine import _ptr, _stream

BLOCK = 128
CODES = torch.float8_e4m3fn
SCALES = torch.float8_e8m0fnu
DTYPES = {torch.float32: _lib.ML_F32, torch.bfloat16: _lib.ML_BF16, torch.float16: _lib.ML_F16}


def _blocks(n):
    return -(-n // BLOCK)


def _need(ok, text, *args):
    if not ok:
        raise ValueError(text % args)


def _device_of(name, *tensors):
    """The one device of the call's tensors."""
    dev = None
    for t in tensors:
        if t is None:
            continue
        _need(isinstance(t, torch.Tensor), "%s: expected tensors, got %s", name, type(t).__name__)
        if t.device.type != 'cuda':
            raise MonolocoHipError("%s runs on HIP devices only, got a tensor on %s (there is no CPU fallback)" % (name, t.device))
        _need(dev is None or t.device == dev, "%s: tensors on %s and on %s", name, dev, t.device)
        dev = t.device
    return dev


def _rows(t):
    """A matrix whose rows are contiguous and do not overlap (a copy where they are not)."""
    if t.numel() and ((t.shape[1] > 1 and t.stride(1) != 1) or (t.shape[0] > 1 and t.stride(0) < t.shape[1])):
        t = t.contiguous()
    return t


def _ld(t):
    """Row stride of such a matrix (of a single row: anything that is long enough)."""
    return t.stride(0) if t.shape[0] > 1 and t.numel() else max(t.shape[1], 1)


def _codes_empty(m, n, dev):
    """(m, n) codes whose rows start on 16 bytes: what the product loads in whole pieces."""
    return torch.empty((m, -(-n // 16) * 16), dtype=CODES, device=dev)[:, :n]


def _quantize(x, tile, straight=True, transposed=False, colsum=False):
    """-> q, scale, qt, scale_t, column sums per 128 rows (None where not asked for)."""
    m, n = x.shape
    dev = x.device
    x = _rows(x)
    q = s = qt = st = part = None
    if straight:
        q = _codes_empty(m, n, dev)
        s = torch.empty((_blocks(m) if tile else m, _blocks(n)), dtype=SCALES, device=dev)
    if transposed:
        qt = _codes_empty(n, m, dev)
        st = torch.empty((_blocks(n) if tile else n, _blocks(m)), dtype=SCALES, device=dev)
    if colsum:
        part = torch.empty((_blocks(m), n), dtype=torch.float32, device=dev)
    if x.numel():
        with torch.cuda.device(dev):
            check_ops(_lib.load().ml_fp8_quantize(
                _ptr(x), DTYPES[x.dtype], m, n, _ld(x), int(tile), _ptr(q), _ld(q) if straight else 0, _ptr(s), s.shape[1] if straight else 0,
                _ptr(qt), _ld(qt) if transposed else 0, _ptr(st), st.shape[1] if transposed else 0, _ptr(part), _stream(dev)))
    return q, s, qt, st, part


def quantize(x, block=(1, BLOCK), transposed=False):
    """x (m, n) in fp32, bf16 or fp16 -> (codes (m, n), scales) in blocks of (1, 128) or (128, 128).

    ``transposed=True``: (codes, scales, codes_t, scales_t) from one read of x: the same, and x^T (n, m) in blocks of ITS rows -- what a
    product needs that reduces over the other axis.  With (128, 128) blocks the transposed codes and scales are the straight ones,
    transposed.  Rows of the codes start on 16 bytes (a view of a wider buffer where n is no multiple of 16).  Not differentiable."""
    _device_of('quantize', x)
    _need(x.dim() == 2 and x.dtype in DTYPES, "quantize: needs a matrix in fp32, bf16 or fp16, got %s %s", tuple(x.shape), x.dtype)
    _need(tuple(block) in ((1, BLOCK), (BLOCK, BLOCK)), "quantize: blocks are (1, 128) or (128, 128), got %r", block)
    _lib.load()
    with torch.no_grad():
        q, s, qt, st, _ = _quantize(x.detach(), tuple(block) == (BLOCK, BLOCK), True, bool(transposed))
    return (q, s, qt, st) if transposed else (q, s)


def _scales_of(name, codes, scale):
    """-> is it a scale per tile (else per row)?"""
    _need(scale.dtype == SCALES, "matmul: %s_scale is %s, not %s", name, scale.dtype, SCALES)
    rows, k = codes.shape
    want = [(rows, _blocks(k)), (_blocks(rows), _blocks(k))]
    _need(tuple(scale.shape) in want, "matmul: %s_scale has shape %s; %s codes take %s (a scale per row and 128 columns) or %s (per 128 x 128)",
          name, tuple(scale.shape), (rows, k), want[0], want[1])
    return tuple(scale.shape) != want[0]


def _matmul(a, sa, a_tile, b, sb, b_tile, bias, out):
    m, n, k = a.shape[0], b.shape[0], a.shape[1]
    if m and n:
        a, b, sa, sb = _rows(a), _rows(b), _rows(sa), _rows(sb)
        dev = out.device
        with torch.cuda.device(dev):
            check_ops(_lib.load().ml_fp8_matmul(
                _ptr(a), _ld(a), _ptr(sa), _ld(sa), int(a_tile), _ptr(b), _ld(b), _ptr(sb), _ld(sb), int(b_tile),
                _ptr(bias), DTYPES[bias.dtype] if bias is not None else 0, _ptr(out), DTYPES[out.dtype], _ld(out), m, n, k, _stream(dev)))
    return out


def matmul(a, a_scale, b, b_scale, bias=None, out_dtype=torch.bfloat16, out=None):
    """a (m, k) . b (n, k)^T [+ bias (n)] of e4m3 codes with their block scales -> (m, n) in ``out_dtype`` (fp32, bf16, fp16), accumulated
    in fp32 and rounded once.  16-bit results come from the 8-bit matrix instructions (1.5e-5 of the result's norm beside the rounding), fp32
    results from exact bf16 operands at half the rate (4e-8; the operands' values have to lie in fp32's normal range, smaller ones count as 0).

    Each scale is (rows, ceil(k / 128)) or (ceil(rows / 128), ceil(k / 128)), as ``quantize`` gives them.  ``out``: an (m, n) tensor of one
    of the three types with contiguous rows to write into (``out_dtype`` is then its type).  Not differentiable: see ``linear``."""
    dev = _device_of('matmul', a, a_scale, b, b_scale, bias, out)
    _need(a.dim() == 2 and b.dim() == 2 and a.dtype == CODES and b.dtype == CODES, "matmul: a and b are matrices of %s, got %s %s and %s %s", CODES,
          tuple(a.shape), a.dtype, tuple(b.shape), b.dtype)
    _need(a.shape[1] == b.shape[1], "matmul: a has rows of %d, b of %d", a.shape[1], b.shape[1])
    a_tile, b_tile = _scales_of('a', a, a_scale), _scales_of('b', b, b_scale)
    m, n = a.shape[0], b.shape[0]
    if bias is not None:
        _need(tuple(bias.shape) == (n,) and bias.dtype in DTYPES, "matmul: the bias is (%d) in fp32, bf16 or fp16, got %s %s", n, tuple(bias.shape), bias.dtype)
        _need(not (bias.requires_grad and torch.is_grad_enabled()), "matmul is not differentiable: use linear, or detach the bias")
        bias = bias.detach().contiguous()
    if out is None:
        _need(out_dtype in DTYPES, "matmul: out_dtype is fp32, bf16 or fp16, got %s", out_dtype)
        out = torch.empty((m, n), dtype=out_dtype, device=dev)
    else:
        _need(tuple(out.shape) == (m, n) and out.dtype in DTYPES, "matmul: out is %s %s, needed (%d, %d) in fp32, bf16 or fp16", tuple(out.shape), out.dtype, m, n)
        _need(_rows(out) is out, "matmul: the rows of out have to be contiguous and apart")
        _need(not (out.requires_grad and torch.is_grad_enabled()), "matmul is not differentiable: out must not require a gradient")
        _matmul(a, a_scale, a_tile, b, b_scale, b_tile, bias, out)
        torch.autograd.graph.increment_version(out)
        return out
    return _matmul(a, a_scale, a_tile, b, b_scale, b_tile, bias, out)


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias):
        x2 = x.reshape(-1, x.shape[-1])
        need_x, need_w = ctx.needs_input_grad[0], ctx.needs_input_grad[1]
        qx, sx, qxt, sxt, _ = _quantize(x2, False, True, need_w)
        qw, sw, qwt, swt, _ = _quantize(weight, True, True, need_x)
        y = torch.empty((x2.shape[0], weight.shape[0]), dtype=x.dtype, device=x.device)
        _matmul(qx, sx, False, qw, sw, True, bias, y)
        ctx.save_for_backward(qxt, sxt, qwt, swt)
        ctx.like = (x.shape, x.dtype, weight.dtype, bias.dtype if bias is not None else None)
        return y.view(x.shape[:-1] + (weight.shape[0],))

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        need_x, need_w, need_b = ctx.needs_input_grad
        qxt, sxt, qwt, swt = ctx.saved_tensors
        xshape, xdt, wdt, bdt = ctx.like
        n, k = dy.shape[-1], xshape[-1]
        dev = dy.device
        dx = dw = db = None
        dy2 = dy.reshape(-1, n)
        m = dy2.shape[0]
        qd, sd, qdt, sdt, part = _quantize(dy2, False, need_x or not need_w, need_w, need_b)
        if need_x:
            dx = _matmul(qd, sd, False, qwt, swt, True, None, torch.empty((m, k), dtype=xdt, device=dev)).view(xshape)
        if need_w:
            dw = _matmul(qdt, sdt, False, qxt, sxt, False, None, torch.empty((n, k), dtype=wdt, device=dev))
        if need_b:
            db = torch.empty((n,), dtype=bdt, device=dev)
            with torch.cuda.device(dev):
                check_ops(_lib.load().ml_sum_rows(_ptr(part), part.shape[0], n, _ptr(db), DTYPES[bdt], _stream(dev)))
        return dx, dw, db


def linear(x, weight, bias=None):
    """x (..., k) . weight (n, k)^T + bias (n) with both operands rounded to 8 bits, forward and backward; the result has x's type.

    Forward: x in 1 x 128 blocks of its rows, the weight in 128 x 128 tiles.  Backward, from dy rounded the same way: dx from the
    transposed tiles of the weight, dw from dy^T and x^T in 1 x 128 blocks along the batch, the bias gradient from dy itself.  What is kept
    for the backward pass are the 8-bit transposed operands, not x.  x, weight and bias may each be fp32, bf16 or fp16."""
    _device_of('linear', x, weight, bias)
    _need(x.dim() >= 1 and weight.dim() == 2 and x.shape[-1] == weight.shape[1], "linear: x %s does not fit weight %s", tuple(x.shape), tuple(weight.shape))
    _need(x.dtype in DTYPES and weight.dtype in DTYPES, "linear: x and weight are fp32, bf16 or fp16, got %s and %s", x.dtype, weight.dtype)
    _need(weight.shape[1] > 0, "linear: the weight has no columns")
    if bias is not None:
        _need(tuple(bias.shape) == (weight.shape[0],) and bias.dtype in DTYPES, "linear: the bias is (%d) in fp32, bf16 or fp16, got %s %s",
              weight.shape[0], tuple(bias.shape), bias.dtype)
        bias = bias.contiguous()
    return _Linear.apply(x, weight, bias)


def _norm_args(name, x, weight, residual, eps):
    _device_of(name, x, weight, residual)
    _need(x.dim() >= 1 and x.dtype in DTYPES, "%s: x is fp32, bf16 or fp16 with at least one axis, got %s %s", name, tuple(x.shape), x.dtype)
    n = x.shape[-1]
    _need(n > 0, "%s: the last axis is empty", name)
    _need(tuple(weight.shape) == (n,) and weight.dtype in (x.dtype, torch.float32), "%s: the weight is (%d) in x's type or fp32, got %s %s", name, n,
          tuple(weight.shape), weight.dtype)
    _need(residual is None or (residual.shape == x.shape and residual.dtype == x.dtype), "%s: the residual has to be like x, %s %s", name, tuple(x.shape), x.dtype)
    _need(eps >= 0, "%s: eps is negative", name)
    _lib.load()


def _norm(x, weight, residual, eps, eight, want_h):
    """-> y or None, h or None, codes, scales."""
    n = x.shape[-1]
    dev = x.device
    x2 = _rows(x.reshape(-1, n))
    r2 = _rows(residual.reshape(-1, n)) if residual is not None else None
    weight = weight.contiguous()
    m = x2.shape[0]
    h = torch.empty((m, n), dtype=x.dtype, device=dev) if want_h else None
    y = q = s = None
    if eight:
        q, s = _codes_empty(m, n, dev), torch.empty((m, _blocks(n)), dtype=SCALES, device=dev)
    else:
        y = torch.empty((m, n), dtype=x.dtype, device=dev)
    if m:
        with torch.cuda.device(dev):
            check_ops(_lib.load().ml_rms_norm(
                _ptr(x2), _ld(x2), _ptr(r2), _ld(r2) if r2 is not None else 0, DTYPES[x.dtype], _ptr(weight), DTYPES[weight.dtype], m, n, float(eps),
                _ptr(h), n, _ptr(y), n, _ptr(q), _ld(q) if eight else 0, _ptr(s), s.shape[1] if eight else 0, _stream(dev)))
    return y, h, q, s


class _RmsNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, residual, eps):
        ctx.set_materialize_grads(False)
        y, h, _, _ = _norm(x, weight, residual, eps, False, residual is not None)
        ctx.eps = eps
        if residual is None:
            ctx.save_for_backward(x, weight)
            return y.view(x.shape)
        h = h.view(x.shape)
        ctx.save_for_backward(h, weight)
        return y.view(x.shape), h

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, dh=None):
        h, weight = ctx.saved_tensors
        need_x, need_w, need_r, _ = ctx.needs_input_grad
        if dy is None:      # only h is used: it is a sum
            return dh if need_x else None, torch.zeros_like(weight) if need_w else None, dh if need_r else None, None
        n, dev = h.shape[-1], h.device
        dy2, h2 = _rows(dy.reshape(-1, n)), _rows(h.reshape(-1, n))
        d2 = _rows(dh.reshape(-1, n)) if dh is not None else None
        weight = weight.contiguous()
        m = h2.shape[0]
        lib = _lib.load()
        dx, dw = torch.empty((m, n), dtype=h.dtype, device=dev), torch.empty((n,), dtype=weight.dtype, device=dev)
        work = torch.empty((int(lib.ml_rms_norm_backward_groups(m, n)) * n,), dtype=torch.float32, device=dev)
        with torch.cuda.device(dev):
            check_ops(lib.ml_rms_norm_backward(
                _ptr(dy2), _ld(dy2), _ptr(h2), _ld(h2), _ptr(d2), _ld(d2) if d2 is not None else 0, DTYPES[h.dtype], _ptr(weight), DTYPES[weight.dtype],
                m, n, float(ctx.eps), _ptr(dx), n, _ptr(dw), _ptr(work), _stream(dev)))
        dx = dx.view(h.shape)
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
    _need(not (torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, residual))),
          "rms_norm_fp8 is not differentiable: use rms_norm and linear, or torch.no_grad()")
    _, h, q, s = _norm(x, weight, residual, eps, True, residual is not None)
    return (q, s, h.view(x.shape)) if residual is not None else (q, s)
