"""Plain 64-bit forms of the 8-bit residual-block operators (CPU tensors), for the tests of monoloco_amd.fp8 and monoloco_amd.train.adamw."""
import torch

B = 128


def pow2(e):
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def floor_log2(x):
    return (x.contiguous().view(torch.int64) >> 52) - 1023


def scale_bytes(amax):
    """e8m0 byte of a block whose largest magnitude is amax (fp64 tensor): 127 for zeros, 255 for what is not finite, at least 1."""
    e = floor_log2(amax.clamp(min=2.0 ** -1000)) - 8
    e = e + (448 * pow2(e) < amax).long()
    b = (e + 127).clamp(min=1)
    b = torch.where(amax == 0, torch.full_like(b, 127), b)
    return torch.where(torch.isfinite(amax), b, torch.full_like(b, 255))


def scale_values(byte):
    byte = byte.long()
    return torch.where(byte == 255, torch.full(byte.shape, float('nan'), dtype=torch.float64), pow2(byte - 127))


def step_of(y):
    return pow2(floor_log2(y.abs().clamp(min=2.0 ** -6)) - 3)


def nearest(y):
    s = step_of(y)
    return torch.round(y / s) * s


def _amax(x, tile):
    m, n = x.shape
    pad = torch.nn.functional.pad(x.abs(), (0, -n % B, 0, -m % B if tile else 0)).nan_to_num(nan=float('inf'), posinf=float('inf'))
    a = pad.view(pad.shape[0], -1, B).amax(-1)
    return a.view(-1, B, a.shape[1]).amax(1) if tile else a


def spread(s, m, n, tile):
    s = s.repeat_interleave(B, 1)[:, :n]
    return s.repeat_interleave(B, 0)[:m] if tile else s


def quantize(x, tile=False):
    """-> code values (fp64; NaN in a block that is not finite), scale bytes."""
    x = x.double()
    b = scale_bytes(_amax(x, tile))
    sv = spread(scale_values(b), *x.shape, tile)
    return torch.where(torch.isnan(sv), sv, nearest(x.nan_to_num() / sv)), b


def values(codes, byte, tile=False):
    return codes.double() * spread(scale_values(byte.long()), codes.shape[0], codes.shape[1], tile)


def rounded(x, tile=False):
    return values(*quantize(x, tile), tile)


def rms_norm(x, w, r, eps):
    h = x.double() + (r.double() if r is not None else 0)
    return h / torch.sqrt((h * h).mean(-1, keepdim=True) + eps) * w.double(), h


def rms_norm_backward(dy, h, w, dh, eps):
    """-> dx, dw, and the sums of magnitudes that their rounding errors are measured against."""
    dy, h, w = dy.double(), h.double(), w.double()
    dh = dh.double() if dh is not None else torch.zeros_like(h)
    rstd = 1 / torch.sqrt((h * h).mean(-1, keepdim=True) + eps)
    g = dy * w
    dx = rstd * (g - h * rstd ** 2 * (g * h).mean(-1, keepdim=True)) + dh
    adx = rstd * (g.abs() + h.abs() * rstd ** 2 * (g * h).abs().mean(-1, keepdim=True)) + dh.abs()
    return dx, (dy * h * rstd).sum(0), adx, (dy * h * rstd).abs().sum(0)


def mix32(x):
    x = x ^ (x >> 16)
    x = (x * 0x7feb352d) & 0xffffffff
    x = x ^ (x >> 15)
    x = ((x >> 16) * 0x846ca68b % 65536 * 65536 + (x & 0xffff) * 0x846ca68b) & 0xffffffff
    return x ^ (x >> 16)


def bits(seed, step, index, n):
    key = mix32((seed + 0x9e3779b9 * mix32((step + 0x85ebca6b * (index + 1)) & 0xffffffff)) & 0xffffffff)
    i = torch.arange(n, dtype=torch.int64)
    blk = torch.tensor([mix32(int((key + b * 0x9e3779b9) & 0xffffffff)) for b in range(-(-n // B))], dtype=torch.int64)
    mul = torch.tensor([(j * 0x85ebca6b) & 0xffffffff for j in range(B)], dtype=torch.int64)
    return mix32((blk.repeat_interleave(B)[:n] + mul.repeat(len(blk))[:n]) & 0xffffffff)


def stochastic(x, u16, positive):
    """-> code values, scale bytes of a flat fp64 tensor."""
    n = x.numel()
    byte = scale_bytes(_amax(torch.nn.functional.pad(x, (0, -n % B)).view(-1, B), False).reshape(-1))
    y = x / scale_values(byte).repeat_interleave(B)[:n]
    s = step_of(y)
    q = torch.floor(y.abs() / s + u16.double() / 65536) * s
    if positive:
        q = torch.where((y > 0) & (q == 0), torch.full_like(q, 2.0 ** -9), q)
    return torch.sign(y) * q, byte


def adamw(p, g, m, v, step, lr, betas, eps, weight_decay):
    b1, b2 = betas
    m2, v2 = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
    den = torch.sqrt(v2 / (1 - b2 ** step)) + eps
    return p * (1 - lr * weight_decay) - lr / (1 - b1 ** step) * m2 / den, m2, v2, (b1 * m).abs() + ((1 - b1) * g).abs(), lr / (1 - b1 ** step) / den
