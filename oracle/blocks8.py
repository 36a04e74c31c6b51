"""Oracle (test infrastructure): rows and weights in 8-bit blocks, the linear layer on them, LayerNorm and GELU with their
gradients, in float64 from the definitions."""
import torch

C2 = 2 * (2 / torch.pi) ** 0.5          # 2 sqrt(2 / pi)
A = 0.044715


def _pow2(n):
    return torch.ldexp(torch.ones_like(n, dtype=torch.float64), n.to(torch.int32))


def exponents(v, square=False):
    """Exponent of every block of v [R, K]: the smallest s >= -126 with max |finite v| <= 448 * 2^s, 0 for a block of zeros."""
    v = v.double()
    R, K = v.shape
    rb = 128 if square else 1
    m = torch.nn.functional.pad(torch.where(v.isfinite(), v.abs(), 0.0), (0, -K % 128, 0, -R % rb))
    top = m.view(m.shape[0] // rb, rb, m.shape[1] // 128, 128).amax((1, 3))
    s = torch.full_like(top, -126)
    for _ in range(400):
        s = torch.where(top > 448 * _pow2(s), s + 1, s)
    return torch.where(top == 0, 0.0, s)


def values(v, square=False):
    """What the blocks of v [R, K] hold, in float64 (NaN where v is not finite; 240 * 2^120 where it would round up to 2^128)."""
    v = v.double()
    R, K = v.shape
    s = exponents(v, square).repeat_interleave(128 if square else 1, 0)[:R].repeat_interleave(128, 1)[:, :K]
    a = v / _pow2(s)
    _, e = torch.frexp(a.abs().clamp_min(2.0 ** -6))
    step = _pow2(e - 4)                   # e4m3: 3 bits behind the leading one, subnormals below 2^-6
    q = torch.round(a / step) * step * _pow2(s)
    q = torch.where(q.abs() >= 2.0 ** 128, q.sign() * 240 * 2.0 ** 120, q)
    return torch.where(v.isfinite(), q, float("nan"))


def gelu(x):
    return x * torch.sigmoid(C2 * (x + A * x ** 3))


def gelu_slope(x):
    p = torch.sigmoid(C2 * (x + A * x ** 3))
    return torch.where(x.abs() > 20, (x > 0).double(), p + x * p * (1 - p) * C2 * (1 + 3 * A * x ** 2))


def ln_parts(x, eps):
    """(xh, r) of rows."""
    mean = x.mean(-1, keepdim=True)
    r = 1 / torch.sqrt(((x - mean) ** 2).mean(-1, keepdim=True) + eps)
    return (x - mean) * r, r


def ln_grads(dy, xh, r, w):
    """(dx, dy xh): dx of y = xh w + b from the normalised rows."""
    g = dy * w
    return r * (g - g.mean(-1, keepdim=True) - xh * (g * xh).mean(-1, keepdim=True)), dy * xh
