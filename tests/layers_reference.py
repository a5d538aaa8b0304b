"""Plain 64-bit forms of the layers on features, with a bound on what a kernel may
be off: values travel with the largest error that the kernel's arithmetic allows.

Roundings counted: an operand's type rounds by at most `half(type)` relative to the
value; a sum of n products in float32 is off by at most (n + 16) 2^-24 of the sum
of their magnitudes, in any order (n - 1 additions and a rounding each; 16 stands
for the products that the split of float32 operands leaves out, 3 at 2^-23 or
less, and for the additions beside the sum); an activation is evaluated to 16
units of float32 in its value and in its argument."""
import math

import torch

F32 = 2.0**-24
SLACK = 16
SLOPE = {torch.bfloat16: torch.float16}


def half(dtype):
    return torch.finfo(dtype).eps / 2


class Off:
    """A value in 64 bits and the most that the kernel's may differ from it."""

    def __init__(self, v, e=None):
        self.v = v.detach().double()
        self.e = torch.zeros_like(self.v) if e is None else e

    def t(self):
        return Off(self.v.t(), self.e.t())

    def rounded(self, dtype):
        # numbers below the type's smallest normal one are rounded by half its smallest step
        step = torch.finfo(dtype).smallest_normal * half(dtype)
        return Off(self.v, self.e + half(dtype) * (self.v.abs() + self.e) + step)

    def __add__(self, other):
        v = self.v + other.v
        return Off(v, self.e + other.e + F32 * v.abs())

    def __mul__(self, other):
        v = self.v * other.v
        return Off(v, self.v.abs() * other.e + self.e * other.v.abs() + self.e * other.e + 2 * F32 * v.abs())

    def __matmul__(self, other):
        a, b = self.v.abs(), other.v.abs()
        n = self.v.shape[1]
        e = a @ other.e + self.e @ b + self.e @ other.e + (n + SLACK) * F32 * (a @ b)
        return Off(self.v @ other.v, e)

    def column_sums(self):
        n = self.v.shape[0]
        return Off(self.v.sum(0), self.e.sum(0) + (n + SLACK) * F32 * self.v.abs().sum(0))


def check(got, want, dtype, what=""):
    """`want` (before it is rounded to the output's type) against the kernel's."""
    want = want.rounded(dtype)
    assert got.dtype == dtype and got.shape == want.v.shape, (what, got.dtype, got.shape, want.v.shape)
    off = (got.detach().double() - want.v).abs()
    worst = float((off / want.e.clamp(min=1e-300)).max()) if off.numel() else 0.0
    assert worst <= 1.0, f"{what}: {worst:.3g} times the bound"
    return worst


def derivatives(z, kind, a):
    """f, f', f'' and the largest magnitudes of f', f'' and f'''."""
    one = torch.ones_like(z)
    if kind == "relu":
        return z.clamp(min=0), (z > 0).double(), 0 * z, (1.0, 0.0, 0.0)
    if kind == "silu":
        p = torch.sigmoid(z)
        d = p * (1 - p)
        return z * p, p + z * d, d * (2 + z * (1 - 2 * p)), (1.1, 0.5, 0.5)
    if kind == "gelu":
        c, d = 0.5 * torch.erfc(-z / math.sqrt(2)), torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
        return z * c, c + z * d, d * (2 - z * z), (1.13, 0.8, 1.0)
    if kind == "softplus":
        p = torch.sigmoid(a * z)
        return torch.logaddexp(a * z, 0 * z) / a, p, a * p * torch.sigmoid(-a * z), (1.0, a / 4, a * a / 10)
    if kind == "sine":
        return torch.sin(a * z), a * torch.cos(a * z), -a * a * torch.sin(a * z), (a, a * a, a**3)
    return z, one, 0 * z, (1.0, 0.0, 0.0)


def activated(z, kind, a):
    f, d, dd, (l1, l2, l3) = derivatives(z.v, kind, a)
    near = z.e + SLACK * F32 * z.v.abs()   # the argument's own error and the evaluation's
    if kind == "relu":                     # the slope jumps where the sign is not certain
        jump = (z.v.abs() <= z.e).double()
        return Off(f, z.e), Off(d, jump), Off(dd)
    size = 1.0 if kind in ("none", "relu", "silu", "gelu") else (1.0 / a if kind == "softplus" else 1.0)
    return (Off(f, l1 * near + SLACK * F32 * (f.abs() + (0 if kind == "none" else size) * 2.0**-6)),
            Off(d, l2 * near + (0 if kind == "none" else SLACK * F32 * l1)),
            Off(dd, l3 * near + SLACK * F32 * l2))


def linear(x, w, b, kind="none", a=1.0, residual=None, x_scales=None, w_scales=None, units8=False):
    """(y, f'(z) as Off, f''(z), z) of operands in any type.  units8: the product of
    8-bit rows in the 8-bit units, which add eight products with the bits below 2^-13
    of the largest cut off: up to 2^-13 of the largest from each of the other seven,
    less than 2^-10 of the sum of their magnitudes."""
    z = Off(x) @ Off(w).t()
    if units8:
        z.e = z.e + 2.0**-10 * (x.double().abs() @ w.double().abs().t())
    if x_scales is not None:
        s = x_scales.double()[:, None] * w_scales.double()
        z = Off(z.v * s, (z.e + 2 * F32 * z.v.abs()) * s)
    if b is not None:
        z = z + Off(b)
    y, d, dd = activated(z, kind, a)
    if residual is not None:
        y = y + Off(residual)
    return y, d, dd, z


def linear_gradients(gy, x, w, d, kind, dtype):
    """(gx, gw, gb, gz): the slope is kept in float32 (fp16 for bf16, of a sine without its
    factor) and its product with gy rounded to the type."""
    gz = Off(gy) if kind == "none" else (Off(gy) * d.rounded(SLOPE.get(dtype, torch.float32))).rounded(dtype)
    return gz @ Off(w), gz.t() @ Off(x), gz.column_sums(), gz


def linear_second(gy, x, w, d, dd, gz, kind, dtype, u, of_w=None, of_b=None):
    """(of gy, of x, of w, of b) of <u, gx> + <of_w, gw> + <of_b, gb>."""
    t = None
    if of_w is not None:
        t = Off(x) @ Off(of_w).t()
        if of_b is not None:
            t = t + Off(of_b)
        t = t.rounded(dtype)
    elif of_b is not None:
        t = Off(of_b.expand(gy.shape))
    if u is not None:
        part = Off(u) @ Off(w).t()
        t = part if t is None else part + t
    q = (t * (Off(gy) * dd)).rounded(dtype)
    gx = q @ Off(w)
    if of_w is not None:
        gx = gx + (gz @ Off(of_w)).rounded(dtype)
    gw = q.t() @ Off(x)
    if u is not None:
        gw = gw + gz.t() @ Off(u)
    return t * d, gx, gw, q.column_sums()


def norm(x, w, residual, eps, dtype):
    """(y, s, 1 / sqrt(mean s^2 + eps)) of the rows."""
    s = Off(x) if residual is None else Off(x) + Off(residual)
    return unit(s, eps, w) + (s,)


def unit(s, eps, w):
    n = s.v.shape[1]
    mean = s.v.square().mean(1, keepdim=True) + eps
    i = mean.rsqrt()
    # half of the mean's own relative error, and a few steps of the root and the quotient
    off = ((n + SLACK) / 2 + 8) * F32 * i + i * (s.e * s.v.abs()).mean(1, keepdim=True) / mean
    i = Off(i.expand_as(s.v).contiguous(), off.expand_as(s.v).contiguous())
    weight = Off((torch.ones(n, device=s.v.device) if w is None else w).expand_as(s.v))
    return s * (i * weight), i
