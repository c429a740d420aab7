"""Root-mean-square norm and gradient clipping in 64 bits, on the CPU."""
import torch


def bf16(v: torch.Tensor) -> torch.Tensor:
    """The bf16 nearest to each f64, rounded once: 8 bits of it, ties to even, steps of 2^-133 below the least normal value."""
    step = torch.ldexp(torch.ones_like(v), torch.frexp(v).exponent.clamp(min=-125) - 8)
    return torch.where(torch.isfinite(v), torch.round(v / step) * step, v).to(torch.bfloat16)


def held(v: torch.Tensor, dtype) -> torch.Tensor:
    return bf16(v) if dtype == torch.bfloat16 else v.to(dtype)


def total(x, residual):
    """h, of the residual's type (of x's without one)."""
    return x if residual is None else held(x.double() + residual.double(), residual.dtype)


def rms_norm(h, weight, eps):
    """-> (y, 1 / sqrt(mean(h^2) + eps)) in f64."""
    h, w = h.double(), weight.double()
    r = 1 / torch.sqrt((h * h).mean(-1, keepdim=True) + eps)
    return h * r * w, r


def rms_norm_backward(h, weight, eps, dy, dh=None):
    """-> (gradient of h, gradient of the weight) in f64."""
    h, w, dy = h.double(), weight.double(), dy.double()
    r = 1 / torch.sqrt((h * h).mean(-1, keepdim=True) + eps)
    g = dy * w
    d = r * (g - h * r * r * (g * h).mean(-1, keepdim=True))
    return d if dh is None else d + dh.double(), (dy * h * r).sum(0)


def gradient_norm(grads):
    return torch.sqrt(sum(((g.double() * g.double()).sum() for g in grads), torch.zeros((), dtype=torch.float64)))


def clipped(grads, max_norm, norm=None):
    c = (max_norm / ((gradient_norm(grads) if norm is None else norm.double()) + 1e-6)).clamp(max=1.0)
    return [g.double() * c for g in grads]
