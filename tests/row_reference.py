"""Plain 64-bit forms of the row operators (gradient norm and clip, RMS norm with residual, 8-bit
rows with block scales and their product), written from their definitions on CPU tensors."""
import torch

BLOCK = 128
MAX8 = {torch.float8_e4m3fn: 448.0, torch.float8_e5m2: 57344.0}
LEAST8 = {torch.float8_e4m3fn: (-6, 3), torch.float8_e5m2: (-14, 2)}  # least exponent, bits behind it


def half_step(dtype):
    """Largest relative error of one rounding to dtype."""
    return torch.finfo(dtype).eps / 2


def two(e):
    return ((e.long() + 1023) << 52).view(torch.float64)


def _scale_exponent(top, dtype):
    """The least e >= -126 with top * 2^-e inside the format; 0 for a block of zeros."""
    x = torch.frexp(top)[1]
    e = x - (9 if dtype == torch.float8_e4m3fn else 16)
    e = torch.where(top > MAX8[dtype] * two(e), e + 1, e)
    return torch.where(top == 0, torch.zeros_like(e), e.clamp(min=-126))


def quantise(v, dtype=torch.float8_e4m3fn, h=1):
    """v [R, C] -> (values on the 8-bit grid [R, C] f64, exponents [ceil(R / h), ceil(C / 128)])."""
    v = v.double().cpu()
    R, C = v.shape
    p = torch.nn.functional.pad(v, (0, -C % BLOCK, 0, -R % h))
    b = p.reshape(p.shape[0] // h, h, p.shape[1] // BLOCK, BLOCK)
    fin = torch.where(torch.isfinite(b), b.abs(), torch.zeros_like(b))
    top = fin.amax(dim=(1, 3))
    e = _scale_exponent(top, dtype)
    u = b * two(-e)[:, None, :, None]
    low, bits = LEAST8[dtype]
    mag = torch.where(torch.isfinite(u), u.abs(), torch.zeros_like(u)).clamp(min=2.0 ** low)
    step = two(torch.frexp(mag)[1] - 1 - bits)
    q = torch.round(u / step) * step
    q = torch.where(torch.isfinite(b), q, torch.full_like(q, float("nan")))
    return q.reshape(p.shape)[:R, :C], e


def value(q, e, h=1):
    """What 8-bit rows stand for."""
    s = two(e).repeat_interleave(BLOCK, 1)[:, :q.shape[1]]
    return q.double().cpu() * s.repeat_interleave(h, 0)[:q.shape[0]]


def rms_norm(x, weight, eps, residual=None):
    h = x.double().cpu()
    if residual is not None:  # the stored sum is what is normed
        h = (h + residual.double().cpu()).to(x.dtype).double()
    inv = (h.pow(2).mean(-1, keepdim=True) + eps) ** -0.5
    y = h * inv
    return (y if weight is None else y * weight.double().cpu()), h, inv


def rms_norm_bwd(h, weight, inv, dy, dh=None):
    dy = dy.double().cpu()
    g = dy if weight is None else dy * weight.double().cpu()
    dx = inv * (g - h * inv ** 2 * (g * h).mean(-1, keepdim=True))
    if dh is not None:
        dx = dx + dh.double().cpu()
    return dx, (dy * h * inv).reshape(-1, h.shape[-1]).sum(0)


def clip(grads, max_norm, p=2.0):
    flat = torch.cat([g.double().cpu().reshape(-1) for g in grads])
    total = flat.abs().max() if p == float("inf") else flat.abs().pow(p).sum() ** (1.0 / p)
    c = torch.clamp(max_norm / (total + 1e-6), max=1.0)
    return total, [g.double().cpu() * c for g in grads]
