"""MXFP4 in 64 bits, for the tests: quantization, values, and the bounds an
fp32-accumulating product may be off by."""
import torch

GRID = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def pow2(e):
    return torch.ldexp(torch.ones(e.shape, dtype=torch.float64), e)


def scale_exponent(amax):
    """floor(log2(amax)) - 2, not below -127; -127 for 0 (fp64 in, int out)."""
    m, ex = torch.frexp(amax)
    return torch.where(amax > 0, (ex - 3).clamp(min=-127), torch.full_like(ex, -127)).int()


def round_e2m1(y):
    """Nearest E2M1 value (ties to the even code), saturating; fp64."""
    a = y.abs()
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0)).double()
    return (torch.round(a / step) * step).clamp(max=6.0) * torch.where(y < 0, -1.0, 1.0)


def quantize(x):
    """(values fp64, scale bytes) of finite ``x`` [R, K] on the CPU."""
    b = x.detach().cpu().double().view(x.shape[0], -1, 32)
    e = scale_exponent(b.abs().amax(-1))
    unit = pow2(e)[..., None]
    return (round_e2m1(b / unit) * unit).view(x.shape), (e + 127).to(torch.uint8)


def unblock(flat, rows, cols):
    rb, cb = -(-rows // 128), -(-cols // 4)
    t = flat.cpu().view(rb, cb, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(rb * 128, cb * 4)
    return t


def values(q, scales):
    """fp64 values of packed codes [R, K/2] and row-major scale bytes [R, K/32]."""
    q = q.cpu()
    c = torch.stack([q & 15, q >> 4], -1).view(q.shape[0], -1).long()
    v = GRID[c & 7].double() * torch.where(c >= 8, -1.0, 1.0)
    return (v.view(q.shape[0], -1, 32) * pow2(scales.int() - 127)[..., None]).view(c.shape)


def product(a, b):
    """(a @ b.T, error bound of its fp32 accumulation): the products are exact
    in fp32, each of the K additions is off by at most one step of the running
    sum (2^-23 of its magnitude, truncation included)."""
    return a @ b.T, a.shape[1] * 2.0 ** -23 * (a.abs() @ b.abs().T)


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def gelu(v):
    return 0.5 * v * (1 + torch.tanh((2 / torch.pi) ** 0.5 * (v + 0.044715 * v ** 3)))


def swiglu_bounded(v, dv, g, dg):
    """h = v * silu(g) and how far an fp32 evaluation may be off: the inputs'
    own errors (|silu'| <= 1.1), and per evaluation the exponential's
    2 + 1.18 |g| steps plus four more roundings of 2^-23."""
    s = g * torch.sigmoid(g)
    h = v * s
    return h, s.abs() * dv + 1.1 * (v.abs() + dv) * dg + (6 + 1.18 * g.abs()) * 2.0 ** -23 * h.abs()


def quantize_bounded(h, dh):
    """Values of h's quantization and, per element, how far those of any
    h' with |h' - h| <= dh may be from them: 0 away from every rounding and
    scale boundary."""
    q, _ = quantize(h)
    far = torch.zeros_like(q)
    hb, db = (t.view(t.shape[0], -1, 32) for t in (h, dh))
    top, slack = hb.abs().amax(-1), db.amax(-1)
    for amax in ((top - slack).clamp(min=0), top + slack):
        unit = pow2(scale_exponent(amax))[..., None]
        for x in (hb - db, hb + db):
            far = torch.maximum(far, (round_e2m1(x / unit) * unit - q.view(hb.shape)).abs()
                                .view(q.shape))
    return q, far
