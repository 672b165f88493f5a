"""Plain 64-bit forms of block quantisation, block-scaled contraction and linear cross entropy, with error bounds."""
import torch

FP8 = {28: (torch.float8_e4m3fn, 448.0, 3, -6), 29: (torch.float8_e5m2, 57344.0, 2, -14)}
TYPES = {0: torch.float32, 2: torch.float16, 14: torch.bfloat16}
FLOOR = 2.0 ** -100


def half_step(kind):
    return torch.finfo(kind).eps / 2


def spread(scale, block, shape):
    """A scale for each element from one for each block."""
    for i, (b, n) in enumerate(zip(block, shape)):
        if b > 1:
            scale = scale.repeat_interleave(b, i).narrow(i, 0, n)
    return scale


def round8(y, kind):
    """The 8-bit numbers (as float64) nearest to y, ties to even, saturated; NaN stays."""
    _, largest, bits, least = FP8[kind]
    _, e = torch.frexp(torch.where(torch.isfinite(y), y, torch.ones_like(y)))
    step = torch.exp2((e - 1).clamp(min=least).double() - bits)
    return (torch.round(y / step) * step).clamp(-largest, largest)


def quantize(x, block, kind):
    """(Q as float64, S as float32): the definition of htBlockQuantize."""
    _, largest, _, _ = FP8[kind]
    pad, view = [], []
    for n, b in zip(x.shape, block):
        pad = [0, -n % b] + pad
        view += [(n + b - 1) // b, b]
    a = torch.nn.functional.pad(x.float().abs(), pad).view(view)
    bad = a.isnan()
    a = torch.where(bad, torch.full_like(a, float("nan")), a).amax([2 * i + 1 for i in range(x.dim())])
    a = torch.where(a.isnan(), a, a.clamp(min=FLOOR)).double()
    s, r = (a / largest).float(), (largest / a).float()
    return round8(x.double() * spread(r, block, x.shape).double(), kind), s


def scaled(a, sa, blockA, b, sb, blockB, alpha, beta, c):
    """(D, bound of the f32 sums' error) of D[m, n] = alpha sum_k A B + beta C, k in blocks of 128."""
    x = a.double() * spread(sa, blockA, a.shape).double()
    y = b.double() * spread(sb, blockB, b.shape).double()
    d, mag = alpha * (x @ y.T), abs(alpha) * (x.abs() @ y.abs().T)
    k = a.shape[1]
    # a block: at most 128 exact products summed in f32, truncated in the worst case (a whole step, 2^-23, each); then two
    # scales, a sum over the blocks, alpha and beta
    bound = (min(k, 128) + (k + 127) // 128 + 6) * 2.0 ** -23 * mag
    if c is not None:
        d = d + beta * c.double()
        bound = bound + 2.0 ** -22 * (beta * c.double()).abs()
    return d, bound


def logits(h, w, alpha):
    """(z, bound of |error of z|): f32 sums of at most D exact products (f32 operands are sums of three bf16 numbers: what is left
    out is at most 2^-24 of a product, for which the bound has room)."""
    z = alpha * (h.double() @ w.double().T)
    mag = abs(alpha) * (h.double().abs() @ w.double().abs().T)
    per = (h.shape[1] + 4) * 2.0 ** -23 + (2.0 ** -20 if h.dtype == torch.float32 else 0)
    return z, per * mag


def loss(h, w, targets, alpha, ignore):
    """(loss, lse, bound of each)."""
    z, dz = logits(h, w, alpha)
    lse = torch.logsumexp(z, 1)
    at = targets.clamp(0, w.shape[0] - 1)[:, None]
    zt, keep = z.gather(1, at)[:, 0], targets != ignore
    # exp and log are good to 2^-21, a sum of V positive terms in pieces to 2^-18; lse is rounded twice
    blse = dz.amax(1) + 2.0 ** -18 + 2.0 ** -22 * lse.abs()
    bloss = blse + dz.gather(1, at)[:, 0] + 2.0 ** -22 * (zt.abs() + lse.abs())
    zero = torch.zeros_like(lse)
    return torch.where(keep, lse - zt, zero), lse, torch.where(keep, bloss, zero), blse


def gradient(h, w, targets, lse, g, alpha, ignore):
    """(dH, dW, bound of each) with lse as given; rows of ignored tokens count for nothing, whatever they hold."""
    kind, (t, _), v = h.dtype, h.shape, w.shape[0]
    keep = (targets != ignore) & (targets >= 0) & (targets < v)
    hz = torch.where(keep[:, None], h, torch.zeros_like(h))
    z, dz = logits(hz, w, alpha)
    x = z - torch.where(keep, lse, torch.zeros_like(lse)).double()[:, None]
    p = torch.exp(x) * keep[:, None]
    f = (torch.where(keep, g, torch.zeros_like(g)).double() * alpha)[:, None]
    hot = torch.zeros_like(p)
    hot[torch.arange(t, device=h.device)[keep], targets[keep]] = 1
    P = (p - hot) * f
    # p: error of the exponent (its own rounding 2^-23 |x|, exp 2^-21); P: rounded to the type (f16: behind a power of two
    # that leaves 2^-38 of the largest factor), f32's split drops 2^-20
    round_p = half_step(kind) if kind != torch.float32 else 2.0 ** -20
    eP = f.abs() * p * (dz + 2.0 ** -21 + 2.0 ** -22 * x.abs()) + P.abs() * (round_p + 2.0 ** -22)
    if kind == torch.float16:
        eP = eP + f.abs().max() * 2.0 ** -38
    else:
        # the smallest step of a bf16 number is 2^-133: a P rounded to one is off by at most half of it, an f32 P as a sum of
        # bf16 numbers by at most half of it in its last one, and another half where the product reads them
        eP = eP + 2.0 ** -133

    def product(P, eP, y, n):
        out, mag = P @ y, P.abs() @ y.abs()
        bound = eP @ y.abs() + (n + 8) * 2.0 ** -23 * mag + half_step(kind) * 1.01 * (out.abs() + eP @ y.abs())
        return out, bound + (2.0 ** -25 if kind == torch.float16 else 2.0 ** -130)

    dh, bh = product(P, eP, w.double(), v)
    dw, bw = product(P.T, eP.T, hz.double(), t)
    return dh, dw, bh, bw
