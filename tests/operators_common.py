"""64-bit references of the operators (deepity_b200/operators.py) with bounds on the rounding of a 32-bit
computation that stores float32 or bfloat16.

Every reference returns (value, bound).  U = 2^-24 is half a step of float32.  A sum of n products in
float32 is off by n * 2U of the sum of their magnitudes at most, whatever its order and even where the adder
truncates; a stored value by half a step of its type, ``half(dtype)`` of its magnitude."""
import torch

U = 2.0 ** -24
BLOCK = 128


def half(dtype):
    return torch.finfo(dtype).eps / 2


def check(got, want, what):
    """got within its bound of want = (value, bound); infinities and NaN in the same places."""
    value, bound = want
    got = got.double()
    assert got.shape == value.shape, (what, got.shape, value.shape)
    same = (got == value) | (got.isnan() & value.isnan())
    off = torch.where(same, 0.0, (got - value).abs())
    bad = ~(off <= torch.where(same, 1.0, bound))
    assert not bad.any(), (what, int(bad.sum()), "of", bad.numel(), "first", [int(i) for i in bad.nonzero()[0]],
                           "got", float(got[bad][0]), "want", float(value[bad][0]), "bound", float(bound[bad][0]))


# ------------------------------------------------------------------------------ vocabulary loss
def vocab_reference(hidden, weight, targets, bias, scale, ignore_index, grad=None):
    """{"loss", "lse"[, "hidden", "weight", "bias"]: (value, bound)} on 2-D tensors."""
    kind, width = hidden.dtype, hidden.shape[1]
    vocab = weight.shape[0]
    valid = (targets >= 0) & (targets < vocab) & (targets != ignore_index)
    h = torch.where(valid[:, None], hidden.double(), 0.0)
    w = weight.double()
    b = torch.zeros(vocab, dtype=torch.float64, device=w.device) if bias is None else bias.double()
    logits = scale * (h @ w.T) + b
    # the products: 6 of planes (or 1), each summed over the width; 16 roundings more for the planes, the scale
    # and log2(e), the bias, and the differences that are exponentiated
    mass = scale * (h.abs() @ w.abs().T)
    off = (6 * width + 16) * 2 * U * mass + 16 * U * torch.where(b.isinf(), 0.0, b.abs())
    top = off.amax(1)
    lse = torch.logsumexp(logits, 1)
    # exponentials good to 2^-21 (ex2 of a rounded argument), 2 roundings a term in sums of up to 32 and in the joins
    level = torch.where(lse.isfinite(), lse.abs(), 0.0)
    peak = logits.amax(1).abs()
    peak = torch.where(peak.isfinite(), peak, 0.0)
    d_lse = top + 2.0 ** -21 + (vocab / 128 + 128) * U + 16 * U * (level + peak)
    at = targets.clamp(0, vocab - 1)[:, None]
    picked = logits.gather(1, at)[:, 0]
    d_picked = off.gather(1, at)[:, 0] + 8 * U * torch.where(picked.isfinite(), picked.abs(), 0.0)
    zero = torch.zeros_like(lse)
    out = {"lse": (torch.where(valid, lse, zero), d_lse + 4 * U * level),
           "loss": (torch.where(valid, lse - picked, zero), d_lse + d_picked + 8 * U * (level + peak))}
    if grad is None:
        return out
    g = torch.where(valid, grad.double().expand_as(lse), 0.0)[:, None]
    p = torch.exp(logits - lse[:, None])
    hot = torch.zeros_like(p).scatter_(1, at, 1.0)
    s = torch.where(valid[:, None], g * (p - hot), 0.0)
    relative = off + (2 * d_lse + 2.0 ** -20)[:, None] + 16 * U * torch.where(logits.isfinite(), logits.abs(), 0.0)
    # (the exponent of an error of a few tenths is still below twice the error)
    d_s = g.abs() * (2 * p * relative) + 4 * U * g.abs() * (p + hot)
    d_s = d_s + (s.abs() + d_s) * (2.0 ** -8 if kind == torch.bfloat16 else 2.0 ** -23)
    d_s = torch.where(valid[:, None], d_s, 0.0)
    magnitude = s.abs() + d_s

    def product(value, mass_, d_, terms):
        bound = d_ + (6 * terms + 32) * 2 * U * mass_
        return value, bound + half(kind) * (value.abs() + bound)

    out["hidden"] = product(scale * (s @ w), scale * (magnitude @ w.abs()), scale * (d_s @ w.abs()), vocab)
    out["weight"] = product(scale * (s.T @ h), scale * (magnitude.T @ h.abs()), scale * (d_s.T @ h.abs()), len(h))
    out["bias"] = product(s.sum(0), magnitude.sum(0), d_s.sum(0), len(h))
    return out


# ------------------------------------------------------------------------------ residual norms
def _statistics(v, kind, eps):
    mean = v.mean(1, keepdim=True) if kind == "layer" else torch.zeros_like(v[:, :1])
    return mean, 1.0 / ((v - mean).square().mean(1, keepdim=True) + eps).sqrt()


def _standard(v, mag, mean, rstd):
    """(v - mean) * rstd with its magnitude."""
    return (v - mean) * rstd, (mag + mean.abs()) * rstd


#: Roundings of a 32-bit sum over a row (32 in a thread, 9 joins) and of the dozen operations around it.
ROW = 64 * U


def norm_reference(stream, branch, norm, post_norm, post_weight, post_bias, gate, a, b, pre_weight, pre_bias, eps):
    kind = stream.dtype
    x, width = stream.double(), stream.shape[1]
    stats = [torch.zeros(len(x), 1, dtype=torch.float64, device=x.device)] * 2
    new, mag = x, x.abs()
    if branch is not None:
        u = branch.double()
        mag_u = u.abs()
        if post_norm:
            stats = list(_statistics(u, norm, eps))
            u, mag_u = _standard(u, mag_u, *stats)
            if post_weight is not None:
                u, mag_u = u * post_weight.double(), mag_u * post_weight.double().abs()
            if post_bias is not None:
                u, mag_u = u + post_bias.double(), mag_u + post_bias.double().abs()
        if gate is not None:
            g = gate.double().reshape(-1, width)
            g = g.repeat_interleave(len(x) // len(g), 0)
            u, mag_u = u * g, mag_u * g.abs()
        new, mag = a * x + b * u, abs(a) * x.abs() + abs(b) * mag_u
    mean, rstd = _statistics(new, norm, eps)
    # an error of e * mag in every element moves the deviation by e * (the root mean square of mag) * rstd
    wide = 1.0 + mag.square().mean(1, keepdim=True).sqrt() * rstd
    h, mag_h = _standard(new, mag, mean, rstd)
    mag_h = (mag_h + mag.mean(1, keepdim=True) * rstd) * wide
    if pre_weight is not None:
        h, mag_h = h * pre_weight.double(), mag_h * pre_weight.double().abs()
    if pre_bias is not None:
        h, mag_h = h + pre_bias.double(), mag_h + pre_bias.double().abs()
    four = torch.cat([*stats, mean, rstd], 1)
    root = lambda v: v.square().mean(1, keepdim=True).sqrt()  # noqa: E731
    first = branch.double().abs() if branch is not None else mag
    d_four = ROW * torch.cat([root(first), stats[1] * (1 + root(first) * stats[1]), root(mag), rstd * wide], 1)
    return {"new": (new, ROW * mag + half(kind) * new.abs()), "normed": (h, 4 * ROW * mag_h + half(kind) * h.abs()),
            "stats": (four, 4 * d_four)}


def norm_backward_reference(d_normed, d_stream, new_stream, branch, stats, norm, post_norm, post_weight, post_bias,
                            gate, a, b, pre_weight, pre_bias):
    kind, (rows, width) = new_stream.dtype, new_stream.shape
    m1, r1, m2, r2 = stats.double().split(1, 1)
    one = torch.ones(width, dtype=torch.float64, device=new_stream.device)
    wn = one if pre_weight is None else pre_weight.double()
    wp = one if post_weight is None else post_weight.double()
    bp = 0 * one if post_bias is None else post_bias.double()
    dh = d_normed.double()

    def pull(q, mag_q, n, mag_n, r):
        mean = (lambda v: v.mean(1, keepdim=True)) if norm == "layer" else (lambda v: 0.0)
        value = r * (q - mean(q) - n * (q * n).mean(1, keepdim=True))
        return value, r * (mag_q + mean(mag_q) + mag_n * (mag_q * mag_n).mean(1, keepdim=True))

    def stored(value, mag):
        return value, 4 * ROW * mag + half(kind) * (value.abs() + 4 * ROW * mag)

    def summed(value, mag, dim=0):
        value, mag, n = value.sum(dim), mag.sum(dim), value.shape[dim]
        bound = (8 * ROW + 2 * n * U) * mag
        return value, bound + half(kind) * (value.abs() + bound)

    n, mag_n = _standard(new_stream.double(), new_stream.double().abs(), m2, r2)
    out = {"pre_weight": summed(dh * n, dh.abs() * mag_n), "pre_bias": summed(dh, dh.abs())}
    d, mag = pull(dh * wn, (dh * wn).abs(), n, mag_n, r2)
    if d_stream is not None:
        d, mag = d + d_stream.double(), mag + d_stream.double().abs()
    out["stream"] = stored(a * d, abs(a) * mag)
    if branch is None:
        return out
    y = branch.double()
    mag_y = y.abs()
    if post_norm:
        y, mag_y = _standard(y, mag_y, m1, r1)
    u, mag_u = (y * wp + bp, mag_y * wp.abs() + bp.abs()) if post_norm else (y, mag_y)
    s, mag_s = b * d, abs(b) * mag
    if gate is not None:
        g = gate.double().reshape(-1, width)
        shape = (len(g), rows // len(g), width)
        value, bound = summed((s * u).view(shape), (mag_s * mag_u).view(shape), 1)
        out["gate"] = value.view(gate.shape), bound.view(gate.shape)
        g = g.repeat_interleave(rows // len(g), 0)
        s, mag_s = s * g, mag_s * g.abs()
    if post_norm:
        out["post_weight"], out["post_bias"] = summed(s * y, mag_s * mag_y), summed(s, mag_s)
        s, mag_s = pull(s * wp, mag_s * wp.abs(), y, mag_y, r1)
    out["branch"] = stored(s, 2 * mag_s)
    return out


# ------------------------------------------------------------------------------ packed activations
def pack_reference(x):
    """Codes and scales by the definition, in float32 operations that round like the definition's."""
    x = x.float().cpu()
    rows, width = x.shape
    count = -(-width // BLOCK)
    blocks = torch.nn.functional.pad(x, (0, count * BLOCK - width)).view(rows, count, BLOCK)
    top = blocks.abs().amax(2)  # NaN where a block holds one
    some = (top >= 2.0 ** -100) & top.isfinite()
    factor = torch.full_like(top, 127.0) / top
    codes = torch.where(some[:, :, None], (blocks * factor[:, :, None]).round(), 0.0)
    scales = torch.where(some, top / torch.full_like(top, 127.0), 0.0)
    scales = torch.where(top.isfinite(), scales, float("nan"))
    return codes.view(rows, -1)[:, :width].to(torch.int8), scales


def unpack_reference(codes, scales):
    """In float64; the product of a code and a float32 scale."""
    return codes.double() * scales.double().repeat_interleave(BLOCK, 1)[:, :codes.shape[1]]


def activation_reference(act, x):
    """f(x), f'(x) in float64 and what a float32 evaluation from an exponential may be off by: tanh and the logistic
    function 2^-20, the others a few roundings."""
    if act == "relu":
        return x.clamp(min=0.0), (x > 0).double(), 0 * x, 0 * x
    if act == "linear":
        return x, torch.ones_like(x), 0 * x, 0 * x
    if act == "hard_tanh":
        return x.clamp(-1, 1), ((x > -1) & (x < 1)).double(), 0 * x, 0 * x
    if act == "esigmoid":
        a = 1 + x.abs()
        return 0.5 + 0.5 * x / a, 0.5 / (a * a), 8 * U + 0 * x, 8 * U / (a * a)
    e = 2.0 ** -20
    if act == "sigmoid":
        f = torch.sigmoid(x)
        return f, f * (1 - f), e + 0 * x, 2 * e + 0 * x
    if act == "tanh":
        f = torch.tanh(x)
        return f, 1 - f * f, e + 0 * x, 4 * e + 0 * x
    root = (2 / torch.pi) ** 0.5
    inner = root * (x + 0.044715 * x ** 3)
    t = torch.tanh(inner)
    slope = root * (1 + 3 * 0.044715 * x * x)
    # the argument's own rounding (constants of 32 bits among it) moves tanh by 8U |inner| (1 - t^2) <= 8U
    return (0.5 * x * (1 + t), 0.5 * (1 + t) + 0.5 * x * slope * (1 - t * t), (e + 8 * U) * (x.abs() + 1),
            (e + 8 * U) * (1 + 2 * x.abs() * slope))
