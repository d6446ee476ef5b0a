"""What the tests of products by expert and of dropout share: definitions in 64 bits with the error that each operator may make.

u is half a step of float32 (2^-24).  A sum of m products held in float: in any order each of the m products and of the m additions is off
by at most u of the running sum of sizes, or by 2 u where the addition cuts instead of rounding; float32 operands that are cut into
three parts leave at most 3 u of each product behind.  2 (m + 8) u of the sum of sizes covers all of it with the second-order terms."""
import torch

U = 2.0 ** -24
MASK32 = 0xFFFFFFFF


def bounds(offsets, num_rows):
    """The experts' rows as the operators take them: offsets brought into range, and none below an earlier one."""
    at = []
    for o in offsets.tolist():
        at.append(max(at[-1:] + [min(max(o, 0), num_rows)]))
    return list(zip(at, at[1:]))


def product(rows, weights, offsets):
    """(exact, error)"""
    out = torch.zeros(rows.shape[0], weights.shape[2], dtype=torch.float64, device=rows.device)
    size = torch.zeros_like(out)
    for e, (a, b) in enumerate(bounds(offsets, rows.shape[0])):
        out[a:b] = rows[a:b].double() @ weights[e].double()
        size[a:b] = rows[a:b].double().abs() @ weights[e].double().abs()
    return out, 2 * (rows.shape[1] + 8) * U * size


def grad_weights(rows, grad, offsets):
    """(exact, error)"""
    spans = bounds(offsets, rows.shape[0])
    out = torch.zeros(len(spans), rows.shape[1], grad.shape[1], dtype=torch.float64, device=rows.device)
    error = torch.zeros_like(out)
    for e, (a, b) in enumerate(spans):
        out[e] = rows[a:b].double().t() @ grad[a:b].double()
        error[e] = 2 * (b - a + 8) * U * (rows[a:b].double().abs().t() @ grad[a:b].double().abs())
    return out, error


def quantized(x):
    """(values, scales): the definition, bit for bit.  (A tensor divided by a Python number is multiplied with its reciprocal, which is not
    the quotient: the divisor is a tensor.)"""
    x = x.float()
    top = x.abs().amax(-1) if x.shape[-1] else torch.zeros(x.shape[:-1], device=x.device)
    scales = torch.where(top.isfinite(), top / torch.full_like(top, 127.0), torch.full_like(top, float("nan")))
    values = torch.round(x / scales[..., None]).clamp(-127, 127)
    return torch.where(scales[..., None] > 0, values, 0.0).to(torch.int8), scales


def product_int8(values, scales, weight_values, weight_scales, offsets):
    """(exact, error): whole numbers below 2^31 exactly, rounded to float once, and two products."""
    out = torch.zeros(values.shape[0], weight_values.shape[1], dtype=torch.float64, device=values.device)
    for e, (a, b) in enumerate(bounds(offsets, values.shape[0])):
        out[a:b] = (values[a:b].double() @ weight_values[e].double().t()) * scales[a:b, None].double() * weight_scales[e].double()
    return out, out.abs() * 3 * U * 1.01


def words(seed, blocks):
    """Philox4x32-10 of the counters (b, b >> 32, 0, 6) of `blocks`, an int64 tensor: [..., 4] 32-bit words."""
    k0, k1 = seed & MASK32, (seed >> 32) & MASK32
    c0, c1, c2, c3 = blocks & MASK32, blocks >> 32, torch.zeros_like(blocks), torch.full_like(blocks, 6)
    for _ in range(10):
        p0, p1 = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = ((p1 >> 32) & MASK32) ^ c1 ^ k0, p1 & MASK32, ((p0 >> 32) & MASK32) ^ c3 ^ k1, p0 & MASK32
        k0, k1 = (k0 + 0x9E3779B9) & MASK32, (k1 + 0xBB67AE85) & MASK32
    return torch.stack((c0, c1, c2, c3), -1)


def kept(seed, first, count, p, device="cuda"):
    """(which of the values first .. first + count stay, their factor)"""
    limit = int(p * 65536 + 0.5)
    blocks = torch.arange(first // 8, (first + count + 7) // 8, device=device)
    w = words(seed, blocks)
    halves = torch.stack((w & 0xFFFF, w >> 16), -1).reshape(-1)
    at = first - first // 8 * 8
    return halves[at:at + count] >= limit, 65536 / (65536 - limit) if limit < 65536 else 0.0


def dropout(x, p, seed):
    """(exact, error): the factor is rounded to float, the product too."""
    stay, factor = kept(seed, 0, x.numel(), p, x.device)
    out = torch.where(stay.view(x.shape), x.double() * factor, 0.0)
    return out, torch.where(out.isfinite(), out.abs() * 2 * U * 1.01, 0.0)
