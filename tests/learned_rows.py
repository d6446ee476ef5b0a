"""What the tests of learned rows share: definitions in 64 bits with the error that each operator may make.

u is half a step of float32 (2^-24), the error of one float operation relative to its result; a result in type t is rounded once more, by at
most half a step of t relative to it, or half the smallest subnormal number."""
import torch

U = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def rounding(exact, dtype):
    """How far a correctly rounded value may be from `exact`; the second term holds below the smallest normal number."""
    info = torch.finfo(dtype)
    return exact.abs() * info.eps / 2 + info.tiny * info.eps / 2


def within(got, exact, error):
    """got is within its rounding of exact +- error (error: of the float32 result before it)."""
    assert got.shape == exact.shape
    diff = (got.double() - exact).abs()
    # the rounding acts on the float result, which is itself `error` off
    allowed = error * (1 + 2 * half_step(got.dtype)) + rounding(exact, got.dtype)
    worst = (diff - allowed).max().item() if diff.numel() else -1.0
    assert worst <= 0, f"{worst} beyond the bound"


def lookup(table, ids, scale, padding):
    flat = ids.reshape(-1)
    dead = torch.zeros_like(flat, dtype=torch.bool) if padding is None else flat == padding
    dead |= (flat < 0) | (flat >= table.shape[0])
    rows = table.double()[flat.masked_fill(dead, 0)] * scale if table.shape[0] else torch.zeros(flat.numel(), table.shape[1], dtype=torch.float64, device=ids.device)
    rows[dead] = 0
    return rows.view(*ids.shape, table.shape[1])


def sums(grad, ids, num_rows, scale, padding):
    """(exact gradient, error of sums in float32): m summands added in any order make at most (m - 1) u of the sum of their
    sizes, the scale and its own float rounding at most 2 u of the result; m u + 2 u covers it with the second-order
    terms below 2^24 / m."""
    flat, g = ids.reshape(-1), grad.reshape(ids.numel(), -1).double()
    live = (flat >= 0) & (flat < num_rows)
    if padding is not None:
        live &= flat != padding
    flat, g = flat[live], g[live]
    total = torch.zeros(num_rows, g.shape[1], dtype=torch.float64, device=g.device).index_add_(0, flat, g)
    size = torch.zeros_like(total).index_add_(0, flat, g.abs())
    count = torch.zeros(num_rows, dtype=torch.float64, device=g.device).index_add_(0, flat, torch.ones_like(flat, dtype=torch.float64))
    return total * scale, (count[:, None] + 2) * U * size * abs(scale) * 1.01


def order(experts, num_experts):
    key = experts.reshape(-1)
    dropped = (key < 0) | (key >= num_experts)
    key = key.masked_fill(dropped, num_experts)
    source = torch.sort(key, stable=True).indices
    place = torch.empty_like(source)
    place[source] = torch.arange(source.numel(), device=key.device)
    place = torch.where(dropped, ~place, place).view_as(experts)
    offsets = torch.searchsorted(key[source].contiguous(), torch.arange(num_experts + 1, device=key.device))
    return offsets, source, place


def brought(rows, place):
    place = place.view(place.shape[0], -1)
    got = rows.double()[place.clamp(min=0)] if rows.shape[0] else torch.zeros(*place.shape, rows.shape[1], dtype=torch.float64, device=rows.device)
    return torch.where((place < 0)[..., None], 0.0, got)


def combine(rows, place, weights):
    """(exact, error): K products, each off by u, and K - 1 additions."""
    b = brought(rows, place)
    K = b.shape[1]
    if weights is not None:
        w = weights.double().view(b.shape[0], K, 1)
        b = torch.where((place.view(b.shape[0], K) < 0)[..., None], 0.0, b * w)
    return b.sum(1), b.abs().sum(1) * (K + 1) * U * 1.01


def spread(x, place, weights):
    """(exact, error): one product."""
    place = place.view(place.shape[0], -1)
    T, K = place.shape
    v = x.double()[:, None, :].expand(T, K, -1)
    if weights is not None:
        v = v * weights.double().view(T, K, 1)
    v = torch.where((place < 0)[..., None], 0.0, v)
    rows = torch.empty(T * K, x.shape[1], dtype=torch.float64, device=x.device)
    rows[torch.where(place < 0, ~place, place).reshape(-1)] = v.reshape(T * K, -1)
    return rows, rows.abs() * U * 1.01


def weight_grads(grad, rows, place):
    """(exact, error): D products and D - 1 additions."""
    p = brought(rows, place) * grad.double()[:, None, :]
    D = grad.shape[1]
    return p.sum(2).view(place.shape), p.abs().sum(2).view(place.shape) * (D + 1) * U * 1.01
