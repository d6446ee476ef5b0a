"""Dropout without a stored mask, against its definition, and a layer of all that runs over rows sorted by expert."""
import pytest
import torch

import expert_products as exact
import learned_rows
from learned_rows import within

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


@pytest.fixture(scope="module")
def ops():
    from graph_sampling_b200 import ops as m
    return m


@pytest.fixture(scope="module")
def nn():
    from graph_sampling_b200.gs import nn as m
    return m


def generator(seed):
    g = torch.Generator("cuda")
    g.manual_seed(seed)
    return g


def normal(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(1,), (7,), (8,), (9,), (1000, 3), (33, 1024), (257, 602), (5, 6, 7, 8), (1, 1_000_003), (4096, 513)])
def test_dropout(ops, dtype, shape):
    x = normal(generator(shape[0]), *shape, dtype=dtype)
    for p in (0.0, 0.1, 0.5, 0.999, 1.0):
        for seed in (0, 12_345, 2 ** 64 - 1):
            out = ops.dropout(x, p, seed)
            assert out.dtype == dtype and out.shape == x.shape
            within(out, *exact.dropout(x, p, seed))
    assert torch.equal(ops.dropout(x, 0.0, 5), x) and int(torch.count_nonzero(ops.dropout(x, 1.0, 5))) == 0


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides_and_addresses(ops, dtype):
    g = generator(2)
    big = normal(g, 300, 120, dtype=dtype)
    for x in (big[:, :64], big[:, 8:72], big[:, 1:66], big[::3, 4:68], big.t(), big[:, ::2], big[:1].expand(9, 120), big[:, :1].expand(300, 7), big[5:6, 3:50],
              big.view(-1)[1:], big.view(30, 10, 120)[:, :, 3:9], big[7, 9]):
        within(ops.dropout(x, 0.3, 99), *exact.dropout(x, 0.3, 99))


@pytest.mark.parametrize("dtype", DTYPES)
def test_widths_of_an_access(ops, dtype):
    """Rows and runs that begin on 32-byte boundaries, on 16-byte ones, and end a block after the last whole access."""
    big = normal(generator(12), 303, 128, dtype=dtype)
    for x in (big[:, 16:80], big[:, 16:88], big[:, 8:72], big.view(-1)[16:], big.view(-1)[8:], big.view(-1)[4:], big.view(-1)[:24], big.view(-1)[:2000 * 8 + 8],
              big.view(-1)[16:16 + 4096 * 8 + 13], big[::2, :64], big[1::2, 64:]):
        within(ops.dropout(x, 0.3, 98), *exact.dropout(x, 0.3, 98))


@pytest.mark.parametrize("dtype", DTYPES)
def test_dropped_values_do_not_count(ops, nn, dtype):
    stay, _ = exact.kept(3, 0, 5000, 0.4)
    for value in (float("nan"), float("inf"), -float("inf")):
        x = torch.where(stay, 1.0, value).to(dtype)
        out = ops.dropout(x, 0.4, 3)
        assert out.isfinite().all() and torch.all(out[~stay] == 0) and torch.all(out[stay] > 1)
        x = torch.where(stay, value, 1.0).to(dtype)
        assert torch.all(ops.dropout(x, 0.4, 3).isfinite() == ~stay)
        leaf = torch.ones(5000, dtype=dtype, device="cuda", requires_grad=True)
        grad, = torch.autograd.grad(nn.dropout(leaf, 0.4, 3), leaf, torch.where(stay, 1.0, value).to(dtype))
        assert grad.isfinite().all() and torch.all(grad[~stay] == 0)


def test_share_of_dropped_values(ops):
    """6.4 M draws with probability p, rounded to 2^-16: their share is within 6 standard deviations of it."""
    x = torch.ones(6_400_000, device="cuda")
    for p in (0.001, 0.1, 0.37, 0.9):
        q = int(p * 65536 + 0.5) / 65536
        dropped = float((ops.dropout(x, p, 17) == 0).double().mean())
        assert abs(dropped - q) < 6 * (q * (1 - q) / x.numel()) ** 0.5
    a, b = ops.dropout(x, 0.5, 1) == 0, ops.dropout(x, 0.5, 2) == 0
    assert abs(float((a & b).double().mean()) - 0.25) < 6 * (0.25 * 0.75 / x.numel()) ** 0.5


def test_seeds(ops, nn):
    x = torch.ones(10_000, device="cuda")
    ops.set_seed(4)
    first, second = ops.dropout(x, 0.5), ops.dropout(x, 0.5)
    assert not torch.equal(first, second)
    ops.set_seed(4)
    assert torch.equal(ops.dropout(x, 0.5), first) and torch.equal(nn.dropout(x, 0.5), second)
    ops.set_seed(7777)
    assert torch.equal(ops.dropout(x, 0.5, 2 ** 64 + 3), ops.dropout(x, 0.5, 3))
    seed = torch.tensor([3], device="cuda")
    assert torch.equal(ops.dropout(x, 0.5, seed), ops.dropout(x, 0.5, 3)) and torch.equal(ops.dropout(x, 0.5, seed[0]), ops.dropout(x, 0.5, 3))
    seed.fill_(-1)
    assert torch.equal(ops.dropout(x, 0.5, seed), ops.dropout(x, 0.5, 2 ** 64 - 1))
    leaf = x.clone().requires_grad_()
    out = nn.dropout(leaf, 0.5, seed)
    grad, = torch.autograd.grad(out, leaf, torch.ones_like(x), retain_graph=True)
    assert torch.equal(grad, out.detach())
    seed.add_(1)                                                              # the backward pass would draw another mask
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(out, leaf, torch.ones_like(x))
    for bad in (seed.float(), seed.int(), torch.zeros(2, dtype=torch.int64, device="cuda"), seed.cpu()):
        with pytest.raises(TypeError, match="seed"):
            ops.dropout(x, 0.5, bad)
    for p in (-0.1, 1.1, float("nan")):
        with pytest.raises(TypeError, match="between 0 and 1"):
            ops.dropout(x, p, 1)
        with pytest.raises(TypeError, match="between 0 and 1"):
            nn.dropout(leaf, p, 1)


@pytest.mark.parametrize("dtype", DTYPES)
def test_gradient(nn, dtype):
    g = generator(4)
    x, up = normal(g, 100, 77, dtype=dtype).requires_grad_(), normal(g, 100, 77, dtype=dtype)
    out = nn.dropout(x, 0.25, 8)
    within(out.detach(), *exact.dropout(x.detach(), 0.25, 8))
    grad, = torch.autograd.grad(out, x, up, create_graph=True)
    within(grad.detach(), *exact.dropout(up, 0.25, 8))
    with pytest.raises(RuntimeError, match="cannot be differentiated again"):
        up.requires_grad_()
        again, = torch.autograd.grad(nn.dropout(x, 0.25, 8), x, up, create_graph=True)
        torch.autograd.grad(again.sum(), up)
    everywhere, = torch.autograd.grad(nn.dropout(x, 0.25, 8).sum(), x)          # a gradient of one value, broadcast
    within(everywhere, *exact.dropout(torch.ones_like(up.detach()), 0.25, 8))


def test_positions_beyond_32_bits(ops):
    if torch.cuda.mem_get_info()[0] < 30 << 30:
        pytest.skip("needs 30 GB")
    count = (1 << 32) + 4099
    x = torch.ones(count, dtype=torch.bfloat16, device="cuda")
    out = ops.dropout(x, 0.5, 21)
    for first, some in ((0, 5000), ((1 << 31) - 100, 300), ((1 << 32) - 100, 4199)):
        stay, factor = exact.kept(21, first, some, 0.5)
        assert torch.equal(out[first:first + some] != 0, stay)


def test_captured_with_a_seed_on_the_device(ops):
    x, seed = torch.ones(70_000, device="cuda"), torch.tensor([1], device="cuda")
    ops.dropout(x, 0.5, seed)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        seed.add_(1)
        out = ops.dropout(x, 0.5, seed)
    for turn in range(3):
        graph.replay()
        assert torch.equal(out, ops.dropout(x, 0.5, int(seed))) and int(seed) == turn + 2


# ---- a layer ---------------------------------------------------------------------------------------------------------------------
def layer(nn, x, experts, weights, up, down, p, seed):
    order = nn.expert_order(experts, up.shape[0])
    hidden = nn.dropout(nn.product(nn.dispatch(x, order), up, order), p, seed)
    return nn.combine(nn.product(hidden, down, order), order, weights), order


def plain_layer(x, order, weights, up, down, p, seed):
    """The same in 64 bits."""
    place = order.place
    T, K = place.shape
    rows = torch.zeros(T * K, x.shape[1], dtype=torch.float64, device="cuda")
    rows = rows.index_copy(0, torch.where(place < 0, ~place, place).flatten(), torch.where((place < 0)[..., None], 0.0, x[:, None].expand(T, K, -1)).flatten(0, 1))
    spans = exact.bounds(order.offsets, T * K)

    def product(r, w):
        rest = torch.zeros(T * K - spans[-1][1], w.shape[2], dtype=torch.float64, device="cuda")
        return torch.cat([r[a:b] @ w[e] for e, (a, b) in enumerate(spans)] + [rest])
    hidden = product(rows, up)
    stay, factor = exact.kept(seed, 0, hidden.numel(), p)
    hidden = torch.where(stay.view_as(hidden), hidden * factor, 0.0)
    out = product(hidden, down)
    back = torch.where((place < 0)[..., None], 0.0, out[place.clamp(min=0)])
    return (back * weights[..., None]).sum(1)


@pytest.mark.parametrize("tokens,per_token,experts,width,inner", [(1, 2, 4, 64, 96), (37, 2, 8, 64, 128), (200, 3, 5, 47, 90), (513, 4, 16, 128, 256)])
def test_layer(nn, tokens, per_token, experts, width, inner):
    """float32 throughout: the loss of accuracy of two products and their gradients is some 1e-6 of the largest values."""
    g = generator(tokens)
    ids = torch.rand(tokens, experts, generator=g, device="cuda").topk(per_token, 1).indices
    ids[torch.rand(tokens, generator=g, device="cuda") < 0.1] = -1
    x = normal(g, tokens, width).requires_grad_()
    weights = torch.rand(tokens, per_token, generator=g, device="cuda").requires_grad_()
    up = (normal(g, experts, width, inner) * width ** -0.5).requires_grad_()
    down = (normal(g, experts, inner, width) * inner ** -0.5).requires_grad_()
    grad = normal(g, tokens, width)
    out, order = layer(nn, x, ids, weights, up, down, 0.2, 77)
    wanted = (x, weights, up, down)
    got = torch.autograd.grad(out, wanted, grad)
    wide = [t.detach().double().requires_grad_() for t in wanted]
    want = plain_layer(wide[0], order, wide[1], wide[2], wide[3], 0.2, 77)
    grads = torch.autograd.grad(want, wide, grad.double())
    # a chain of sums of at most 2 max(width, inner, rows) products each: every one adds 2 (m + 8) u of what it sums in sizes, which are
    # at most some m^1/2 times the result's own size
    m = max(width, inner, tokens * per_token)
    for a, b in zip((out.detach(), *got), (want.detach(), *grads)):
        assert (a.double() - b).abs().max() <= 8 * (m + 8) * exact.U * max(1.0, b.abs().max().item()) * m ** 0.5


def test_layer_captured_and_replayed(nn):
    g = generator(12)
    ids = torch.randint(-1, 6, (64, 2), generator=g, device="cuda")
    x, weights = normal(g, 64, 64), torch.rand(64, 2, generator=g, device="cuda")
    up, down, grad = normal(g, 6, 64, 96) * 0.1, normal(g, 6, 96, 64) * 0.1, normal(g, 64, 64)

    def step():
        leaves = [t.detach().requires_grad_() for t in (x, weights, up, down)]
        out, _ = layer(nn, leaves[0], ids, leaves[1], leaves[2], leaves[3], 0.3, 5)
        return (out.detach(), *torch.autograd.grad(out, leaves, grad))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for turn in range(3):
        x.copy_(normal(g, 64, 64))
        ids.copy_(torch.randint(-1, 6, (64, 2), generator=g, device="cuda"))
        graph.replay()
        for a, b in zip(held, step()):
            assert torch.equal(a, b)


def test_layer_in_8_bits(ops, nn):
    """Serving: rows quantized, the product in whole numbers, and back."""
    g = generator(13)
    ids = torch.randint(-1, 5, (50, 2), generator=g, device="cuda")
    x, w = normal(g, 50, 96, dtype=torch.bfloat16), normal(g, 5, 96, 64)
    weights = torch.rand(50, 2, generator=g, device="cuda")
    weight_values, weight_scales = ops.quantize_rows(w.transpose(1, 2))
    order = nn.expert_order(ids, 5)
    rows = nn.dispatch(x, order)
    values, scales = ops.quantize_rows(rows)
    product = ops.expert_product_int8(values, scales, weight_values, weight_scales, order.offsets, torch.float32)
    within(product, *exact.product_int8(*exact.quantized(rows), *exact.quantized(w.transpose(1, 2)), order.offsets))
    within(nn.combine(product, order, weights), *learned_rows.combine(product, order.place, weights))
