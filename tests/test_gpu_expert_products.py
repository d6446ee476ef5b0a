"""Products of rows sorted by expert, in float types and in 8 bits, with their gradients, against their definition in 64 bits."""
import pytest
import torch

import expert_products as exact
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


def offsets_of(counts):
    return torch.tensor([0] + counts, device="cuda").cumsum(0)


# rows of the experts, rows of no expert behind them, k, n
SHAPES = [([1], 0, 1, 1), ([0, 1, 0], 3, 8, 8), ([5, 0, 7], 2, 16, 40), ([64, 64], 0, 64, 64), ([1, 2, 3, 4], 0, 1024, 64), ([127, 128, 129], 5, 72, 136),
          ([256, 0, 257], 1, 64, 256), ([300], 0, 128, 384), ([33] * 9, 7, 200, 264), ([31, 97, 500], 0, 1000, 1016), ([3, 0, 60], 0, 7, 5),
          ([130, 1], 9, 63, 65), ([100, 200], 0, 101, 47), ([700], 0, 602, 100), ([2, 2], 600, 15, 17), ([2000, 0, 1, 1500], 0, 256, 250),
          ([16, 0, 5, 17, 32, 1], 0, 2048, 512), ([0, 0], 40, 64, 64), ([1030], 0, 33, 1)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("counts,rest,k,n", SHAPES)
def test_product_and_gradients(ops, dtype, counts, rest, k, n):
    g = generator(k * 7 + n)
    offsets = offsets_of(counts)
    rows = normal(g, sum(counts) + rest, k, dtype=dtype)
    weights, grad = normal(g, len(counts), k, n, dtype=dtype), normal(g, sum(counts) + rest, n, dtype=dtype)
    out = ops.expert_product(rows, weights, offsets)
    assert out.dtype == dtype
    within(out, *exact.product(rows, weights, offsets))
    within(ops.expert_product(grad, weights.transpose(1, 2), offsets), *exact.product(grad, weights.transpose(1, 2), offsets))
    got = ops.expert_product_grad(rows, grad, offsets)
    assert got.dtype == dtype
    within(got, *exact.grad_weights(rows, grad, offsets))
    assert torch.equal(got, ops.expert_product_grad(rows, grad, offsets)) and torch.equal(out, ops.expert_product(rows, weights, offsets))
    ops.default_context().check_device()


@pytest.mark.parametrize("dtype", DTYPES)
def test_many_experts(ops, dtype):
    g = generator(3)
    counts = torch.randint(0, 5, (2500,), generator=g, device="cuda").tolist()
    counts[1023] = counts[1024] = 0
    offsets = offsets_of(counts)
    rows, grad = normal(g, sum(counts) + 3, 24, dtype=dtype), normal(g, sum(counts) + 3, 16, dtype=dtype)
    weights = normal(g, 2500, 24, 16, dtype=dtype)
    within(ops.expert_product(rows, weights, offsets), *exact.product(rows, weights, offsets))
    within(ops.expert_product_grad(rows, grad, offsets), *exact.grad_weights(rows, grad, offsets))
    for E in (1023, 1024, 1025):
        within(ops.expert_product(rows, weights[:E], offsets[:E + 1]), *exact.product(rows, weights[:E], offsets[:E + 1]))
        within(ops.expert_product_grad(rows, grad, offsets[:E + 1]), *exact.grad_weights(rows, grad, offsets[:E + 1]))


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides_and_addresses(ops, dtype):
    g = generator(5)
    offsets = offsets_of([70, 0, 130, 3])
    big, wide = normal(g, 210, 300, dtype=dtype), normal(g, 4, 200, 300, dtype=dtype)
    for first in (0, 1, 2, 8, 64):
        rows, weights = big[:, first:first + 96], wide[:, first:first + 96, first:first + 72]
        within(ops.expert_product(rows, weights, offsets), *exact.product(rows, weights, offsets))
        turned = wide[:, first:first + 72, first:first + 96].transpose(1, 2)
        within(ops.expert_product(rows, turned, offsets), *exact.product(rows, turned, offsets))
        grad = big[:, first + 101:first + 101 + 80]
        within(ops.expert_product_grad(rows, grad, offsets), *exact.grad_weights(rows, grad, offsets))
    same = big[:1, :64].expand(210, 64)                                       # one row for all
    one = wide[:1, :64, :40].expand(4, 64, 40)                                # one matrix for all
    within(ops.expert_product(same, one, offsets), *exact.product(same, one, offsets))
    within(ops.expert_product_grad(same, big[:, :64], offsets), *exact.grad_weights(same, big[:, :64], offsets))
    column = big.t().contiguous().t()[:, :64]                                 # columns that are runs of memory
    within(ops.expert_product(column, wide[:, :64, :64], offsets), *exact.product(column, wide[:, :64, :64], offsets))
    scattered = wide.permute(2, 0, 1).contiguous().permute(1, 2, 0)[:, :64, ::2]
    within(ops.expert_product(column, scattered, offsets), *exact.product(column, scattered, offsets))
    ops.default_context().check_device()


@pytest.mark.parametrize("dtype", DTYPES)
def test_experts_do_not_touch_each_other(ops, dtype):
    """Infinities and NaN of one expert, and in the rows of none, stay there."""
    g = generator(6)
    counts = [50, 77, 0, 20, 130]
    offsets = offsets_of(counts)
    rows, grad, weights = normal(g, 300, 72, dtype=dtype), normal(g, 300, 40, dtype=dtype), normal(g, 5, 72, 40, dtype=dtype)
    clean = rows.clone(), grad.clone(), weights.clone()
    for e, value in ((1, float("nan")), (3, float("inf"))):
        rows[offsets[e]:offsets[e + 1]] = value
        grad[offsets[e]:offsets[e + 1]] = value
    rows[int(offsets[-1]):] = float("nan")
    grad[int(offsets[-1]):] = float("inf")
    weights[3] = float("inf")
    out, back, of_weights = ops.expert_product(rows, weights, offsets), ops.expert_product(grad, weights.transpose(1, 2), offsets), ops.expert_product_grad(rows, grad, offsets)
    want, want_back, want_weights = exact.product(clean[0], clean[2], offsets), exact.product(clean[1], clean[2].transpose(1, 2), offsets), exact.grad_weights(clean[0], clean[1], offsets)
    for e in range(5):
        a, b = int(offsets[e]), int(offsets[e + 1])
        if e in (1, 3):
            assert not out[a:b].isfinite().any() and not back[a:b].isfinite().any() and not of_weights[e].isfinite().any()
        else:
            within(out[a:b], want[0][a:b], want[1][a:b])
            within(back[a:b], want_back[0][a:b], want_back[1][a:b])
            within(of_weights[e], want_weights[0][e], want_weights[1][e])
    assert torch.all(out[int(offsets[-1]):] == 0) and torch.all(back[int(offsets[-1]):] == 0)


def test_offsets_out_of_range(ops):
    from graph_sampling_b200.cabi import GsbError
    g = generator(7)
    ctx = ops.Context()
    for dtype in DTYPES:
        rows, grad, weights = normal(g, 100, 64, dtype=dtype), normal(g, 100, 64, dtype=dtype), normal(g, 3, 64, 64, dtype=dtype)
        good = torch.tensor([3, 20, 20, 90], device="cuda")                   # rows in front of the first expert's
        within(ops.expert_product(rows, weights, good, ctx=ctx), *exact.product(rows, weights, good))
        within(ops.expert_product_grad(rows, grad, good, ctx=ctx), *exact.grad_weights(rows, grad, good))
        ctx.check_device()
        for bad in ([0, 50, 101, 105], [-5, 10, 40, 100]):
            offsets = torch.tensor(bad, device="cuda")
            within(ops.expert_product(rows, weights, offsets, ctx=ctx), *exact.product(rows, weights, offsets))
            with pytest.raises(GsbError) as e:
                ctx.check_device()
            assert e.value.status == -8
            within(ops.expert_product_grad(rows, grad, offsets, ctx=ctx), *exact.grad_weights(rows, grad, offsets))
            with pytest.raises(GsbError):
                ctx.check_device()
        offsets = torch.tensor([0, 60, 30, 100], device="cuda")               # decreasing: the middle one has no rows
        within(ops.expert_product(rows, weights, offsets, ctx=ctx), *exact.product(rows, weights, offsets))
        with pytest.raises(GsbError):
            ctx.check_device()
        within(ops.expert_product_grad(rows, grad, offsets, ctx=ctx), *exact.grad_weights(rows, grad, offsets))
        with pytest.raises(GsbError):
            ctx.check_device()


def test_shapes_without_values(ops, nn):
    offsets = torch.tensor([0, 2, 4], device="cuda")
    rows, weights = torch.ones(5, 3, device="cuda"), torch.ones(2, 3, 4, device="cuda")
    assert ops.expert_product(rows[:0], weights, offsets * 0).shape == (0, 4)
    assert ops.expert_product(rows, weights[:, :, :0], offsets).shape == (5, 0)
    assert torch.equal(ops.expert_product(rows[:, :0], weights[:, :0], offsets), torch.zeros(5, 4, device="cuda"))
    assert torch.equal(ops.expert_product_grad(rows[:0], rows[:0], offsets * 0), torch.zeros(2, 3, 3, device="cuda"))
    assert ops.expert_product_grad(rows[:, :0], rows, offsets).shape == (2, 0, 3)
    for bad in ((rows, weights[0], offsets), (rows, weights, offsets[:2]), (rows, weights.half(), offsets), (rows[:, :2], weights, offsets),
                (rows, weights, offsets.int()), (rows, weights[:0], offsets[:1]), (rows, weights.cpu(), offsets), (rows, weights, offsets.cpu())):
        with pytest.raises(TypeError):
            ops.expert_product(*bad)
        with pytest.raises(TypeError):
            nn.product(bad[0].clone().requires_grad_(), *bad[1:])
    for bad in ((rows, rows[:3], offsets), (rows, rows.half(), offsets), (rows, rows, offsets[:1]), (rows, rows[0], offsets)):
        with pytest.raises(TypeError):
            ops.expert_product_grad(*bad)


# ---- autograd ------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", DTYPES)
def test_gradients(ops, nn, dtype):
    g = generator(8)
    order = nn.expert_order(torch.randint(-1, 4, (90, 2), generator=g, device="cuda"), 4)
    rows, weights = normal(g, 180, 40, dtype=dtype).requires_grad_(), normal(g, 4, 40, 24, dtype=dtype).requires_grad_()
    up = normal(g, 180, 24, dtype=dtype)
    out = nn.product(rows, weights, order)
    assert torch.equal(out, ops.expert_product(rows, weights, order.offsets))
    a, b = torch.autograd.grad(out, (rows, weights), up, retain_graph=True)
    within(a, *exact.product(up, weights.detach().transpose(1, 2), order.offsets))
    within(b, *exact.grad_weights(rows.detach(), up, order.offsets))
    assert torch.equal(torch.autograd.grad(out, weights, up, retain_graph=True)[0], b)
    assert torch.equal(torch.autograd.grad(out, rows, up)[0], a)
    turned = weights.detach().transpose(1, 2).contiguous().requires_grad_()      # weights held as [experts, n, k]
    c, = torch.autograd.grad(nn.product(rows, turned.transpose(1, 2), order.offsets), turned, up)
    assert torch.equal(c.transpose(1, 2), b)
    shared = weights.detach()[:1].clone().requires_grad_()                       # one matrix for all experts
    d, = torch.autograd.grad(nn.product(rows.float(), shared.float().expand(4, 40, 24), order.offsets).sum(), shared)
    assert d.shape == shared.shape and d.isfinite().all()


def test_gradient_against_differences(nn):
    """The product is linear in each operand: a difference over any step is the gradient, but for rounding."""
    g = generator(9)
    offsets = offsets_of([9, 0, 14])
    rows, weights = normal(g, 25, 12).requires_grad_(), normal(g, 3, 12, 10).requires_grad_()
    up = normal(g, 25, 10)

    def loss(r, w):
        return (nn.product(r, w, offsets).double() * up).sum()
    got = torch.autograd.grad(loss(rows, weights), (rows, weights))
    for tensor, of in ((rows, got[0]), (weights, got[1])):
        step = normal(g, *tensor.shape)
        others = (rows.detach(), weights.detach())
        plus = [o + step if t is tensor else o for t, o in zip((rows, weights), others)]
        minus = [o - step if t is tensor else o for t, o in zip((rows, weights), others)]
        difference = (loss(*plus) - loss(*minus)).item() / 2
        # operands below 6 in size, 12 of them to a product and 250 products of the loss: 2 (12 + 8) u 12 * 36 * 6 * 250 < 1.6 at the very most;
        # errors of random signs are some hundredth of it
        assert abs(difference - (of.double() * step.double()).sum().item()) < 1.6


def test_only_once_and_no_tangents(nn):
    offsets = offsets_of([3, 4])
    rows, weights = torch.randn(7, 8, device="cuda", requires_grad=True), torch.randn(2, 8, 8, device="cuda", requires_grad=True)
    grads = torch.autograd.grad(nn.product(rows, weights, offsets).sum(), (rows, weights), create_graph=True)
    for grad in grads:
        with pytest.raises(RuntimeError, match="cannot be differentiated again"):
            torch.autograd.grad(grad.sum(), (rows, weights), allow_unused=True, retain_graph=True)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(rows.detach(), torch.ones_like(rows))
        with pytest.raises(RuntimeError, match="tangent"):
            nn.product(dual, weights, offsets)
        with pytest.raises(RuntimeError, match="tangent"):
            nn.dropout(dual, 0.5)


def test_changed_operands_are_noticed(nn):
    offsets = offsets_of([3, 4])
    rows, weights = torch.randn(7, 8, device="cuda", requires_grad=True), torch.randn(2, 8, 8, device="cuda", requires_grad=True)
    out = nn.product(rows, weights, offsets)
    with torch.no_grad():
        weights += 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("width,stride", [(602, 602), (601, 601), (604, 604), (64, 66), (1, 3), (7, 7), (65, 67), (130, 132), (191, 193), (9, 1201), (100, 100)])
def test_rows_at_distances_that_no_line_has(ops, dtype, width, stride):
    """Rows 2, 4 and 8 of which begin a 16-byte line: few and many, experts that begin at any of them, NaN and infinities in the row before and behind."""
    for rows in (7, 8, 9, 127, 129, 300, 1111, 5000):
        g = generator(rows + width)
        x = normal(g, rows * stride, dtype=dtype).view(rows, stride)[:, :width]
        offsets = torch.tensor([0, rows // 3, rows // 3, rows // 2 + 1, rows - rows // 7], device="cuda")
        for n in (100, 300):
            w = normal(g, 4, width, n, dtype=dtype)
            want = exact.product(x, w, offsets)
            within(ops.expert_product(x, w, offsets), *want)
        spoiled = x.clone()                                 # contiguous: its distances are the width
        spoiled[rows // 2 - 1, -1], spoiled[rows // 2 + 1, 0] = float("nan"), float("inf")
        out, clean = ops.expert_product(spoiled, w, offsets), ops.expert_product(x.contiguous(), w, offsets)
        other = torch.ones(rows, dtype=torch.bool, device="cuda")
        other[rows // 2 - 1] = other[rows // 2 + 1] = False
        assert torch.equal(out[other], clean[other])


# ---- 8 bits ----------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,width", [(1, 1), (3, 5), (33, 1024), (200, 100), (65, 602), (70, 2048), (40, 2056), (9, 4099), (1000, 16), (2, 70_000)])
def test_quantize(ops, dtype, rows, width):
    g = generator(width)
    x = normal(g, rows, width, dtype=dtype) * torch.logspace(-3, 3, rows, device="cuda")[:, None].to(dtype)
    if rows > 2:
        x[1] = 0
        x[2, width // 2] = float("inf")
    if rows > 8:
        x[3, width - 1] = float("nan")
        x[4] = torch.finfo(dtype).tiny * torch.finfo(dtype).eps * 3            # the smallest numbers there are
        x[5, 0] = torch.finfo(dtype).max
        x[6] = torch.arange(width, device="cuda") % 127 + 0.5                  # halves: ties
        x[6, 0] = 127
    values, scales = ops.quantize_rows(x)
    want_values, want_scales = exact.quantized(x)
    assert values.dtype == torch.int8 and scales.dtype == torch.float32 and values.stride(0) % 16 == 0
    assert torch.equal(values, want_values) and torch.equal(scales.nan_to_num(-1), want_scales.nan_to_num(-1))
    wide = torch.empty(rows, width + 5, dtype=dtype, device="cuda")
    wide[:, 3:3 + width] = x
    again = ops.quantize_rows(wide[:, 3:3 + width])
    assert torch.equal(again[0], values) and torch.equal(again[1].nan_to_num(-1), scales.nan_to_num(-1))


def test_quantize_shapes(ops):
    g = generator(1)
    w = normal(g, 4, 24, 20, dtype=torch.bfloat16)
    values, scales = ops.quantize_rows(w.transpose(1, 2))
    want = exact.quantized(w.transpose(1, 2))
    assert values.shape == (4, 20, 24) and scales.shape == (4, 20) and torch.equal(values, want[0]) and torch.equal(scales, want[1])
    values, scales = ops.quantize_rows(w[0, 0])
    assert values.shape == (20,) and scales.shape == ()
    assert ops.quantize_rows(w[:0])[0].shape == (0, 24, 20)
    values, scales = ops.quantize_rows(w[0, :, :0])
    assert values.shape == (24, 0) and torch.all(scales == 0)


@pytest.mark.parametrize("counts,rest,k,n", SHAPES)
def test_product_int8(ops, counts, rest, k, n):
    g = generator(k + n)
    offsets = offsets_of(counts)
    values, scales = ops.quantize_rows(normal(g, sum(counts) + rest, k))
    weight_values, weight_scales = ops.quantize_rows(normal(g, len(counts), k, n).transpose(1, 2))
    for dtype in DTYPES:
        out = ops.expert_product_int8(values, scales, weight_values, weight_scales, offsets, dtype)
        assert out.dtype == dtype
        within(out, *exact.product_int8(values, scales, weight_values, weight_scales, offsets))
    assert ops.expert_product_int8(values, scales, weight_values, weight_scales, offsets).dtype == torch.bfloat16


def test_product_int8_limits_and_layouts(ops):
    g = generator(11)
    k = 131_071
    values = torch.full((3, k + 1), -128, dtype=torch.int8, device="cuda")[:, :k]
    weight_values = torch.full((1, 8, k + 1), -128, dtype=torch.int8, device="cuda")[:, :, :k]
    scales, weight_scales, offsets = torch.ones(3, device="cuda"), torch.ones(1, 8, device="cuda"), offsets_of([3])
    out = ops.expert_product_int8(values, scales, weight_values, weight_scales, offsets, torch.float32)
    assert torch.all(out == float(128 * 128 * k))                              # the largest sum there is, rounded to float
    with pytest.raises(TypeError, match="131071"):
        ops.expert_product_int8(torch.zeros(1, k + 1, dtype=torch.int8, device="cuda"), scales[:1], torch.zeros(1, 8, k + 1, dtype=torch.int8, device="cuda"),
                                weight_scales, offsets_of([1]))
    values = torch.randint(-128, 128, (50, 300), generator=g, device="cuda").to(torch.int8)
    weight_values = torch.randint(-128, 128, (2, 300, 300), generator=g, device="cuda").to(torch.int8)
    offsets = offsets_of([20, 25])
    scales, weight_scales = torch.rand(50, generator=g, device="cuda"), torch.rand(2, 40, generator=g, device="cuda")
    for v, w in ((values[:, 3:80], weight_values[:, 5:45, 7:84]), (values[:, :64], weight_values.transpose(1, 2)[:, :40, :64]),
                 (values[:1, :48].expand(50, 48), weight_values[:1, :40, :48].expand(2, 40, 48)), (values[:, ::5], weight_values[:, :40, ::5])):
        within(ops.expert_product_int8(v, scales, w, weight_scales, offsets, torch.float32), *exact.product_int8(v, scales, w, weight_scales, offsets))
    scales[7] = float("nan")
    out = ops.expert_product_int8(values, scales, weight_values[:, :40], weight_scales, offsets)
    assert out[7].isnan().all() and out[:7].isfinite().all() and out[8:].isfinite().all() and torch.all(out[45:] == 0)
    for bad in ((values, scales[:3], weight_values[:, :40], weight_scales, offsets), (values[:, :8], scales, weight_values[:, :40], weight_scales, offsets),
                (values, scales, weight_values[:, :40], weight_scales[:, :3], offsets), (values, scales.half(), weight_values[:, :40], weight_scales, offsets),
                (values, scales, weight_values[:, :40], weight_scales, offsets[:2])):
        with pytest.raises(TypeError):
            ops.expert_product_int8(*bad)


def test_first_call_of_a_thread(ops, nn):
    """A thread that has made no other call of CUDA's runtime yet (autograd's, a new one) has no context of the driver's."""
    import threading
    g = generator(21)
    offsets = offsets_of([3000, 2000, 1000])
    rows, weights = normal(g, 6000, 256, dtype=torch.bfloat16), normal(g, 3, 256, 256, dtype=torch.bfloat16)
    want = ops.expert_product(rows, weights, offsets)
    want_grad = ops.expert_product_grad(rows, want, offsets)
    kept = [torch.empty_like(want) for _ in range(4)], [torch.empty_like(want_grad) for _ in range(4)]
    torch.cuda.synchronize()
    del kept                                                                    # memory that needs no call to be had
    got = {}

    def call(k):
        got[k] = ops.expert_product_grad(rows, want, offsets) if k % 2 else ops.expert_product(rows, weights, offsets)
    for k in range(4):
        thread = threading.Thread(target=call, args=(k,))
        thread.start()
        thread.join()
        assert torch.equal(got[k], want_grad if k % 2 else want)
    leaf = rows.clone().requires_grad_()
    back, = torch.autograd.grad(nn.product(leaf, weights, offsets), leaf, want)
    assert torch.equal(back, ops.expert_product(want, weights.transpose(1, 2), offsets))
