"""Rows sorted by expert and back, against their definition in 64 bits."""
import pytest
import torch

import learned_rows as exact

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


def draw(g, shape, experts, dropped=0.1):
    ids = torch.randint(0, experts, shape, generator=g, device="cuda")
    ids[torch.rand(shape, generator=g, device="cuda") < dropped] = -1
    return ids


def same_order(got, want):
    for x, y in zip(got, want):
        assert torch.equal(x, y)


# ---- order -----------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("shape,experts", [((1,), 1), ((1, 1), 7), ((3, 2), 8), ((16, 2), 8), ((255,), 3), ((257, 8), 64), ((1000, 1), 256),
                                           ((2047, 4), 255), ((4097,), 1000), ((5000, 6), 2048), ((8191, 8), 64), ((40_000,), 5000), ((70_001,), 65_536),
                                           ((300_000, 2), 4), ((2_000_000,), 12), ((1024,), 30), ((1025,), 30), ((16_384,), 100), ((16_385,), 100)])
def test_order(ops, shape, experts):
    g = generator(experts)
    ids = draw(g, shape, experts)
    same_order(ops.expert_order(ids, experts), exact.order(ids, experts))
    for ids in (torch.full(shape, experts - 1, device="cuda"), torch.full(shape, -1, device="cuda")):
        same_order(ops.expert_order(ids, experts), exact.order(ids, experts))


def test_order_shapes_and_errors(ops):
    from graph_sampling_b200.cabi import GsbError
    ctx = ops.Context()
    offsets, source, place = ops.expert_order(torch.empty(0, 2, dtype=torch.int64, device="cuda"), 3, ctx=ctx)
    assert offsets.tolist() == [0, 0, 0, 0] and source.numel() == 0 and place.shape == (0, 2)
    ids = draw(generator(2), (6, 50), 9).t()                               # not contiguous
    same_order(ops.expert_order(ids, 9, ctx=ctx), exact.order(ids, 9))
    ctx.check_device()
    ids = torch.tensor([[0, 5], [2, 3], [-2, 1]], device="cuda")          # 5, 3 and -2 are no experts
    same_order(ops.expert_order(ids, 3, ctx=ctx), exact.order(ids, 3))
    with pytest.raises(GsbError) as e:
        ctx.check_device()
    assert e.value.status == -8


# ---- dispatch and combine ----------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens,per_token,width", [(1, 1, 1), (1, 8, 1024), (16, 2, 1024), (33, 3, 7), (257, 5, 100), (1000, 1, 602), (129, 13, 64),
                                                    (4000, 4, 31), (511, 2, 2056)])
def test_there_and_back(ops, dtype, tokens, per_token, width):
    g = generator(tokens + width)
    _, _, place = ops.expert_order(draw(g, (tokens, per_token), 10, 0.2), 10)
    x, y = normal(g, tokens, width, dtype=dtype), normal(g, tokens * per_token, width, dtype=dtype)
    up = normal(g, tokens, width, dtype=dtype)
    for weights in (None, torch.rand(tokens, per_token, generator=g, device="cuda"), normal(g, tokens, per_token, dtype=dtype)):
        rows = ops.expert_dispatch(x, place, weights)
        assert rows.dtype == dtype
        exact.within(rows, *exact.spread(x, place, weights))
        if weights is None:
            assert torch.equal(rows.double(), exact.spread(x, place, None)[0])                 # a copy
        exact.within(ops.expert_combine(y, place, weights), *exact.combine(y, place, weights))
        grad_rows, grad_weights = ops.expert_combine_grad(up, y, place, weights)
        exact.within(grad_rows, *exact.spread(up, place, weights))
        if weights is None:
            assert grad_weights is None
        else:
            assert grad_weights.dtype == weights.dtype
            exact.within(grad_weights, *exact.weight_grads(up, y, place))
    if per_token == 1:
        flat = place.view(-1)
        assert torch.equal(ops.expert_dispatch(x, flat), ops.expert_dispatch(x, place))
        assert torch.equal(ops.expert_combine(y, flat), ops.expert_combine(y, place))


def test_strides_and_short_rows(ops):
    g = generator(5)
    offsets, _, place = ops.expert_order(draw(g, (60, 3), 6, 0.3), 6)
    big, wide = normal(g, 60, 90), normal(g, 180, 70)
    exact.within(ops.expert_dispatch(big[:, 5:69], place), *exact.spread(big[:, 5:69], place, None))
    exact.within(ops.expert_dispatch(big[:1].expand(60, 90), place), *exact.spread(big[:1].expand(60, 90), place, None))
    exact.within(ops.expert_combine(wide[:, 2:66], place), *exact.combine(wide[:, 2:66], place, None))
    exact.within(ops.expert_combine(wide.t().contiguous().t(), place), *exact.combine(wide, place, None))
    kept = int(offsets[-1])
    w = torch.rand(60, 3, generator=g, device="cuda")
    out = ops.expert_combine(wide[:kept], place, w)                           # without the rows of dropped slots
    exact.within(out, *exact.combine(wide, place, w))
    a, b = ops.expert_combine_grad(big[:, :70], wide[:kept], place, w), ops.expert_combine_grad(big[:, :70], wide, place, w)
    assert torch.equal(a[0], b[0][:kept]) and torch.equal(a[1], b[1])
    ops.default_context().check_device()


def test_all_dropped_and_empty(ops):
    place = ops.expert_order(torch.full((5, 2), -1, device="cuda"), 4)[2]
    x = torch.full((5, 12), float("nan"), device="cuda")
    y = torch.full((10, 12), float("inf"), device="cuda")
    w = torch.full((5, 2), float("nan"), device="cuda")
    assert torch.all(ops.expert_dispatch(x, place, w) == 0) and torch.all(ops.expert_combine(y, place, w) == 0)
    assert torch.all(ops.expert_combine(y[:0], place, w) == 0)
    grad_rows, grad_weights = ops.expert_combine_grad(x, y, place, w)
    assert torch.all(grad_rows == 0) and torch.all(grad_weights == 0)
    none = place[:0]
    assert ops.expert_dispatch(x[:0], none).shape == (0, 12) and ops.expert_combine(y[:0], none).shape == (0, 12)
    assert ops.expert_combine(torch.empty(10, 0, device="cuda"), place).shape == (5, 0)
    ops.default_context().check_device()


def test_values_of_dropped_slots_do_not_count(ops):
    g = generator(7)
    ids = torch.tensor([[0, -1], [-1, 1], [1, 0]], device="cuda")
    _, _, place = ops.expert_order(ids, 2)
    y, w = normal(g, 6, 9), torch.rand(3, 2, generator=g, device="cuda")
    y[4:] = float("nan")
    w[0, 1] = w[1, 0] = float("nan")
    exact.within(ops.expert_combine(y, place, w), *exact.combine(y, place, w))
    _, grad_weights = ops.expert_combine_grad(normal(g, 3, 9), y, place, w)
    assert grad_weights[0, 1] == 0 and grad_weights[1, 0] == 0 and torch.all(grad_weights.isfinite())


def test_places_out_of_range_are_not_followed(ops):
    from graph_sampling_b200.cabi import GsbError
    ctx = ops.Context()
    x = torch.ones(2, 6, device="cuda")
    place = torch.tensor([[0, 4], [1 << 40, -100]], device="cuda")
    for call in (lambda: ops.expert_dispatch(x, place, ctx=ctx), lambda: ops.expert_combine(torch.ones(4, 6, device="cuda"), place, ctx=ctx),
                 lambda: ops.expert_combine_grad(x, torch.ones(4, 6, device="cuda"), place, torch.ones(2, 2, device="cuda"), ctx=ctx)):
        call()
        with pytest.raises(GsbError) as e:
            ctx.check_device()
        assert e.value.status == -8


def test_offsets_beyond_32_bits(ops):
    """4.6e9 values in the sorted rows."""
    tokens, per_token, width = 280_000, 8, 2048
    ids = torch.arange(tokens * per_token, device="cuda").view(tokens, per_token).remainder_(7)
    _, source, place = ops.expert_order(ids, 7)
    x = torch.arange(tokens, device="cuda").remainder_(251).to(torch.bfloat16)[:, None].expand(tokens, width).contiguous()
    rows = ops.expert_dispatch(x, place)
    assert torch.equal(rows[:, 2047], x[source // per_token, 2047]) and torch.equal(rows[-1], x[source[-1] // per_token])
    out = ops.expert_combine(rows, place, torch.full((tokens, per_token), 0.125, device="cuda"))
    assert torch.equal(out, x)                                                # eight equal values, an eighth of each
    del rows, out
    torch.cuda.empty_cache()


# ---- autograd --------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("weighted", [None, "float32", "same"])
def test_autograd(nn, dtype, weighted):
    g = generator(12)
    order = nn.expert_order(draw(g, (50, 3), 5, 0.2), 5)
    x, y = normal(g, 50, 40, dtype=dtype).requires_grad_(), normal(g, 150, 40, dtype=dtype).requires_grad_()
    w = None if weighted is None else torch.rand(50, 3, generator=g, device="cuda").to(dtype if weighted == "same" else torch.float32).requires_grad_()
    up, up_rows = normal(g, 50, 40, dtype=dtype), normal(g, 150, 40, dtype=dtype)
    rows, out = nn.dispatch(x, order), nn.combine(y, order, w)
    wd = None if w is None else w.detach()
    exact.within(rows.detach(), *exact.spread(x.detach(), order.place, None))
    exact.within(out.detach(), *exact.combine(y.detach(), order.place, wd))
    torch.autograd.backward((rows, out), (up_rows, up))
    exact.within(x.grad, *exact.combine(up_rows, order.place, None))
    exact.within(y.grad, *exact.spread(up, order.place, wd))
    if w is not None:
        exact.within(w.grad, *exact.weight_grads(up, y.detach(), order.place))
        only, = torch.autograd.grad(nn.combine(y.detach(), order, w), w, up)         # one of the two gradients alone
        assert torch.equal(only, w.grad)
        only, = torch.autograd.grad(nn.combine(y, order, w.detach()), y, up)
        assert torch.equal(only, y.grad)


def test_gradients_against_differences(nn):
    """Combine is linear in its rows and in its weights: central differences are exact up to rounding, 8 u of the summands."""
    g = generator(13)
    order = nn.expert_order(draw(g, (20, 4), 5, 0.2), 5)
    y, w, up = normal(g, 80, 16).requires_grad_(), torch.rand(20, 4, generator=g, device="cuda").requires_grad_(), normal(g, 20, 16)
    nn.combine(y, order, w).backward(up)
    for leaf, step in ((y, normal(g, 80, 16)), (w, normal(g, 20, 4))):
        with torch.no_grad():
            plus, minus = ((nn.combine(leaf + s * step, order, w) if leaf is y else nn.combine(y, order, leaf + s * step)).double() for s in (1.0, -1.0))
            diff = ((plus - minus) * up.double()).sum() / 2
            got = torch.where(leaf.grad == 0, 0.0, leaf.grad.double() * step.double()).sum()
            size = exact.combine(y.abs() + step.abs() if leaf is y else y.abs(), order.place, w.abs() if leaf is y else w.abs() + step.abs())[0]
            # sums of 4 products and of 16: at most 17 u of the sum of the sizes each way, four times over
            assert abs(diff - got) <= (size * up.double().abs()).sum() * 68 * exact.U


def test_second_derivative_is_refused(nn):
    order = nn.expert_order(torch.tensor([1, 0], device="cuda"), 2)
    for leaf, f in ((torch.ones(2, 4, device="cuda", requires_grad=True), lambda t: nn.dispatch(t, order)),
                    (torch.ones(2, 4, device="cuda", requires_grad=True), lambda t: nn.combine(t, order)),
                    (torch.ones(2, device="cuda", requires_grad=True), lambda t: nn.combine(torch.ones(2, 4, device="cuda"), order, t))):
        grad, = torch.autograd.grad(f(leaf).square().sum(), leaf, create_graph=True)
        with pytest.raises(RuntimeError):
            grad.sum().backward()


def test_capture_and_replay(nn, ops):
    """A whole step, order to gradients, captured once and replayed with other experts."""
    g = generator(14)
    ids = draw(g, (64, 2), 8, 0.1)
    x, w = normal(g, 64, 32, dtype=torch.bfloat16).requires_grad_(), torch.rand(64, 2, generator=g, device="cuda").requires_grad_()
    up = normal(g, 64, 32, dtype=torch.bfloat16)

    def step():
        order = nn.expert_order(ids, 8)
        out = nn.combine(nn.dispatch(x, order), order, w)
        return (order.place, out.detach()) + torch.autograd.grad(out, (x, w), up)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        place, out, grad_x, grad_w = step()
    for turn in range(3):
        ids.copy_(draw(g, (64, 2), 8, 0.3 * turn))
        graph.replay()
        same_order((place,), exact.order(ids, 8)[2:])
        rows = exact.spread(x.detach(), place, None)[0].bfloat16()
        exact.within(out, *exact.combine(rows, place, w.detach()))
        exact.within(grad_x, *exact.combine(exact.spread(up, place, w.detach())[0].bfloat16(), place, None))
        exact.within(grad_w, *exact.weight_grads(up, rows, place))
    alive = nn.combine(x, nn.expert_order(torch.arange(64, device="cuda"), 64))
    with pytest.raises(RuntimeError, match="still alive"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            nn.dispatch(x, place)
    del alive


def test_together_on_a_sampled_frontier(nn, oracle):
    """Sample, look the frontier's embeddings up, project them by node type, bring them back, and train: every gradient against
    the same model written with torch's own operations in 64 bits."""
    import graph_sampling_b200.gs as gs
    from graph_sampling_b200.synthetic import rmat_csc
    g = generator(15)
    indptr, indices = rmat_csc(3000, 40_000, seed=5, device="cpu")
    A = gs.Matrix().load_csc(indptr.cuda(), indices.cuda())
    sub = A._graph._CAPI_fused_columnwise_slicing_sampling(torch.arange(200, device="cuda"), 8, False)
    frontier = sub._CAPI_all_indices()
    types = frontier % 4
    table, kernels = normal(g, 3000, 24).requires_grad_(), normal(g, 4, 24, 16).requires_grad_()
    order = nn.expert_order(types, 4)
    rows = nn.dispatch(nn.embedding(table, frontier, 0.5), order)
    ends = order.offsets.tolist()
    projected = torch.cat([rows[a:b].double() @ kernels[e].double() for e, (a, b) in enumerate(zip(ends, ends[1:]))]).float()
    out = nn.combine(projected, order)
    up = normal(g, *out.shape)
    out.backward(up)
    t64, k64 = table.detach().double().requires_grad_(), kernels.detach().double().requires_grad_()
    want = torch.einsum("nd,nde->ne", t64[frontier] * 0.5, k64[types])
    want.backward(up.double())
    # scale 0.5 and copies are exact; the float32 roundings of the projection and of the gradients on the way: 2 u each,
    # the sums over equal ids none (a frontier's ids are distinct), that of the products' gradients in 64 bits
    size = torch.einsum("nd,nde->ne", t64.detach()[frontier].abs(), k64.detach()[types].abs())
    assert torch.all((out.detach().double() - want.detach()).abs() <= 2 * exact.U * size)
    assert torch.allclose(table.grad.double(), t64.grad, rtol=0, atol=4 * exact.U * t64.grad.abs().max().item())
    assert torch.allclose(kernels.grad.double(), k64.grad, rtol=0, atol=4 * exact.U * k64.grad.abs().max().item() * 30)
