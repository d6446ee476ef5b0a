"""Embedding rows against their definition in 64 bits: lookup, the dense and the row-wise gradient, autograd, capture."""
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


def draw_ids(g, n, rows, kind):
    if kind == "same":
        return torch.full((n,), rows - 1, device="cuda")
    if kind == "distinct":
        return torch.randperm(rows, generator=g, device="cuda")[:n]
    u = torch.rand(n, generator=g, device="cuda", dtype=torch.float64)
    return (u.pow(1 if kind == "uniform" else 6) * rows).long().clamp_(0, rows - 1)


# ---- lookup ----------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("width", [1, 2, 3, 5, 8, 31, 64, 100, 257, 602, 1024, 2056])
def test_lookup(ops, dtype, width):
    g = generator(width)
    table = normal(g, 777, width, dtype=dtype)
    for n in (1, 63, 3001):
        ids = torch.randint(0, 777, (n,), generator=g, device="cuda")
        for scale, padding in ((1.0, None), (-3.3, 5), (float(width) ** 0.5, -1)):
            out = ops.embedding_lookup(table, ids, scale, padding)
            assert out.dtype == dtype
            want = exact.lookup(table, ids, torch.tensor(scale, dtype=torch.float32).double().item(), padding)
            exact.within(out, want, want.abs() * exact.U)
    assert torch.equal(ops.embedding_lookup(table, ids), table[ids])        # scale 1: a copy


def test_lookup_shapes_strides_and_offsets(ops):
    g = generator(1)
    table = normal(g, 50, 24)
    ids = torch.randint(0, 50, (4, 3, 2), generator=g, device="cuda")
    assert torch.equal(ops.embedding_lookup(table, ids), table[ids])
    assert torch.equal(ops.embedding_lookup(table, ids.transpose(0, 2)), table[ids.transpose(0, 2)])
    assert torch.equal(ops.embedding_lookup(table, ids[0, 0, 0]), table[ids[0, 0, 0]])                # no dimension
    assert ops.embedding_lookup(table, ids[:0]).shape == (0, 3, 2, 24)
    assert torch.equal(ops.embedding_lookup(table[:, 3:20], ids), table[:, 3:20][ids])                 # rows at a stride, odd start
    assert torch.equal(ops.embedding_lookup(table.t(), ids % 24), table.t()[ids % 24])                 # copied
    assert torch.equal(ops.embedding_lookup(table[7:8].expand(50, 24), ids), table[7].expand(4, 3, 2, 24))
    assert ops.embedding_lookup(table[:, :0], ids).shape == (4, 3, 2, 0)
    pinned = torch.randn(60, 20).pin_memory()
    ids = torch.randint(0, 60, (33,), generator=g, device="cuda")
    assert torch.equal(ops.embedding_lookup(pinned, ids).cpu(), pinned[ids.cpu()])


def test_lookup_out_of_range_is_zero_and_reported(ops):
    from graph_sampling_b200.cabi import GsbError
    ctx = ops.Context()
    table = torch.ones(10, 6, device="cuda")
    ids = torch.tensor([3, 10, -1, -(1 << 62), 9], device="cuda")
    out = ops.embedding_lookup(table, ids, ctx=ctx)
    assert torch.equal(out[:, 0], torch.tensor([1.0, 0, 0, 0, 1], device="cuda"))
    with pytest.raises(GsbError) as e:
        ctx.check_device()
    assert e.value.status == -8
    ops.embedding_lookup(table, torch.tensor([3, -1], device="cuda"), 1.0, -1, ctx=ctx)     # padding may be out of range
    ops.embedding_lookup(table, torch.tensor([3, 1 << 40], device="cuda"), 1.0, 1 << 40, ctx=ctx)
    ctx.check_device()
    assert torch.equal(ops.embedding_lookup(table[:0], torch.tensor([0, 1], device="cuda"), 1.0, 0, ctx=ctx), torch.zeros(2, 6, device="cuda"))
    with pytest.raises(GsbError):
        ctx.check_device()


def test_special_values_pass(ops):
    table = torch.tensor([[float("inf"), float("nan"), -0.0, 65504.0]], device="cuda").repeat(3, 1)
    for dtype in DTYPES:
        out = ops.embedding_lookup(table.to(dtype), torch.tensor([2, 1], device="cuda"), 1.0, 1)
        assert out[0, 0] == float("inf") and out[0, 1].isnan() and torch.signbit(out[0, 2]) and torch.all(out[1] == 0)


@pytest.mark.parametrize("rows,width", [(4_300_000, 1024)])
def test_offsets_beyond_32_bits(ops, rows, width):
    """4.4e9 values in the table and in its gradient."""
    table = torch.zeros(rows, width, dtype=torch.bfloat16, device="cuda")
    ids = torch.tensor([rows - 1, 0, rows - 2, rows - 1], device="cuda")
    table[rows - 1] = 3.0
    table[rows - 2] = 2.0
    assert ops.embedding_lookup(table, ids)[:, 0].tolist() == [3.0, 0.0, 2.0, 3.0]
    del table
    grad = ops.embedding_grad(torch.ones(4, width, dtype=torch.bfloat16, device="cuda"), ids, rows)
    assert torch.all(grad[rows - 1] == 2) and torch.all(grad[rows - 2] == 1) and torch.all(grad[0] == 1)
    assert int(torch.count_nonzero(grad[:, 0])) == 3
    del grad
    torch.cuda.empty_cache()


# ---- gradients -------------------------------------------------------------------------------------------------------------
SHAPES = [(1, 1, 1, "same"), (2, 1, 7, "same"), (31, 7, 3, "uniform"), (33, 40, 16, "distinct"), (1000, 10, 64, "skewed"),
          (1024, 100_000, 100, "uniform"), (2049, 2049, 257, "distinct"), (20_000, 3, 33, "same"), (20_011, 5000, 602, "skewed"),
          (70_001, 70_000, 8, "uniform"), (300_007, 1_000_000, 4, "skewed"), (300_007, 4, 130, "skewed"), (4096, 300, 2056, "skewed"),
          (600_000, 2, 1, "uniform"), (1_300_000, 9000, 3, "skewed"), (2_500_000, 300_000, 2, "uniform"),
          # one CTA, a cluster, the grid: the last of the one and the first of the next
          (1024, 5000, 4, "uniform"), (1025, 5000, 4, "uniform"), (2048, 500, 4, "uniform"), (2049, 500, 4, "uniform"), (32_768, 70_000, 4, "uniform"), (32_769, 70_000, 4, "uniform")]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,rows,width,kind", SHAPES)
def test_gradients(ops, dtype, n, rows, width, kind):
    g = generator(n + width)
    ids = draw_ids(g, n, rows, kind)
    grad = normal(g, n, width, dtype=dtype)
    for scale, padding in ((1.0, None), (0.5, int(ids[n // 2]))):
        want, error = exact.sums(grad, ids, rows, scale, padding)
        dense = ops.embedding_grad(grad, ids, rows, scale, padding)
        assert dense.dtype == dtype
        exact.within(dense, want, error)
        assert torch.equal(dense, ops.embedding_grad(grad, ids, rows, scale, padding))                 # the same bits
        row_ids, some = ops.embedding_grad_rows(grad, ids, rows, scale, padding)
        live = ids if padding is None else ids[ids != padding]
        assert torch.equal(row_ids, torch.unique(live)) and torch.equal(some, dense[row_ids])
        wide = ops.embedding_grad(grad, ids, rows, scale, padding, dtype=torch.float32)
        assert wide.dtype == torch.float32
        exact.within(wide, want, error)
        if dtype != torch.float32:
            assert torch.equal(wide.to(dtype), dense)
        row_ids2, some2, number = ops.embedding_grad_rows(grad, ids, rows, scale, padding, torch.float32, sync=False)
        assert int(number) == row_ids.numel() and torch.equal(row_ids2[:int(number)], row_ids)
        assert torch.equal(some2[:int(number)], wide[row_ids])


@pytest.mark.parametrize("ids", [[5, 5, 5, 0, 9, 0], [9, 8, 7], [0] * 65, list(range(10)) * 40, [3] * 31 + [4] * 33 + [5] * 64 + [6]])
def test_chunk_borders(ops, ids):
    """Runs that begin and end at every place of a chunk, whole numbers: exact whatever the order of the sums."""
    ids = torch.tensor(ids, device="cuda")
    n = ids.numel()
    grad = torch.arange(n, device="cuda", dtype=torch.float32)[:, None] + torch.arange(70, device="cuda") * 100
    want = torch.zeros(10, 70, dtype=torch.float64, device="cuda").index_add_(0, ids, grad.double())
    assert torch.equal(ops.embedding_grad(grad, ids, 10).double(), want)


def test_gradient_padding_out_of_range_and_empty(ops):
    from graph_sampling_b200.cabi import GsbError
    ctx = ops.Context()
    grad = torch.full((5, 3), float("nan"), device="cuda")
    grad[1] = 2.0
    ids = torch.tensor([-1, 1, -1, -1, -1], device="cuda")
    out = ops.embedding_grad(grad, ids, 4, 1.0, -1, ctx=ctx)                     # what padding holds does not count
    assert torch.equal(out[1], torch.full((3,), 2.0, device="cuda")) and int(torch.count_nonzero(out)) == 3
    ctx.check_device()
    out = ops.embedding_grad(grad, torch.tensor([4, 1, -7, 1 << 40, 99], device="cuda"), 4, ctx=ctx)
    assert torch.equal(out[1], torch.full((3,), 2.0, device="cuda")) and int(torch.count_nonzero(out)) == 3
    with pytest.raises(GsbError) as e:
        ctx.check_device()
    assert e.value.status == -8
    with pytest.raises(GsbError):                                                # a call that waits for its size says so itself
        ops.embedding_grad_rows(grad, torch.tensor([4, 1, 1, 1, 1], device="cuda"), 4, ctx=ctx)
    row_ids, rows = ops.embedding_grad_rows(grad, torch.full((5,), 7, device="cuda"), 10, 1.0, 7, ctx=ctx)
    assert row_ids.numel() == 0 and rows.shape == (0, 3)
    row_ids, rows = ops.embedding_grad_rows(grad[:0], ids[:0], 10, ctx=ctx)
    assert row_ids.numel() == 0 and rows.shape == (0, 3)
    assert torch.equal(ops.embedding_grad(grad[:0], ids[:0], 6, ctx=ctx), torch.zeros(6, 3, device="cuda"))
    assert ops.embedding_grad(grad[:0], ids[:0], 0, ctx=ctx).shape == (0, 3)
    ctx.check_device()


def test_ids_of_a_very_large_table(ops):
    """Ids of 32 bits: no array of the table's size is made."""
    g = generator(3)
    rows = 2 ** 32 - 2
    ids = torch.randint(rows - 5000, rows, (9000,), generator=g, device="cuda")
    ids[:10] = torch.arange(10, device="cuda")
    grad = normal(g, 9000, 20)
    row_ids, out = ops.embedding_grad_rows(grad, ids, rows)
    unique, inverse = torch.unique(ids, return_inverse=True)
    want, error = exact.sums(grad, inverse, unique.numel(), 1.0, None)
    assert torch.equal(row_ids, unique)
    exact.within(out, want, error)


def test_rows_behind_the_last_stay(ops):
    grad = torch.ones(6, 4, device="cuda")
    ids = torch.tensor([2, 2, 7, 7, 7, 1], device="cuda")
    ctx = ops.default_context()
    out_ids, out_rows = torch.full((6,), -5, device="cuda"), torch.full((6, 4), -5.0, device="cuda")
    count = torch.zeros(1, dtype=torch.int64, device="cuda")
    work = torch.empty(ctx.lib.gsb_embedding_grad_workspace(6, 10, 4), dtype=torch.uint8, device="cuda")
    assert ctx.lib.gsb_embedding_grad_rows(ctx.handle, torch.cuda.current_stream().cuda_stream, grad.data_ptr(), 0, 4, 4, ids.data_ptr(),
                                           6, 10, 1.0, 0, 0, out_ids.data_ptr(), out_rows.data_ptr(), 0, count.data_ptr(),
                                           work.data_ptr(), work.numel(), None) == 0
    assert out_ids.tolist() == [1, 2, 7, -5, -5, -5] and out_rows[:, 0].tolist() == [1, 2, 3, -5, -5, -5] and int(count) == 3
    assert ctx.lib.gsb_embedding_grad_rows(ctx.handle, torch.cuda.current_stream().cuda_stream, grad.data_ptr(), 0, 4, 4, ids.data_ptr(),
                                           6, 10, 1.0, 0, 0, out_ids.data_ptr(), out_rows.data_ptr(), 0, count.data_ptr(),
                                           work.data_ptr(), work.numel() - 1, None) == -4


def test_strided_and_broadcast_gradients(ops):
    g = generator(9)
    ids = torch.randint(0, 20, (15, 4), generator=g, device="cuda")
    big = normal(g, 15, 4, 40)
    for grad in (big[..., 3:14], big[..., :8], big[:, :, 0:1].expand(15, 4, 12), big[:1].expand(15, 4, 40), big.transpose(0, 1).contiguous().transpose(0, 1)):
        want, error = exact.sums(grad, ids, 20, 1.0, None)
        exact.within(ops.embedding_grad(grad, ids, 20), want, error)


# ---- autograd --------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("sparse", [False, True])
def test_autograd(nn, dtype, sparse):
    g = generator(4)
    table = normal(g, 300, 48, dtype=dtype).requires_grad_()
    ids = draw_ids(g, 500, 300, "skewed").view(20, 25)
    out = nn.embedding(table, ids, 2.0, 7, sparse)
    up = normal(g, 20, 25, 48, dtype=dtype)
    out.backward(up)
    want, error = exact.sums(up, ids, 300, 2.0, 7)
    assert table.grad.is_sparse == sparse
    if sparse:                                            # torch's accumulation forgets that it is coalesced
        alone, = torch.autograd.grad(nn.embedding(table, ids, 2.0, 7, True), table, up)
        assert alone.is_coalesced() and torch.equal(alone.indices(), table.grad._indices())
        assert torch.equal(alone.indices()[0], torch.unique(ids[ids != 7]))
    exact.within(table.grad.to_dense() if sparse else table.grad, want, error)
    with torch.no_grad():
        assert not nn.embedding(table, ids).requires_grad
    assert not nn.embedding(table.detach(), ids).requires_grad


def test_gradient_against_differences(nn):
    """The loss is linear in the table, so a central difference is exact up to the rounding of the two lookups, u each."""
    g = generator(6)
    table = normal(g, 40, 12).requires_grad_()
    ids = torch.randint(0, 40, (90,), generator=g, device="cuda")
    up, step = normal(g, 90, 12), normal(g, 40, 12)
    nn.embedding(table, ids, 1.5, 3).backward(up)
    with torch.no_grad():
        plus, minus = (nn.embedding((table + s * step), ids, 1.5, 3).double() for s in (1.0, -1.0))
        diff = ((plus - minus) * up.double()).sum() / 2
        want = (table.grad.double() * step.double()).sum()
        # table +- step and the lookup round once each (2 u of |out| + |step| ...), the gradient's sums at most 92 u
        size = ((plus.abs() + minus.abs()) * up.double().abs()).sum() * 2 + (exact.sums(up.abs(), ids, 40, 1.5, 3)[0] * step.double().abs()).sum() * 92
        assert abs(diff - want) <= size * exact.U


def test_sum_and_accumulation(nn):
    table = torch.ones(5, 8, device="cuda", requires_grad=True)
    ids = torch.tensor([1, 1, 4], device="cuda")
    for _ in range(2):
        nn.embedding(table, ids).sum().backward()        # the incoming gradient is broadcast from one value
    assert table.grad[:, 0].tolist() == [0, 4, 0, 0, 2]


def test_second_derivative_is_refused(nn):
    table = torch.ones(5, 8, device="cuda", requires_grad=True)
    out = nn.embedding(table, torch.tensor([1, 2], device="cuda"))
    grad, = torch.autograd.grad((out * out).sum(), table, create_graph=True)
    assert grad[1, 0] == 2
    with pytest.raises(RuntimeError):
        grad.sum().backward()


@pytest.mark.parametrize("n", [700, 3000, 50_000])
def test_capture_and_replay(nn, ops, n):
    g = generator(8)
    table = normal(g, 1000, 64).requires_grad_()
    ids = draw_ids(g, n, 1000, "skewed")
    up = normal(g, n, 64)
    streams = torch.cuda.Stream()
    streams.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(streams):
        for _ in range(2):
            torch.autograd.grad(nn.embedding(table, ids, 2.0, 5), table, up)
            ops.embedding_grad_rows(up, ids, 1000, sync=False)
    torch.cuda.current_stream().wait_stream(streams)
    graphs = []
    for _ in range(2):                                    # two graphs over the same inputs, from one pool
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=graphs[0][0].pool() if graphs else None):
            out = nn.embedding(table, ids, 2.0, 5)
            dense, = torch.autograd.grad(out, table, up)
            rows = ops.embedding_grad_rows(up, ids, 1000, sync=False)
        graphs.append((graph, out.detach(), dense, rows))
        del out
    for turn in range(3):
        ids.copy_(draw_ids(g, n, 1000, "uniform" if turn else "same"))
        up.copy_(normal(g, n, 64))
        for graph, out, dense, (row_ids, rows, number) in graphs:
            graph.replay()
            want = exact.lookup(table.detach(), ids, 2.0, 5)
            exact.within(out, want, want.abs() * exact.U)
            exact.within(dense, *exact.sums(up, ids, 1000, 2.0, 5))
            unique = torch.unique(ids)
            assert int(number) == unique.numel() and torch.equal(row_ids[:int(number)], unique)
            exact.within(rows[:int(number)], *(x[unique] for x in exact.sums(up, ids, 1000, 1.0, None)))
    with pytest.raises(RuntimeError):                     # a size cannot be waited for in a capture
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            ops.embedding_grad_rows(up, ids, 1000)


def test_capture_beside_an_eager_graph_of_the_same_leaf_is_refused(nn):
    table = torch.ones(50, 16, device="cuda", requires_grad=True)
    ids = torch.arange(20, device="cuda")
    alive = nn.embedding(table, ids)                      # made on the default stream and still held
    with pytest.raises(RuntimeError, match="still alive"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            nn.embedding(table, ids)
    alive.sum().backward()
    assert torch.all(table.grad[:20] == 1)


def test_streams_do_not_share_scratch(ops):
    g = generator(11)
    jobs = []
    for i in range(4):
        n, rows, width = 30_000 + i, 2000, 40 + i
        jobs.append((draw_ids(g, n, rows, "skewed"), normal(g, n, width), rows))
    want = [exact.sums(grad, ids, rows, 1.0, None) for ids, grad, rows in jobs]
    streams = [torch.cuda.Stream() for _ in jobs]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for s, (ids, grad, rows) in zip(streams, jobs):
            with torch.cuda.stream(s):
                got.append(ops.embedding_grad(grad, ids, rows))
        torch.cuda.synchronize()
        for out, (w, error) in zip(got, want):
            exact.within(out, w, error)


def test_another_device_than_the_current_one(nn, ops):
    if torch.cuda.device_count() < 2:
        pytest.skip("needs two GPUs")
    table = torch.randn(30, 8, device="cuda:1", requires_grad=True)
    ids = torch.tensor([3, 3, 29], device="cuda:1")
    out = nn.embedding(table, ids)
    out.sum().backward()
    assert torch.equal(out.detach(), table.detach()[ids]) and table.grad[3, 0] == 2
    with pytest.raises(TypeError):
        ops.embedding_lookup(table.detach(), ids.to("cuda:0"))
