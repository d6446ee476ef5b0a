"""Learned rows where calls meet other things: waits that run out, memory at odd addresses, other streams, timing in a capture."""
import pytest
import torch

import learned_rows as exact

pytestmark = pytest.mark.gpu
TIMEOUT = -5


@pytest.fixture(scope="module")
def ops():
    from graph_sampling_b200 import ops as m
    return m


def generator(seed):
    g = torch.Generator("cuda")
    g.manual_seed(seed)
    return g


def stream():
    return torch.cuda.current_stream().cuda_stream


# ---- the sort of more than 32 768 positions meets at a word in memory --------------------------------------------------------
@pytest.mark.parametrize("kind", ["dense", "rows", "order", "order of many"])
def test_waits_that_run_out(ops, kind):
    from graph_sampling_b200.cabi import GsbError
    g = generator(1)
    n, rows = 400_000, 30_000
    ids = torch.randint(0, rows, (n,), generator=g, device="cuda")
    grad = torch.randn(n, 8, generator=g, device="cuda")
    ctx = ops.Context()

    def call():
        if kind == "dense":
            return (ops.embedding_grad(grad, ids, rows, ctx=ctx),)
        if kind == "rows":
            return ops.embedding_grad_rows(grad, ids, rows, sync=False, ctx=ctx)
        return ops.expert_order(ids if kind == "order of many" else ids % 50, rows if kind == "order of many" else 50, ctx=ctx)

    want = call()
    ctx.check_device()
    usual, expired = ctx.get_option("max_polls"), 0
    ctx.set_option("max_polls", 1)
    for _ in range(100):
        got = call()
        try:
            ctx.check_device()
            number = int(got[2]) if kind == "rows" else None
            for x, y in zip(got, want):
                assert torch.equal(x[:number], y[:number])     # whoever gets through all the same is right
        except GsbError as e:
            assert e.status == TIMEOUT
            expired += 1
            if kind.startswith("order"):                       # what is left can be used as indexes
                offsets, source, place = got
                assert 0 <= int(offsets.min()) and int(offsets.max()) <= n and 0 <= int(source.min()) and int(source.max()) < n
                assert -n <= int(place.min()) and int(place.max()) < n
            if expired == 5:
                break
    # (they may come to the barriers so close to each other that no wait runs out, whatever its limit)
    ctx.set_option("max_polls", usual)
    for x, y in zip(call(), want):
        number = int(want[2]) if kind == "rows" else None
        assert torch.equal(x[:number], y[:number])
    ctx.check_device()


# ---- memory at odd addresses ---------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype,code", [(torch.float32, 0), (torch.float16, 1), (torch.bfloat16, 2)])
@pytest.mark.parametrize("n", [50, 40_000])
@pytest.mark.parametrize("shift", [1, 2, 3, 5])
def test_results_at_any_address(ops, dtype, code, n, shift):
    """Tables, gradients and results that begin in the middle of a unit, with nothing written around them."""
    g = generator(shift)
    rows, width = 333, 24
    ctx = ops.default_context()
    ids = torch.randint(0, rows - 30, (n,), generator=g, device="cuda")
    room = torch.randn(n * width + 16, generator=g, device="cuda").to(dtype)
    grad = room[shift:shift + n * width].view(n, width)
    guard = torch.full((rows * width + 32,), 7.0, dtype=dtype, device="cuda")
    work = torch.empty(ctx.lib.gsb_embedding_grad_workspace(n, rows, width), dtype=torch.uint8, device="cuda")
    out = guard[shift:shift + rows * width].view(rows, width)
    assert ctx.lib.gsb_embedding_grad(ctx.handle, stream(), grad.data_ptr(), code, width, width, ids.data_ptr(), n, rows, 1.0, 0, 0,
                                      out.data_ptr(), code, work.data_ptr(), work.numel()) == 0
    exact.within(out, *exact.sums(grad, ids, rows, 1.0, None))
    assert torch.all(guard[:shift] == 7) and torch.all(guard[shift + rows * width:] == 7)
    wide = torch.full((rows * width + 32,), 7.0, device="cuda")
    out = wide[shift:shift + rows * width].view(rows, width)
    assert ctx.lib.gsb_embedding_grad(ctx.handle, stream(), grad.data_ptr(), code, width, width, ids.data_ptr(), n, rows, 1.0, 0, 0,
                                      out.data_ptr(), 0, work.data_ptr(), work.numel()) == 0
    exact.within(out, *exact.sums(grad, ids, rows, 1.0, None))
    assert torch.all(wide[:shift] == 7) and torch.all(wide[shift + rows * width:] == 7)
    guard = torch.full((n * width + 32,), 7.0, dtype=dtype, device="cuda")
    out = guard[shift:shift + n * width].view(n, width)
    assert ctx.lib.gsb_embedding_lookup(ctx.handle, stream(), grad.data_ptr(), code, n, width, width, ids.data_ptr(), n, 1.0, 0, 0,
                                        out.data_ptr()) == 0
    assert torch.all(guard[:shift] == 7) and torch.all(guard[shift + n * width:] == 7)
    keep = ids < n                                             # ids beyond the n rows of this table are zeros, and recorded
    assert torch.equal(out[keep], grad[ids[keep]]) and torch.all(out[~keep] == 0)
    if not bool(keep.all()):
        from graph_sampling_b200.cabi import GsbError
        with pytest.raises(GsbError):
            ctx.check_device()


def test_no_rows_and_all_padding(ops):
    from graph_sampling_b200.cabi import GsbError
    ctx = ops.Context()
    for n in (5, 50_000):
        grad = torch.ones(n, 6, device="cuda")
        ids = torch.zeros(n, dtype=torch.int64, device="cuda")
        assert ops.embedding_grad(grad, ids, 0, 1.0, 0, ctx=ctx).shape == (0, 6)
        assert int(torch.count_nonzero(ops.embedding_grad(grad, ids, 9, 1.0, 0, ctx=ctx))) == 0
        assert ops.embedding_grad_rows(grad, ids, 9, 1.0, 0, ctx=ctx)[0].numel() == 0
        ctx.check_device()
        ops.embedding_grad(grad, ids, 0, ctx=ctx)
        with pytest.raises(GsbError):
            ctx.check_device()


# ---- other streams ---------------------------------------------------------------------------------------------------------------
def test_inputs_made_on_another_stream(ops):
    """Kernels are set up before the one in front of them has ended: what an event orders still comes first."""
    g = generator(3)
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    table = torch.randn(5000, 128, generator=g, device="cuda")
    other = torch.randn(40_000, 128, generator=g, device="cuda")
    ids = torch.randint(0, 5000, (40_000,), generator=g, device="cuda")
    filler = torch.randn(4096, 4096, device="cuda")
    torch.cuda.synchronize()
    for turn in range(10):
        n = 20_000 if turn % 2 else 40_000
        value = float(turn + 1)
        with torch.cuda.stream(b):
            ops.embedding_lookup(table, ids)                                  # something of ours in front
        with torch.cuda.stream(a):
            filler @ filler                                                   # long enough for b to get ahead
            made = other[:n] * 0 + value
            event = a.record_event()
        with torch.cuda.stream(b):
            b.wait_event(event)
            made.record_stream(b)
            grad = ops.embedding_grad(made, ids[:n], 5000)
            back = ops.embedding_lookup(grad, ids[:n])
        torch.cuda.synchronize()
        count = torch.bincount(ids[:n], minlength=5000).float() * value
        assert torch.equal(grad, count[:, None].expand(5000, 128)) and torch.equal(back, count[ids[:n], None].expand(n, 128))


def test_results_used_on_the_spot_by_other_kernels(ops):
    """Ours behind torch's and torch's behind ours, in one stream, many times over."""
    g = generator(4)
    table = torch.randn(300, 64, generator=g, device="cuda")
    ids = torch.randint(0, 300, (1000,), generator=g, device="cuda")
    for _ in range(50):
        table.add_(1.0)
        rows = ops.embedding_lookup(table, ids)
        rows.mul_(2.0)
        grad = ops.embedding_grad(rows, ids, 300, 0.5)
        count = torch.bincount(ids, minlength=300).double()[:, None]
        want = table.double() * count                      # 2 * 0.5: exact scalings, sums of equal values
        assert torch.all((grad.double() - want).abs() <= (count + 2) * exact.U * want.abs() * 1.01)


def test_profiling_does_not_enter_a_capture(ops):
    ctx = ops.Context()
    g = generator(5)
    ids = torch.randint(0, 100, (500,), generator=g, device="cuda")
    grad = torch.randn(500, 16, generator=g, device="cuda")
    ops.embedding_grad(grad, ids, 100, ctx=ctx)
    ctx.profile_enable(True)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.embedding_grad(grad, ids, 100, ctx=ctx)
    ops.embedding_grad(grad, ids, 100, ctx=ctx)
    graph.replay()
    times = ctx.profile_read()
    ctx.profile_enable(False)
    assert times["key_sort"][1] == 1 and times["embed_grad"][1] == 1 and times["key_sort"][0] > 0
    exact.within(out, *exact.sums(grad, ids, 100, 1.0, None))


def test_large_sorts_on_several_streams_at_once(ops):
    """More than 32 768 positions each: launches of which every one wants the whole GPU."""
    g = generator(6)
    jobs = []
    for i in range(4):
        n, rows, width = 60_000 + 50_000 * i, 20_000, 24
        jobs.append((torch.randint(0, rows, (n,), generator=g, device="cuda"), torch.randn(n, width, generator=g, device="cuda"), rows))
    want = [exact.sums(grad, ids, rows, 1.0, None) for ids, grad, rows in jobs]
    streams = [torch.cuda.Stream() for _ in jobs]
    ctx = ops.Context()
    torch.cuda.synchronize()
    for _ in range(20):
        got = []
        for s, (ids, grad, rows) in zip(streams, jobs):
            with torch.cuda.stream(s):
                got.append((ops.embedding_grad(grad, ids, rows, ctx=ctx), ops.expert_order(ids, rows, ctx=ctx)[1]))
        torch.cuda.synchronize()
        ctx.check_device()
        for (out, source), (w, error), (ids, _, _) in zip(got, want, jobs):
            exact.within(out, w, error)
            assert torch.equal(source, torch.sort(ids, stable=True).indices)


def test_threads_that_wait_for_numbers_at_once():
    """Backward passes of several threads through one context, each with a number of rows of its own."""
    import threading

    import graph_sampling_b200.gs as gs
    g = generator(7)
    tables = [torch.randn(2000, 16, generator=g, device="cuda").requires_grad_() for _ in range(4)]
    ids = [torch.randint(0, 100 * (i + 1), (3000,), generator=g, device="cuda") for i in range(4)]
    gs.nn.embedding(tables[0], ids[0])
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(30):
                grad, = torch.autograd.grad(gs.nn.embedding(tables[i], ids[i], sparse=True).sum(), tables[i])
                if not torch.equal(grad.indices()[0], torch.unique(ids[i])):
                    wrong.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(120)
    assert not any(t.is_alive() for t in threads) and not wrong


@pytest.mark.parametrize("dtype,code", [(torch.float32, 0), (torch.bfloat16, 2)])
def test_addresses_that_no_tensor_has_are_refused(ops, dtype, code):
    """Nothing is launched for an address that is not a multiple of its type's size, or for a workspace off its boundary."""
    ctx, refused = ops.default_context(), -1
    lib, h, s = ctx.lib, ctx.handle, stream()
    ids = torch.zeros(8, dtype=torch.int64, device="cuda")
    rows = torch.zeros(16, 8, dtype=dtype, device="cuda")
    out = torch.full((16, 8), 5.0, dtype=dtype, device="cuda")
    long = torch.full((32,), 5, dtype=torch.int64, device="cuda")
    work = torch.empty(1 << 20, dtype=torch.uint8, device="cuda")
    r, o, i, q, w, size = rows.data_ptr(), out.data_ptr(), ids.data_ptr(), long.data_ptr(), work.data_ptr(), 1 << 19
    for a, b, c in ((1, 0, 0), (0, 1, 0), (0, 0, 4)):
        assert lib.gsb_embedding_lookup(h, s, r + a, code, 8, 8, 8, i + c, 4, 1.0, 0, 0, o + b) == refused
        assert lib.gsb_expert_spread(h, s, r + a, code, 4, 2, 8, 8, i + c, None, 0, o + b) == refused
        assert lib.gsb_expert_combine(h, s, r + a, code, 8, 4, 2, 8, 8, i + c, None, 0, o + b) == refused
        assert lib.gsb_expert_combine_grad(h, s, r + a, code, 4, 2, 8, 8, r, 8, 8, i + c, None, 0, o + b, None) == refused
    for a, b, c, d in ((1, 0, 0, 0), (0, 1, 0, 0), (0, 0, 4, 0), (0, 0, 0, 16)):
        assert lib.gsb_embedding_grad(h, s, r + a, code, 8, 8, i + c, 4, 8, 1.0, 0, 0, o + b, code, w + d, size) == refused
        assert lib.gsb_embedding_grad_rows(h, s, r + a, code, 8, 8, i + c, 4, 8, 1.0, 0, 0, q, o + b, code, q + 128, w + d, size,
                                           None) == refused
    for a, d in ((4, 0), (0, 16)):
        assert lib.gsb_expert_order(h, s, i + a, 4, 4, q, q + 64, q + 128, w + d, size) == refused
    weights = r                                                       # of the rows' type, off by a byte
    assert lib.gsb_expert_spread(h, s, r, code, 4, 2, 8, 8, i, weights + 1, code, o) == refused
    assert lib.gsb_expert_combine_grad(h, s, r, code, 4, 2, 8, 8, r, 8, 8, i, weights, code, o, o + 1) == refused
    assert torch.all(out == 5) and torch.all(long == 5)
    ctx.check_device()


@pytest.mark.parametrize("n,rows,width,dtype,kind", [
    (500_000, 410_007, 128, torch.float32, "spread"), (1_700_000, 1_600_005, 32, torch.float32, "spread"),
    (900_001, 2_000_000, 128, torch.bfloat16, "front"), (1500, 1700, 36_032, torch.float32, "spread"),
    (600_000, 420_000, 192, torch.bfloat16, "hub"), (420_000, 420_000, 128, torch.float32, "last"),
    (420_000, 420_000, 128, torch.float32, "none"), (100_000, 98_000, 2048, torch.float16, "front")])
def test_rows_without_a_sum_in_large_gradients(ops, n, rows, width, dtype, kind):
    """More than 200 MB of rows: zeros wherever no position is, whatever was in the memory before."""
    g = generator(8)
    ids = torch.randint(0, rows, (n,), generator=g, device="cuda")
    if kind == "front":
        ids //= 64
    elif kind == "hub":
        ids = torch.where(ids % 3 > 0, 77_777, ids)
    elif kind == "last":
        ids = torch.full_like(ids, rows - 1)
    elif kind == "none":
        ids = torch.full_like(ids, 5)
    grad = torch.randint(-3, 4, (n, width), generator=g, device="cuda").to(dtype)
    for scale, pad in ((1.0, 5), (0.5, None)):
        before = torch.full((rows, width), float("nan"), dtype=dtype, device="cuda")
        del before                                         # whose memory the result gets
        out = ops.embedding_grad(grad, ids, rows, scale, pad)
        keep = torch.ones_like(ids, dtype=torch.bool) if pad is None else ids != pad
        want = torch.zeros(rows, width, device="cuda").index_add_(0, ids[keep], grad[keep].float()) * scale
        assert torch.equal(out, want.to(dtype))            # sums of small integers: exact in float, one rounding
        again = ops.embedding_grad(grad, ids, rows, scale, pad)
        assert torch.equal(out, again)
        del out, want, again
    torch.cuda.empty_cache()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("width,n", [(301, 40_000), (601, 20_000), (1433, 7000), (2047, 4999), (4095, 2100), (4097, 2100),
                                     (401, 45_000), (601, 30_000), (1433, 12_001), (2047, 8000), (4095, 4000), (4097, 4000), (51, 3001), (131, 3001)])
@pytest.mark.parametrize("shift,gap", [(0, 0), (1, 0), (3, 1), (5, 7)])
def test_large_lookups_of_odd_rows(ops, dtype, width, n, shift, gap):
    """Short and long lists of rows whose values are no whole words, from tables that begin and end anywhere; nothing is written around."""
    g = generator(9)
    rows, stride = 501, width + gap
    ctx = ops.Context()
    room = torch.randn(shift + rows * stride, generator=g, device="cuda").to(dtype)
    table = room[shift:].as_strided((rows, width), (stride, 1))
    ids = torch.randint(0, rows, (n,), generator=g, device="cuda")
    ids[:4] = torch.tensor([0, rows - 1, -1, 0])
    ids[-3:] = torch.tensor([rows - 1, 7, 0])
    for scale, pad in ((1.0, None), (0.5, 7)):
        guard = torch.full((n * width + 16,), 7.0, dtype=dtype, device="cuda")
        out = guard[shift:shift + n * width].view(n, width)
        code = 1 if dtype == torch.float16 else 2
        assert ctx.lib.gsb_embedding_lookup(ctx.handle, stream(), table.data_ptr(), code, rows, width, stride, ids.data_ptr(), n, scale,
                                            int(pad is not None), pad or 0, out.data_ptr()) == 0
        want = table[ids.clamp(0)] * scale                     # exact: a power of two
        want[ids < 0] = 0
        if pad is not None:
            want[ids == pad] = 0
        assert torch.equal(out, want)
        assert torch.all(guard[:shift] == 7) and torch.all(guard[shift + n * width:] == 7)
        with pytest.raises(Exception):
            ctx.check_device()                                 # id -1
    out = ops.embedding_lookup(table, ids.clamp(0), ctx=ctx)
    assert torch.equal(out, table[ids.clamp(0)])
    ctx.check_device()


@pytest.mark.parametrize("n,keys", [(16_384, 1023), (16_385, 1023), (16_385, 1024), (32_768, 1024), (32_769, 2047), (40_000, 511),
                                    (40_000, 512), (40_000, 1023), (40_000, 1024), (40_000, 65_536), (600_000, 65_536), (600_001, 65_536),
                                    (1_300_000, 1023)])
def test_widths_of_digits(ops, n, keys):
    """Both sides of where a sort takes another digit, another number of passes, or more than one tile; the largest key is `keys`."""
    g = generator(10)
    ids = torch.randint(-1, keys, (n,), generator=g, device="cuda")
    ids[:2] = torch.tensor([keys - 1, -1])
    offsets, source, place = ops.expert_order(ids, keys)
    key = torch.where(ids < 0, keys, ids)
    want = torch.sort(key, stable=True).indices
    assert torch.equal(source, want) and torch.equal(offsets[1:], torch.bincount(key, minlength=keys + 1)[:keys].cumsum(0))
    row = torch.empty_like(want)
    row[want] = torch.arange(n, device="cuda")
    assert int(offsets[0]) == 0 and torch.equal(place, torch.where(ids < 0, ~row, row))


@pytest.mark.parametrize("n", [900, 30_000, 599_999, 600_001])
@pytest.mark.parametrize("bits", [1, 10, 11, 19, 20, 21, 22, 28, 30, 32])
def test_widths_of_ids(ops, n, bits):
    g = generator(bits)
    rows = min(2 ** bits, 2 ** 32 - 2) - (1 if bits < 32 else 0)
    ids = torch.randint(0, rows, (n,), generator=g, device="cuda")
    ids[:2] = torch.tensor([rows - 1, 0])
    grad = torch.randint(-3, 4, (n, 2), generator=g, device="cuda").float()
    row_ids, got = ops.embedding_grad_rows(grad, ids, rows)
    unique, at = torch.unique(ids, return_inverse=True)
    assert torch.equal(row_ids, unique)
    assert torch.equal(got, torch.zeros_like(got).index_add_(0, at, grad))     # sums of small integers are exact


def test_large_calls_captured_and_replayed(ops):
    """A gradient whose rows without a sum are cleared behind the sums, and rows that are looked up through shared memory; two graphs
    that share a pool."""
    g = generator(11)
    n, rows, width = 420_000, 420_003, 128
    ids = torch.randint(0, rows, (n,), generator=g, device="cuda")
    grad = torch.randint(-3, 4, (n, width), generator=g, device="cuda").float()
    table = torch.randn(5000, 1433, generator=g, device="cuda").half()
    few = torch.randint(0, 5000, (12_000,), generator=g, device="cuda")
    for _ in range(2):
        ops.embedding_grad(grad, ids, rows), ops.embedding_lookup(table, few, 0.5, 3)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=graphs[0][0].pool() if graphs else None):
            out = ops.embedding_grad(grad, ids, rows), ops.embedding_lookup(table, few, 0.5, 3)
        graphs.append((graph, out))
    for turn in range(3):
        ids.copy_(torch.randint(0, rows if turn != 1 else 1000, (n,), generator=g, device="cuda"))
        few.copy_(torch.randint(0, 5000, (12_000,), generator=g, device="cuda"))
        want = torch.zeros(rows, width, device="cuda").index_add_(0, ids, grad)       # small integers: exact in any order
        looked = table[few] * 0.5 * (few != 3)[:, None]
        for graph, (dense, found) in graphs:
            dense.fill_(float("nan"))
            found.fill_(float("nan"))
            graph.replay()
            assert torch.equal(dense, want) and torch.equal(found, looked)
