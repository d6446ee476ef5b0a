"""Products by expert and dropout beside other callers and in calls that the documentation allows and few make: threads, captured graphs, kinds of
tensors, addresses, waits that run out, memory that held something else."""
import ctypes
import threading

import pytest
import torch

import expert_products as exact
from learned_rows import within

pytestmark = pytest.mark.gpu
TIMEOUT, INVALID, CAPACITY = -5, -1, -4
CODES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}


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


def stream():
    return ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)


def offsets_of(counts):
    return torch.tensor([0] + counts, device="cuda").cumsum(0)


def all_kinds(ops, ctx=None):
    """(name, call, its result): one call per kernel."""
    g = generator(1)
    few, many, more = offsets_of([2, 0, 3]), offsets_of([300, 0, 1000, 500]), offsets_of([3001, 0, 9000, 5])
    jobs = []
    for dtype in (torch.float32, torch.bfloat16):
        for name, offsets, n, k, m in (("few", few, 8, 64, 40), ("tiles", many, 1900, 1024, 512), ("odd tiles", more, 12_100, 602, 250)):
            rows, w, grad = normal(g, n, k, dtype=dtype), normal(g, offsets.numel() - 1, k, m, dtype=dtype), normal(g, n, m, dtype=dtype)
            jobs.append((f"{name} {dtype}", lambda rows=rows, w=w, offsets=offsets: ops.expert_product(rows, w, offsets, ctx=ctx)))
            jobs.append((f"{name} back {dtype}", lambda grad=grad, w=w, offsets=offsets: ops.expert_product(grad, w.transpose(1, 2), offsets, ctx=ctx)))
            jobs.append((f"{name} weights {dtype}", lambda rows=rows, grad=grad, offsets=offsets: ops.expert_product_grad(rows, grad, offsets, ctx=ctx)))
    rows, w = normal(g, 1900, 1024), normal(g, 4, 1024, 512)
    wv, ws = ops.quantize_rows(w.transpose(1, 2))

    def int8():
        v, s = ops.quantize_rows(rows, ctx=ctx)
        return ops.expert_product_int8(v, s, wv, ws, many, torch.float32, ctx=ctx)
    jobs.append(("int8", int8))
    jobs.append(("dropout", lambda: ops.dropout(rows, 0.3, 7, ctx=ctx)))
    return jobs


def at_once(*jobs):
    raised = []
    torch.cuda.synchronize()

    def run(job):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                job()
                torch.cuda.current_stream().synchronize()
        except BaseException as e:
            raised.append(e)
    threads = [threading.Thread(target=run, args=(job,)) for job in jobs]
    for t in threads:
        t.start()
    for t in threads:
        t.join(240)
    assert not any(t.is_alive() for t in threads)
    if raised:
        raise raised[0]


def test_threads(ops):
    kinds = all_kinds(ops)
    want = [call() for _, call in kinds]
    got = {}

    def job(shift):
        def run():
            for turn in range(3):
                for i in range(len(kinds)):
                    at = (i + shift) % len(kinds)
                    got[shift, at, turn] = kinds[at][1]()
        return run
    at_once(*(job(shift) for shift in (0, 5, 11, 17)))
    for (_, at, _), result in got.items():
        assert torch.equal(result, want[at]), kinds[at][0]
    ops.default_context().check_device()


def test_graphs_replayed_at_once(ops):
    kinds = all_kinds(ops)
    want = [call() for _, call in kinds]
    graphs, held = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held.append([call() for _, call in kinds])
        graphs.append(graph)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for turn in range(3):
        for results in held:
            for r in results:
                r.fill_(float("nan"))
        torch.cuda.synchronize()
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for results in held:
            for (name, _), r, w in zip(kinds, results, want):
                assert torch.equal(r, w), name


def test_one_behind_the_other(ops):
    """Hundreds of calls that nothing waits between, of kernels that are set up while the one in front ends and of some that are not."""
    kinds = all_kinds(ops)
    want = [call() for _, call in kinds]
    torch.cuda.synchronize()
    for turn in range(20):
        got = [call() for _, call in kinds]
    for (name, _), r, w in zip(kinds, got, want):
        assert torch.equal(r, w), name


def test_memory_that_held_something_else(ops):
    kinds = all_kinds(ops)
    want = [call() for _, call in kinds]
    for (name, call), w in zip(kinds, want):
        junk = [torch.full((w.numel(),), float("nan"), device="cuda") for _ in range(3)] + [torch.full((1 << 22,), float("nan"), device="cuda")]
        del junk
        assert torch.equal(call(), w), name


def test_waits_that_run_out(ops):
    """Waits of half a microsecond, which some kernels never need: calls that give up say so, and the next ones are right."""
    from graph_sampling_b200.cabi import GsbError
    ctx = ops.Context()
    usual, gave_up = ctx.get_option("max_polls"), set()
    for name, call in all_kinds(ops, ctx):
        if "tiles" not in name and name != "int8":
            continue
        want = call()
        ctx.check_device()
        ctx.set_option("max_polls", 1)
        expired = 0
        for _ in range(20):
            got = call()
            try:
                ctx.check_device()
            except GsbError as e:
                assert e.status == TIMEOUT
                expired += 1
                gave_up.add(name)
                if expired == 3:
                    break
            else:
                assert torch.equal(got, want), name
        ctx.set_option("max_polls", usual)
        for _ in range(2):
            assert torch.equal(call(), want), name
            ctx.check_device()
    assert len(gave_up) >= 3, gave_up


def test_negated_views(ops, nn):
    g = generator(2)
    offsets = offsets_of([20, 30])
    rows, w, grad = normal(g, 50, 24), normal(g, 2, 24, 40), normal(g, 50, 40)
    assert torch.equal(ops.expert_product(torch._neg_view(rows), w, offsets), ops.expert_product(-rows, w, offsets))
    assert torch.equal(ops.expert_product(rows, torch._neg_view(w), offsets), ops.expert_product(rows, -w, offsets))
    assert torch.equal(ops.expert_product_grad(rows, torch._neg_view(grad), offsets), ops.expert_product_grad(rows, -grad, offsets))
    assert torch.equal(ops.dropout(torch._neg_view(rows), 0.5, 3), ops.dropout(-rows, 0.5, 3))
    assert torch.equal(ops.expert_product(rows, w, torch._neg_view(-offsets)), ops.expert_product(rows, w, offsets))
    values, scales = ops.quantize_rows(torch._neg_view(rows))
    assert torch.equal(values, ops.quantize_rows(-rows)[0])


@pytest.mark.parametrize("dtype", list(CODES))
@pytest.mark.parametrize("n,k,m", [(40, 24, 33), (2000, 256, 264), (2000, 250, 99)])
def test_addresses(ops, dtype, n, k, m):
    """Through the C interface: results at any address of their type, nothing written beside them."""
    g, ctx = generator(3), ops.default_context()
    lib, code, size = ctx.lib, CODES[dtype], torch.empty(0, dtype=dtype).element_size()
    offsets = offsets_of([n // 4, 0, n // 2])
    rows, w, grad = normal(g, n, k, dtype=dtype), normal(g, 3, k, m, dtype=dtype), normal(g, n, m, dtype=dtype)
    for shift in (0, 1, 3, 8):
        guard = torch.full((n * m + 64,), 7.0, dtype=dtype, device="cuda")
        out = guard[16 + shift:16 + shift + n * m].view(n, m)
        need = lib.gsb_expert_product_workspace(rows.data_ptr(), code, n, k, k, w.data_ptr(), k * m, m, 1, m, 3)
        work = torch.empty(max(need, 256) + 256, dtype=torch.uint8, device="cuda")
        call = lambda to, room, bytes: lib.gsb_expert_product(ctx.handle, stream(), rows.data_ptr(), code, n, k, k, w.data_ptr(), k * m, m, 1, m,
                                                              offsets.data_ptr(), 3, to, room, bytes)
        assert call(out.data_ptr(), work.data_ptr(), need) == 0
        within(out, *exact.product(rows, w, offsets))
        assert torch.all(guard[:16 + shift] == 7) and torch.all(guard[16 + shift + n * m:] == 7)
        if size > 1:
            assert call(out.data_ptr() + 1, work.data_ptr(), need) == INVALID
        if need > 0:
            assert call(out.data_ptr(), work.data_ptr(), need - 1) == CAPACITY and call(out.data_ptr(), work.data_ptr() + 16, need) == INVALID
            assert call(out.data_ptr(), None, 0) == INVALID
        guard = torch.full((3 * k * m + 64,), 7.0, dtype=dtype, device="cuda")
        out = guard[16 + shift:16 + shift + 3 * k * m].view(3, k, m)
        need = lib.gsb_expert_product_grad_workspace(rows.data_ptr(), code, n, k, k, grad.data_ptr(), m, m, 3)
        work = torch.empty(max(need, 256), dtype=torch.uint8, device="cuda")
        assert lib.gsb_expert_product_grad(ctx.handle, stream(), rows.data_ptr(), code, n, k, k, grad.data_ptr(), m, m, offsets.data_ptr(), 3,
                                           out.data_ptr(), work.data_ptr(), need) == 0
        within(out, *exact.grad_weights(rows, grad, offsets))
        assert torch.all(guard[:16 + shift] == 7) and torch.all(guard[16 + shift + 3 * k * m:] == 7)
        guard = torch.full((n * k + 64,), 7.0, dtype=dtype, device="cuda")
        out = guard[16 + shift:16 + shift + n * k].view(n, k)
        assert lib.gsb_dropout(ctx.handle, stream(), rows.data_ptr(), code, n, k, k, 0.25, 5, None, out.data_ptr()) == 0
        within(out, *exact.dropout(rows, 0.25, 5))
        assert torch.all(guard[:16 + shift] == 7) and torch.all(guard[16 + shift + n * k:] == 7)
        values, scales = torch.full((n * (k + 5) + 64,), 9, dtype=torch.int8, device="cuda"), torch.full((n,), -1.0, device="cuda")
        assert lib.gsb_quantize_rows(ctx.handle, stream(), rows.data_ptr(), code, n, k, k, values.data_ptr() + shift, k + 5, scales.data_ptr()) == 0
        want = exact.quantized(rows)
        assert torch.equal(values[shift:shift + n * (k + 5)].view(n, k + 5)[:, :k], want[0]) and torch.equal(scales, want[1])
        assert torch.all(values[:shift] == 9) and torch.all(values[shift:shift + n * (k + 5)].view(n, k + 5)[:, k:] == 9)
    ctx.check_device()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("width", [65, 72, 129, 257, 264, 602, 1319, 3057, 3064, 3065, 3066])
def test_quantize_from_and_to_any_address(ops, dtype, width):
    """Rows that begin at every value of a line, written to bytes at every distance, with what is around them left as it was."""
    ctx, code = ops.default_context(), CODES[dtype]
    n, flat = 19, normal(generator(width), 20 * (width + 9) + 16, dtype=dtype)
    for start in range(8):
        for more, out_more in ((0, 0), (1, 3), (8, 1), (3, 2)):
            rows = flat[start:start + n * (width + more)].view(n, width + more)[:, :width]
            wide = width + out_more
            values, scales = torch.full((n * wide + 64,), 9, dtype=torch.int8, device="cuda"), torch.full((n + 2,), -1.0, device="cuda")
            assert ctx.lib.gsb_quantize_rows(ctx.handle, stream(), rows.data_ptr(), code, n, width, width + more, values.data_ptr() + start, wide,
                                             scales.data_ptr() + 4) == 0
            want, got = exact.quantized(rows), values[start:start + n * wide].view(n, wide)
            assert torch.equal(got[:, :width], want[0]) and torch.equal(scales[1:-1], want[1]) and scales[0] == scales[-1] == -1
            assert torch.all(values[:start] == 9) and torch.all(values[start + n * wide:] == 9) and torch.all(got[:, width:] == 9)


def test_arguments_that_the_c_interface_refuses(ops):
    ctx = ops.default_context()
    lib, x = ctx.lib, torch.zeros(4096, device="cuda")
    o = offsets_of([4])
    p = x.data_ptr()
    good = dict(rows=p, dtype=0, n=4, k=8, stride=8, w=p, we=64, wk=8, wn=1, m=8, offsets=o.data_ptr(), experts=1, out=p + 8192)

    def product(**change):
        a = {**good, **change}
        return lib.gsb_expert_product(ctx.handle, stream(), a["rows"], a["dtype"], a["n"], a["k"], a["stride"], a["w"], a["we"], a["wk"], a["wn"], a["m"],
                                      a["offsets"], a["experts"], a["out"], None, 0)
    assert product() == 0
    for change in (dict(dtype=3), dict(n=-1), dict(n=1 << 31), dict(k=0), dict(k=(1 << 20) + 1), dict(m=0), dict(stride=-8), dict(wk=2, wn=2), dict(wn=-1),
                   dict(offsets=None), dict(offsets=o.data_ptr() + 4), dict(experts=0), dict(experts=65_537), dict(rows=None), dict(w=None), dict(out=None),
                   dict(rows=p + 2), dict(w=p + 1)):
        assert product(**change) == INVALID, change
    assert lib.gsb_dropout(ctx.handle, stream(), p, 0, 4, 8, 8, 1.5, 1, None, p + 8192) == INVALID
    assert lib.gsb_dropout(ctx.handle, stream(), p, 0, 4, 8, 8, float("nan"), 1, None, p + 8192) == INVALID
    assert lib.gsb_dropout(ctx.handle, stream(), p, 0, 4, 8, 8, 0.5, 1, p + 4, p + 8192) == INVALID
    assert lib.gsb_quantize_rows(ctx.handle, stream(), p, 0, 4, 8, 8, p + 8192, 7, p + 4096) == INVALID
    for change in (dict(stride=24), dict(k=131_072), dict(values=p + 8)):
        assert lib.gsb_expert_product_int8(ctx.handle, stream(), change.get("values", p), 4, change.get("k", 16), change.get("stride", 16), p, p, 128, 16, p, 8,
                                           o.data_ptr(), 1, p + 8192, 0) == INVALID
    ctx.check_device()


def test_captured_backward_beside_an_eager_graph(nn):
    """As for the other functions of learned rows: refused, where it would end the process."""
    g = generator(4)
    offsets = offsets_of([20, 30])
    rows, w = normal(g, 50, 24).requires_grad_(), normal(g, 2, 24, 40).requires_grad_()
    for call in (lambda: nn.product(rows, w, offsets), lambda: nn.dropout(rows, 0.5, 3)):
        eager = call()
        with pytest.raises(RuntimeError, match="made outside the capture"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                call()
        del eager


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_largest_values(ops, dtype):
    """Sums that leave the type are infinite, and what does not leave it is right, up to the largest number there is."""
    offsets = offsets_of([600])
    top = torch.finfo(dtype).max
    rows, w = torch.zeros(600, 256, dtype=dtype, device="cuda"), torch.zeros(1, 256, 256, dtype=dtype, device="cuda")
    rows[:, 0], rows[5, 1], rows[7, 3] = top, top, -float("inf")
    w[0, 0, 0], w[0, 1, :], w[0, 0, 3], w[0, 3, 9] = 1, 1, 0.5, 2
    out = ops.expert_product(rows, w, offsets)
    assert float(out[0, 0]) == top and float(out[0, 3]) == top / 2 and float(out[5, 0]) == float("inf") and float(out[5, 1]) == top
    assert float(out[7, 9]) == -float("inf") and out[7, 1].isnan() and float(out[0, 1]) == 0


def test_rows_of_a_large_call(ops):
    """Offsets of values beyond 32 bits: 2.3 M rows of 1 024."""
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("needs 24 GB")
    g, n = generator(5), 2_300_000
    rows = torch.randn(n, 1024, generator=g, device="cuda", dtype=torch.bfloat16)
    w = normal(g, 3, 1024, 136, dtype=torch.bfloat16)
    ends = [0, 700_001, 700_001, n - 5]
    out = ops.expert_product(rows, w, torch.tensor(ends, device="cuda"))
    for first in (0, 700_000, n - 300, n - 6):
        some = slice(first, min(first + 290, n))
        part = torch.tensor([min(max(e - first, 0), some.stop - first) for e in ends], device="cuda")
        within(out[some], *exact.product(rows[some], w, part))
    back = ops.expert_product_grad(rows[:, :64], out, torch.tensor(ends, device="cuda"))
    want, error = exact.grad_weights(rows[:700_001, :64], out[:700_001], torch.tensor(ends[:2], device="cuda"))
    within(back[:1], want, error)
    assert int(torch.count_nonzero(back[1])) == 0
