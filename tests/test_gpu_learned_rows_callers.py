"""Learned rows beside other callers and in calls that the documentation allows and few make: threads, kinds of tensors, addresses,
waits that run out, values that are no numbers."""
import ctypes
import threading

import pytest
import torch

import learned_rows as exact

pytestmark = pytest.mark.gpu
TIMEOUT = -5


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


def stream():
    return ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)


def at_once(*jobs):
    """Runs the jobs on threads, each on a stream of its own, and raises what one of them raised."""
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


# ---- several threads -----------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("blocking", [0, 1])
def test_sparse_gradients_beside_a_thread_that_samples(ops, nn, blocking):
    """Both wait for sizes through the default context, whatever each finds."""
    import graph_sampling_b200.gs as gs
    from graph_sampling_b200.synthetic import rmat_csc
    g = generator(1)
    indptr, indices = rmat_csc(3000, 40_000, seed=5, device="cpu")
    A = gs.Matrix().load_csc(indptr.cuda(), indices.cuda())
    seeds = [torch.arange(10 * (i + 1), device="cuda") for i in range(20)]
    degree = indptr.diff().clamp(max=8).cuda()
    tables = [torch.randn(2000, 16, generator=g, device="cuda").requires_grad_() for _ in range(2)]
    ids = [torch.randint(0, 150 * (i + 1), (3000,), generator=g, device="cuda") for i in range(2)]
    unique = [torch.unique(i) for i in ids]

    def sampler():
        for turn in range(300):
            s = seeds[turn % len(seeds)]
            sub = A._graph._CAPI_fused_columnwise_slicing_sampling(s, 8, False)
            found = sub._CAPI_all_indices()
            assert s.numel() <= found.numel() <= s.numel() + int(degree[s].sum()) and bool((found < 3000).all())

    def trainer(i):
        def work():
            for _ in range(300):
                grad, = torch.autograd.grad(nn.embedding(tables[i], ids[i], sparse=True).sum(), tables[i])
                assert torch.equal(grad.indices()[0], unique[i]) and grad.values().shape == (unique[i].numel(), 16)
        return work

    ctx = ops.default_context()
    usual = ctx.get_option("blocking_wait")
    ctx.set_option("blocking_wait", blocking)
    try:
        at_once(sampler, trainer(0), trainer(1))
    finally:
        ctx.set_option("blocking_wait", usual)
    ctx.check_device()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_long_odd_rows_of_two_widths_looked_up_by_two_threads(ops, dtype):
    """Launches with much shared memory and with less, a context each: what one asks for is not taken back by the other."""
    g = generator(2)

    def job(width, n):
        table = torch.randn(60, width, generator=g, device="cuda").to(dtype)
        ids = torch.randint(0, 60, (n,), generator=g, device="cuda")
        want, ctx = table[ids], ops.Context()

        def work():
            for _ in range(400):
                out = ops.embedding_lookup(table, ids, ctx=ctx)
            assert torch.equal(out, want)
        return work

    at_once(job(4095, 4000), job(2047, 8000))


def test_timers_and_counts_of_two_threads(ops):
    """Every launch is counted and timed as what it is, whoever else launches through the context meanwhile."""
    g = generator(10)
    table = torch.randn(500, 64, generator=g, device="cuda")
    ids = torch.randint(0, 500, (20_000,), generator=g, device="cuda")
    grad = torch.randn(20_000, 64, generator=g, device="cuda")
    ctx = ops.Context()
    ops.embedding_lookup(table, ids, ctx=ctx), ops.embedding_grad(grad, ids, 500, ctx=ctx)
    before = ctx.launch_count()
    ops.embedding_lookup(table, ids, ctx=ctx)
    of_lookup = ctx.launch_count() - before
    ops.embedding_grad(grad, ids, 500, ctx=ctx)
    of_grad = ctx.launch_count() - before - of_lookup
    ctx.profile_enable(True)
    ctx.profile_reset()
    before = ctx.launch_count()
    at_once(lambda: [ops.embedding_lookup(table, ids, ctx=ctx) for _ in range(600)],
            lambda: [ops.embedding_grad(grad, ids, 500, ctx=ctx) for _ in range(400)])
    times = ctx.profile_read()
    ctx.profile_enable(False)
    assert ctx.launch_count() - before == 600 * of_lookup + 400 * of_grad
    assert {name: n for name, (ms, n) in times.items()} == {"embed_lookup": 600, "key_sort": 400, "embed_grad": 400}
    assert all(ms > 0 for ms, n in times.values())


# ---- kinds of tensors ----------------------------------------------------------------------------------------------------------
def test_forward_mode_is_refused(nn):
    """Tangents of what goes in, and of the gradients that come back, are not dropped without a word."""
    import torch.autograd.forward_ad as fw
    g = generator(3)
    table, y, w = (torch.randn(*shape, generator=g, device="cuda") for shape in ((10, 8), (6, 8), (3, 2)))
    ids, order = torch.tensor([3, 1, 3], device="cuda"), nn.expert_order(torch.tensor([[0, 1], [1, -1], [0, 0]], device="cuda"), 2)
    x = torch.randn(3, 8, generator=g, device="cuda")
    calls = [(table, lambda t: nn.embedding(t, ids)), (table, lambda t: nn.embedding(t, ids, sparse=True)), (x, lambda t: nn.dispatch(t, order)),
             (y, lambda t: nn.combine(t, order)), (y, lambda t: nn.combine(t, order, w)), (w, lambda t: nn.combine(y, order, t))]
    with fw.dual_level():
        for leaf, call in calls:
            for primal in (leaf, leaf.clone().requires_grad_()):
                with pytest.raises(RuntimeError):
                    call(fw.make_dual(primal, torch.ones_like(leaf)))
            back = leaf.clone().requires_grad_()
            out = call(back)
            with pytest.raises(RuntimeError):
                torch.autograd.grad(out, back, fw.make_dual(torch.ones_like(out), torch.ones_like(out)))
            assert torch.autograd.grad(call(back), back, torch.ones_like(out))[0] is not None
    for leaf, call in calls:
        call(leaf)


def test_second_derivatives_are_refused_for_whatever_they_are_taken(nn):
    """Not only where a backward pass meets the gradient: also towards the gradient that came in, or one operand alone."""
    from torch.autograd import functional
    g = generator(4)
    table, y, w = (torch.randn(*shape, generator=g, device="cuda") for shape in ((10, 8), (6, 8), (3, 2)))
    ids, order = torch.tensor([3, 1, 3], device="cuda"), nn.expert_order(torch.tensor([[0, 1], [1, -1], [0, 0]], device="cuda"), 2)
    x = torch.randn(3, 8, generator=g, device="cuda")
    for leaf, call in ((table, lambda t: nn.embedding(t, ids)), (x, lambda t: nn.dispatch(t, order)), (y, lambda t: nn.combine(t, order)),
                       (y, lambda t: nn.combine(t, order, w)), (w, lambda t: nn.combine(y, order, t))):
        for twice in (lambda: functional.jvp(call, leaf, torch.ones_like(leaf)),
                      lambda: functional.hvp(lambda t: call(t).square().sum(), leaf, torch.ones_like(leaf)),
                      lambda: functional.vhp(lambda t: call(t).square().sum(), leaf, torch.ones_like(leaf))):
            with pytest.raises(RuntimeError, match="cannot be differentiated again"):
                twice()
        assert functional.vjp(call, leaf, torch.ones_like(call(leaf)))[1].shape == leaf.shape
    rows, weights = y.clone().requires_grad_(), w.clone().requires_grad_()
    of_rows, of_weights = torch.autograd.grad(nn.combine(rows, order, weights).sum(), (rows, weights), create_graph=True)
    for grad, other in ((of_rows, weights), (of_weights, rows)):
        with pytest.raises(RuntimeError, match="cannot be differentiated again"):
            torch.autograd.grad(grad.sum(), other, allow_unused=True, retain_graph=True)


@pytest.mark.parametrize("width", [1, 6])
def test_views_that_stand_for_their_negative(ops, nn, width):
    """The imaginary part of a conjugate shares its memory and differs in sign."""
    g = generator(5)
    negative = lambda n, w=width: torch.view_as_complex(torch.randn(n, w, 2, generator=g, device="cuda")).conj().imag
    flat = lambda n, w=width: torch._neg_view(torch.randn(n, w, generator=g, device="cuda"))
    ids = torch.randint(0, 9, (40,), generator=g, device="cuda")
    order = ops.expert_order(torch.randint(0, 4, (20, 2), generator=g, device="cuda"), 4)[2]
    for make in (negative, flat):
        table, x, y, w, up, ups = make(9), make(20), make(40), make(20, 2), make(40), make(20)
        assert table.is_neg() and w.is_neg()
        plain = lambda t: t.resolve_neg().clone().contiguous()
        assert torch.equal(ops.embedding_lookup(table, ids), plain(table)[ids])
        assert torch.equal(ops.embedding_grad(up, ids, 9), ops.embedding_grad(plain(up), ids, 9))
        assert torch.equal(ops.embedding_grad_rows(up, ids, 9)[1], ops.embedding_grad_rows(plain(up), ids, 9)[1])
        assert torch.equal(ops.expert_dispatch(x, order, w), ops.expert_dispatch(plain(x), order, plain(w)))
        assert torch.equal(ops.expert_combine(y, order, w), ops.expert_combine(plain(y), order, plain(w)))
        for a, b in zip(ops.expert_combine_grad(ups, y, order, w), ops.expert_combine_grad(plain(ups), plain(y), order, plain(w))):
            assert torch.equal(a, b)
        leaf = plain(table).requires_grad_()
        assert torch.equal(torch.autograd.grad(nn.embedding(leaf, ids), leaf, up)[0], ops.embedding_grad(plain(up), ids, 9))


def test_captured_backward_passes_to_leaves_behind_a_view(nn):
    """With an eager graph of the leaf alive the backward pass is refused, the forward call is not; without one both are captured."""
    g = generator(15)
    ids, order = torch.tensor([3, 1, 3], device="cuda"), nn.expert_order(torch.tensor([[0, 1], [1, -1], [0, 0]], device="cuda"), 2)
    y = torch.randn(6, 8, generator=g, device="cuda")
    for shape, call in (((10, 8), lambda t: nn.embedding(t, ids)), ((3, 8), lambda t: nn.dispatch(t, order)),
                        ((6, 8), lambda t: nn.combine(t, order)), ((3, 2), lambda t: nn.combine(y, order, t))):
        leaf = torch.randn(*shape, generator=g, device="cuda").requires_grad_()
        up = torch.randn_like(call(leaf.detach()))
        alive = leaf * 1
        with pytest.raises(RuntimeError, match="behind this operand.*still alive"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                out = call(leaf.view_as(leaf)[:] * 2)
                torch.autograd.grad(out, leaf, up)
        del out
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            kept = call(leaf * 2).detach()                    # no backward pass: nothing to refuse
        graph.replay()
        assert torch.equal(kept, call(leaf.detach() * 2))
        del alive
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            torch.autograd.grad(call(leaf * 2), leaf, up)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            grad, = torch.autograd.grad(call(leaf * 2), leaf, up)
        graph.replay()
        assert torch.equal(grad, torch.autograd.grad(call(leaf * 2), leaf, up)[0])


# ---- addresses and waits ----------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype,code", [(torch.float32, 0), (torch.float16, 1), (torch.bfloat16, 2)])
@pytest.mark.parametrize("n,rows,width", [(60_000, 40, 256), (300_007, 4, 130), (9000, 2, 1032), (200_000, 70, 24)])
def test_the_same_bits_at_any_address_and_stride(ops, dtype, code, n, rows, width):
    """Long sums, whose pieces decide about the last bits."""
    g = generator(4)
    ids = torch.randint(0, rows, (n,), generator=g, device="cuda")
    grad = torch.randn(n, width, generator=g, device="cuda").to(dtype)
    want = ops.embedding_grad(grad, ids, rows), ops.embedding_grad(grad, ids, rows, dtype=torch.float32)
    for shift, gap in ((1, 0), (2, 0), (4, 0), (0, 1), (0, 2), (3, 5), (0, 8)):
        room = torch.empty(shift + n * (width + gap), dtype=dtype, device="cuda")
        there = room[shift:].as_strided((n, width), (width + gap, 1))
        there.copy_(grad)
        assert torch.equal(ops.embedding_grad(there, ids, rows), want[0])
        assert torch.equal(ops.embedding_grad(there, ids, rows, dtype=torch.float32), want[1])
        row_ids, some = ops.embedding_grad_rows(there, ids, rows)
        assert torch.equal(some, want[0][row_ids])
    ctx = ops.default_context()
    work = torch.empty(ctx.lib.gsb_embedding_grad_workspace(n, rows, width), dtype=torch.uint8, device="cuda")
    for shift in (1, 2, 4):
        out = torch.empty(shift + rows * width, dtype=dtype, device="cuda")[shift:].view(rows, width)
        assert ctx.lib.gsb_embedding_grad(ctx.handle, stream(), grad.data_ptr(), code, width, width, ids.data_ptr(), n, rows, 1.0, 0, 0,
                                          out.data_ptr(), code, work.data_ptr(), work.numel()) == 0
        assert torch.equal(out, want[0])


@pytest.mark.parametrize("kind", ["dense", "rows", "order", "order of many"])
def test_a_wait_that_does_run_out(ops, kind):
    """Ids read in place from host memory: the sort's CTAs come to their barrier one after the other, and the first gives up."""
    g = generator(6)
    n, rows, width, pad = 400_000, 30_000, 8, 64
    experts = rows if kind == "order of many" else 50
    ids = torch.randint(0, experts if kind.startswith("order") else rows, (n,), generator=g, device="cuda")
    there = ids.cpu().pin_memory()
    grad = torch.randn(n, width, generator=g, device="cuda")
    ctx = ops.Context()
    lib, h, s = ctx.lib, ctx.handle, stream()
    size = lib.gsb_expert_order_workspace(n, experts) if kind.startswith("order") else lib.gsb_embedding_grad_workspace(n, rows, width)
    work = torch.empty(size, dtype=torch.uint8, device="cuda")

    def room(count, dtype):
        return torch.full((count + pad,), -7, dtype=dtype, device="cuda")

    def call(count_host=None):
        if kind == "dense":
            out = [room(rows * width, torch.float32)]
            st = lib.gsb_embedding_grad(h, s, grad.data_ptr(), 0, width, width, there.data_ptr(), n, rows, 1.0, 0, 0, out[0].data_ptr(), 0,
                                        work.data_ptr(), size)
        elif kind == "rows":
            out = [room(n, torch.int64), room(n * width, torch.float32), room(1, torch.int64)]
            st = lib.gsb_embedding_grad_rows(h, s, grad.data_ptr(), 0, width, width, there.data_ptr(), n, rows, 1.0, 0, 0, out[0].data_ptr(),
                                             out[1].data_ptr(), 0, out[2].data_ptr(), work.data_ptr(), size, count_host)
        else:
            out = [room(experts + 1, torch.int64), room(n, torch.int64), room(n, torch.int64)]
            st = lib.gsb_expert_order(h, s, there.data_ptr(), n, experts, *(t.data_ptr() for t in out), work.data_ptr(), size)
        assert all(bool((t[-pad:] == -7).all()) for t in out)       # nothing is written behind a result, wait or no wait
        return st, [t[:-pad] for t in out]

    st, want = call()
    assert st == 0 and lib.gsb_check_device_status(h, s) == 0
    usual = ctx.get_option("max_polls")
    ctx.set_option("max_polls", 1)
    for _ in range(3):
        st, got = call()
        assert st == 0 and lib.gsb_check_device_status(h, s) == TIMEOUT
        if kind == "dense":
            continue                                                # anything at all
        if kind == "rows":
            assert int(got[2]) == 0
            number = ctypes.c_int64(-1)
            assert call(ctypes.byref(number))[0] == TIMEOUT and number.value == 0
        else:
            offsets, source, place = got
            assert 0 <= int(offsets.min()) and int(offsets.max()) <= n and 0 <= int(source.min()) and int(source.max()) < n
            assert -n <= int(place.min()) and int(place.max()) < n
    ctx.set_option("max_polls", usual)
    st, got = call()
    assert st == 0 and lib.gsb_check_device_status(h, s) == 0
    number = int(want[2]) if kind == "rows" else None
    if kind == "rows":
        got, want = [got[0][:number], got[1][:number * width], got[2]], [want[0][:number], want[1][:number * width], want[2]]
    assert all(torch.equal(x, y) for x, y in zip(got, want))


def test_what_places_out_of_range_leave(ops):
    """Rows that no place names are not written; the others are right; sums leave bad places out."""
    g = generator(7)
    ctx = ops.Context()
    tokens, per_token, width = 50, 3, 20
    slots = tokens * per_token
    place = torch.randperm(slots, generator=g, device="cuda").view(tokens, per_token)
    bad = torch.rand(tokens, per_token, generator=g, device="cuda") < 0.2
    given = torch.where(bad, torch.where(torch.rand(tokens, per_token, generator=g, device="cuda") < 0.5, slots, -(1 << 40)), place)
    x, y = torch.randn(tokens, width, generator=g, device="cuda"), torch.randn(slots, width, generator=g, device="cuda")
    w = torch.rand(tokens, per_token, generator=g, device="cuda")
    named = torch.zeros(slots, dtype=torch.bool, device="cuda")
    named[place[~bad]] = True
    lib, h, s = ctx.lib, ctx.handle, stream()
    out = torch.full((slots, width), 7.0, device="cuda")
    assert lib.gsb_expert_spread(h, s, x.data_ptr(), 0, tokens, per_token, width, width, given.data_ptr(), None, 0, out.data_ptr()) == 0
    want = torch.full((slots, width), 7.0, device="cuda")
    want[place.reshape(-1)] = x.repeat_interleave(per_token, 0)
    want[~named] = 7.0
    assert torch.equal(out, want) and lib.gsb_check_device_status(h, s) == -8
    rows, weights = torch.full((slots, width), 7.0, device="cuda"), torch.full((tokens, per_token), 7.0, device="cuda")
    up = torch.randn(tokens, width, generator=g, device="cuda")
    assert lib.gsb_expert_combine_grad(h, s, up.data_ptr(), 0, tokens, per_token, width, width, y.data_ptr(), slots, width, given.data_ptr(),
                                       w.data_ptr(), 0, rows.data_ptr(), weights.data_ptr()) == 0
    assert bool((rows[~named] == 7).all()) and bool((weights[bad] == 0).all()) and lib.gsb_check_device_status(h, s) == -8
    left_out = torch.where(bad, -1, place)
    exact.within(rows[named], *(t[named] for t in exact.spread(up, place, w)))
    exact.within(weights, *exact.weight_grads(up, y, left_out))
    exact.within(ops.expert_combine(y, given, w, ctx=ctx), *exact.combine(y, left_out, w))
    assert lib.gsb_check_device_status(h, s) == -8
    assert torch.equal(ops.expert_dispatch(x, given, ctx=ctx)[named], want[named])
    assert lib.gsb_check_device_status(h, s) == -8


@pytest.mark.parametrize("n,experts", [(20_000, 50), (40_001, 7), (300_000, 1000), (123_457, 60_000), (700_001, 2000)])
@pytest.mark.parametrize("most", [1, 2, 7, 100, 147, 148, 1000])
def test_orders_by_fewer_ctas(ops, n, experts, most):
    """A GPU, or a part of one, that holds fewer CTAs at once than a B200."""
    g = generator(11)
    ids = torch.randint(-1, experts, (n,), generator=g, device="cuda")
    ctx = ops.Context()
    size = ctx.lib.gsb_expert_order_workspace(n, experts)
    work = torch.full((size + 256,), 77, dtype=torch.uint8, device="cuda")
    offsets, source, place = (torch.full((m + 8,), -7, dtype=torch.int64, device="cuda") for m in (experts + 1, n, n))
    assert ctx.lib.gsb_selftest_expert_order(ctx.handle, stream(), ids.data_ptr(), n, experts, most, offsets.data_ptr(), source.data_ptr(),
                                             place.data_ptr(), work.data_ptr(), size) == 0
    for got, want in zip((offsets, source, place), exact.order(ids, experts)):
        assert torch.equal(got[:-8], want) and bool((got[-8:] == -7).all())
    assert bool((work[size:] == 77).all())
    ctx.check_device()
    assert ctx.lib.gsb_selftest_expert_order(ctx.handle, stream(), ids.data_ptr(), n, experts, 0, offsets.data_ptr(), source.data_ptr(),
                                             place.data_ptr(), work.data_ptr(), size) == -1


@pytest.mark.parametrize("n", [1, 5, 33, 1030, 4100, 32_768, 40_003])
@pytest.mark.parametrize("experts", [3, 2048, 2055, 65_535, 65_536])
def test_offsets_of_experts_without_slots(ops, n, experts):
    """Runs of them of any length in front, in between and behind."""
    g = generator(12)
    few = torch.randint(0, experts, (n,), generator=g, device="cuda") // 9 * 9
    for ids in (few, few.clamp(min=experts // 2), few.clamp(max=experts // 3), torch.full_like(few, experts - 1), torch.zeros_like(few),
                torch.full_like(few, -1), torch.where(few % 2 == 0, experts // 2, -1)):
        for got, want in zip(ops.expert_order(ids, experts), exact.order(ids, experts)):
            assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("width,n", [(399, 82_000), (401, 79_000), (401, 80_001), (601, 60_000), (799, 40_000), (799, 41_003), (801, 19_000), (801, 21_001)])
def test_odd_rows_on_both_sides_of_the_staged_lookup(ops, dtype, width, n):
    g = generator(13)
    room = torch.randn(3 + 700 * (width + 4), generator=g, device="cuda").to(dtype)
    table = room[3:].as_strided((700, width), (width + 4, 1))
    ids = torch.randint(0, 700, (n,), generator=g, device="cuda")
    ids[:2] = torch.tensor([0, 699])
    assert torch.equal(ops.embedding_lookup(table, ids), table[ids])
    want = table[ids] * 0.5
    want[ids == 7] = 0
    assert torch.equal(ops.embedding_lookup(table, ids, 0.5, 7), want)


def test_a_wait_of_the_sampler_that_ran_out_is_read_by_a_call_on_rows(ops):
    """The next cooperative call of the context works again, without anybody else reading the error."""
    g = generator(14)
    n, keys = 300_001, 1_000_000
    key = torch.randint(0, keys, (n,), generator=g, device="cuda")
    there, rows_in = key.cpu().pin_memory(), torch.arange(n, device="cuda")
    ctx = ops.Context()
    lib, h, s = ctx.lib, ctx.handle, stream()

    def convert():
        out = [torch.empty(m, dtype=torch.int64, device="cuda") for m in (keys + 1, n, n)]
        assert lib.gsb_coo2csc(h, s, there.data_ptr(), rows_in.data_ptr(), n, keys, 0, *(t.data_ptr() for t in out)) == 0
        return out

    want = convert()
    ctx.check_device()
    usual = ctx.get_option("max_polls")
    ids, grad = torch.tensor([3, 1, 3], device="cuda"), torch.ones(3, 4, device="cuda")
    for _ in range(3):
        ctx.set_option("max_polls", 1)
        convert()
        ctx.set_option("max_polls", usual)
        torch.cuda.synchronize()
        with pytest.raises(Exception) as e:
            ops.embedding_grad_rows(grad, ids, 5, ctx=ctx)
        assert e.value.status == TIMEOUT
        assert ops.embedding_grad_rows(grad, ids, 5, ctx=ctx)[0].tolist() == [1, 3]
        assert all(torch.equal(x, y) for x, y in zip(convert(), want))
        ctx.check_device()


# ---- values -------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_infinities_and_nan_that_count(ops, dtype):
    """They reach the sums that they belong to and no other, in short sums and in those that many chunks share."""
    g = generator(8)
    n, rows, width = 5000, 6, 40
    ids = torch.randint(0, 3, (n,), generator=g, device="cuda") * 2
    grad = torch.randn(n, width, generator=g, device="cuda").to(dtype)
    grad[ids == 0] = 1.0
    grad[int((ids == 0).nonzero()[7]), 3] = float("inf")
    at = (ids == 2).nonzero().flatten()
    grad[at[5], 4], grad[at[900], 4] = float("inf"), float("-inf")
    grad[at[11], 5] = float("nan")
    out = ops.embedding_grad(grad, ids, rows, 0.5)
    want = torch.zeros(rows, width, dtype=torch.float64, device="cuda").index_add_(0, ids, grad.double()) * 0.5
    assert torch.equal(out.isnan(), want.isnan()) and torch.equal(out.isposinf(), want.isposinf()) and not out.isneginf().any()
    assert out[0, 3] == float("inf") and out[2, 4].isnan() and out[2, 5].isnan()
    row_ids, some = ops.embedding_grad_rows(grad, ids, rows, 0.5)
    assert row_ids.tolist() == [0, 2, 4] and torch.equal(some.nan_to_num(3.0), out[::2].nan_to_num(3.0))
    order = torch.tensor([[0, 2], [1, 3], [4, ~5]], device="cuda")
    y = torch.ones(6, width, dtype=dtype, device="cuda")
    y[0, 1], y[2, 1], y[3, 2], y[5] = float("inf"), float("-inf"), float("nan"), float("nan")
    got = ops.expert_combine(y, order)
    assert got[0, 1].isnan() and got[1, 2].isnan() and int(got.isnan().sum()) == 2 and torch.all(got[2] == 1)
    grad_rows, grad_weights = ops.expert_combine_grad(torch.ones(3, width, dtype=dtype, device="cuda"), y, order,
                                                      torch.tensor([[2.0, 1.0], [float("inf"), 1.0], [1.0, float("nan")]], device="cuda"))
    assert grad_weights[0].tolist() == [float("inf"), float("-inf")] and grad_weights[1, 1].isnan() and grad_weights[2].tolist() == [width, 0]
    assert torch.all(grad_rows[1].isposinf()) and torch.all(grad_rows[5] == 0) and torch.all(grad_rows[0] == 2)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("width,n", [(1, 500), (33, 3000), (101, 40_000), (601, 30_000), (4095, 4000)])
def test_odd_rows_out_of_pinned_host_memory(ops, nn, dtype, width, n):
    table = torch.randn(501, width).to(dtype).pin_memory()
    g = generator(9)
    ids = torch.randint(0, 501, (n,), generator=g, device="cuda")
    there = table.cuda()
    assert torch.equal(ops.embedding_lookup(table, ids), there[ids])
    want = there[ids] * 0.5
    want[ids == 7] = 0
    assert torch.equal(ops.embedding_lookup(table, ids, 0.5, 7), want) and torch.equal(nn.embedding(table, ids, 0.5, 7), want)
    assert torch.equal(ops.embedding_lookup(table[3:], ids.clamp(max=497)), there[3:][ids.clamp(max=497)])


def test_pinned_tables_that_go_at_once(ops):
    """A table may be dropped behind the call: its memory is not handed out again while the lookup is still to come."""
    ids = torch.arange(2000, device="cuda")
    filler = torch.randn(4096, 4096, device="cuda")
    ops.embedding_lookup(torch.zeros(2000, 64).pin_memory(), ids)
    torch.cuda.synchronize()
    for turn in range(5):
        for _ in range(20):
            filler @ filler                                   # long enough for the host to get ahead
        out = ops.embedding_lookup(torch.full((2001, 64), float(turn)).pin_memory()[1:], ids)
        later = [torch.full((2001, 64), -1.0).pin_memory() for _ in range(4)]
        assert bool((out == turn).all())
        del later
