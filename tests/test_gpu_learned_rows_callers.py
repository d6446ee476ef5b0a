"""Learned rows beside other callers and in calls that the documentation allows and few make: threads, kinds of tensors, addresses,
waits that run out, values that are no numbers."""
import ctypes
import threading

import pytest
import torch

import learned_rows as exact

pytestmark = pytest.mark.gpu


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
