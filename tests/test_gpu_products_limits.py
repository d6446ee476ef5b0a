"""Products by expert and quantized rows at the ends of what they take: more rows than 32 bits count lanes of, offsets that fall from one launch's experts to the
next's, views, float32 on the tensor cores near the largest and the smallest numbers, sums over hundreds of thousands of values."""
import ctypes

import pytest
import torch

import expert_products as exact
from learned_rows import within

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
CODES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}


@pytest.fixture(scope="module")
def ops():
    from graph_sampling_b200 import ops as m
    return m


def generator(seed):
    g = torch.Generator("cuda")
    g.manual_seed(seed)
    return g


def normal(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def stream():
    return ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)


@pytest.mark.parametrize("dtype,width", [(torch.bfloat16, 65), (torch.float32, 65)])
def test_more_rows_than_32_bits_count_lanes_of(ops, dtype, width):
    """A warp a row: 2^27 rows are 2^32 lanes.  One row in memory stands for all."""
    n = (1 << 27) + 41
    if torch.cuda.mem_get_info()[0] < 12 << 30:
        pytest.skip("needs 12 GB")
    ctx = ops.default_context()
    row = normal(generator(1), 1, width, dtype=dtype)
    want, want_scale = exact.quantized(row)
    values, scales = torch.full((n, width), 99, dtype=torch.int8, device="cuda"), torch.full((n,), -1.0, device="cuda")
    assert 99 not in want.tolist()[0]
    assert ctx.lib.gsb_quantize_rows(ctx.handle, stream(), row.data_ptr(), CODES[dtype], n, width, 0, values.data_ptr(), width, scales.data_ptr()) == 0
    assert torch.all(scales == want_scale)
    for first in range(0, n, 1 << 23):
        assert torch.all(values[first:first + (1 << 23)] == want), first


def test_negated_views_in_8_bits(ops):
    """Rows and weights that lie on 16-byte boundaries and are read in place, and some that do not and are copied."""
    g = generator(2)
    offsets = torch.tensor([0, 20, 50], device="cuda")
    scales, weight_scales = torch.rand(50, generator=g, device="cuda"), torch.rand(2, 40, generator=g, device="cuda")
    for k in (32, 27):
        values = torch.randint(-127, 128, (50, k), generator=g, device="cuda").to(torch.int8)
        weight_values = torch.randint(-127, 128, (2, 40, k), generator=g, device="cuda").to(torch.int8)
        minus = ops.expert_product_int8(-values, scales, weight_values, weight_scales, offsets)
        assert torch.count_nonzero(minus) > 0
        assert torch.equal(ops.expert_product_int8(torch._neg_view(values), scales, weight_values, weight_scales, offsets), minus)
        assert torch.equal(ops.expert_product_int8(values, scales, torch._neg_view(weight_values), weight_scales, offsets), minus)


@pytest.mark.parametrize("rows_of_all,k,n", [(6_000, 24, 16), (40_000, 256, 128), (40_001, 250, 99)])
def test_offsets_that_fall_from_one_launch_to_the_next(ops, rows_of_all, k, n):
    """A launch takes 1 024 experts.  An offset below one of an earlier launch is raised to it as it is within a launch: no row is in two experts, and those
    behind the last expert's are zeros."""
    from graph_sampling_b200.cabi import GsbError
    g, ctx, experts = generator(k), ops.Context(), 2500
    good = torch.randint(0, rows_of_all + 1, (experts + 1,), generator=g, device="cuda").sort().values
    falls = good.clone()
    falls[500], falls[1024] = good[1100], good[3]                                # the second launch's first is below
    far = good.clone()
    far[10], far[1025:2049] = good[2300], good[1025:2049] // 2                   # the third's are below one of the first
    end = good.clone()
    end[-1] = end[2049] = 5                                                      # the last launch ends below where an earlier one does
    for dtype in DTYPES:
        rows, grad, weights = normal(g, rows_of_all, k, dtype=dtype), normal(g, rows_of_all, n, dtype=dtype), normal(g, experts, k, n, dtype=dtype)
        values, scales = ops.quantize_rows(rows)
        weight_values, weight_scales = ops.quantize_rows(weights.transpose(1, 2))
        for offsets in (good, falls, far, end):
            for call in (lambda: within(ops.expert_product(rows, weights, offsets, ctx=ctx), *exact.product(rows, weights, offsets)),
                         lambda: within(ops.expert_product(grad, weights.transpose(1, 2), offsets, ctx=ctx),
                                        *exact.product(grad, weights.transpose(1, 2), offsets)),
                         lambda: within(ops.expert_product_grad(rows, grad, offsets, ctx=ctx), *exact.grad_weights(rows, grad, offsets)),
                         lambda: within(ops.expert_product_int8(values, scales, weight_values, weight_scales, offsets, dtype, ctx=ctx),
                                        *exact.product_int8(values, scales, weight_values, weight_scales, offsets))):
                call()
                if offsets is good:
                    ctx.check_device()
                else:
                    with pytest.raises(GsbError) as e:
                        ctx.check_device()
                    assert e.value.status == -8


def test_workspace_of_many_experts(ops):
    """More than 1 024 experts want room for where each launch ends, whatever kernels the call goes to."""
    ctx, g = ops.default_context(), generator(4)
    rows, grad, weights = normal(g, 1500, 8), normal(g, 1500, 8), normal(g, 1500, 8, 8)
    offsets = torch.arange(1501, device="cuda")
    need = ctx.lib.gsb_expert_product_workspace(rows.data_ptr(), 0, 1500, 8, 8, weights.data_ptr(), 64, 8, 1, 8, 1500)
    need_grad = ctx.lib.gsb_expert_product_grad_workspace(rows.data_ptr(), 0, 1500, 8, 8, grad.data_ptr(), 8, 8, 1500)
    assert need > 0 and need_grad > 0
    work, out, out_grad = torch.empty(max(need, need_grad), dtype=torch.uint8, device="cuda"), torch.empty_like(rows), torch.empty_like(weights)

    def product(room, size):
        return ctx.lib.gsb_expert_product(ctx.handle, stream(), rows.data_ptr(), 0, 1500, 8, 8, weights.data_ptr(), 64, 8, 1, 8, offsets.data_ptr(), 1500,
                                          out.data_ptr(), room, size)

    def product_grad(room, size):
        return ctx.lib.gsb_expert_product_grad(ctx.handle, stream(), rows.data_ptr(), 0, 1500, 8, 8, grad.data_ptr(), 8, 8, offsets.data_ptr(), 1500,
                                               out_grad.data_ptr(), room, size)
    for call, size in ((product, need), (product_grad, need_grad)):
        assert call(None, 0) == -1 and call(work.data_ptr(), size - 1) == -4 and call(work.data_ptr(), size) == 0
    within(out, *exact.product(rows, weights, offsets))
    within(out_grad, *exact.grad_weights(rows, grad, offsets))


class MappedMemory:
    """`size` bytes (a multiple of 2 MiB) with nothing mapped behind them, as a tensor of bytes."""
    GRANULE = 2 << 20

    def __init__(self, size):
        self.cuda, self.size, self.address = ctypes.CDLL("libcuda.so.1"), size, ctypes.c_uint64(0)
        self.handle = ctypes.c_uint64(0)
        # CUmemAllocationProp: pinned memory of the current device; CUmemAccessDesc: to be read and written by it
        device = torch.cuda.current_device()
        prop, access = (ctypes.c_int32 * 8)(1, 0, 1, device, 0, 0, 0, 0), (ctypes.c_int32 * 3)(1, device, 3)
        self.do("cuMemAddressReserve", ctypes.byref(self.address), ctypes.c_size_t(size + self.GRANULE), ctypes.c_size_t(0), ctypes.c_uint64(0), ctypes.c_uint64(0))
        self.do("cuMemCreate", ctypes.byref(self.handle), ctypes.c_size_t(size), ctypes.byref(prop), ctypes.c_uint64(0))
        self.do("cuMemMap", self.address, ctypes.c_size_t(size), ctypes.c_size_t(0), self.handle, ctypes.c_uint64(0))
        self.do("cuMemSetAccess", self.address, ctypes.c_size_t(size), ctypes.byref(access), ctypes.c_size_t(1))
        self.__cuda_array_interface__ = {"shape": (size,), "typestr": "|u1", "data": (self.address.value, False), "version": 3}
        self.bytes = torch.as_tensor(self, device="cuda")
        assert self.bytes.data_ptr() == self.address.value

    def do(self, name, *args):
        status = getattr(self.cuda, name)(*args)
        assert status == 0, (name, status)

    def last(self, rows, width, dtype):
        """A matrix that ends where the memory does."""
        size = torch.empty(0, dtype=dtype).element_size()
        return self.bytes[self.size - rows * width * size:].view(dtype).view(rows, width)

    def free(self):
        torch.cuda.synchronize()
        del self.bytes
        self.do("cuMemUnmap", self.address, ctypes.c_size_t(self.size))
        self.do("cuMemRelease", self.handle)
        self.do("cuMemAddressFree", self.address, ctypes.c_size_t(self.size + self.GRANULE))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("k,n,counts", [(64, 64, [1] * 16384), (256, 320, [5000, 0, 3191]), (128, 64, [64] * 128 + [8191]), (512, 512, [2, 63, 65, 3966])])
def test_rows_that_end_where_memory_does(ops, dtype, k, n, counts):
    """Nothing is mapped behind the rows and the gradient's rows of an expert that ends inside a tile."""
    g, offsets, rows = generator(k), torch.tensor([0] + counts, device="cuda").cumsum(0), sum(counts)
    size = [(rows * width * 2 + (4 << 20) - 1) // (2 << 20) * (2 << 20) for width in (k, n)]
    memory, other = MappedMemory(size[0]), MappedMemory(size[1])
    x, d = memory.last(rows, k, dtype), other.last(rows, n, dtype)
    x.copy_(normal(g, rows, k, dtype=dtype))
    d.copy_(normal(g, rows, n, dtype=dtype))
    got = ops.expert_product_grad(x, d, offsets)
    out = ops.expert_product(x, normal(generator(1), len(counts), k, n, dtype=dtype), offsets)
    torch.cuda.synchronize()
    want = torch.zeros(got.shape, dtype=torch.float64, device="cuda")
    error = torch.zeros_like(want)
    if len(counts) == rows:  # one row each
        want = x.double()[:, :, None] * d.double()[:, None, :]
        error = 18 * exact.U * want.abs()
    else:
        want, error = exact.grad_weights(x, d, offsets)
    within(got, want, error)
    some = slice(0, offsets.numel() - 1) if len(counts) < 200 else slice(len(counts) - 50, len(counts))
    weights = normal(generator(1), len(counts), k, n, dtype=dtype)
    first, part = int(offsets[some.start]), offsets[some.start:some.stop + 1] - offsets[some.start]
    within(out[first:], *exact.product(x[first:], weights[some], part))
    x = d = None
    memory.free()
    other.free()


@pytest.mark.parametrize("dtype", DTYPES)
def test_gradients_of_experts_that_end_inside_a_tile(ops, dtype):
    """The next expert's rows, infinities and NaN among them, are none of an expert's, wherever in a line of 64 rows it ends."""
    g = generator(6)
    counts = [64 * (i % 3) + i for i in range(1, 64)] + [0, 64, 128, 1, 700, 3000]
    offsets, n = torch.tensor([5] + counts, device="cuda").cumsum(0), sum(counts) + 5 + 70
    for k, m in ((64, 64), (200, 136), (264, 520)):
        rows, grad = normal(g, n, k, dtype=dtype), normal(g, n, m, dtype=dtype)
        want, error = exact.grad_weights(rows, grad, offsets)
        within(ops.expert_product_grad(rows, grad, offsets), want, error)
        spoiled, spoiled_grad = rows.clone(), grad.clone()
        for e in range(1, len(counts), 2):
            spoiled[offsets[e]:offsets[e + 1]] = float("nan")
            spoiled_grad[offsets[e]:offsets[e + 1]] = float("inf")
        for at in (slice(0, 5), slice(int(offsets[-1]), n)):
            spoiled[at], spoiled_grad[at] = float("inf"), float("nan")
        within(ops.expert_product_grad(spoiled, spoiled_grad, offsets)[::2], want[::2], error[::2])


# ---- float32 on the tensor cores -------------------------------------------------------------------------------------------------------
# Operands are taken apart into three parts, a = a0 + a1 + a2 exactly, the first towards zero: |a1| < 2^-7 |a|, |a2| <= 2^-16 |a|.  Left out are a1 b2,
# a2 b1 and a2 b2, below 2^-22 (1 + 2^-10) |a b| together.  Where a sum has one product that is not zero, a0 b0 is exact, the five others, 2^-6 of it in
# size, are added in five additions that cut less than 2^-23 of them each, and the two sums meet in one rounding of 2^-24.
ONE_PRODUCT = 2.0 ** -22 + 2.0 ** -24 + 2.0 ** -26
ROWS, K, N = 3000, 520, 512
ENDS = [0, 1100, 1100, 2990]


def by_tiles(ops, rows, weights, grad):
    """All three calls of these operands go to the tensor cores: of float32 they want room for the weights' parts and for the rows' descriptions."""
    lib, (n, k), (experts, _, m) = ops.default_context().lib, rows.shape, weights.shape
    forward = lib.gsb_expert_product_workspace(rows.data_ptr(), 0, n, k, k, weights.data_ptr(), k * m, m, 1, m, experts)
    back = lib.gsb_expert_product_workspace(grad.data_ptr(), 0, n, m, m, weights.data_ptr(), k * m, 1, m, k, experts)
    return min(forward, back, lib.gsb_expert_product_grad_workspace(rows.data_ptr(), 0, n, k, k, grad.data_ptr(), m, m, experts)) > 0


def one_product_each(g, near):
    """Rows, weights and gradient rows of which every sum of a product, of the rows' gradient and of the weights' has one product that is not zero.  `near`:
    all of those within 2^-9 of the largest number, above it none; else numbers of 24 bits around 1."""
    def number(*shape):
        x = 1 + torch.rand(*shape, generator=g, device="cuda") * (2 ** -10 if near else 1)
        return x * torch.where(torch.rand(*shape, generator=g, device="cuda") < 0.5, -1.0, 1.0)
    top = torch.finfo(torch.float32).max
    low, high = (2.0 ** 63 * (1.25 + 0.75 / 128), 0.0) if near else (1.0, 1.0)  # to nearest in 8 bits both are larger
    if near:  # (1 + 2^-10)^2 (1 + 2^-20) low high is the largest number
        high = top / (low * (1 + 2 ** -10) ** 2 * (1 + 2 ** -20))
    weights = number(3, K, N) * low
    rows, grad = torch.zeros(ROWS, K, device="cuda"), torch.zeros(ROWS, N, device="cuda")
    at = torch.arange(ROWS, device="cuda")
    rows[at, at * 7 % K] = number(ROWS) * high
    grad[at, at * 5 % N] = number(ROWS) * high
    # of the weights' gradient: one row of each expert with numbers, the others zeros
    alone, alone_grad = torch.zeros(ROWS, K, device="cuda"), torch.zeros(ROWS, N, device="cuda")
    for a, b in ((0, 1100), (1100, 2990)):
        alone[(a + 2 * b) // 3], alone_grad[(a + 2 * b) // 3] = number(K) * high, number(N) * low
    return rows, weights, grad, alone, alone_grad


def all_close(got, want, relative):
    assert want.float().isfinite().all() and got.isfinite().all()
    assert ((got.double() - want).abs() - relative * want.abs()).max().item() <= 0


@pytest.mark.parametrize("near", [False, True])
def test_float32_products_of_24_bits(ops, near):
    """Every part of both operands counts: losing a product of a third part, or of two second ones, would be off by up to 2^-16 and 2^-14.  And a product that is
    not infinite is none, however near the largest number it and its factors' first parts are."""
    g, offsets = generator(11 + near), torch.tensor(ENDS, device="cuda")
    rows, weights, grad, alone, alone_grad = one_product_each(g, near)
    assert by_tiles(ops, rows, weights, grad)
    all_close(ops.expert_product(rows, weights, offsets), exact.product(rows, weights, offsets)[0], ONE_PRODUCT)
    turned = weights.transpose(1, 2)
    all_close(ops.expert_product(grad, turned, offsets), exact.product(grad, turned, offsets)[0], ONE_PRODUCT)
    all_close(ops.expert_product_grad(alone, alone_grad, offsets), exact.grad_weights(alone, alone_grad, offsets)[0], ONE_PRODUCT)


def same_numbers(got, want, error):
    """NaN and infinities where the definition in 64 bits has them, and numbers within the bound."""
    narrow = want.float()
    assert torch.equal(got.isnan(), narrow.isnan()) and torch.equal(got == float("inf"), narrow == float("inf"))
    assert torch.equal(got == -float("inf"), narrow == -float("inf"))
    fine = narrow.isfinite()
    within(got[fine], want[fine], error[fine])


def test_float32_infinities_and_nan(ops):
    """In rows, weights and gradient rows, by ones and by whole rows, of some experts and of rows of none."""
    g, offsets, inf, nan = generator(13), torch.tensor(ENDS, device="cuda"), float("inf"), float("nan")
    rows, weights, grad = normal(g, ROWS, K), normal(g, 3, K, N), normal(g, ROWS, N)
    assert by_tiles(ops, rows, weights, grad)
    clean = rows.clone(), weights.clone(), grad.clone()

    def all_three(rows, weights, grad):
        for got, (want, _), (_, error) in ((ops.expert_product(rows, weights, offsets), exact.product(rows, weights, offsets), exact.product(clean[0], clean[1], offsets)),
                                           (ops.expert_product(grad, weights.transpose(1, 2), offsets), exact.product(grad, weights.transpose(1, 2), offsets),
                                            exact.product(clean[2], clean[1].transpose(1, 2), offsets)),
                                           (ops.expert_product_grad(rows, grad, offsets), exact.grad_weights(rows, grad, offsets),
                                            exact.grad_weights(clean[0], clean[2], offsets))):
            same_numbers(got, want, error)
    all_three(*clean)
    for x, width in ((rows, K), (grad, N)):
        x[7, 3], x[8, width - 1], x[130, 64], x[131, 63] = inf, -inf, nan, inf
        x[1500, 5], x[1500, 6] = inf, -inf
        x[2000], x[2995] = 0, nan
        x[2000, 9] = inf
    all_three(rows, clean[1], clean[2])
    all_three(clean[0], clean[1], grad)
    weights[0, 5, 7], weights[0, :, 100], weights[2, K - 1, N - 1], weights[2, 64, 64], weights[1] = inf, 0, -inf, nan, nan
    all_three(clean[0], weights, clean[2])
    all_three(rows, weights, grad)
    weights[0, 5, 7] = weights[2, K - 1, N - 1] = torch.finfo(torch.float32).max  # and next to it the largest number alone
    weights[2, 64, 64] = 0
    rows[:, 5], rows[:, K - 1], grad[:, 7], grad[:, N - 1] = 0.5, -0.25, 0.125, 0.5
    got, want = ops.expert_product(rows, weights, offsets), exact.product(rows, weights, offsets)[0]
    assert torch.equal(got.isfinite(), want.float().isfinite())
    got, want = ops.expert_product(grad, weights.transpose(1, 2), offsets), exact.product(grad, weights.transpose(1, 2), offsets)[0]
    assert torch.equal(got.isfinite(), want.float().isfinite())


def test_float32_root_mean_square(ops):
    """What the documents say of the error of sums: 3e-7 of the result (rms).  Each of the six products of parts that are summed is above it."""
    g, offsets = generator(14), torch.tensor(ENDS, device="cuda")
    rows, weights, grad = normal(g, ROWS, K), normal(g, 3, K, N), normal(g, ROWS, N)
    assert by_tiles(ops, rows, weights, grad)
    for got, (want, _) in ((ops.expert_product(rows, weights, offsets), exact.product(rows, weights, offsets)),
                           (ops.expert_product(grad, weights.transpose(1, 2), offsets), exact.product(grad, weights.transpose(1, 2), offsets)),
                           (ops.expert_product_grad(rows, grad, offsets), exact.grad_weights(rows, grad, offsets))):
        assert ((got.double() - want).pow(2).mean().sqrt() / want.pow(2).mean().sqrt()).item() < 6e-7




@pytest.mark.parametrize("exponent", [-149, -142, -134, -133, -130, -126])
def test_float32_infinity_times_the_smallest_weights(ops, exponent):
    """Infinity times a weight is NaN where the weight is 0, and else infinity, however small it is."""
    g, offsets, inf = generator(15), torch.tensor(ENDS, device="cuda"), float("inf")
    rows, weights, grad = torch.zeros(ROWS, K, device="cuda"), torch.zeros(3, K, N, device="cuda"), torch.zeros(ROWS, N, device="cuda")
    sign = torch.where(torch.rand(3, 64, 64, generator=g, device="cuda") < 0.5, -1.0, 1.0)
    weights[:, :64, :64] = (sign.double() * torch.randint(1, 3, (3, 64, 64), generator=g, device="cuda") * 2.0 ** exponent).float()
    at = torch.arange(ROWS, device="cuda")
    rows[at, at % 64] = grad[at, at % 64] = inf
    assert by_tiles(ops, rows, weights, grad)
    turned = weights.transpose(1, 2)
    for got, want in ((ops.expert_product(rows, weights, offsets), exact.product(rows, weights, offsets)[0]),
                      (ops.expert_product(grad, turned, offsets), exact.product(grad, turned, offsets)[0])):
        assert (want == inf).any() and (want == -inf).any() and want.isnan().any()
        assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got == inf, want == inf) and torch.equal(got == -inf, want == -inf)


# ---- long sums of 16-bit types -----------------------------------------------------------------------------------------------------------
# Tensor memory cuts what an addition of 16 products leaves below the sum's last bits.  By what was measured an instruction's products are held with two bits
# more than the sum, whose last is 2^-23 of it at most: 16 products cut by 2^-25 and the sum by 2^-23 are 5 * 2^-23 of the running sum at the very most, half of that on average,
# and of the final one, where all are positive, half again.  Sums leave it after 16 384 values, 1 024 instructions: 1 024 * 5 / 4 * 2^-23 = 1.5e-4 of the result
# (1.1e-4 was measured).  The float additions of 62 such sums to a million values are below 62 / 2 * 2^-24 < 2^-19.
LONG = 1024 * 5 / 4 * 2.0 ** -23 + 2.0 ** -19


def positive(g, dtype, *shape):
    return (torch.rand(*shape, generator=g, device="cuda") * 0.03 + 0.001).to(dtype)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("k,first", [(300_032, 0), (1_000_000, 0), (999_996, 0), (999_001, 0), (600_000, 1), (600_000, 2)])
def test_products_over_long_rows(ops, dtype, k, first):
    """By TMA, by TMA class by class, copied and read by warps (`first`: values in front of the first row, off 16-byte boundaries)."""
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("needs 24 GB")
    g = generator(k)
    rows = positive(g, dtype, 500 * k + 8)[first:first + 500 * k].view(500, k)
    offsets = torch.tensor([0, 150, 150, 490], device="cuda")
    for n, turned in ((120, False), (250, True)):
        weights = positive(g, dtype, 3, n, k).transpose(1, 2) if turned else positive(g, dtype, 3, k, n)
        out = ops.expert_product(rows, weights, offsets)
        want = exact.product(rows, weights, offsets)[0]
        within(out, want, want.abs() * LONG)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("width", [512, 508])
def test_gradients_over_long_experts(ops, dtype, width):
    """So many matrices that there is no room for sums of chunks: an expert's million rows are summed in one."""
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("needs 24 GB")
    g, n, experts = generator(width), 1_000_000, 1040
    rows, grad = positive(g, dtype, n, width), positive(g, dtype, n, width)
    offsets = torch.full((experts + 1,), n - 3, dtype=torch.long, device="cuda")
    offsets[:3] = torch.tensor([0, 0, 990_001], device="cuda")
    out = ops.expert_product_grad(rows, grad, offsets)
    for e, a, b in ((1, 0, 990_001), (2, 990_001, n - 3)):
        want = sum(rows[i:min(i + 100_000, b)].double().t() @ grad[i:min(i + 100_000, b)].double() for i in range(a, b, 100_000))
        within(out[e], want, want.abs() * LONG)
    assert not out[0].any() and not out[3:].any()
