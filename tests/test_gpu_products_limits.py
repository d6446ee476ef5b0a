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
