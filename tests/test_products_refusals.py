"""What products by expert and dropout refuse before anything is launched, and the definitions that their tests use; no GPU is needed."""
import pytest
import torch

import expert_products as exact
from graph_sampling_b200 import cabi
from graph_sampling_b200 import build as gsb_build


@pytest.fixture(scope="module")
def native():
    gsb_build.build()
    gsb_build.build_native()
    from graph_sampling_b200 import ops
    return ops._load_native()


rows, weights, offsets = torch.zeros(6, 4), torch.zeros(2, 4, 3), torch.tensor([0, 2, 6])
values, scales = torch.zeros(6, 4, dtype=torch.int8), torch.zeros(6)
weight_values, weight_scales = torch.zeros(2, 3, 4, dtype=torch.int8), torch.zeros(2, 3)


@pytest.mark.parametrize("name,args,message", [
    ("expert_product", (None, weights, offsets), "rows must be a tensor"),
    ("expert_product", (rows.double(), weights, offsets), "float32, float16 or bfloat16"),
    ("expert_product", (rows[0], weights, offsets), "two dimensions"),
    ("expert_product", (rows, weights, offsets), "rows must be a CUDA tensor"),
    ("expert_product_grad", (rows, rows.long(), offsets), "rows must be a CUDA tensor"),
    ("expert_product_grad", (rows, None, offsets), "grad must be a tensor"),
    ("quantize_rows", (rows.double(),), "float32, float16 or bfloat16"),
    ("quantize_rows", (torch.tensor(1.0),), "at least one dimension"),
    ("quantize_rows", (rows,), "x must be a CUDA tensor"),
    ("expert_product_int8", (rows, scales, weight_values, weight_scales, offsets, torch.float32), "values must be int8"),
    ("expert_product_int8", (values[0], scales, weight_values, weight_scales, offsets, torch.float32), "two dimensions"),
    ("expert_product_int8", (values, scales, weight_values, weight_scales, offsets, torch.int8), "result's dtype"),
    ("expert_product_int8", (values, scales, weight_values, weight_scales, offsets, None), "torch.dtype"),
    ("expert_product_int8", (values, scales, weight_values, weight_scales, offsets, torch.float32), "values must be a CUDA tensor"),
    ("dropout", (rows.long(), 0.5, 1, None), "float32, float16 or bfloat16"),
    ("dropout", (rows, "x", 1, None), "real number"),
    ("dropout", (rows, 0.5, 1.5, None), "int"),
    ("dropout", (rows, 0.5, 1, 3), "seed must be a tensor"),
    ("dropout", (rows, 0.5, 1, None), "x must be a CUDA tensor"),
    ("nn_product", (rows, weights, offsets), "CUDA tensor"),
    ("nn_dropout", (rows, 0.5, 1, None), "CUDA tensor"),
])
def test_refusals(native, name, args, message):
    with pytest.raises(TypeError, match=message):
        getattr(native, name)(0, *args)


def test_calls_without_a_context():
    lib = cabi.load()
    assert lib.gsb_expert_product(None, None, None, 0, 1, 1, 1, None, 1, 1, 1, 1, None, 1, None, None, 0) == -1
    assert lib.gsb_expert_product_grad(None, None, None, 0, 1, 1, 1, None, 1, 1, None, 1, None, None, 0) == -1
    assert lib.gsb_expert_product_int8(None, None, None, 1, 1, 16, None, None, 16, 16, None, 1, None, 1, None, 0) == -1
    assert lib.gsb_quantize_rows(None, None, None, 0, 1, 1, 1, None, 1, None) == -1
    assert lib.gsb_dropout(None, None, None, 0, 1, 1, 1, 0.5, 1, None, None) == -1


def test_generator_of_the_definition():
    """Known answers of Philox4x32-10 (published with it): counter and key of zeros, and of ones."""
    def plain(c, k):
        c, k = list(c), list(k)
        for _ in range(10):
            p0, p1 = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
            c = [p1 >> 32 ^ c[1] ^ k[0], p1 & exact.MASK32, p0 >> 32 ^ c[3] ^ k[1], p0 & exact.MASK32]
            k = [(k[0] + 0x9E3779B9) & exact.MASK32, (k[1] + 0xBB67AE85) & exact.MASK32]
        return c
    assert plain([0] * 4, [0] * 2) == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    assert plain([exact.MASK32] * 4, [exact.MASK32] * 2) == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]
    blocks = torch.tensor([0, 1, 7, 2 ** 32 - 1, 2 ** 32, 2 ** 40 + 3])
    for seed in (0, 1, 0x123456789ABCDEF0, 2 ** 64 - 1):
        for b, w in zip(blocks.tolist(), exact.words(seed, blocks).tolist()):
            assert w == plain([b & exact.MASK32, b >> 32, 0, 6], [seed & exact.MASK32, seed >> 32])
