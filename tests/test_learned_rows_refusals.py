"""What the operators of learned rows refuse before anything is launched; no GPU is needed for it."""
import pytest
import torch

from graph_sampling_b200 import cabi
from graph_sampling_b200 import build as gsb_build


@pytest.fixture(scope="module")
def native():
    gsb_build.build()
    gsb_build.build_native()
    from graph_sampling_b200 import ops
    return ops._load_native()


ids, table, grad = torch.zeros(3, dtype=torch.int64), torch.zeros(5, 4), torch.zeros(3, 4)
place, weights = torch.zeros(3, 2, dtype=torch.int64), torch.zeros(3, 2)


@pytest.mark.parametrize("name,args,message", [
    ("embedding_lookup", (None, ids, 1.0, None), "table must be a tensor"),
    ("embedding_lookup", (table.double(), ids, 1.0, None), "float32, float16 or bfloat16"),
    ("embedding_lookup", (table[0], ids, 1.0, None), "two dimensions"),
    ("embedding_lookup", (table, ids, 1.0, None), "on the GPU or in pinned host memory"),
    ("embedding_lookup", (table, ids, "x", None), "real number"),
    ("embedding_lookup", (table, ids, 1.0, 1.5), "integer"),
    ("embedding_grad", (grad, ids, -1, 1.0, None, None), "num_rows"),
    ("embedding_grad", (grad, ids[:2], 5, 1.0, None, None), "shape of ids"),
    ("embedding_grad", (grad.long(), ids, 5, 1.0, None, None), "float32, float16 or bfloat16"),
    ("embedding_grad", (grad, ids, 5, 1.0, None, torch.float16), "result's dtype"),
    ("embedding_grad", (grad, ids, 5, 1.0, None, "float32"), "torch.dtype"),
    ("embedding_grad", (grad, ids.int(), 5, 1.0, None, None), "ids must be int64"),
    ("embedding_grad", (grad, ids, 5, 1.0, None, None), "CUDA tensor"),
    ("embedding_grad_rows", (grad, ids, 5, 1.0, None, torch.bfloat16, True), "result's dtype"),
    ("expert_order", (ids, 0), "num_experts"),
    ("expert_order", (ids, 65_537), "num_experts"),
    ("expert_order", (ids.float(), 4), "expert_ids must be int64"),
    ("expert_order", (ids, 4), "CUDA tensor"),
    ("expert_dispatch", (grad[0], place, None), "two dimensions"),
    ("expert_dispatch", (grad, place, None), "CUDA tensor"),
    ("expert_combine", (grad.int(), place, None), "float32, float16 or bfloat16"),
    ("expert_combine_grad", (grad, grad, place, None), "CUDA tensor"),
    ("nn_embedding", (table, ids, 1.0, None, False), "GPU or in pinned"),
    ("nn_embedding", (table.clone().requires_grad_(), ids, 1.0, None, False), "table must be a CUDA tensor"),
    ("nn_dispatch", (grad, place), "CUDA tensor"),
    ("nn_combine", (grad, place, weights), "CUDA tensor"),
])
def test_refusals(native, name, args, message):
    with pytest.raises(TypeError, match=message):
        getattr(native, name)(0, *args)


def test_wrong_number_of_arguments(native):
    with pytest.raises(TypeError):
        native.embedding_lookup(0, table, ids)


def test_scratch_sizes_and_calls_without_a_context():
    lib = cabi.load()
    assert lib.gsb_embedding_grad_workspace(0, 10, 4) >= 0
    small, large = lib.gsb_embedding_grad_workspace(1000, 10, 4), lib.gsb_embedding_grad_workspace(1_000_000, 2 ** 32 - 2, 4)
    assert 0 < small < large
    assert lib.gsb_embedding_grad_workspace(2 ** 31, 10, 4) == -1 and lib.gsb_embedding_grad_workspace(5, 2 ** 32 - 1, 4) == -1
    assert lib.gsb_embedding_grad_workspace(5, 10, 0) == -1 and lib.gsb_embedding_grad_workspace(-1, 10, 4) == -1
    assert lib.gsb_expert_order_workspace(100, 8) > 0
    assert lib.gsb_expert_order_workspace(100, 0) == -1 and lib.gsb_expert_order_workspace(100, 65_537) == -1
    assert lib.gsb_embedding_lookup(None, None, None, 0, 1, 1, 1, None, 1, 1.0, 0, 0, None) == -1
    assert lib.gsb_embedding_grad(None, None, None, 0, 1, 1, None, 1, 1, 1.0, 0, 0, None, 0, None, 0) == -1
    assert lib.gsb_embedding_grad_rows(None, None, None, 0, 1, 1, None, 1, 1, 1.0, 0, 0, None, None, 0, None, None, 0, None) == -1
    assert lib.gsb_expert_order(None, None, None, 1, 1, None, None, None, None, 0) == -1
    assert lib.gsb_expert_spread(None, None, None, 0, 1, 1, 1, 1, None, None, 0, None) == -1
    assert lib.gsb_expert_combine(None, None, None, 0, 1, 1, 1, 1, 1, None, None, 0, None) == -1
    assert lib.gsb_expert_combine_grad(None, None, None, 0, 1, 1, 1, 1, None, 1, 1, None, None, 0, None, None) == -1


def test_no_cpu_path():
    if torch.cuda.is_available():
        pytest.skip("GPU present")
    import graph_sampling_b200.gs as gs
    with pytest.raises(RuntimeError):
        gs.nn.embedding(table, ids)
