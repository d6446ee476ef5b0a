"""Forward-mode tangents are refused before anything else is looked at; no GPU is needed for it."""
import pytest
import torch
import torch.autograd.forward_ad as fw

from graph_sampling_b200 import build as gsb_build


@pytest.fixture(scope="module")
def native():
    gsb_build.build()
    gsb_build.build_native()
    from graph_sampling_b200 import ops
    return ops._load_native()


rows, place = torch.zeros(3, 4), torch.zeros(3, 1, dtype=torch.int64)


@pytest.mark.parametrize("name,call", [
    ("table", lambda m, dual: m.nn_embedding(0, dual, place, 1.0, None, False)), ("x", lambda m, dual: m.nn_dispatch(0, dual, place)),
    ("rows", lambda m, dual: m.nn_combine(0, dual, place, None)), ("weights", lambda m, dual: m.nn_combine(0, rows, place, dual))])
@pytest.mark.parametrize("requires_grad", [False, True])
def test_tangents_are_refused(native, name, call, requires_grad):
    with fw.dual_level():
        dual = fw.make_dual(rows.clone().requires_grad_(requires_grad), torch.ones_like(rows))
        with pytest.raises(RuntimeError, match=name + " carries a forward-mode tangent"):
            call(native, dual)
        with pytest.raises(TypeError, match="GPU|CUDA"):
            call(native, fw.unpack_dual(dual).primal)
