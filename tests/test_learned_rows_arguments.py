"""Arguments of learned rows that are neither true nor false; no GPU is needed for it."""
import pytest
import torch

from graph_sampling_b200 import build as gsb_build


@pytest.fixture(scope="module")
def native():
    gsb_build.build()
    gsb_build.build_native()
    from graph_sampling_b200 import ops
    return ops._load_native()


def test_what_has_no_truth_value_is_refused(native):
    neither, ids, rows = torch.zeros(2), torch.zeros(3, dtype=torch.int64), torch.zeros(3, 4)
    for call in (lambda: native.nn_embedding(0, rows, ids, 1.0, None, neither),
                 lambda: native.embedding_grad_rows(0, rows, ids, 5, 1.0, None, None, neither)):
        with pytest.raises(RuntimeError, match="more than one value is ambiguous"):
            call()
