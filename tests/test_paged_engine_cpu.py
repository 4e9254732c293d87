"""What PagedDecoder works out on tensors of its own, without a GPU."""

import importlib

import pytest
import torch


@pytest.mark.parametrize("cu,tokens,want", [
    ([0, 2, 2, 5], 5, [0, 0, 2, 2, 2]),
    ([0, 2, 2, 5], 8, [0, 0, 2, 2, 2, 2, 2, 2]),  # tokens that no sequence owns
    ([0, 0], 3, [0, 0, 0]),
])
def test_owners_stay_within_the_batch(b200, cu, tokens, want):
    pe = importlib.import_module(b200.__name__ + ".paged_engine")
    cu = torch.tensor(cu, dtype=torch.int32)
    owner = pe._owners(cu, torch.arange(tokens))
    assert owner.tolist() == want
    torch.zeros(cu.numel() - 1)[owner]  # (an index beyond it would be an error here, an assertion on a GPU)
