"""What PagedDecoder works out on tensors of its own, without a GPU."""

import importlib
import types

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


def test_the_decoders_device_is_current_while_it_launches(b200, monkeypatch):
    """The C entry points launch on the current device: it is the model's own, whichever the caller's is."""
    pe = importlib.import_module(b200.__name__ + ".paged_engine")
    inside, seen = [], []

    class Device:
        def __init__(self, device):
            self.device = device

        def __enter__(self):
            inside.append(self.device)

        def __exit__(self, *error):
            inside.pop()

    monkeypatch.setattr(pe.torch.cuda, "device", Device)

    def head(hidden, weight, **how):
        seen.append(list(inside))
        return hidden, None

    monkeypatch.setattr(pe, "b200_lm_head", head)
    dec = pe.PagedDecoder.__new__(pe.PagedDecoder)
    dec.device = torch.device("cpu")
    dec.batch, dec.prefix_len, dec._room = 2, 0, 4
    dec.lengths = torch.zeros(2, dtype=torch.int32)
    dec.prefix_table = torch.zeros(1, dtype=torch.int32)
    dec.model = types.SimpleNamespace(lm_head=types.SimpleNamespace(weight=None))

    def layers(*args):
        seen.append(list(inside))
        return torch.zeros(2, 8)

    dec._layers = layers
    dec.forward(torch.zeros(2, 1, dtype=torch.int64))
    dec.set_prefix(torch.zeros(3, dtype=torch.int64))
    dec.logits(torch.zeros(2, 8))
    assert seen == [[dec.device]] * 3 and not inside
