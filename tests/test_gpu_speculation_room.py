"""speculative_generate in the smallest caches that it accepts: sequences that are done early outgrow nothing."""

import importlib
from types import SimpleNamespace

import pytest
import torch

pytestmark = pytest.mark.gpu

CONFIG = dict(hidden_size=256, intermediate_size=512, num_hidden_layers=2, num_attention_heads=4,
              num_key_value_heads=2, head_dim=64, vocab_size=512)


@pytest.fixture(scope="module")
def pe(b200):
    return importlib.import_module(b200.__name__ + ".paged_engine")


@pytest.fixture(scope="module")
def models(b200, pe):
    q2 = importlib.import_module(b200.__name__ + ".qwen2")
    return [pe.random_decoder(q2.qwen2_config(**CONFIG), seed=s) for s in (5, 6)]


@pytest.mark.parametrize("prefix", [0, 24])
@pytest.mark.parametrize("drafts", [2, 7])
@pytest.mark.parametrize("seed", range(4))
def test_the_smallest_caches_are_large_enough(b200, pe, models, cuda_device, seed, drafts, prefix):
    """Batches whose sequences differ in the drafts that stand; pages of 8 tokens without a slot to spare. Every key
    finds its place (no report), and the caches hold the tokens that were returned."""
    longest, new = 12, 35 - drafts
    room = longest + new + drafts + 1
    assert room % 8 == 0
    lib = importlib.import_module(b200.__name__ + "._lib").load()
    status = lambda: lib.qi4_device_status(torch.cuda.current_stream().cuda_stream)  # noqa: E731
    assert status() == 0
    target, draft = (pe.PagedDecoder(m, 6, room, page_size=8, prefix_len=prefix) for m in (models[0], models[seed % 2]))
    g = torch.Generator().manual_seed(seed)
    if prefix:
        system = torch.randint(0, 512, (prefix,), generator=g).to(cuda_device)
        target.set_prefix(system)
        draft.set_prefix(system)
    prompts = [torch.randint(0, 512, (longest,), generator=g) for _ in range(6)]
    gen = torch.Generator(device=cuda_device).manual_seed(seed)
    tokens, _ = pe.speculative_generate(target, draft, prompts, new, drafts=drafts, temperature=0.7, generator=gen)
    assert status() == 0
    assert tokens.shape == (6, new) and int(tokens.min()) >= 0 and int(tokens.max()) < 512
    # One step from the last token but one, for the caches as they are and for caches filled anew.
    again = pe.PagedDecoder(models[0], 6, room, page_size=8, prefix_len=prefix)
    if prefix:
        again.set_prefix(system)
    again.forward(torch.cat((torch.stack(prompts).to(cuda_device), tokens[:, :new - 2]), dim=1))
    target.lengths = again.lengths.clone()
    x, y = (dec.logits(dec.forward(tokens[:, new - 2:new - 1])).float() for dec in (target, again))
    # (other tiles and batch shapes: bf16 roundings of two layers, some 1% of the norm)
    assert float((x - y).norm() / y.norm()) < 0.05
    assert status() == 0


def test_generation_goes_on_from_what_the_caches_hold(b200, pe, models, cuda_device):
    """A second call on the same decoders continues their sequences."""
    target, draft = (pe.PagedDecoder(m, 3, 96) for m in models)
    g = torch.Generator().manual_seed(9)
    prompts = [torch.randint(0, 512, (n,), generator=g) for n in (5, 1, 12)]
    gen = torch.Generator(device=cuda_device).manual_seed(9)
    first, _ = pe.speculative_generate(target, draft, prompts, 9, drafts=3, temperature=0.7, generator=gen)
    second, _ = pe.speculative_generate(target, draft, [row[-1:] for row in first], 8, drafts=3, temperature=0.7,
                                        generator=gen)
    for dec, m in ((target, models[0]), (draft, models[1])):
        assert dec.lengths.tolist() == [p.numel() - 1 + 17 for p in prompts]
        again = pe.PagedDecoder(m, 3, 96)
        seqs = [torch.cat((p.to(cuda_device), a, b))[:-1] for p, a, b in zip(prompts, first, second)]
        cu = torch.tensor([0, *(s.numel() for s in seqs)], device=cuda_device).cumsum(0).to(torch.int32)
        hidden = again.forward(torch.cat(seqs), cu_tokens=cu, max_tokens=max(s.numel() for s in seqs))
        want = again.logits(hidden)[cu[1:].long() - 1].float()
        dec.lengths = dec.lengths - 1
        got = dec.logits(dec.forward(torch.stack([s[-1:] for s in seqs]))).float()
        assert float((got - want).norm() / want.norm()) < 0.05


def _broken(model):
    """The model with a final norm that makes every logit NaN."""
    top = SimpleNamespace(weight=torch.full_like(model.model.norm.weight, float("nan")))
    return SimpleNamespace(config=model.config, lm_head=model.lm_head, model=SimpleNamespace(
        embed_tokens=model.model.embed_tokens, layers=model.model.layers, norm=top))


def test_logits_that_are_no_numbers(b200, pe, models, cuda_device):
    """A draft without probabilities is refused throughout; of a target without them every token is -1."""
    prompts = [torch.tensor([3, 4, 5]), torch.tensor([6])]
    for broken in ("draft", "target", "both"):
        target = pe.PagedDecoder(_broken(models[0]) if broken != "draft" else models[0], 2, 32)
        draft = pe.PagedDecoder(_broken(models[0]) if broken != "target" else models[0], 2, 32)
        tokens, stood = pe.speculative_generate(target, draft, prompts, 6, drafts=2)
        torch.cuda.synchronize()
        if broken == "draft":
            assert int(tokens.min()) >= 0 and int(tokens.max()) < 512 and stood == 0
        else:
            assert bool((tokens == -1).all())
