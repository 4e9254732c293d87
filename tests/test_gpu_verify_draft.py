"""b200_verify_draft on a GPU: equal to the rule in whole numbers, and distributed as the target."""

import importlib

import pytest
import torch

import _paged as pg

pytestmark = pytest.mark.gpu


def _inputs(dev, B, K, V, dtype, seed, close=0.5):
    g = torch.Generator(device=dev).manual_seed(seed)
    logits = torch.randn(B, K + 1, V, generator=g, device=dev) * 2
    target = torch.softmax(logits, -1).to(dtype)
    draft = torch.softmax(logits[:, :K] + close * torch.randn(B, K, V, generator=g, device=dev), -1).to(dtype)
    tokens = torch.multinomial(draft.float().view(-1, V), 1, generator=g).view(B, K) if K else torch.zeros(
        B, 0, dtype=torch.int64, device=dev)
    u = torch.rand(B, K + 1, generator=g, device=dev)
    return tokens, target, draft, u


def _same(got, want):
    assert torch.equal(got[1].cpu(), want[1]) and torch.equal(got[0].cpu(), want[0])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,K,V", [(1, 1, 1), (1, 4, 7), (3, 0, 130), (5, 3, 1000), (2, 6, 50257), (9, 5, 32000),
                                   (4, 2, 151936), (33, 40, 515)])
def test_verify_equals_the_rule(b200, cuda_device, dtype, B, K, V):
    tokens, target, draft, u = _inputs(cuda_device, B, K, V, dtype, seed=B * 100 + K)
    _same(b200.b200_verify_draft(tokens, target, u, draft_probs=draft), pg.verify_plain(tokens, target, u, draft, None))
    counts = torch.tensor([(3 * b) % (K + 2) - 1 for b in range(B)], dtype=torch.int32, device=cuda_device)
    _same(b200.b200_verify_draft(tokens, target, u, draft_probs=draft, draft_counts=counts),
          pg.verify_plain(tokens, target, u, draft, counts))
    _same(b200.b200_verify_draft(tokens, target, u), pg.verify_plain(tokens, target, u, None, None))


def test_verify_edges(b200, cuda_device):
    """u = 0 and just below 1, equal distributions, nothing left to draw from, NaN and infinite weights, strides."""
    B, K, V = 6, 3, 777
    tokens, target, draft, u = _inputs(cuda_device, B, K, V, torch.float32, seed=3)
    for value in (0.0, 1 - 2.0 ** -24):
        w = torch.full_like(u, value)
        _same(b200.b200_verify_draft(tokens, target, w, draft_probs=draft), pg.verify_plain(tokens, target, w, draft, None))
    got = b200.b200_verify_draft(tokens, target, u, draft_probs=target[:, :K].contiguous())
    assert bool((got[1] == K).all()) and torch.equal(got[0][:, :K], tokens)  # p = q: every draft stands
    gone = target.clone()
    gone[1] = 0
    gone[2, :, 5:] = float("nan")
    gone[3] *= 1e-14
    gone[4, 0, 9] = float("inf")
    high = draft.clone()
    high[5] = 1.0  # p <= q everywhere: drawn from p
    _same(b200.b200_verify_draft(tokens, gone, u, draft_probs=high), pg.verify_plain(tokens, gone, u, high, None))
    assert int(b200.b200_verify_draft(tokens, gone, u, draft_probs=high)[0][1, 0]) == -1
    wide = torch.zeros(B, K + 2, V + 3, device=cuda_device)
    wide[:, :K + 1, :V] = target
    _same(b200.b200_verify_draft(tokens, wide[:, :K + 1, :V], u, draft_probs=draft),
          pg.verify_plain(tokens, target, u, draft, None))
    turned = target.transpose(1, 2).contiguous().transpose(1, 2)
    _same(b200.b200_verify_draft(tokens, turned, u, draft_probs=draft), pg.verify_plain(tokens, target, u, draft, None))
    odd = tokens.clone()
    odd[0, 0], odd[1, 1], odd[2, 0] = -1, V, 2 ** 40
    _same(b200.b200_verify_draft(odd, target, u, draft_probs=draft), pg.verify_plain(odd, target, u, draft, None))
    lib = importlib.import_module(b200.__name__ + "._lib").load()
    assert lib.qi4_device_status(torch.cuda.current_stream().cuda_stream) == 16
    assert b200.b200_verify_draft(tokens[:0], target[:0], u[:0])[0].shape == (0, K + 1)


def test_verified_tokens_are_distributed_as_the_target(b200, cuda_device):
    """200,000 independent sequences over 24 tokens: counts of the first token against the target's probabilities, a
    chi-square of 23 degrees of freedom, above 65 with probability below 1e-5 (seeded: one fixed draw)."""
    N, V = 200000, 24
    g = torch.Generator(device=cuda_device).manual_seed(11)
    p = torch.softmax(torch.randn(2, V, generator=g, device=cuda_device), -1)
    q = torch.softmax(torch.randn(1, V, generator=g, device=cuda_device), -1)
    tokens = torch.multinomial(q.expand(N, V), 1, generator=g)
    u = torch.rand(N, 2, generator=g, device=cuda_device)
    out, acc = b200.b200_verify_draft(tokens, p.expand(N, 2, V), u, draft_probs=q.expand(N, 1, V))
    counts = torch.bincount(out[:, 0], minlength=V).double()
    want = N * p[0].double()
    assert float(((counts - want) ** 2 / want).sum()) < 65
    second = out[acc == 1, 1]
    want = len(second) * p[1].double()
    assert float(((torch.bincount(second, minlength=V).double() - want) ** 2 / want).sum()) < 65


def test_verify_refuses(b200, cuda_device):
    tokens, target, draft, u = _inputs(cuda_device, 2, 3, 50, torch.float32, seed=1)
    good = dict(draft_tokens=tokens, target_probs=target, uniforms=u, draft_probs=draft)
    counts = torch.zeros(2, dtype=torch.int32, device=cuda_device)
    for error, kw in [
        (TypeError, dict(draft_tokens=tokens.int())), (TypeError, dict(target_probs=target.double())),
        (TypeError, dict(draft_probs=draft.half())), (TypeError, dict(uniforms=u.double())),
        (TypeError, dict(draft_counts=counts.long())), (ValueError, dict(draft_counts=counts[:1])),
        (ValueError, dict(draft_tokens=tokens[:, :2])), (ValueError, dict(uniforms=u[:, :3])),
        (ValueError, dict(draft_probs=draft[..., :9])), (ValueError, dict(target_probs=target[0])),
        (ValueError, dict(uniforms=u.cpu())), (ValueError, dict(draft_probs=draft.cpu())),
    ]:
        with pytest.raises(error):
            b200.b200_verify_draft(**{**good, **kw})
