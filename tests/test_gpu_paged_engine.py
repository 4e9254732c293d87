"""PagedDecoder and speculative decoding on a GPU, against a plain FP32 forward of the same weights.

A plain forward keeps FP32 throughout; the decoder rounds activations to bf16
some ten times per layer (relative 2^-8 each, uniformly spread: rms 2^-8 /
sqrt(3)) over two layers: sqrt(20) 2^-8 / sqrt(3) = 1% of the logits' norm is
expected, 5% is the bound.
"""

import importlib
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

CONFIG = dict(hidden_size=256, intermediate_size=512, num_hidden_layers=2, num_attention_heads=4,
              num_key_value_heads=2, head_dim=64, vocab_size=512)


@pytest.fixture(scope="module")
def pe(b200):
    return importlib.import_module(b200.__name__ + ".paged_engine")


@pytest.fixture(scope="module")
def model(b200, pe):
    q2 = importlib.import_module(b200.__name__ + ".qwen2")
    return pe.random_decoder(q2.qwen2_config(**CONFIG), seed=5)


def _plain(b200, model, tokens):
    """Logits [n, vocabulary] of one sequence, FP32."""
    cfg = model.config
    D, n = cfg.head_dim, tokens.numel()

    def lin(m, x):
        w = b200.dequantize_canonical_w4g64_b200(m.qweight, m.scales, m.zeros, out_features=m.out_features,
                                                 in_features=m.in_features)
        return x @ w.t() + (0 if m.bias is None else m.bias.float())

    def norm(x, w):
        return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + cfg.rms_norm_eps) * w.weight.float()

    cos, sin = b200.rope_table(n, D, base=cfg.rope_theta, device=tokens.device)

    def turn(x):
        a, b = x[..., :D // 2], x[..., D // 2:]
        return torch.cat((a * cos[:, None] - b * sin[:, None], b * cos[:, None] + a * sin[:, None]), dim=-1)

    h = model.model.embed_tokens.weight[tokens].float()
    hidden = torch.arange(n, device=tokens.device) > torch.arange(n, device=tokens.device)[:, None]
    for layer in model.model.layers:
        x, a, f = norm(h, layer.input_layernorm), layer.self_attn, layer.mlp
        q, k, v = (lin(m, x).view(n, -1, D) for m in (a.q_proj, a.k_proj, a.v_proj))
        q, k = turn(q), turn(k)
        k, v = (t.repeat_interleave(q.shape[1] // k.shape[1], dim=1) for t in (k, v))
        s = torch.einsum("ihd,jhd->hij", q, k) / math.sqrt(D)
        w = torch.softmax(s.masked_fill(hidden, -math.inf), dim=-1)
        h = h + lin(a.o_proj, torch.einsum("hij,jhd->ihd", w, v).reshape(n, -1))
        x = norm(h, layer.post_attention_layernorm)
        h = h + lin(f.down_proj, torch.nn.functional.silu(lin(f.gate_proj, x)) * lin(f.up_proj, x))
    return norm(h, model.model.norm) @ model.lm_head.weight.float().t()


def _close(got, want):
    assert float((got.float() - want).norm() / want.norm()) < 0.05


def _tokens(n, seed):
    return torch.randint(0, CONFIG["vocab_size"], (n,), generator=torch.Generator().manual_seed(seed)).cuda()


def test_prompts_chunks_and_steps_match_a_plain_forward(b200, pe, model, cuda_device):
    sizes = [70, 1, 200, 33]
    seqs = [_tokens(n + 12, i) for i, n in enumerate(sizes)]
    want = [_plain(b200, model, s) for s in seqs]
    dec = pe.PagedDecoder(model, 4, 220)
    cu = torch.tensor([0, *sizes], device=cuda_device).cumsum(0).to(torch.int32)
    hidden = dec.forward(torch.cat([s[:n] for s, n in zip(seqs, sizes)]), cu_tokens=cu, max_tokens=max(sizes))
    for b, n in enumerate(sizes):
        _close(dec.logits(hidden[cu[b]:cu[b + 1]]), want[b][:n])
    # A ragged chunk (the second sequence pauses), then single tokens, then five at once.
    step = [3, 0, 2, 1]
    cu = torch.tensor([0, *step], device=cuda_device).cumsum(0).to(torch.int32)
    hidden = dec.forward(torch.cat([s[n:n + k] for s, n, k in zip(seqs, sizes, step)]), cu_tokens=cu, max_tokens=3)
    at = [n + k for n, k in zip(sizes, step)]
    assert dec.lengths.tolist() == at
    _close(dec.logits(hidden), torch.cat([w[n:e] for w, n, e in zip(want, sizes, at)]))
    for _ in range(3):
        hidden = dec.forward(torch.stack([s[e] for s, e in zip(seqs, at)])[:, None])
        _close(dec.logits(hidden), torch.stack([w[e] for w, e in zip(want, at)]))
        at = [e + 1 for e in at]
    hidden = dec.forward(torch.stack([s[e:e + 5] for s, e in zip(seqs, at)]))
    _close(dec.logits(hidden).view(4, 5, -1), torch.stack([w[e:e + 5] for w, e in zip(want, at)]))


def test_a_shared_prefix_is_the_sequences_beginning(b200, pe, model, cuda_device):
    prefix = _tokens(150, 50)
    own = [_tokens(n, 60 + n) for n in (9, 3, 17)]
    dec = pe.PagedDecoder(model, 3, 40, prefix_len=160)
    first = dec.set_prefix(prefix)
    want = [_plain(b200, model, torch.cat((prefix, s))) for s in own]
    _close(dec.logits(first), want[0][:150])
    cu = torch.tensor([0, 8, 10, 26], dtype=torch.int32, device=cuda_device)
    hidden = dec.forward(torch.cat([s[:-1] for s in own]), cu_tokens=cu, max_tokens=16)
    _close(dec.logits(hidden), torch.cat([w[150:-1] for w in want]))
    hidden = dec.forward(torch.stack([s[-1:] for s in own]))
    _close(dec.logits(hidden), torch.stack([w[-1] for w in want]))
    with pytest.raises(ValueError):
        dec.set_prefix(_tokens(161, 1))


@pytest.mark.parametrize("prefix", [0, 40])
def test_speculation_keeps_the_caches_with_the_tokens(b200, pe, model, cuda_device, prefix):
    """Drafts from the target itself nearly all stand; whatever stood or fell, both caches end with the tokens that
    were returned, so the next token's logits are those of a plain forward over them."""
    prompts = [_tokens(n, 80 + n) for n in (5, 1, 12)]
    system = _tokens(prefix, 90) if prefix else None
    made = {}
    for kind in ("itself", "another"):
        q2 = importlib.import_module(b200.__name__ + ".qwen2")
        other = model if kind == "itself" else pe.random_decoder(q2.qwen2_config(**CONFIG), seed=6)
        target, draft = (pe.PagedDecoder(m, 3, 64, prefix_len=prefix) for m in (model, other))
        if prefix:
            target.set_prefix(system)
            draft.set_prefix(system)
        gen = torch.Generator(device=cuda_device).manual_seed(3)
        tokens, stood = pe.speculative_generate(target, draft, prompts, 20, drafts=4, temperature=0.7, generator=gen)
        assert tokens.shape == (3, 20) and int(tokens.min()) >= 0 and int(tokens.max()) < 512
        made[kind] = stood
        for b, p in enumerate(prompts):
            # The cache holds the prompt and all returned tokens but, at most, those after the last step's start.
            n = int(target.lengths[b])
            assert n == int(draft.lengths[b]) and p.numel() - 1 + 20 <= n <= p.numel() + 20 + 4
        # Back to the 19th token of each: the 20th's logits.
        for dec, m in ((target, model), (draft, other)):
            dec.lengths = torch.tensor([p.numel() + 18 for p in prompts], dtype=torch.int32, device=cuda_device)
            hidden = dec.forward(tokens[:, 18:19])
            for b, p in enumerate(prompts):
                seq = torch.cat(([system] if prefix else []) + [p, tokens[b, :19]])
                _close(dec.logits(hidden)[b], _plain(b200, m, seq)[-1])
    assert made["itself"] > 0.9 > made["another"]


def test_speculation_refuses(pe, model):
    target, draft = (pe.PagedDecoder(model, 2, 32) for _ in range(2))
    prompts = [_tokens(3, 1), _tokens(4, 2)]
    for args, kw in (((prompts[:1], 5), {}), ((prompts, 0), {}), ((prompts, 5), dict(temperature=0.0)),
                     ((prompts, 5), dict(drafts=0)), ((prompts, 30), {}), (([prompts[0], prompts[0][:0]], 5), {})):
        with pytest.raises(ValueError):
            pe.speculative_generate(target, draft, *args, **kw)
    with pytest.raises(ValueError):
        target.forward(_tokens(6, 3))
