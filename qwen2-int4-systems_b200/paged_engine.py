"""A Qwen2-like W4G64 decoder over a paged cache, and speculative decoding with it.

``PagedDecoder`` takes a model laid out as the reference's
``QwenInt4ForCausalLM`` (src/qwen_int4/model.py: its QuantLinear buffers,
norms, tied embedding; ``random_decoder`` builds one without a checkpoint) and
runs its layers on this library's kernels over pages: one ``forward`` serves
whole prompts, prompt chunks, single tokens and drafts, a different number for
every sequence. Per layer: residual add + RMSNorm, q/k/v in one call, rotary
append, paged (or shared-prefix) attention, o_proj, residual add + RMSNorm,
gate/up + SwiGLU, down_proj. A prompt that all sequences share is cached once
(``set_prefix``) and read once per layer for the whole batch.

``speculative_generate`` drafts with a second, smaller decoder and verifies all
drafts of a step in one ``forward`` of the target (``b200_verify_draft``); the
tokens are distributed as the target's own. Taking drafts back is setting the
sequences' lengths.
"""

from __future__ import annotations

from types import SimpleNamespace

import torch

from . import _lib
from .backends import _require_cuda, _stream, b200_w4g64_gate_up_silu, b200_w4g64_linear, b200_w4g64_linear_multi
from .lm_head import b200_lm_head
from .paged import b200_paged_attention, b200_rope_paged_append, b200_shared_prefix_attention, rope_table
from .qwen2 import quantize_symmetric_rtn_torch
from .speculative import b200_verify_draft


@torch.no_grad()
def random_decoder(config, *, device="cuda", seed: int = 0):
    """A model of ``config`` (``qwen2.qwen2_config``) with random symmetric W4G64 weights, laid out as PagedDecoder
    reads it; every tensor as ``qwen2.build_random_qwen2`` makes it."""
    gen = torch.Generator(device=device).manual_seed(seed)
    heads, kv, dim = config.num_attention_heads, config.num_key_value_heads, config.head_dim
    hidden, inter = config.hidden_size, config.intermediate_size

    def randn(*shape):
        return (torch.randn(shape, device=device, generator=gen) * 0.02).to(torch.bfloat16)

    def linear(n, k, bias=False):
        qw, sc = quantize_symmetric_rtn_torch(randn(n, k).float())
        zeros = torch.zeros((n * (k // 64) + 1) // 2, 1, dtype=torch.uint8, device=device)
        return SimpleNamespace(qweight=qw, scales=sc, zeros=zeros, bias=randn(n) if bias else None, in_features=k,
                               out_features=n, group_size=64, packing="canonical")

    def norm():
        return SimpleNamespace(weight=torch.ones(hidden, dtype=torch.bfloat16, device=device))

    embed = SimpleNamespace(weight=randn(config.vocab_size, hidden))
    layers = [SimpleNamespace(
        input_layernorm=norm(), post_attention_layernorm=norm(),
        self_attn=SimpleNamespace(q_proj=linear(heads * dim, hidden, True), k_proj=linear(kv * dim, hidden, True),
                                  v_proj=linear(kv * dim, hidden, True), o_proj=linear(hidden, heads * dim)),
        mlp=SimpleNamespace(gate_proj=linear(inter, hidden), up_proj=linear(inter, hidden),
                            down_proj=linear(hidden, inter))) for _ in range(config.num_hidden_layers)]
    return SimpleNamespace(config=config, lm_head=embed,
                           model=SimpleNamespace(embed_tokens=embed, layers=layers, norm=norm()))


def _owners(cu_tokens, t):
    """The sequence of each of the tokens t; tokens behind the last sequence's, whose results are not defined, count as
    that one's, so that they index nothing beyond the batch."""
    return torch.searchsorted(cu_tokens[1:], t, right=True).clamp_max(cu_tokens.numel() - 2)


def _sample(p, generator):
    """One token of each row of p [batch, vocabulary]: the first of p / (exponential numbers), as torch.multinomial draws
    it. Rows that are no numbers give some token, not an assertion on the GPU, after which nothing runs there."""
    return (p / torch.empty_like(p).exponential_(1, generator=generator)).argmax(dim=-1)


class PagedDecoder:
    """``batch`` sequences of up to ``max_len`` keys each (a shared prefix not counted) in pages of ``page_size``."""

    def __init__(self, model, batch: int, max_len: int, *, page_size: int = 16, prefix_len: int = 0):
        self.lib = _require_cuda()
        self.model, cfg = model, model.config
        self.heads, self.kv_heads = cfg.num_attention_heads, cfg.num_key_value_heads
        self.head_dim = getattr(cfg, "head_dim", cfg.hidden_size // cfg.num_attention_heads)
        self.eps = float(cfg.rms_norm_eps)
        self.embed = model.model.embed_tokens.weight
        self.device = self.embed.device
        self.batch, self.max_len = int(batch), int(max_len)
        own = -(-max_len // page_size)
        shared = -(-prefix_len // page_size)
        shape = (len(model.model.layers), batch * own + shared, self.kv_heads, page_size, self.head_dim)
        self.k_cache = torch.zeros(shape, dtype=torch.bfloat16, device=self.device)
        self.v_cache = torch.zeros(shape, dtype=torch.bfloat16, device=self.device)
        pages = torch.arange(shape[1], dtype=torch.int32, device=self.device)
        self.table = pages[:batch * own].view(batch, own)
        self.prefix_table, self.prefix_len, self._room = pages[batch * own:], 0, int(prefix_len)
        self.lengths = torch.zeros(batch, dtype=torch.int32, device=self.device)  # keys cached of each sequence
        self.cos, self.sin = rope_table(max_len + prefix_len, self.head_dim, base=cfg.rope_theta, device=self.device)

    def _norm(self, h, delta, weight):
        out = torch.empty_like(h)
        rc = self.lib.qi4_add_rmsnorm(
            h.data_ptr(), None if delta is None else delta.data_ptr(),
            _lib.DTYPE_NONE if delta is None else _lib.DTYPE_F32 if delta.dtype == torch.float32 else _lib.DTYPE_BF16,
            weight.data_ptr(), out.data_ptr(), h.shape[0], h.shape[1], self.eps, _stream(h.device))
        _lib.check(rc, "qi4_add_rmsnorm")
        return out

    @staticmethod
    def _linear(x, lin):
        return b200_w4g64_linear(x, lin.qweight, lin.scales, lin.zeros, lin.bias, out_features=lin.out_features,
                                 in_features=lin.in_features, group_size=64, packing="canonical")

    def _layers(self, tokens, append, attend):
        h = self.embed.index_select(0, tokens.reshape(-1))
        delta = None
        for i, layer in enumerate(self.model.model.layers):
            a, f = layer.self_attn, layer.mlp
            x = self._norm(h, delta, layer.input_layernorm.weight)
            q, k, v = b200_w4g64_linear_multi(x, [a.q_proj, a.k_proj, a.v_proj])
            q, k, v = (t.view(t.shape[0], -1, self.head_dim) for t in (q, k, v))
            q = append(q, k, v, self.k_cache[i], self.v_cache[i])
            o = attend(q, self.k_cache[i], self.v_cache[i])
            delta = self._linear(o.flatten(1), a.o_proj)
            x = self._norm(h, delta, layer.post_attention_layernorm.weight)
            delta = self._linear(b200_w4g64_gate_up_silu(x, f.gate_proj, f.up_proj), f.down_proj)
        return self._norm(h, delta, self.model.model.norm.weight)

    @torch.inference_mode()
    def forward(self, tokens, *, cu_tokens=None, max_tokens: int | None = None) -> torch.Tensor:
        """Hidden states [T, hidden] of the new tokens, which are appended to the sequences.

        tokens [batch, n] (n new tokens each), or [T] with cu_tokens [batch +
        1] int32 on the device, sequence b owning tokens cu_tokens[b] to
        cu_tokens[b + 1]; max_tokens: no sequence has more (a host number).
        """
        T = tokens.numel()
        if cu_tokens is None:
            if tokens.ndim != 2 or tokens.shape[0] != self.batch:
                raise ValueError("tokens must be [batch, n], or come with cu_tokens")
            count, max_tokens = tokens.shape[1], tokens.shape[1]
            first = torch.arange(self.batch, device=self.device) * count
        else:
            count, first = cu_tokens[1:] - cu_tokens[:-1], cu_tokens[:-1]
        before, after = self.lengths, self.lengths + count
        positions = None
        if self.prefix_len:  # rotary positions run on from the prefix's
            t = torch.arange(T, device=self.device)
            owner = t // max(max_tokens, 1) if cu_tokens is None else _owners(cu_tokens, t)
            positions = (self.prefix_len + before[owner] + t - first[owner]).to(torch.int32)

        def append(q, k, v, kc, vc):
            return b200_rope_paged_append(q, k, v, kc, vc, self.table, before, self.cos, self.sin, cu_tokens=cu_tokens,
                                          positions=positions, q_out=q)

        def attend(q, kc, vc):
            if self.prefix_len:
                return b200_shared_prefix_attention(q, kc, vc, self.prefix_table, self.prefix_len, self.table, after,
                                                    cu_tokens=cu_tokens, max_tokens=max_tokens)
            return b200_paged_attention(q, kc, vc, self.table, after, cu_tokens=cu_tokens, max_tokens=max_tokens)

        with torch.cuda.device(self.device):
            out = self._layers(tokens, append, attend)
        self.lengths = after.to(torch.int32)
        return out

    @torch.inference_mode()
    def set_prefix(self, tokens) -> torch.Tensor:
        """Cache ``tokens`` [P] as the beginning of every sequence; its hidden states. The sequences start anew."""
        n = tokens.numel()
        if n > self._room:
            raise ValueError(f"the decoder was built for a prefix of {self._room} tokens")
        table = self.prefix_table.view(1, -1)
        none, all_ = (torch.tensor([x], dtype=torch.int32, device=self.device) for x in (0, n))

        def append(q, k, v, kc, vc):
            return b200_rope_paged_append(q, k, v, kc, vc, table, none, self.cos, self.sin, q_out=q)

        with torch.cuda.device(self.device):
            out = self._layers(tokens, append, lambda q, kc, vc: b200_paged_attention(q, kc, vc, table, all_))
        self.prefix_len = n
        self.lengths = torch.zeros_like(self.lengths)
        return out

    @torch.inference_mode()
    def logits(self, hidden) -> torch.Tensor:
        """Logits [..., vocabulary] (bf16) over the tied embedding."""
        if hidden.numel() // hidden.shape[-1] <= 8:
            with torch.cuda.device(self.device):
                out, _ = b200_lm_head(hidden, self.model.lm_head.weight, return_argmax=False)
            return out.view(*hidden.shape[:-1], -1)
        return hidden @ self.model.lm_head.weight.t()


@torch.inference_mode()
def speculative_generate(target: PagedDecoder, draft: PagedDecoder, prompts, max_new_tokens: int, *, drafts: int = 4,
                         temperature: float = 1.0, generator: torch.Generator | None = None):
    """(tokens [batch, max_new_tokens], share of the drafts that stood) sampled from the target at ``temperature``.

    ``prompts``: one 1-D tensor of at least one token per sequence (what
    follows a shared prefix, if ``set_prefix`` was called on both decoders).
    Each step the draft proposes ``drafts`` tokens per sequence; the target
    reads them in one pass, and ``b200_verify_draft`` keeps those that stand
    and draws the next. Both caches then go back to the tokens that stand. A
    token is -1 where the target's probabilities for it are no numbers.
    """
    if temperature <= 0 or drafts < 1 or max_new_tokens < 1:
        raise ValueError("temperature must be positive, with at least one draft and one new token")
    B, dev = target.batch, target.device
    if len(prompts) != B or draft.batch != B or min(p.numel() for p in prompts) < 1:
        raise ValueError("one prompt of at least one token per sequence is needed")
    longest = max(p.numel() for p in prompts)
    if longest + max_new_tokens + drafts + 1 > min(target.max_len, draft.max_len):
        raise ValueError("the sequences would outgrow the decoders' caches")
    # All but each prompt's last token go into both caches; the last is the first step's input.
    sizes = [p.numel() - 1 for p in prompts]
    cu = torch.tensor([0, *sizes], device=dev).cumsum(0).to(torch.int32)
    if longest > 1:
        body = torch.cat([p[:-1] for p in prompts]).to(dev)
        for model in (target, draft):
            model.forward(body, cu_tokens=cu, max_tokens=longest - 1)
    last = torch.stack([p[-1] for p in prompts]).to(dev)
    # Where the caches end with all but the last returned token. A sequence may go beyond it by `drafts` as it finishes;
    # it is taken back to it, so that what later steps still append to it needs no more room than an open sequence's.
    end_t, end_d = target.lengths + max_new_tokens, draft.lengths + max_new_tokens

    def probs(model, hidden):
        return torch.softmax(model.logits(hidden).float() / temperature, dim=-1)

    vocab = target.model.lm_head.weight.shape[0]
    out = torch.full((B, max_new_tokens + drafts + 1), -1, dtype=torch.int64, device=dev)
    made = torch.zeros(B, dtype=torch.int64, device=dev)
    place = torch.arange(drafts + 1, device=dev)
    stood = tried = 0
    while True:
        open_ = made < max_new_tokens
        if not bool(open_.any()):
            break
        start_t, start_d = target.lengths, draft.lengths
        tokens = torch.empty(B, drafts + 1, dtype=torch.int64, device=dev)
        tokens[:, 0] = last
        q = torch.empty(B, drafts, vocab, device=dev)
        for i in range(drafts):
            q[:, i] = probs(draft, draft.forward(tokens[:, i:i + 1]))
            tokens[:, i + 1] = _sample(q[:, i], generator)
        draft.forward(tokens[:, drafts:])  # (the last draft's key, for when it stands)
        p = probs(target, target.forward(tokens)).view(B, drafts + 1, vocab)
        u = torch.rand(B, drafts + 1, device=dev, generator=generator)
        found, accepted = b200_verify_draft(tokens[:, 1:], p, u, draft_probs=q)
        # Sequences that have all their tokens stay where they are.
        step = torch.where(open_, accepted + 1, 0)
        out.scatter_(1, torch.where(open_[:, None], made[:, None] + place, out.shape[1] - 1), found)
        # (-1 where the target's probabilities are no numbers: the sequence goes on from token 0)
        last = torch.where(open_, found.gather(1, accepted.long()[:, None])[:, 0].clamp_min(0), last)
        made += step
        target.lengths = torch.minimum(start_t + step, end_t).to(torch.int32)
        draft.lengths = torch.minimum(start_d + step, end_d).to(torch.int32)
        stood += int(accepted[open_].sum())
        tried += drafts * int(open_.sum())
    return out[:, :max_new_tokens], stood / max(tried, 1)
