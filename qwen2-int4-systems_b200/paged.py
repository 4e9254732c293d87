"""Paged KV cache: rotary append, ragged attention and attention behind a shared prefix.

The cache of one layer is two pools ``[pages, kv_heads, page_size, head_dim]``
(BF16 or FP16; any strides with ``head_dim`` contiguous, so a
``[pages, page_size, kv_heads, head_dim]`` pool is passed transposed). Row
``b`` of ``block_table`` names the pages of sequence ``b``'s positions in
order. A batch is ragged: its new tokens are the rows of ``[T, heads, dim]``
tensors, sequence ``b`` owning rows ``cu_tokens[b]`` to ``cu_tokens[b + 1]``
(without ``cu_tokens``, ``T / B`` rows each); decode steps, drafts, prompt
chunks and whole prompts mix freely. All index tensors are int32 on the
device and are read by the kernels alone, so captured graphs advance with
them; ``qi4_device_status`` reports positions beyond a table, pages outside
the pool and rotary positions outside the table.

A step per layer is ``b200_rope_paged_append`` (lengths: keys cached so far),
then ``b200_paged_attention`` (lengths: the new ones included).
C ABI: ``qi4_rope_paged_append``, ``qi4_paged_attention``,
``qi4_shared_prefix_attention``. For a paged cache they stand for the
rotation, cache growth, head expansion and masked attention of the reference's
src/qwen_int4/model.py:74-118.
"""

from __future__ import annotations

import torch

from .backends import _fast, _require_cuda


def _ops():
    _require_cuda()
    if _fast is None:
        raise RuntimeError("the _qi4_torch extension is not built; run the package's build step (build.py)")
    return _fast


def rope_table(positions: int, rotary_dim: int, *, base: float = 10000.0, scaling: float = 1.0,
               attention_scaling: float = 1.0, device=None) -> tuple[torch.Tensor, torch.Tensor]:
    """(cos, sin) FP32 ``[positions, rotary_dim / 2]`` of position / ``scaling`` for b200_rope_paged_append:
    angles in 64 bits, so that far positions keep their accuracy; both times ``attention_scaling``."""
    if positions <= 0 or rotary_dim < 0 or rotary_dim % 16 or scaling <= 0:
        raise ValueError("rope_table needs positions > 0, a rotary_dim that is a multiple of 16 and scaling > 0")
    freq = float(base) ** (-torch.arange(0, rotary_dim, 2, dtype=torch.float64, device=device) / max(rotary_dim, 1))
    angle = torch.arange(positions, dtype=torch.float64, device=device)[:, None] / scaling * freq
    return (angle.cos() * attention_scaling).float(), (angle.sin() * attention_scaling).float()


def b200_rope_paged_append(q, k, v, k_cache, v_cache, block_table, lengths, cos=None, sin=None, *, cu_tokens=None,
                           positions=None, interleaved: bool = False, q_out=None) -> torch.Tensor:
    """Rotate the new queries and keys, append the new keys and values; returns the rotated queries.

    q [T, Hq, D], k / v [T, kv_heads, D] (views of a joint projection are read
    in place); lengths [B]: keys already cached, token i of sequence b goes to
    position lengths[b] + i. cos / sin: FP32 [rows, rotary_dim / 2] (see
    ``rope_table``), row ``positions[t]`` or the token's position; the first
    rotary_dim dimensions are turned in pairs (m, m + rotary_dim / 2), or
    (2m, 2m + 1) when ``interleaved``; without cos / sin nothing is turned.
    ``q_out`` may be ``q``. lengths is not changed.
    """
    return _ops().rope_paged_append(q, k, v, k_cache, v_cache, block_table, lengths, cos, sin, cu_tokens, positions,
                                    interleaved, q_out)


def b200_paged_attention(q, k_cache, v_cache, block_table, lengths, *, cu_tokens=None, max_tokens=None, scale=None,
                         causal: bool = True, out=None, workspace=None) -> torch.Tensor:
    """out [T, Hq, D]: every new token's queries over its sequence's pages.

    lengths [B]: the sequences' keys, the new tokens' included. Causal: token
    i of a sequence's n sees the keys up to position lengths[b] - n + i; else
    all of them. A token that sees no key gets zeros. ``max_tokens`` (a host
    number: no sequence has more new tokens, which ``qi4_device_status``
    checks) lets a batch given by ``cu_tokens`` run on the kernel and the
    tiles for its row count. A block_table may be wider than the lengths need;
    one that covers at most 512 keys (up to 4096 for few sequences) saves a
    launch.
    ``workspace``: a uint8 tensor of ``qi4_paged_attention_workspace`` bytes,
    for callers that own their memory.
    """
    return _ops().attend(q, k_cache, v_cache, None, 0, block_table, lengths, cu_tokens, max_tokens, scale, causal, out,
                         workspace)


def b200_shared_prefix_attention(q, k_cache, v_cache, prefix_table, prefix_length: int, block_table, lengths, *,
                                 cu_tokens=None, max_tokens=None, scale=None, out=None,
                                 workspace=None) -> torch.Tensor:
    """b200_paged_attention (causal) for sequences that share their first ``prefix_length`` keys.

    prefix_table [pages] holds the prefix in the same pool, read once for the
    whole batch; block_table and lengths cover each sequence's own keys after
    it. Every token sees the whole prefix.
    """
    return _ops().attend(q, k_cache, v_cache, prefix_table, prefix_length, block_table, lengths, cu_tokens, max_tokens,
                         scale, True, out, workspace)
