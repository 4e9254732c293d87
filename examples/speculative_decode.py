"""Speculative decoding over a paged cache with a shared system prompt, on random weights.

    python examples/speculative_decode.py --batch 16 --prefix 1000 --new 64

Builds a Qwen2-1.5B-shaped target with random W4G64 weights and a draft made
of its first layers, caches one common prompt for the whole batch, and samples
from the target through drafts of four tokens. Random weights draft badly: the
share of drafts that stand says nothing about a trained pair.
"""

import argparse
import importlib
import sys
import time
from pathlib import Path
from types import SimpleNamespace

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))
PACKAGE = "qwen2-int4-systems_b200"


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--batch", type=int, default=16)
    ap.add_argument("--prefix", type=int, default=1000, help="tokens of the shared prompt (0: none)")
    ap.add_argument("--prompt", type=int, default=50, help="tokens of each sequence's own prompt, at most")
    ap.add_argument("--new", type=int, default=64)
    ap.add_argument("--drafts", type=int, default=4)
    ap.add_argument("--layers", type=int, default=28)
    ap.add_argument("--draft-layers", type=int, default=4)
    ap.add_argument("--temperature", type=float, default=1.0)
    args = ap.parse_args()
    pe = importlib.import_module(PACKAGE + ".paged_engine")
    q2 = importlib.import_module(PACKAGE + ".qwen2")
    model = pe.random_decoder(q2.qwen2_config(num_hidden_layers=args.layers), seed=0)
    small = SimpleNamespace(config=model.config, lm_head=model.lm_head, model=SimpleNamespace(
        embed_tokens=model.model.embed_tokens, layers=model.model.layers[:args.draft_layers], norm=model.model.norm))
    room = args.prompt + args.new + args.drafts + 1
    target, draft = (pe.PagedDecoder(m, args.batch, room, prefix_len=args.prefix) for m in (model, small))
    gen = torch.Generator().manual_seed(1)
    vocab = model.config.vocab_size
    prompts = [torch.randint(0, vocab, (args.prompt - i % max(args.prompt // 2, 1),), generator=gen)
               for i in range(args.batch)]
    if args.prefix:
        system = torch.randint(0, vocab, (args.prefix,), generator=gen).cuda()
        target.set_prefix(system)
        draft.set_prefix(system)
    device_gen = torch.Generator(device="cuda").manual_seed(2)
    torch.cuda.synchronize()
    start = time.perf_counter()
    tokens, stood = pe.speculative_generate(target, draft, prompts, args.new, drafts=args.drafts,
                                            temperature=args.temperature, generator=device_gen)
    torch.cuda.synchronize()
    spent = time.perf_counter() - start
    print(f"{tokens.numel()} tokens in {spent:.2f} s ({tokens.numel() / spent:.0f} tokens/s), "
          f"{100 * stood:.1f}% of the drafts stood")
    print("first sequence:", tokens[0, :16].tolist())


if __name__ == "__main__":
    main()
