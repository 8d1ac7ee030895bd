"""Candidates from one prompt, served from a paged cache.

A prompt is scored once; candidates fork from it, each token's log probability
is kept, and at intervals the less likely half is dropped and the others are
forked in their place. At the end the cache is made contiguous. The model is a
small random one; a bundle's directory loads a compressed model instead:

    python examples/serve_paged.py [bundle]
"""

from __future__ import annotations

import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "s-salaad_amd"))

from ssalaad_amd import PagedEngine, build_efficient_model, token_logprobs  # noqa: E402


def small_model():
    from transformers import LlamaConfig, LlamaForCausalLM

    torch.manual_seed(0)
    cfg = LlamaConfig(vocab_size=1000, hidden_size=256, intermediate_size=512, num_hidden_layers=2,
                      num_attention_heads=4, num_key_value_heads=2, max_position_embeddings=512)
    return LlamaForCausalLM(cfg).to("cuda", torch.bfloat16).eval()


def candidates(engine: PagedEngine, prompt, n: int, new_tokens: int, every: int = 8, seed: int = 0):
    """n continuations of `prompt` with their log probabilities, best first."""
    gen = torch.Generator(device=engine.device).manual_seed(seed)
    logits = engine.feed([0], [prompt])
    engine.fork([0] * (n - 1), range(1, n))
    logits = logits.expand(n, -1)
    seqs = list(range(n))
    total = torch.zeros(n, device=engine.device)
    out = torch.empty(n, 0, dtype=torch.int64, device=engine.device)
    for t in range(new_tokens):
        token = torch.multinomial(torch.softmax(logits.float(), -1), 1, generator=gen)[:, 0]
        total = total + token_logprobs(logits.contiguous(), token).logprobs
        out = torch.cat([out, token[:, None]], 1)
        if t + 1 == new_tokens:
            break
        logits = engine.step(seqs, token)
        if (t + 1) % every == 0:  # the likelier half goes on twice
            order = total.argsort(descending=True).tolist()
            keep, drop = order[: n - n // 2], order[n - n // 2:]
            engine.free(drop)
            engine.fork(keep[: len(drop)], drop)
            at = torch.arange(n, device=engine.device)
            at[drop] = torch.tensor(keep[: len(drop)], device=engine.device)
            logits, total, out = logits[at], total[at], out[at]
    order = total.argsort(descending=True)
    return out[order], total[order]


def main() -> None:
    model = build_efficient_model(sys.argv[1], device="cuda") if len(sys.argv) > 1 else small_model()
    engine = PagedEngine(model, max_seqs=9, pages=256, page=16, max_context=512)
    prompt = torch.randint(0, model.config.vocab_size, (100,), generator=torch.Generator().manual_seed(1))
    tokens, logprobs = candidates(engine, prompt, n=8, new_tokens=32)
    used = int((engine.refs > 0).sum())
    live = int(engine.compact())
    print(f"8 candidates of 32 tokens, log probabilities {logprobs[0]:.1f} to {logprobs[-1]:.1f}; "
          f"{used} pages in use, {live} after packing")
    scores = engine.score(8, torch.cat([prompt.to(tokens.device), tokens[0]]), top=3)
    again = float(scores.logprobs[-32:].sum())
    print(f"the best one scored as a prompt: {again:.1f}; its last token's alternatives: "
          f"{scores.top_ids[-1].tolist()}")


if __name__ == "__main__":
    main()
