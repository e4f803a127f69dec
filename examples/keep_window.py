"""From a long cleartext prompt to the few tokens that the encrypted decode step keeps.

    python examples/keep_window.py [--tokens 4096] [--keep 256]

One attention layer of the decode step's shape (32 query heads over 8 key heads of 128) with random weights runs in the
clear: queries and keys get their rotary positions, the prompt's attention over the keys as they came gives the softmax's
shift and intervals, the keys and values go into 4-bit pages, and every key head keeps the tokens to which its queries gave
most, beside the last ones: two pages, as the encrypted step holds them.  Their keys and values as they came, from before the 4
bits, are the history that ``encrypt_kv_history`` encrypts for it.  The next token's attention over the pages that are kept is compared
with the one over the whole prompt.  Random weights attend almost evenly, so what is kept here is not much of the whole; a model's
is.
"""

import argparse
import math
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))

from holmes_amd import clear  # noqa: E402
from holmes_amd.decode import DecodeSpec  # noqa: E402


def run(tokens: int = 4096, keep: int = 256, recent: int = 64, seed: int = 0) -> dict:
    base = DecodeSpec()
    hidden, heads, kv_heads, dim = base.hidden_dim, base.query_heads, base.kv_heads, base.head_dim
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def weight(rows, cols):
        return (torch.randn((rows, cols), generator=gen, device="cuda") / math.sqrt(rows)).to(torch.bfloat16)

    wq, wk, wv = weight(hidden, heads * dim), weight(hidden, kv_heads * dim), weight(hidden, kv_heads * dim)
    x = torch.randn((tokens + 1, hidden), generator=gen, device="cuda").to(torch.bfloat16)
    rotary = clear.RotaryPositions(dim, base=base.rope_theta)
    queries, keys = rotary.rotate(torch.arange(tokens + 1, device="cuda"), (x @ wq).view(-1, heads, dim),
                                  (x @ wk).view(-1, kv_heads, dim))
    values = (x @ wv).view(-1, kv_heads, dim)

    # the prompt, over keys that nothing has rounded: the softmax's intervals, from rows that see a page or more (the last, of less)
    prompt = clear.prompt_attention(queries[:tokens], keys[:tokens], values[:tokens], ranges=True)
    rows = slice(min(clear.PAGE_TOKENS, tokens) - 1, None)
    ranges = clear.softmax_ranges(prompt.low[rows], prompt.high[rows], prompt.lse[rows])

    # its keys and values in 4-bit pages, and what every cached token was given
    columns, few = -(-tokens // clear.PAGE_TOKENS), -(-(keep + 1) // clear.PAGE_TOKENS)
    pool = clear.ClearKVPages(columns + few, kv_heads=kv_heads, head_dim=dim)
    pages = torch.randperm(columns + few, generator=gen, device="cuda").to(torch.int32)[None]
    table, window = pages[:, :columns].contiguous(), pages[:, columns:].contiguous()

    def slots(table, first, n):
        place = torch.arange(first, first + n, device="cuda")
        return table[0].long()[place // clear.PAGE_TOKENS] * clear.PAGE_TOKENS + place % clear.PAGE_TOKENS

    pool.append(keys[:tokens], values[:tokens], slots(table, 0, tokens))
    lengths = torch.tensor([tokens], dtype=torch.int32, device="cuda")
    starts = torch.tensor([0, tokens], dtype=torch.int32, device="cuda")
    cached = pool.attend(queries[:tokens], table, lengths, starts=starts, most=tokens)
    weights = pool.weigh(queries[:tokens], table, lengths, cached.lse, starts=starts, most=tokens)

    # every key head's heaviest tokens, and the last ones
    kept = pool.evict(table, lengths, weights, window, keep, recent=min(recent, keep))
    held = pool.read(slots(window, 0, min(keep, tokens)), torch.float32)

    # the same tokens as they came, as ``encrypt_kv_history`` takes them: [tokens][kv_heads * head_dim], each head's its own
    at = kept.kept[0, :, :min(keep, tokens)].T.long()[..., None].expand(-1, -1, dim)
    history = keys[:tokens].gather(0, at).flatten(1), values[:tokens].gather(0, at).flatten(1)

    # the next token over the whole prompt and over what was kept
    whole = pool.attend(queries[tokens:], table, lengths)
    part = pool.attend(queries[tokens:], window, kept.lengths)
    after = pool.weigh(queries[tokens:], window, kept.lengths, part.lse, prior=kept.weights)
    return {"ranges": ranges, "weights": weights, "kept": kept, "held": held, "history": history, "whole": whole, "part": part, "after": after,
            "queries": queries, "keys": keys, "values": values, "prompt": prompt, "cached": cached}


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    ap.add_argument("--tokens", type=int, default=4096)
    ap.add_argument("--keep", type=int, default=256)
    args = ap.parse_args()
    got = run(args.tokens, args.keep)
    r = got["ranges"]
    print(f"score_shift {r.score_shift:.4f}, exp_interval {r.exp_interval}, rsqrt_interval {r.rsqrt_interval}")
    share = got["kept"].weights.sum() / got["weights"].sum()
    print(f"{args.keep} of {args.tokens} tokens for each key head hold {100 * share:.1f} % of the attention")
    off = (got["part"].out.float() - got["whole"].out.float()).norm() / got["whole"].out.float().norm()
    print(f"the next token's attention over those is {off:.2f} of its size off the whole's")


if __name__ == "__main__":
    main()
