"""From a cleartext prompt to the encrypted decode step's softmax, and from answers to scores.

    python examples/calibrate_decode.py [--tokens 2048] [--vocab 32000]

One attention layer of the decode step's shape (32 query heads over 8 key heads of 128) with random
weights runs in the clear: the prompt's keys and values go into 4-bit pages, its attention gives the
outputs and the range of every row's scores, and ``DecodeSpec`` takes the softmax's shift and intervals
from them, widened by what the keys' 4 bits can have moved them by.  Then single tokens follow, as they would be served, and the answers are scored: log
probabilities of the tokens that came, entropies, the most likely alternatives.  Random weights say
nothing about language; what the example shows is which call follows which.
"""

import argparse
import math
import sys
from pathlib import Path

import numpy as np
import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))

from holmes_amd import clear  # noqa: E402
from holmes_amd.decode import DecodePolynomials, DecodeSpec  # noqa: E402


def run(tokens: int = 2048, steps: int = 4, vocab: int = 32000, seed: int = 0) -> dict:
    base = DecodeSpec()
    hidden, heads, kv_heads, dim = base.hidden_dim, base.query_heads, base.kv_heads, base.head_dim
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def weight(rows, cols):
        return (torch.randn((rows, cols), generator=gen, device="cuda") / math.sqrt(rows)).to(torch.bfloat16)

    embed = torch.randn((vocab, hidden), generator=gen, device="cuda").to(torch.bfloat16)
    wq, wk, wv, wo = weight(hidden, heads * dim), weight(hidden, kv_heads * dim), weight(hidden, kv_heads * dim), weight(heads * dim, hidden)
    text = torch.randint(0, vocab, (tokens + steps + 1,), generator=gen, device="cuda")

    # a pool of pages, handed out in any order
    columns = -(-(tokens + steps) // clear.PAGE_TOKENS)
    pool = clear.ClearKVPages(columns + 2, kv_heads=kv_heads, head_dim=dim)
    table = torch.randperm(columns + 2, generator=gen, device="cuda")[:columns].to(torch.int32)[None]

    def write(first, x):
        place = torch.arange(first, first + x.shape[0], device="cuda")
        slots = table[0].long()[place // clear.PAGE_TOKENS] * clear.PAGE_TOKENS + place % clear.PAGE_TOKENS
        keys = (x @ wk).view(-1, kv_heads, dim)
        pool.append(keys, (x @ wv).view(-1, kv_heads, dim), slots)
        return keys, slots

    def logits(x, attended):
        return (x + attended.out.flatten(1) @ wo) @ (embed.T / math.sqrt(hidden))

    # the prompt
    x = embed[text[:tokens]]
    keys, slots = write(0, x)
    queries = (x @ wq).view(-1, heads, dim)
    lengths = torch.tensor([tokens], dtype=torch.int32, device="cuda")
    starts = torch.tensor([0, tokens], dtype=torch.int32, device="cuda")
    prompt = pool.attend(queries, table, lengths, starts=starts, most=tokens, ranges=True)
    scores = clear.token_logprobs(logits(x, prompt), text[1:tokens + 1], top=4)

    # the encrypted softmax's shift and intervals, from the rows that see at least a page as its steps do
    rows = slice(clear.PAGE_TOKENS - 1, None)
    rounding = clear.score_rounding(queries[rows], keys, pool.read(slots, torch.float32)[0])
    ranges = clear.softmax_ranges(prompt.low[rows], prompt.high[rows], prompt.lse[rows], rounding=rounding)
    spec = DecodeSpec(score_shift=ranges.score_shift, exp_interval=ranges.exp_interval, rsqrt_interval=ranges.rsqrt_interval)
    exp_series = DecodePolynomials.fit(spec).exp

    # how well the series does on the last token's scores: its first query head, against the keys as they came
    s = (keys[:, 0].float() @ queries[-1, 0].float()).double().cpu().numpy() / math.sqrt(dim)
    mapped = (s - ranges.score_shift) / 2
    lo, hi = ranges.exp_interval
    e = np.polynomial.chebyshev.chebval((2 * mapped - lo - hi) / (hi - lo), exp_series) ** 2
    exact = np.exp(2 * mapped)
    error = float(np.abs(e / e.sum() - exact / exact.sum()).max() / (exact / exact.sum()).max())

    # single tokens behind the prompt
    answers = []
    for i in range(steps):
        x = embed[text[tokens + i:tokens + i + 1]]
        write(tokens + i, x)
        lengths += 1
        step = pool.attend((x @ wq).view(-1, heads, dim), table, lengths)
        answers.append(clear.token_logprobs(logits(x, step), text[tokens + i + 1:tokens + i + 2], top=4))
    return {"ranges": ranges, "rounding": rounding, "softmax_error": error, "prompt": scores, "answers": answers,
            "cache_bytes": pool.nbytes, "mapped": mapped, "total": exact.sum(), "queries": queries, "keys": keys}


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    ap.add_argument("--tokens", type=int, default=2048)
    ap.add_argument("--vocab", type=int, default=32000)
    args = ap.parse_args()
    got = run(args.tokens, vocab=args.vocab)
    r = got["ranges"]
    print(f"{args.tokens} tokens in {got['cache_bytes'] / 2**20:.1f} MiB of 4-bit pages")
    print(f"score_shift {r.score_shift:.4f}, exp_interval {r.exp_interval}, rsqrt_interval {r.rsqrt_interval}")
    print(f"of which up to {got['rounding']:.3f} either way for the scores' rounding by 4-bit keys")
    print(f"degree-15 exponential on those: {got['softmax_error']:.1e} of the largest probability")
    print(f"prompt: mean log probability {got['prompt'].logprobs.mean():.3f}, entropy {got['prompt'].entropy.mean():.3f}")
    for a in got["answers"]:
        print(f"next token: log probability {a.logprobs[0]:.3f}, alternatives {a.top_ids[0].tolist()}")


if __name__ == "__main__":
    main()
