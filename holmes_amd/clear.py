"""The cleartext model's operators that stand beside the encrypted layer.

An encrypted layer is set up from what the cleartext model does: ``DecodeSpec`` takes the shift and
the interval of the softmax's scores and the interval of their exponentials' sum from calibrated
ranges, and the decrypted answers are judged by the probabilities that they give to known tokens.  The
operators here run that model's attention over real prompts at their full length:

* ``ClearKVPages``: a key/value cache in 4 bits on the GPU, in pages of 128 tokens like the encrypted
  cache's; ``append`` quantises keys and values as they are written, ``read`` gives back what is held,
  ``attend`` is the attention of queries over it, with the log of every row's sum of exponentials and
  the least and largest of its scores;
* ``softmax_ranges``: the encrypted softmax's shift and intervals from those, and ``score_rounding`` what the keys'
  4 bits can have moved them by;
* ``token_logprobs``: log probabilities of given tokens, entropy and top alternatives of logits.

Values are held as a sign and one of 0, .5, 1, 1.5, 2, 3, 4, 6 units.  A unit is 2^(b - 127) with one byte
b for each run of 32 values along the head dimension: b is the exponent of the run's largest magnitude
rounded to one mantissa bit, less 2 (kept in 2..252), so the largest becomes 4 or 6 units and no value is
off by more than half a step (a step of 2 above 4; magnitudes beyond 7 2^125 become 6 2^125).  A run that holds an infinity or a NaN is held, and read, as NaN.

Everything but ``softmax_ranges`` and ``score_rounding`` runs in libholmes_ckks on the current stream of its
tensors' device without synchronising; there is no CPU path.
Nothing has a backward pass: an input that requires a gradient is refused, but under ``torch.no_grad()``.
"""

from __future__ import annotations

import importlib.util
import math
import sys
from typing import NamedTuple

import torch

from . import _native as nat

__all__ = ["PAGE_TOKENS", "Attended", "ClearKVPages", "SoftmaxRanges", "TokenScores", "score_rounding", "softmax_ranges",
           "token_logprobs"]

PAGE_TOKENS = 128


class Attended(NamedTuple):
    """Outputs [tokens][query heads][head_dim] in the queries' type; log sum exp of the scaled scores and,
    where asked for, the least and largest of them, [tokens][query heads] float32.  A row that sees no
    token gives 0, -inf, +inf and -inf."""

    out: torch.Tensor
    lse: torch.Tensor
    low: torch.Tensor | None
    high: torch.Tensor | None


class TokenScores(NamedTuple):
    """Of every row of logits: the given token's log probability, the entropy in nats, and the ``top`` most
    likely tokens (the lower one first where they tie) with their log probabilities."""

    logprobs: torch.Tensor | None
    entropy: torch.Tensor
    top_ids: torch.Tensor | None
    top_logprobs: torch.Tensor | None


class SoftmaxRanges(NamedTuple):
    """``DecodeSpec``'s ``score_shift``, ``exp_interval`` and ``rsqrt_interval``."""

    score_shift: float
    exp_interval: tuple
    rsqrt_interval: tuple


_binding = None


def _bound():
    """The extension module of csrc/clear_bind.cpp: a call on a few tokens costs what the host does for it, so
    the checks of tensors, the outputs' allocation and the launch are one native call."""

    global _binding
    if _binding is None:
        nat.lib()  # the library it calls; raises if it has not been built
        path = nat.LIB_PATH.with_name("_clear.so")
        if not path.exists():
            raise RuntimeError(f"{path} is missing: build the HIP extension first (python -m holmes_amd.build)")
        spec = importlib.util.spec_from_file_location("_clear", path)
        module = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(module)
        _binding = module
    return _binding


class ClearKVPages:
    """``pages`` pages of 128 tokens for ``kv_heads`` heads, keys and values: 136 bytes a token and head of
    128 dims.  Slots are numbered page * 128 + place; which sequence holds which pages is the caller's
    table."""

    def __init__(self, pages: int, kv_heads: int = 8, head_dim: int = 128, device="cuda"):
        if head_dim not in (64, 128):
            raise ValueError("head_dim must be 64 or 128")
        if pages < 1 or not 1 <= kv_heads <= 65535:
            raise ValueError("a pool needs pages >= 1 and 1 <= kv_heads <= 65535")
        if torch.device(device).type != "cuda" or not torch.cuda.is_available():
            raise RuntimeError("cleartext pages live on a GPU: there is no CPU path")
        self.pages, self.kv_heads, self.head_dim = int(pages), int(kv_heads), int(head_dim)
        self._lib = nat.lib()
        self.buf = torch.zeros((self.pages, self.kv_heads, self._lib.hck_kv4_page_bytes(self.head_dim)),
                               dtype=torch.uint8, device=device)
        self._native = _bound()
        self._shape = (self.pages, self.kv_heads, self.head_dim, self.buf.device.index)

    @property
    def device(self) -> torch.device:
        return self.buf.device

    @property
    def nbytes(self) -> int:
        return int(self.buf.numel())

    def append(self, keys: torch.Tensor, values: torch.Tensor, slots: torch.Tensor) -> None:
        """Writes ``keys`` and ``values`` [tokens][kv_heads][head_dim] (bf16, fp16 or fp32, any strides but
        the last axis contiguous) into ``slots`` [tokens].  A slot outside the pool, as -1 for padding, leaves
        its token out; the slots of one call must differ (what one named twice holds is undefined)."""

        err = self._native.append(self.buf, *self._shape, keys, values, slots)
        if err:
            nat.check(err, "hck_kv4_append")

    def read(self, slots: torch.Tensor, dtype: torch.dtype = torch.bfloat16) -> tuple:
        """What ``slots`` hold, as ``(keys, values)`` [tokens][kv_heads][head_dim] in ``dtype``: exact in bf16
        and fp32; in fp16 rounded, with its largest value for any above.  Zeros for a slot outside the pool."""

        got = self._native.read(self.buf, *self._shape, slots, dtype)
        if type(got) is int:
            nat.check(got, "hck_kv4_read")
        return got

    def attend(self, queries: torch.Tensor, table: torch.Tensor, lengths: torch.Tensor, *,
               starts: torch.Tensor | None = None, most: int | None = None, causal: bool = True,
               scale: float | None = None, ranges: bool = False) -> Attended:
        """Attention of ``queries`` [tokens][query heads][head_dim] (bf16 or fp16, any strides but the last
        axis contiguous; query heads a multiple of kv_heads, neighbours sharing a key head) over the cache.

        Sequence b holds the pages ``table[b]`` (int32 [sequences][columns]) and ``lengths[b]`` (int32) tokens.
        Its queries are rows ``starts[b] .. starts[b + 1]`` (int32 [sequences + 1]; without ``starts`` the one
        row b), and stand for its last tokens: query i of n sees the tokens up to length - n + i, or, with
        ``causal`` off, all.  ``most`` bounds the queries of one sequence (default: 1 without ``starts``, else
        all rows) and only saves work, as does a table without spare columns (32 sequences of 2000 tokens and one
        query: 20 us, 42 us with ``starts`` and no ``most``, 23 us with 1024 columns); a sequence with more has the rest left unwritten, as has any row that no
        sequence covers.  A page outside the pool counts as tokens that are not there.  ``scale`` multiplies
        the scores (default head_dim^-1/2; at most 2^126); ``ranges`` asks for their least and largest."""

        got = self._native.attend(self.buf, *self._shape, queries, table, lengths, starts, most, causal, scale, ranges)
        if type(got) is int:
            nat.check(got, "hck_kv4_attend")
        return Attended._make(got)


def score_rounding(queries: torch.Tensor, keys: torch.Tensor, held: torch.Tensor, scale: float | None = None) -> float:
    """How far scores over the pages are from those of ``keys`` [tokens][kv_heads][head_dim] where nothing rounds
    them to 4 bits, as in the encrypted layer: the largest |scale q.(k - held)| of all ``queries`` [rows][query
    heads][head_dim] and tokens, with ``held`` what ``read`` gives for the keys, and the products' own rounding in
    32 bits on top.  Plain products of rows by tokens, some 64 M of them at a time.  Waits for the device."""

    heads = keys.shape[1]
    if keys.shape != held.shape or queries.shape[2] != keys.shape[2] or queries.shape[1] % max(heads, 1):
        raise ValueError("queries must be [rows][query heads][head_dim], and keys and held [tokens][kv_heads][head_dim]")
    if keys.numel() == 0 or queries.numel() == 0:
        return 0.0
    most = torch.zeros((), device=keys.device)
    for q, off in zip(queries.float().chunk(heads, 1), (keys.float() - held.float()).unbind(1)):
        q, size = q.flatten(0, 1), torch.linalg.vector_norm(off, dim=1).max()
        for rows in q.split(max(1, (1 << 26) // len(off))):
            slack = keys.shape[2] * 2.0**-24 * torch.linalg.vector_norm(rows, dim=1).max() * size
            most = torch.maximum(most, torch.matmul(rows, off.T.contiguous()).abs().max() + slack)
    return float(most) * (1.0 / math.sqrt(keys.shape[2]) if scale is None else scale)


def softmax_ranges(low: torch.Tensor, high: torch.Tensor, lse: torch.Tensor, margin: float = 0.05,
                   rounding: float = 0.0) -> SoftmaxRanges:
    """The encrypted softmax's shift U and intervals for the rows that ``attend(..., ranges=True)`` saw:
    mapped = (s - U) / 2 runs over ``exp_interval``, made even about 0, and sum exp(2 mapped) over
    ``rsqrt_interval``, both widened by ``margin`` of their width (of their logarithm's, for the sum).  Scores
    and the sums' logarithms are moreover taken up to ``rounding`` further out: ``attend`` measures the keys as
    the pages hold them, the encrypted layer has them unrounded, and ``score_rounding`` gives the difference.
    These are ``DecodeSpec``'s fields; ``PrefillSpec``'s are of scores less their row's mean, which the ranges
    do not tell.  Rows that see no token do not count; a row with a NaN or an infinity, and sums beyond float64, are refused.
    Waits for the device, and so cannot be captured."""

    if not 0.0 <= rounding < math.inf:
        raise ValueError("rounding must be finite and not negative")
    empty = torch.isneginf(lse) & torch.isposinf(low)
    odd = ~empty & ~(torch.isfinite(low) & torch.isfinite(high) & torch.isfinite(lse))
    if lse.numel() == 0:
        raise ValueError("no row saw a token")
    inf = torch.full((), math.inf, dtype=torch.float64, device=lse.device)
    sums = lse.double()
    empties, odds, lo, hi, a, b = torch.stack([
        empty.sum().double(), odd.sum().double(), torch.where(empty, inf, low.double()).min(),
        torch.where(empty, -inf, high.double()).max(), torch.where(empty, inf, sums).min(),
        torch.where(empty, -inf, sums).max()]).tolist()
    if empties == lse.numel():
        raise ValueError("no row saw a token")
    if odds:
        raise ValueError(f"{int(odds)} rows have a score or a sum that is NaN or infinite")
    shift = 0.5 * (lo + hi)
    lo, hi, a, b = lo - rounding, hi + rounding, a - rounding, b + rounding
    half = max(0.25 * (hi - lo) * (1.0 + 2.0 * margin), 1e-3)
    a, b = a - shift, b - shift
    pad = max(margin * (b - a), 1e-3)
    if a - pad < math.log(sys.float_info.min) or b + pad > math.log(sys.float_info.max):
        raise ValueError(f"scores from {lo:.6g} to {hi:.6g}: the sums of their exponentials are beyond float64")
    return SoftmaxRanges(shift, (-half, half), (math.exp(a - pad), math.exp(b + pad)))


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor | None = None, *, top: int = 0) -> TokenScores:
    """Scores of ``logits`` [rows][vocabulary] (bf16, fp16 or fp32, rows any distance apart) in float32: log
    probabilities of ``tokens`` [rows] int64 (a negative one, as of padding, gives 0; one past the vocabulary
    NaN), the entropies, and the ``top`` (up to 32) most likely tokens, int64 and log probabilities.  A logit
    of -inf is a token that cannot be; a row of nothing else gives -inf, and 0 for the entropy."""

    got = (_binding or _bound()).scores(logits, tokens, top)
    if type(got) is int:
        nat.check(got, "hck_token_scores")
    return TokenScores._make(got)
