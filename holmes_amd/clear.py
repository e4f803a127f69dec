"""The cleartext model's operators that stand beside the encrypted layer.

An encrypted layer is set up from what the cleartext model does: ``DecodeSpec`` takes the shift and
the interval of the softmax's scores and the interval of their exponentials' sum from calibrated
ranges, and the decrypted answers are judged by the probabilities that they give to known tokens.  The
operators here run that model's attention over real prompts at their full length:

* ``RotaryPositions``: rotary positions on queries and keys;
* ``prompt_attention``: attention over whole prompts whose keys and values are as they came, as the encrypted layer has
  them, with the log of every row's sum of exponentials and the least and largest of its scores;
* ``ClearKVPages``: a key/value cache in 4 bits on the GPU, in pages of 128 tokens like the encrypted
  cache's; ``append`` quantises keys and values as they are written, ``read`` gives back what is held,
  ``attend`` is the attention of queries over it, with the same numbers of every row; ``weigh`` sums what attention has
  given each cached token, and ``evict`` brings a sequence down to its heaviest ones and says which they are, for
  the few pages of the encrypted layer's cache;
* ``softmax_ranges``: the encrypted softmax's shift and intervals from those, and ``score_rounding`` what the keys'
  4 bits can have moved them by;
* ``token_logprobs``: log probabilities of given tokens, entropy and top alternatives of logits.

Values are held as a sign and one of 0, .5, 1, 1.5, 2, 3, 4, 6 units.  A unit is 2^(b - 127) with one byte
b for each run of 32 values along the head dimension: b is the exponent of the run's largest magnitude
rounded to one mantissa bit, less 2 (kept in 2..252), so the largest becomes 4 or 6 units and no value is
off by more than half a step (a step of 2 above 4; magnitudes beyond 7 2^125 become 6 2^125).  A run that holds an infinity or a NaN is held, and read, as NaN.

Everything but ``softmax_ranges`` and ``score_rounding`` runs in libholmes_ckks on the current stream of its
tensors' device without synchronising; there is no CPU path.
Nothing has a backward pass: an input that requires a gradient is refused, but under ``torch.no_grad()``; nor has anything a
forward-mode derivative: an input with a tangent is refused.
"""

from __future__ import annotations

import importlib.util
import math
import sys
from typing import NamedTuple

import torch

from . import _native as nat

__all__ = ["PAGE_TOKENS", "Attended", "ClearKVPages", "Evicted", "RotaryPositions", "RotaryScaling", "SoftmaxRanges",
           "TokenScores", "prompt_attention", "score_rounding", "softmax_ranges", "token_logprobs"]

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


class Evicted(NamedTuple):
    """Of every sequence and key head the places that the kept tokens had, in order (int32, -1 behind the last);
    of every sequence their number (int32); and their weights (float32, 0 behind the last), which ``weigh`` takes as
    ``prior`` from there on."""

    kept: torch.Tensor
    lengths: torch.Tensor
    weights: torch.Tensor


class RotaryScaling(NamedTuple):
    """Rotary frequencies for more tokens than the ``original`` they were made for, ``factor`` times as many:

    * "linear": all divided by ``factor``;
    * "base": the base times factor^(d / (d - 2)) for d rotated dims, so that the last pair is divided and the first
      is as it was;
    * "wavelength": a pair that makes fewer than ``low`` turns in the original length is divided, one that makes more
      than ``high`` is as it was, and between them the two are blended evenly over the turns;
    * "ramp": the same ends, but blended evenly over the pairs' numbers, whose first is the whole number below the
      (fractional) pair of ``high`` turns and whose last the one above that of ``low``; and the rotated values are
      multiplied by 0.1 log(factor) + 1."""

    kind: str
    factor: float
    original: int = 8192
    low: float = 1.0
    high: float = 4.0


class SoftmaxRanges(NamedTuple):
    """``DecodeSpec``'s ``score_shift``, ``exp_interval`` and ``rsqrt_interval``."""

    score_shift: float
    exp_interval: tuple
    rsqrt_interval: tuple


_modules: dict = {}


def _load(name: str):
    nat.lib()  # the library it calls; raises if it has not been built
    path = nat.LIB_PATH.with_name(f"{name}.so")
    if not path.exists():
        raise RuntimeError(f"{path} is missing: build the HIP extension first (python -m holmes_amd.build)")
    spec = importlib.util.spec_from_file_location(name, path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return _modules.setdefault(name, module)


def _bound():
    """The extension module of csrc/clear_bind.cpp: a call on a few tokens costs what the host does for it, so
    the checks of tensors, the outputs' allocation and the launch are one native call."""

    return _modules.get("_clear") or _load("_clear")


def _window():
    """The extension module of csrc/window_bind.cpp, likewise."""

    return _modules.get("_window") or _load("_window")


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
        self._native, self._more = _bound(), _window()
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


    def weigh(self, queries: torch.Tensor, table: torch.Tensor, lengths: torch.Tensor, lse: torch.Tensor, *,
              starts: torch.Tensor | None = None, most: int | None = None, causal: bool = True,
              scale: float | None = None, prior: torch.Tensor | None = None) -> torch.Tensor:
        """What the attention of ``queries`` has given each cached token: the sum of exp(score - lse) over the rows that
        see it, of the queries of one key head, [sequences][kv_heads][columns * 128] float32.  The arguments are
        ``attend``'s, and ``lse`` is what it returned for them (a row of -inf gives nothing).  Half a step of its 32 bits is a factor of
        exp(|lse| 2^-24) to all that a row gives: rows with scores beyond some 2^22 give their tokens an order rather than shares.
        ``prior`` [sequences][kv_heads][places], what
        earlier calls gave, is added, as 0 where it has no place; places behind a sequence's end are 0.  (``most`` saves
        more here than there: sequences of few queries each are taken another way than prompts.)"""

        got = self._more.weigh(self.buf, *self._shape, queries, table, lengths, lse, starts, most, causal, scale, prior)
        if type(got) is int:
            nat.check(got, "hck_kv4_weigh")
        return got

    def evict(self, table: torch.Tensor, lengths: torch.Tensor, weights: torch.Tensor, into: torch.Tensor, keep: int, *,
              recent: int = 0) -> Evicted:
        """Brings every sequence down to ``keep`` tokens for each key head: its last ``recent`` ones, and of the others
        those of the largest ``weights`` [sequences][kv_heads][places] (float32; 0 behind the last place, NaN above
        all, the earlier one where they tie).  They are copied, in their order, to the pages ``into`` (int32
        [sequences][at least keep / 128]), of which each head then holds tokens of its own choice; the pages of ``table`` stay as they are.
        A sequence of fewer tokens keeps all.  How a call is run goes by the table's columns, not by the lengths, which are on the
        device: a view without spare columns (``table[:, :columns]``) saves work, and beyond 128 columns a workspace of 24.6 KB for
        every 64 of them, sequence and head (32 sequences of 384 tokens to 256, 8 heads: 10 us through 3 columns, 14 through 128, 39 and 19 MB
        through 129, 211 and 101 MB through 1024).  A token whose page is outside the pool is not kept, and a page of ``into``
        outside it takes nothing.  The pages of ``into`` must be none of the tables' and differ (else what they hold is undefined);
        places in them behind the kept tokens stay as they were."""

        got = self._more.evict(self.buf, *self._shape, table, lengths, weights, into, keep, recent)
        if type(got) is int:
            nat.check(got, "hck_kv4_evict")
        return Evicted._make(got)


_PI = 0x3243F6A8885A308D313198A2E03707344A4093822299F3   # times 2^-180


def _turns(frequency: float) -> int:
    """Radians per token as turns per token in units of 2^-64, modulo a turn."""

    n, d = frequency.as_integer_ratio()
    return ((n << 244) // (d * _PI) + 1 >> 1) % (1 << 64)


def _rotary_frequencies(rotated: int, base: float, scaling: RotaryScaling | None) -> tuple:
    """Radians per token of every pair, and what the rotated values are multiplied by."""

    def plain(base):
        return [base ** (-2 * i / rotated) for i in range(rotated // 2)]

    if scaling is None:
        return plain(base), 1.0
    kind, factor, original, low, high = scaling
    if not 1.0 <= factor <= 1 << 20:
        raise ValueError("the factor of a scaling must be in 1..2^20")
    if kind == "linear":
        return [f / factor for f in plain(base)], 1.0
    if kind == "base":
        if rotated < 4:
            raise ValueError("a scaled base needs two pairs")
        return plain(base * factor ** (rotated / (rotated - 2))), 1.0
    if kind not in ("wavelength", "ramp"):
        raise ValueError('the kind of a scaling must be "linear", "base", "wavelength" or "ramp"')
    if not (1 <= original < math.inf and 0.0 < low < high < math.inf):
        raise ValueError("a blended scaling needs original >= 1 and 0 < low < high, all finite")

    if kind == "wavelength":
        def whole(i, f):
            return (original * f / (2.0 * math.pi) - low) / (high - low)
        amount = 1.0
    else:
        if base <= 1.0:
            raise ValueError("a ramp needs a base above 1")

        def pair(turns):
            return rotated * math.log(original / (2.0 * math.pi * turns)) / (2.0 * math.log(base))
        first, last = max(math.floor(pair(high)), 0), min(math.ceil(pair(low)), rotated - 1)

        def whole(i, f):
            return 1.0 - (i - first) / max(last - first, 0.001)
        amount = 0.1 * math.log(factor) + 1.0
    got = []
    for i, f in enumerate(plain(base)):
        w = min(max(whole(i, f), 0.0), 1.0)
        got.append(w * f + (1.0 - w) * (f / factor))
    return got, amount


class RotaryPositions:
    """Rotary positions: of the first ``rotated`` dims of a head (default: all), pairs (i, i + rotated / 2), or, with
    ``interleaved``, (2 i, 2 i + 1), are turned by position * base^(-2 i / rotated) radians; the dims behind stay.  The
    default is what ``DecodeSpec`` and ``PrefillSpec`` take (pairs of halves, rope_theta 500000).  ``scaling``: for long
    contexts.  Frequencies are held as float64 (``frequencies``) and turned into whole units of 2^-64 turns a token, which
    adds 2^-34 turns to an angle at position 2^31; the float64's own rounding is up to 2^-25 turns there.  Sine, cosine and
    products are of 32 bits."""

    def __init__(self, head_dim: int = 128, *, base: float = 500000.0, rotated: int | None = None,
                 interleaved: bool = False, scaling: RotaryScaling | None = None, device="cuda"):
        rotated = head_dim if rotated is None else rotated
        if not 2 <= head_dim <= nat.HCK_ROTARY_MAX or head_dim % 2:
            raise ValueError(f"head_dim must be even, in 2..{nat.HCK_ROTARY_MAX}")
        if not 2 <= rotated <= head_dim or rotated % 2:
            raise ValueError("rotated must be even, in 2..head_dim")
        if not 1.0 <= base <= 1e30:
            raise ValueError("base must be in 1..1e30")
        self.frequencies, self.amount = _rotary_frequencies(rotated, float(base), scaling)
        if torch.device(device).type != "cuda" or not torch.cuda.is_available():
            raise RuntimeError("positions are rotated on a GPU: there is no CPU path")
        self.head_dim, self.rotated, self.interleaved = int(head_dim), int(rotated), bool(interleaved)
        # turns per token in units of 2^-64: position times that, modulo 2^64, is the angle's part of a turn
        turns = map(_turns, self.frequencies)
        self._turns = torch.tensor([t - (1 << 64) if t >= 1 << 63 else t for t in turns], dtype=torch.int64, device=device)
        self._native = _window()

    def rotate(self, positions: torch.Tensor, queries: torch.Tensor, keys: torch.Tensor | None = None, *,
               inverse: bool = False):
        """``queries`` [tokens][heads][head_dim] (bf16, fp16 or fp32, any strides but the last axis contiguous), and
        ``keys`` [tokens][kv_heads][head_dim] of the same type in the same launch, turned by ``positions`` [tokens] (int64 or
        int32, any, also negative): new dense tensors, one or both.  ``inverse`` turns back (times the same amount, if ``scaling`` has one)."""

        got = self._native.rotate(self._turns, self.head_dim, self.rotated, self.interleaved, self.amount, positions,
                                  queries, keys, inverse)
        if type(got) is int:
            nat.check(got, "hck_rotary")
        return got


def prompt_attention(queries: torch.Tensor, keys: torch.Tensor, values: torch.Tensor,
                     starts: torch.Tensor | None = None, *, most: int | None = None, causal: bool = True,
                     scale: float | None = None, ranges: bool = False) -> Attended:
    """Attention over whole prompts: ``queries`` [tokens][query heads][head_dim] and ``keys`` and ``values``
    [tokens][kv_heads][head_dim] of 64 or 128 dims, all bf16 or all fp16 (any strides but the last axis contiguous; tensors that
    16 bytes cannot be loaded from at a time are copied first; query heads a multiple of kv_heads, neighbours sharing a key head).

    Sequence b is the tokens ``starts[b] .. starts[b + 1]`` (int32 [sequences + 1], not decreasing; without ``starts`` there
    is one of all tokens), and query i of it sees its tokens up to i, or, with ``causal`` off, all.  ``most`` bounds the queries
    of one sequence (default: all) and only saves work; a longer one has the rest left unwritten, as has any row that no sequence
    covers.  Scores, statistics and sums are of 32 bits; a probability goes into its product with the values in their 16 bits (in two
    parts where a row sees few tokens), which can add as much to an output's error as its own rounding does; in fp16 those below 2^-32 of
    the row's largest may count as 0.  An infinite value makes its dim infinite or NaN in all rows that see it.  ``scale`` and ``ranges`` as
    for ``ClearKVPages.attend``: the ranges here are those of keys that nothing has rounded, so ``softmax_ranges`` needs no ``rounding`` for them."""

    got = _window().prompt(queries, keys, values, starts, most, causal, scale, ranges)
    if type(got) is int:
        nat.check(got, "hck_prompt_attend")
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

    got = _bound().scores(logits, tokens, top)
    if type(got) is int:
        nat.check(got, "hck_token_scores")
    return TokenScores._make(got)
