"""The cleartext model's operators that stand beside the encrypted layer.

An encrypted layer is set up from what the cleartext model does: ``DecodeSpec`` takes the shift and
the interval of the softmax's scores and the interval of their exponentials' sum from calibrated
ranges, and the decrypted answers are judged by the probabilities that they give to known tokens.  The
operators here run that model's attention over real prompts at their full length:

* ``ClearKVPages``: a key/value cache in 4 bits on the GPU, in pages of 128 tokens like the encrypted
  cache's; ``append`` quantises keys and values as they are written, ``read`` gives back what is held,
  ``attend`` is the attention of queries over it, with the log of every row's sum of exponentials and
  the least and largest of its scores;
* ``softmax_ranges``: the encrypted softmax's shift and intervals from those;
* ``token_logprobs``: log probabilities of given tokens, entropy and top alternatives of logits.

Values are held as a sign and one of 0, .5, 1, 1.5, 2, 3, 4, 6 units.  A unit is 2^(b - 127) with one byte
b for each run of 32 values along the head dimension: b is the exponent of the run's largest magnitude
rounded to one mantissa bit, less 2 (kept in 2..252), so the largest becomes 4 or 6 units and no value is
off by more than half a step.  A run that holds an infinity or a NaN is held, and read, as NaN.

Everything runs in libholmes_ckks on the current stream without synchronising; there is no CPU path.
"""

from __future__ import annotations

import math
from typing import NamedTuple

import torch

from . import _native as nat

__all__ = ["PAGE_TOKENS", "Attended", "ClearKVPages", "SoftmaxRanges", "TokenScores", "softmax_ranges",
           "token_logprobs"]

PAGE_TOKENS = 128

_TYPES = {torch.bfloat16: nat.HCK_BF16, torch.float16: nat.HCK_F16, torch.float32: nat.HCK_F32}


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


def _type(dtype: torch.dtype, allowed, what: str) -> int:
    if dtype not in allowed:
        raise ValueError(f"{what} must be {', '.join(str(d).replace('torch.', '') for d in allowed)}, not {dtype}")
    return _TYPES[dtype]


def _check(cond: bool, message: str) -> None:
    if not cond:
        raise ValueError(message)


def _stream(device: torch.device) -> int:
    return torch.cuda.current_stream(device).cuda_stream


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

    @property
    def device(self) -> torch.device:
        return self.buf.device

    @property
    def nbytes(self) -> int:
        return int(self.buf.numel())

    def _slots(self, slots) -> torch.Tensor:
        _check(slots.dim() == 1 and slots.dtype == torch.int64 and slots.device == self.buf.device,
               "slots must be a 1-d int64 tensor on the pool's device")
        return slots if slots.is_contiguous() else slots.contiguous()

    def append(self, keys: torch.Tensor, values: torch.Tensor, slots: torch.Tensor) -> None:
        """Writes ``keys`` and ``values`` [tokens][kv_heads][head_dim] (bf16, fp16 or fp32, any strides but
        the last axis contiguous) into ``slots`` [tokens].  A slot outside the pool, as -1 for padding, leaves
        its token out; the slots of one call must differ."""

        slots = self._slots(slots)
        shape = (slots.numel(), self.kv_heads, self.head_dim)
        kind = _type(keys.dtype, _TYPES, "keys")
        for name, x in (("keys", keys), ("values", values)):
            _check(x.shape == shape and x.dtype == keys.dtype and x.device == self.buf.device and x.stride(2) == 1,
                   f"{name} must be {list(shape)}, contiguous along the last axis, in one type on the pool's device")
        nat.check(self._lib.hck_kv4_append(
            self.buf.data_ptr(), self.pages, self.kv_heads, self.head_dim, kind, keys.data_ptr(), keys.stride(0),
            keys.stride(1), values.data_ptr(), values.stride(0), values.stride(1), slots.data_ptr(), shape[0],
            _stream(self.buf.device)), "hck_kv4_append")

    def read(self, slots: torch.Tensor, dtype: torch.dtype = torch.bfloat16) -> tuple:
        """What ``slots`` hold, as ``(keys, values)`` [tokens][kv_heads][head_dim] in ``dtype``: exact in bf16
        and fp32; in fp16 rounded, with its largest value for any above.  Zeros for a slot outside the pool."""

        slots = self._slots(slots)
        kind = _type(dtype, _TYPES, "dtype")
        keys = torch.empty((slots.numel(), self.kv_heads, self.head_dim), dtype=dtype, device=self.buf.device)
        values = torch.empty_like(keys)
        nat.check(self._lib.hck_kv4_read(
            self.buf.data_ptr(), self.pages, self.kv_heads, self.head_dim, kind, slots.data_ptr(), slots.numel(),
            keys.data_ptr(), values.data_ptr(), _stream(self.buf.device)), "hck_kv4_read")
        return keys, values

    def attend(self, queries: torch.Tensor, table: torch.Tensor, lengths: torch.Tensor, *,
               starts: torch.Tensor | None = None, most: int | None = None, causal: bool = True,
               scale: float | None = None, ranges: bool = False) -> Attended:
        """Attention of ``queries`` [tokens][query heads][head_dim] (bf16 or fp16, any strides but the last
        axis contiguous; query heads a multiple of kv_heads, neighbours sharing a key head) over the cache.

        Sequence b holds the pages ``table[b]`` (int32 [sequences][columns]) and ``lengths[b]`` (int32) tokens.
        Its queries are rows ``starts[b] .. starts[b + 1]`` (int32 [sequences + 1]; without ``starts`` the one
        row b), and stand for its last tokens: query i of n sees the tokens up to length - n + i, or, with
        ``causal`` off, all.  ``most`` bounds the queries of one sequence (default: 1 without ``starts``, else
        all rows) and only saves work; a sequence with more has the rest left unwritten, as has any row that no
        sequence covers.  A page outside the pool counts as tokens that are not there.  ``scale`` multiplies
        the scores (default head_dim^-1/2); ``ranges`` asks for their least and largest."""

        _check(queries.dim() == 3 and queries.shape[2] == self.head_dim and queries.stride(2) == 1,
               f"queries must be [tokens][query heads][{self.head_dim}], contiguous along the last axis")
        kind = _type(queries.dtype, (torch.bfloat16, torch.float16), "queries")
        tokens, heads = int(queries.shape[0]), int(queries.shape[1])
        _check(heads > 0 and heads % self.kv_heads == 0, f"query heads must be a multiple of {self.kv_heads}")
        _check(table.dim() == 2 and lengths.dim() == 1 and table.shape[0] == lengths.shape[0],
               "table must be [sequences][columns] and lengths [sequences]")
        seqs = int(lengths.shape[0])
        _check(starts.shape == (seqs + 1,) if starts is not None else tokens == seqs,
               "starts must be [sequences + 1], or there is one query for each sequence")
        dev = self.buf.device
        for name, x in (("table", table), ("lengths", lengths), ("starts", starts)):
            _check(x is None or (x.dtype == torch.int32 and x.device == dev and (x.numel() == 0 or x.stride(-1) == 1)),
                   f"{name} must be int32 on the pool's device, contiguous along the last axis")
        _check(queries.device == dev, "queries must be on the pool's device")
        most = (1 if starts is None else tokens) if most is None else min(int(most), tokens)
        _check(most >= 0, "most must not be negative")
        scale = 1.0 / math.sqrt(self.head_dim) if scale is None else float(scale)
        _check(0.0 < scale < math.inf, "scale must be positive and finite")
        out = torch.empty((tokens, heads, self.head_dim), dtype=queries.dtype, device=dev)
        sums = torch.empty((3 if ranges else 1, tokens, heads), dtype=torch.float32, device=dev)
        group, cols = heads // self.kv_heads, int(table.shape[1])
        need = self._lib.hck_kv4_attend_workspace_bytes(tokens, seqs, self.kv_heads, group, self.head_dim, most, cols)
        work = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
        at = [sums[i].data_ptr() if i < len(sums) else None for i in range(3)]
        nat.check(self._lib.hck_kv4_attend(
            self.buf.data_ptr(), self.pages, self.kv_heads, self.head_dim, kind, queries.data_ptr(), tokens, group,
            queries.stride(0), queries.stride(1), table.data_ptr(), table.stride(0), cols, lengths.data_ptr(),
            None if starts is None else starts.data_ptr(), seqs, most, int(causal), scale, out.data_ptr(), at[0], at[1],
            at[2], None if work is None else work.data_ptr(), need, _stream(dev)), "hck_kv4_attend")
        return Attended(out, sums[0], *((sums[1], sums[2]) if ranges else (None, None)))


def softmax_ranges(low: torch.Tensor, high: torch.Tensor, lse: torch.Tensor, margin: float = 0.05) -> SoftmaxRanges:
    """The encrypted softmax's shift U and intervals for the rows that ``attend(..., ranges=True)`` saw:
    mapped = (s - U) / 2 runs over ``exp_interval``, made even about 0, and sum exp(2 mapped) over
    ``rsqrt_interval``, both widened by ``margin`` of their width (of their logarithm's, for the sum).  Rows
    that see no token do not count."""

    seen = torch.isfinite(lse)
    if not bool(seen.any()):
        raise ValueError("no row saw a token")
    lo, hi = float(low[seen].min()), float(high[seen].max())
    shift = 0.5 * (lo + hi)
    half = max(0.25 * (hi - lo) * (1.0 + 2.0 * margin), 1e-3)
    a, b = float(lse[seen].min()) - shift, float(lse[seen].max()) - shift
    pad = max(margin * (b - a), 1e-3)
    return SoftmaxRanges(shift, (-half, half), (math.exp(a - pad), math.exp(b + pad)))


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor | None = None, *, top: int = 0) -> TokenScores:
    """Scores of ``logits`` [rows][vocabulary] (bf16, fp16 or fp32, rows any distance apart) in float32: log
    probabilities of ``tokens`` [rows] int64 (a negative one, as of padding, gives 0; one past the vocabulary
    NaN), the entropies, and the ``top`` (up to 32) most likely tokens, int64 and log probabilities.  A logit
    of -inf is a token that cannot be; a row of nothing else gives -inf, and 0 for the entropy."""

    kind = _type(logits.dtype, _TYPES, "logits")
    _check(logits.dim() == 2 and logits.shape[1] >= 1 and (logits.stride(1) == 1 or logits.shape[1] == 1),
           "logits must be [rows][vocabulary], contiguous along the last axis")
    rows, vocab = int(logits.shape[0]), int(logits.shape[1])
    _check(0 <= top <= min(nat.HCK_TOP_MAX, vocab), f"top must be in 0..{min(nat.HCK_TOP_MAX, vocab)}")
    if tokens is not None:
        _check(tokens.shape == (rows,) and tokens.dtype == torch.int64 and tokens.device == logits.device,
               "tokens must be [rows] int64 on the logits' device")
        tokens = tokens if tokens.is_contiguous() else tokens.contiguous()
    if logits.device.type != "cuda":
        raise RuntimeError("token scores run on a GPU: there is no CPU path")
    dev, lib = logits.device, nat.lib()
    floats = torch.empty((2 + top, rows), dtype=torch.float32, device=dev)
    logs = floats[2:].view(rows, top)
    ids = torch.empty((rows, top), dtype=torch.int64, device=dev)
    need = lib.hck_token_scores_workspace_bytes(rows, vocab, kind, top)
    work = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
    nat.check(lib.hck_token_scores(
        logits.data_ptr(), kind, rows, vocab, logits.stride(0), None if tokens is None else tokens.data_ptr(), top,
        floats[0].data_ptr(), floats[1].data_ptr(), ids.data_ptr(), logs.data_ptr(),
        None if work is None else work.data_ptr(), need, _stream(dev)), "hck_token_scores")
    return TokenScores(None if tokens is None else floats[0], floats[1], ids if top else None, logs if top else None)
